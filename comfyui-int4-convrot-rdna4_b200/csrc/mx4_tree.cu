// C entry of the attention of drafted tokens that form a tree over the paged MX4
// cache. Conventions of include/convrot_b200.h.
#include <algorithm>
#include <cstring>

#include "mx4_host.cuh"
#include "mx4_attn.cuh"
#include "mx4_attn_host.cuh"

#define CONVROT_API extern "C" __attribute__((visibility("default")))

using namespace convrot;

CONVROT_API size_t ck_mx4_tree_attention_workspace_size(int B, int tq, int hq, int hkv, int d, long long longest) {
    if (B <= 0 || tq <= 0 || hkv <= 0 || hq <= 0 || hq % hkv || d <= 0) return 0;
    const AttnPlan p = attn_plan(B, tq, hq, hkv, d, longest);
    return align256(p.partials() * d * 4) + align256(p.partials() * 8);
}

CONVROT_API int ck_mx4_tree_attention(const void* q, int dtype, long long q_seq, long long q_token, long long q_head, const void* codes,
                                      const void* scales, long long pages, int page, const void* table, long long table_ld, int table_pages,
                                      const void* lens, const void* nodes, const void* mask, long long mask_seq, long long mask_row, void* out,
                                      int B, int tq, int hq, int hkv, int d, int G, float softmax_scale, void* workspace,
                                      size_t workspace_bytes, void* stream) {
    if (int rc = check_cache(codes, scales, pages, hkv, d, page, G)) return rc;
    if (dtype != 1 && dtype != 2) return fail("queries must be bf16 (1) or f16 (2)");
    if (B < 0 || tq <= 0 || hq <= 0 || hq % hkv) return fail("query heads must be a positive multiple of the cache's heads");
    if (table_pages < 0 || table_ld < table_pages) return fail("bad block table shape");
    if (static_cast<long long>(table_pages) * page > kMx4MostTokens) return fail("block table longer than 2^31 - 1024 tokens");
    if (mask_seq < 0 || mask_row < 0) return fail("mask strides must not be negative");
    if (B == 0) return 0;
    if (static_cast<long long>(B) * tq * hq > 0x7FFFFFFFll) return fail("too many query rows");
    if (!q || !lens || !mask || !out || (table_pages && !table)) return fail("null pointer");
    if (!aligned_to(q, 2) || !aligned_to(table, 4) || !aligned_to(lens, 4) || !aligned_to(nodes, 4) || !aligned16(out))
        return fail("queries, table or lengths not aligned to their type, or out not to 16 bytes");
    if (pages * 2 * hkv * page > 0xFFFFFFFEll) return fail("the cache holds more than 2^32 - 2 rows");
    const long long longest = static_cast<long long>(table_pages) * page;
    const AttnPlan p = attn_plan(B, tq, hq, hkv, d, longest);
    if (p.tiles > 0x7FFFFFFF) return fail("too many query rows");
    const size_t need = ck_mx4_tree_attention_workspace_size(B, tq, hq, hkv, d, longest);
    if (need && (!workspace || !aligned_to(workspace, 256))) return fail("the workspace must be 256-byte aligned");
    if (workspace_bytes < need) return fail("workspace smaller than ck_mx4_tree_attention_workspace_size");
    Mx4AttnArgs a{q, q_seq, q_token, q_head, static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales),
                  static_cast<const int*>(table), table_ld, longest, static_cast<const int*>(lens), out, static_cast<float*>(workspace),
                  need ? reinterpret_cast<float2*>(static_cast<unsigned char*>(workspace) + align256(p.partials() * d * 4)) : nullptr,
                  B, tq, hq, hkv, page_bits(page), static_cast<int>(pages), G, p.row_tiles, p.splits, p.clustered,
                  softmax_scale * 1.4426950408889634f, static_cast<const uint8_t*>(mask), static_cast<const int*>(nodes), mask_seq, mask_row};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == 1) return run_attention<__nv_bfloat16, true>(a, d, p, st);
    return run_attention<__half, true>(a, d, p, st);
}
