// C entry of the attention of drafted tokens that form a tree over the paged MX4
// cache. Conventions of include/convrot_b200.h.
#include <algorithm>
#include <cstring>

#include "mx4_host.cuh"
#include "mx4_attn.cuh"
#include "mx4_attn_host.cuh"

namespace convrot {

// Status word of the kernels of this file (a bounded wait that gave up).
static __device__ int g_tree_status;

enum : int { kMx4TimeoutProducer = 1, kMx4TimeoutMma = 2, kMx4TimeoutEpilogue = 4 };

__device__ __forceinline__ void tree_record_status(int code) { atomicCAS(&g_tree_status, 0, code); }

cudaError_t tree_take_status(cudaStream_t stream, int* status) {
    cudaError_t e = cudaMemcpyFromSymbolAsync(status, g_tree_status, sizeof(int), 0, cudaMemcpyDeviceToHost, stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
    const int zero = 0;
    if (e == cudaSuccess) e = cudaMemcpyToSymbolAsync(g_tree_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
    return e;
}

}  // namespace convrot

#include "mx4_tree.cuh"

#define CONVROT_API extern "C" __attribute__((visibility("default")))

using namespace convrot;

namespace {

// How a call is cut. `tensor`: the kernel of this file's header, with 256 rows of a cache head a
// block (pair) or 128; otherwise the one for few rows, in tiles of 8 or 16.
struct TreePlan {
    AttnPlan p;
    bool tensor, pair;
};

// Whether blocks take the sequences in the order of their lengths: more of them than multiprocessors, and no
// more sequences than a block has threads.
bool tree_order(int B, long long blocks) { return B > 1 && B <= kTreeThreads && blocks > sm_count(); }

TreePlan tree_plan(int B, int tq, int hq, int hkv, int d, long long longest) {
    TreePlan t{};
    const long long rows = static_cast<long long>(tq) * (hq / hkv);
    // What is least by what was measured: a start, and a time for each tile of rows and 128 tokens. Tiles of
    // 8 rows start first, and read the cache anew for each 8; 128 rows of the tensor kernel take as long
    // as 22 of them. In ns; heads of 128: 1 x 777 tokens of 32 rows 8.9 us
    // in tiles of 8, 19 in one tile of 32, 20 by the tensor kernel; 16 x 4096 tokens of 32 rows 112, 94 and 78 us; of
    // 16 rows (tiles of 16) 57 against 78 us; heads of 64, 32 rows: 72 against 58 us.
    const double units = static_cast<double>(B) * hkv * ((longest + kTreeTile - 1) / kTreeTile), per = d == 64 ? 0.57 : d / 128.0;
    const double few8 = 8000 + 7 * per * units * ((rows + 7) / 8), few16 = 11000 + 14 * per * units * ((rows + 15) / 16);
    const double many = 18000 + (d == 64 ? 10 : 19) * units * (rows <= kTreeTile ? 1.0 : 1.5 * ((rows + 2 * kTreeTile - 1) / (2 * kTreeTile)));
    t.tensor = d <= 128 && many < std::min(few8, few16);
    if (!t.tensor) {
        t.p = attn_plan_rows(B, rows, rows <= 8 || few8 <= few16 ? 8 : 16, hkv, d, longest);
        return t;
    }
    t.pair = rows > kTreeTile;
    t.p.tile_rows = t.pair ? 2 * kTreeTile : kTreeTile;
    t.p.row_tiles = static_cast<int>((rows + t.p.tile_rows - 1) / t.p.tile_rows);
    t.p.tiles = static_cast<long long>(B) * hkv * t.p.row_tiles;
    // Splits by the estimated time of two batches of that longest length, in us (a block's start and end 13, a split's
    // mean on its way out 3, the join 9 and memory's time). All sequences that long: waves of blocks; whole
    // sequences where blocks go by length and are enough. Lengths evenly spread: the longest
    // one's blocks, or the work and a part of a block at the end. One split where more are not a
    // tenth better. Two instead of one, three draws of lengths each: 8 sequences of up to 16384 tokens of 512 rows 344, 376
    // and 446 against 441 to 446 us, all of 16384 465 against 444 to 460 (it takes two); up to 4096 153 to 165 against 132 to
    // 138, all of 4096 153 against 136; 37 of up to 4096, heads of 64, 93 to 105 against 84 to 94 (it takes one in both).
    const long long groups = std::max(1LL, (longest + kTreeTile - 1) / kTreeTile), sms = sm_count();
    const double tile = 3.6 * d / 128 * (t.pair ? 1.0 : 0.5), join = static_cast<double>(t.p.tiles) * t.p.tile_rows * d * 8 / 6.5e6;
    double best = -1;
    for (long long s = 1; s <= std::min(groups, 64LL) && t.p.tiles * s <= 16 * sms + t.p.tiles; ++s) {
        const double block = (groups + s - 1) / s * tile + (s > 1 ? 16 : 13);
        const bool whole = tree_order(B, t.p.tiles * s) && t.p.tiles * 5 >= sms * 4;
        const double equal = whole ? (t.p.tiles + sms - 1) / sms * (groups * tile + 13) : (t.p.tiles * s + sms - 1) / sms * block;
        const double spread = std::max(block, t.p.tiles * s * (block - (groups + s - 1) / s * tile / 2) / sms + block / 6);
        const double both = equal + (B > 1 ? spread : equal), cost = s > 1 ? both + 18 + join * s : 0.9 * both;
        if (best < 0 || cost < best) {
            best = cost;
            t.p.splits = static_cast<int>(s);
        }
    }
    return t;
}

template <typename T, int D, bool PAIR>
int launch_tree(const Mx4AttnArgs& a, const AttnPlan& p, int vec_q, cudaStream_t stream) {
    using Cfg = Mx4TreeCfg<D, PAIR>;
    auto kernel = mx4_tree_kernel<T, D, PAIR>;
    cudaError_t e = ensure_smem(kernel, Cfg::kSmemBytes);
    if (e != cudaSuccess) return static_cast<int>(e);
    e = launch_pdl(kernel, dim3(static_cast<unsigned>(p.tiles), p.splits), dim3(kTreeThreads), Cfg::kSmemBytes, stream, a, vec_q,
                   tree_order(a.B, p.tiles * p.splits) ? sm_count() : 0);
    if (e == cudaSuccess && p.splits > 1) {
        const unsigned rows = static_cast<unsigned>(a.B * a.tq * a.hq);
        const int wide = p.splits > 16;
        e = launch_pdl(mx4_attn_join_kernel<T, D>, dim3(wide ? rows : (rows + 7) / 8), dim3(256), 0, stream, a, p.tile_rows, wide);
    }
    return static_cast<int>(e);
}

template <typename T>
int run_tree(const Mx4AttnArgs& a, int d, const TreePlan& t, cudaStream_t stream) {
    if (!t.tensor) return run_attention<T, true>(a, d, t.p, stream);
    const int vec_q = aligned16(a.q) && (a.qsb | a.qst | a.qsh) % 8 == 0;
    if (d == 128) return t.pair ? launch_tree<T, 128, true>(a, t.p, vec_q, stream) : launch_tree<T, 128, false>(a, t.p, vec_q, stream);
    return t.pair ? launch_tree<T, 64, true>(a, t.p, vec_q, stream) : launch_tree<T, 64, false>(a, t.p, vec_q, stream);
}

}  // namespace

CONVROT_API size_t ck_mx4_tree_attention_workspace_size(int B, int tq, int hq, int hkv, int d, long long longest) {
    if (B <= 0 || tq <= 0 || hkv <= 0 || hq <= 0 || hq % hkv || d <= 0) return 0;
    const AttnPlan p = tree_plan(B, tq, hq, hkv, d, longest).p;
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
    const TreePlan t = tree_plan(B, tq, hq, hkv, d, longest);
    const AttnPlan& p = t.p;
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
    if (dtype == 1) return run_tree<__nv_bfloat16>(a, d, t, st);
    return run_tree<__half>(a, d, t, st);
}
