// C entries of the rotary positions: on their own, and on the way into the paged MX4
// cache. Conventions of include/convrot_b200.h.
#include <algorithm>

#include "mx4_host.cuh"
#include "mx4_cache.cuh"
#include "rope.cuh"
#include "mx4_cache_rope.cuh"

#define CONVROT_API extern "C" __attribute__((visibility("default")))

using namespace convrot;

namespace {

// Fills `r`; `rot` pairs must fit a head of D channels.
int rope_args(RopeArgs& r, const void* positions, int pos_type, long long p_batch, long long p_token, long long p_axis, const void* freqs,
              const int* sections, int axes, int interleaved, int inverse, int D) {
    if (axes <= 0 || axes > kRopeMostAxes) return fail("positions must have 1 to 8 axes");
    if (!sections) return fail("null sections");
    if (pos_type < 0 || pos_type > 2) return fail("positions must be int32 (0), int64 (1) or f32 (2)");
    long long pairs = 0;
    for (int i = 0; i < axes; ++i) {
        if (sections[i] < 0) return fail("sections must not be negative");
        pairs += sections[i];
        if (2 * pairs > D) return fail("the sections hold more pairs than a head");
        r.ends[i] = static_cast<int>(pairs);
    }
    r.pos = positions;
    r.freqs = static_cast<const double*>(freqs);
    r.pb = p_batch;
    r.pt = p_token;
    r.pa = p_axis;
    r.pos_type = pos_type;
    r.pairs = static_cast<int>(pairs);
    r.axes = axes;
    r.interleaved = interleaved != 0;
    r.sign = inverse ? -1.0f : 1.0f;
    return 0;
}

int rope_pointers(const RopeArgs& r) {
    if (r.pairs && (!r.pos || !r.freqs)) return fail("null positions or frequencies");
    if (!aligned_to(r.pos, r.pos_type == 1 ? 8 : 4) || !aligned_to(r.freqs, 8)) return fail("positions or frequencies not aligned to their type");
    return 0;
}

// Chunks of 16 bytes: sections of whole chunks, every row on a 16-byte boundary.
bool whole_chunks(const RopeArgs& r, int D, size_t size, long long strides) {
    const int vp = static_cast<int>(16 / size);
    return r.pairs % vp == 0 && D % (2 * vp) == 0 && strides * static_cast<long long>(size) % 16 == 0;
}

template <typename T, int VP>
int launch_rope(const void* x, void* out, RopeShape s, const RopeArgs& r, cudaStream_t stream) {
    const long long chunks = s.D / (2 * VP);
    // heads a thread: all that leave one wave of blocks full (a token's angles serve a thread's heads)
    const long long places = static_cast<long long>(kRopeResident) * kRopeThreads * sm_count();
    s.runs = static_cast<int>(std::max(1LL, std::min(static_cast<long long>(s.H), places / std::max(1LL, s.tokens * chunks))));
    s.heads = (s.H + s.runs - 1) / s.runs;
    s.runs = (s.H + s.heads - 1) / s.heads;
    const long long per = chunks * s.runs;                        // threads of a token
    s.slice = static_cast<int>(std::max(1LL, std::min(s.tokens, (0x7FFFFFFFll - kRopeThreads) / per)));
    const long long rows = (s.tokens + s.slice - 1) / s.slice;
    if (rows > 65535 || per > 0x7FFFFFFFll - kRopeThreads) return fail("tensor too large");
    const dim3 grid(static_cast<unsigned>((s.slice * per + kRopeThreads - 1) / kRopeThreads), static_cast<unsigned>(rows));
    return static_cast<int>(launch_pdl(rope_kernel<T, VP>, grid, dim3(kRopeThreads), 0, stream, static_cast<const T*>(x), static_cast<T*>(out), s, r));
}

}  // namespace

CONVROT_API int ck_rope(const void* x, int dtype, long long x_batch, long long x_token, long long x_head, void* out, int B, int T, int H,
                        int D, const void* positions, int pos_type, long long p_batch, long long p_token, long long p_axis, const void* freqs,
                        const int* sections, int axes, int interleaved, int inverse, void* stream) {
    if (dtype < 0 || dtype > 2) return fail("dtype must be 0 (f32), 1 (bf16) or 2 (f16)");
    if (B < 0 || T < 0 || H < 0 || D <= 0 || D % 2) return fail("sizes must not be negative, D even");
    RopeArgs r;
    if (int rc = rope_args(r, positions, pos_type, p_batch, p_token, p_axis, freqs, sections, axes, interleaved, inverse, D)) return rc;
    const long long tokens = static_cast<long long>(B) * T;
    if (tokens == 0 || H == 0) return 0;
    if (tokens > (1ll << 62) / (static_cast<long long>(H) * D)) return fail("tensor too large");
    if (!x || !out) return fail("null pointer");
    if (int rc = rope_pointers(r)) return rc;
    if (!aligned_to(x, type_size(dtype)) || !aligned_to(out, type_size(dtype))) return fail("x or out is not aligned to its type");
    const RopeShape s{x_batch, x_token, x_head, tokens, T, H, D, 0, 0, 0};
    return with_type(dtype, [&](auto* t) {
        using E = std::remove_pointer_t<decltype(t)>;
        const bool wide = aligned16(x) && aligned16(out) && whole_chunks(r, D, sizeof(E), x_batch | x_token | x_head);
        if (wide) return launch_rope<E, 16 / sizeof(E)>(x, out, s, r, static_cast<cudaStream_t>(stream));
        return launch_rope<E, 1>(x, out, s, r, static_cast<cudaStream_t>(stream));
    });
}

CONVROT_API int ck_mx4_cache_append_rope(void* codes, void* scales, long long pages, int heads, int d, int page, int G, const void* q,
                                         const void* k, const void* v, int dtype, int q_heads, long long q_token, long long q_head,
                                         long long k_token, long long k_head, long long v_token, long long v_head, void* q_out,
                                         const void* slots, int T, const void* positions, int pos_type, long long p_token, long long p_axis,
                                         const void* freqs, const int* sections, int axes, int interleaved, void* stream) {
    if (int rc = check_cache(codes, scales, pages, heads, d, page, G)) return rc;
    if (T < 0 || q_heads < 0) return fail("T and the query heads must not be negative");
    if (dtype < 0 || dtype > 2) return fail("dtype must be 0 (f32), 1 (bf16) or 2 (f16)");
    RopeArgs r;
    if (int rc = rope_args(r, positions, pos_type, 0, p_token, p_axis, freqs, sections, axes, interleaved, 0, d)) return rc;
    if (T == 0) return 0;
    if (!k || !v || !slots || (q_heads && (!q || !q_out))) return fail("null pointer");
    if (int rc = rope_pointers(r)) return rc;
    const size_t size = type_size(dtype);
    if (!aligned_to(k, size) || !aligned_to(v, size) || !aligned_to(slots, 8)) return fail("keys, values or slots are not aligned to their type");
    if (q_heads && (!aligned_to(q, size) || !aligned_to(q_out, size))) return fail("queries are not aligned to their type");
    const Mx4CacheShape c{pages * page, heads, d, page_bits(page)};
    return with_type(dtype, [&](auto* t) {
        using E = std::remove_pointer_t<decltype(t)>;
        return with_head(d, G, [&](auto dim, auto g) {
            constexpr int D = decltype(dim)::value;
            const long long units = static_cast<long long>(T) * mx4_cache_units<D>(heads);
            long long q_items = static_cast<long long>(T) * q_heads;
            if (2 * units > kMx4MostUnits || q_items > 0x7FFFFFFFll - 4096) return fail("too many tokens in one call");
            Mx4AppendRope a{};
            a.q = q;
            a.k = k;
            a.v = v;
            a.q_out = q_out;
            a.qst = q_token; a.qsh = q_head; a.kst = k_token; a.ksh = k_head; a.vst = v_token; a.vsh = v_head;
            a.slots = static_cast<const long long*>(slots);
            a.codes = static_cast<uint8_t*>(codes);
            a.scales = static_cast<uint8_t*>(scales);
            a.tokens = T;
            a.hq = q_heads;
            a.units = static_cast<int>(units);
            // Few tokens: one launch, in small tasks, so that every warp has little to do (7 tokens of 32 query heads
            // on 8 of 128: 5.5 us; queries apart 9). Many: queries and values by the kernels that do nothing
            // else, which hold more loads (32768 tokens: 164 us; in one launch 178).
            const bool apart = (2 * units + q_items * D / 128) / 32 > 64LL * sm_count();
            cudaStream_t st = static_cast<cudaStream_t>(stream);
            if (apart && q_items) {
                const RopeShape shape{0, q_token, q_head, T, T, q_heads, D, 0, 0, 0};
                const bool wide = aligned16(q) && aligned16(q_out) && whole_chunks(r, d, sizeof(E), q_token | q_head);
                const int rc = wide ? launch_rope<E, 16 / sizeof(E)>(q, q_out, shape, r, st) : launch_rope<E, 1>(q, q_out, shape, r, st);
                if (rc) return rc;
                q_items = 0;
            }
            if (apart)
                if (int rc = run_cache_append(codes, scales, pages, heads, d, page, G, v, v, dtype, v_token, v_head, v_token, v_head, slots, T, true, st)) return rc;
            int size = 32;
            while (size > 8 && (2 * units + q_items * D / 128) / size < 4LL * sm_count()) size /= 2;
            a.size = size;
            a.k_tasks = static_cast<int>((units + size - 1) / size);
            a.v_tasks = apart ? 0 : a.k_tasks;
            a.tasks = a.k_tasks + a.v_tasks + static_cast<int>((q_items * D + 128 * size - 1) / (128 * size));
            const long long strides = k_token | k_head | v_token | v_head | (q_items ? q_token | q_head : 0);
            const bool wide = aligned16(k) && aligned16(v) && (!q_items || (aligned16(q) && aligned16(q_out))) && whole_chunks(r, d, sizeof(E), strides);
            const int smem = kMx4QuantWarps * Mx4Slab<float>::kBytes, blocks = (a.tasks + kMx4QuantWarps - 1) / kMx4QuantWarps;
            auto launch = [&](auto kernel) {
                cudaError_t e = ensure_smem(kernel, smem);
                if (e != cudaSuccess) return static_cast<int>(e);
                return static_cast<int>(launch_pdl(kernel, dim3(blocks), dim3(kMx4QuantWarps * 32), smem, st, a, c, r));
            };
            if (wide) return launch(mx4_cache_append_rope_kernel<E, D, decltype(g)::value, 16 / sizeof(E)>);
            return launch(mx4_cache_append_rope_kernel<E, D, decltype(g)::value, 1>);
        });
    });
}
