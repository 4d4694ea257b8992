// Attention of the newest tokens' queries over the paged MX4 cache.
//
// Included by mx4.cu. For one sequence and cache head, the tq * (hq / hkv) query
// rows that read it are taken together (16 or 32 a block), so the cache is read
// once for all of them; the sequence is split over blocks, and each warp of a
// block walks its own chunks of 32 tokens with a running maximum and sum. Warps
// are joined through shared memory, splits by mx4_attn_join_kernel.
//
// Rotated cache: q k = (H q) (H k), so the query rows are rotated once, and the
// output, a mean of rotated values, is rotated back at the end.
//
// Products run on mma.m16n8k16 (f16 operands, fp32 sums; the contraction over a
// token's channels and the one over tokens are too small a share of the work for
// more). A code is an f16 value exactly.
//   Scores: one MMA pair per block of 32 channels, its result times the block's
//   scale in fp32. Query rows are f16 times a power of two that brings the row's
//   largest value to 2^8.
//   Values: a token's codes times 2^(E_b - E), E the token's largest scale
//   exponent, are f16 values exactly (down to 2^-24 of the token's largest); the
//   rest, 2^E, goes to the probabilities: the numerator's weights are
//   2^(s + E - max(s + E)), with a maximum of their own, so that they are f16
//   values in [0, 1] whatever the values' range. The denominator keeps the usual
//   weights 2^(s - max s) in fp32.
//
// Columns. The contraction's order is free, so a thread's operands are whole
// words of codes: in a tile of 8 tokens column c is token (c >> 1) + 4 (c & 1); a
// thread (g = lane / 4, t = lane % 4) takes word t of each block of its token for
// the scores, and word g (8 channels) of tokens t and t + 4 for the values, whose
// nibbles are interleaved so that one conversion gives both tokens' value of a
// channel. 16-byte chunks of a token are XORed so that neither read meets a bank
// conflict.
#pragma once

namespace convrot {

struct Mx4AttnArgs {
    const void* q;
    long long qsb, qst, qsh;       // strides of the query in elements: sequence, token, head
    const uint8_t* codes;
    const uint8_t* scales;
    const int* table;              // [B, table_ld] page numbers
    long long table_ld;
    long long cap;                 // tokens a table row holds
    const int* lens;
    void* out;
    float* part;                   // per (tile, split, row): D floats ...
    float2* part_ml;               // ... and {maximum, sum}
    int B, tq, hq, hkv, page_bits, pages, group, row_tiles, splits;
    float scale;                   // softmax scale times log2(e)
};

constexpr int kMx4AttnWarps = 4;
constexpr int kMx4AttnChunk = 32;              // tokens a warp takes at a time
constexpr int kMx4AttnGroup = kMx4AttnWarps * kMx4AttnChunk;   // tokens a block takes at a time

template <int D, int MT>
struct Mx4AttnCfg {
    static constexpr int kRows = 16 * MT;
    static constexpr int kCodeBytes = kMx4AttnChunk * D / 2;
    static constexpr int kScaleSlot = D == 256 ? 8 : 4;           // bytes kept of a token's scales
    static constexpr int kScaleBytes = kMx4AttnChunk * kScaleSlot;
    static constexpr int kStageBytes = 2 * kCodeBytes + 2 * kScaleBytes + kMx4AttnChunk * 4;   // + the tokens' places
    static constexpr int kStages = 3;
    static constexpr int kBlocks = D / 32;
    static constexpr int kTableBytes = kMx4AttnChunk * (kBlocks * 4 + kBlocks * 2 + 8);
    static constexpr int kWarpBytes = kStages * kStageBytes + kTableBytes;
    static constexpr int kQStride = D * 2 + 64;                   // bytes; + 64: two rows in distinct banks
    static constexpr int kQBytes = kRows * kQStride;
    static constexpr int kPartStride = D + 4;                     // floats of a joined row
    static constexpr int kPartBytes = kMx4AttnWarps * kRows * kPartStride * 4;
    static constexpr int kRing = kMx4AttnWarps * kWarpBytes;
    static constexpr int kSmemBytes = kQBytes + (kRing > kPartBytes ? kRing : kPartBytes);
};

// Chunk position of a token's 16-byte chunk c.
template <int D>
__device__ __forceinline__ int mx4_chunk_pos(int tok, int c) {
    if constexpr (D == 64) return c ^ ((tok >> 2) & 1);
    if constexpr (D == 128) return c ^ ((tok & 2) | ((tok >> 2) & 1));
    return c ^ (((tok & 3) << 1) | ((tok >> 2) & 1));
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Four bytes of code pairs to four f16 pairs.
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 c0, c1, c2, c3;\n\t"
        "mov.b32 {c0, c1, c2, c3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, c0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, c1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, c3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}

__device__ __forceinline__ uint32_t hmul2_bits(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

__device__ __forceinline__ uint32_t f16x2_bits(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    uint32_t r;
    memcpy(&r, &h, 4);
    return r;
}

template <int BYTES>
__device__ __forceinline__ void cp_async_small(void* dst, const void* src, bool held) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;"
                 :: "r"(smem_u32(dst)), "l"(src), "n"(BYTES), "r"(held ? BYTES : 0) : "memory");
}

// Chunks [first, end) of 32 tokens of a sequence of `n` tokens that `split` of
// `splits` takes: whole groups of a block, evenly.
__device__ __forceinline__ int mx4_split_groups(int n, int splits) {
    const int groups = (n + kMx4AttnGroup - 1) / kMx4AttnGroup;
    return (groups + splits - 1) / splits;
}

template <typename T, int D, int MT>
__global__ void __launch_bounds__(kMx4AttnWarps * 32, MT == 1 && D <= 128 ? 3 : 2)
mx4_attn_kernel(Mx4AttnArgs a) {
    using Cfg = Mx4AttnCfg<D, MT>;
    constexpr int kB = Cfg::kBlocks, kR16 = D / 32;               // blocks; 16-byte chunks of a token
    extern __shared__ __align__(128) unsigned char mx4att[];
    __shared__ float row_scale[Cfg::kRows], pm[kMx4AttnWarps][Cfg::kRows], pl[kMx4AttnWarps][Cfg::kRows];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int tile = blockIdx.x, split = blockIdx.y;
    const int rt = tile % a.row_tiles, hk = tile / a.row_tiles % a.hkv, b = tile / a.row_tiles / a.hkv;
    const int per_head = a.hq / a.hkv, rows_all = a.tq * per_head, row0 = rt * Cfg::kRows;
    const int rows = min(Cfg::kRows, rows_all - row0);
    griddep_wait();
    griddep_launch_dependents();
    const int n = max(0, static_cast<int>(min(static_cast<long long>(a.lens[b]), a.cap)));
    const int per_split = mx4_split_groups(n, a.splits) * kMx4AttnWarps;      // chunks
    const int chunks = (n + kMx4AttnChunk - 1) / kMx4AttnChunk;
    const int c_begin = split * per_split, c_end = min(chunks, c_begin + per_split);
    if (a.splits > 1 && c_begin >= c_end) return;                 // (the join knows how many splits hold tokens)

    unsigned char* q_smem = mx4att;
    unsigned char* ring = mx4att + Cfg::kQBytes + warp * Cfg::kWarpBytes;
    float* kf = reinterpret_cast<float*>(ring + Cfg::kStages * Cfg::kStageBytes);          // [blocks][32]
    float2* info = reinterpret_cast<float2*>(kf + kB * kMx4AttnChunk);                     // [32] {0 or -inf, E}
    __half* vf = reinterpret_cast<__half*>(info + kMx4AttnChunk);                          // [blocks][32]
    // a token's place in the factor tables: columns 2t and 2t + 1 next to each other
    const int my_pos = (lane & ~7) + 2 * (lane & 3) + ((lane >> 2) & 1);

    // ---------------- the pipeline of this warp's chunks
    const int* table = a.table + b * a.table_ld;
    auto page_of = [&](int chunk) -> int {                        // page of this lane's token, -1: none
        const int j = chunk * kMx4AttnChunk + lane;
        return chunk < c_end && j < n ? __ldg(table + (j >> a.page_bits)) : -1;
    };
    const uint32_t v_off = static_cast<uint32_t>(a.hkv) << a.page_bits;       // from a key's place to its value's
    auto issue = [&](int stage, int chunk, int page) {
        unsigned char* st = ring + stage * Cfg::kStageBytes;
        const bool held = page >= 0 && page < a.pages;
        const uint32_t off = (chunk * kMx4AttnChunk + lane) & ((1 << a.page_bits) - 1);
        const uint32_t place = held ? (((static_cast<uint32_t>(page) * 2) * a.hkv + hk) << a.page_bits) + off : 0xFFFFFFFFu;
        #pragma unroll
        for (int i = 0; i < kR16; ++i) {
            const int tok = (i * 32 + lane) / kR16, c = (i * 32 + lane) % kR16;
            const uint32_t p = __shfl_sync(0xFFFFFFFFu, place, tok);
            const bool h = p != 0xFFFFFFFFu;
            const uint8_t* src = a.codes + (h ? static_cast<size_t>(p) * (D / 2) + c * 16 : 0);
            const uint8_t* vsrc = h ? src + static_cast<size_t>(v_off) * (D / 2) : a.codes;
            unsigned char* dst = st + tok * (D / 2) + mx4_chunk_pos<D>(tok, c) * 16;
            cp_async16(dst, src, h);
            cp_async16(dst + Cfg::kCodeBytes, vsrc, h);
        }
        // (heads of 64 have two scale bytes: the aligned word that holds them)
        const size_t sp = held ? (D == 64 ? static_cast<size_t>(place & ~1u) * 2 : static_cast<size_t>(place) * kB) : 0;
        const size_t svp = held ? (D == 64 ? static_cast<size_t>((place + v_off) & ~1u) * 2 : static_cast<size_t>(place + v_off) * kB) : 0;
        unsigned char* sc = st + 2 * Cfg::kCodeBytes + lane * Cfg::kScaleSlot;
        cp_async_small<Cfg::kScaleSlot>(sc, a.scales + sp, held);
        cp_async_small<Cfg::kScaleSlot>(sc + Cfg::kScaleBytes, a.scales + svp, held);
        reinterpret_cast<uint32_t*>(st + 2 * Cfg::kCodeBytes + 2 * Cfg::kScaleBytes)[lane] = place;
    };
    int ci = c_begin + warp, ahead = ci;                          // chunk at work, next chunk to load
    int page = page_of(ahead);
    #pragma unroll
    for (int s = 0; s < Cfg::kStages - 1; ++s) {
        if (ahead < c_end) issue(s, ahead, page);
        cp_async_commit();
        ahead += kMx4AttnWarps;
        page = page_of(ahead);
    }

    // ---------------- query rows: rotated, scaled to f16
    {
        __shared__ float qrow[kMx4AttnWarps][D];                  // (the ring's space is in use: a row at a time)
        for (int r = warp; r < Cfg::kRows; r += kMx4AttnWarps) {
            float* v = qrow[warp];
            const int row = row0 + r;
            if (r < rows) {
                const T* q = static_cast<const T*>(a.q) + b * a.qsb + (row / per_head) * a.qst +
                             (hk * per_head + row % per_head) * a.qsh;
                for (int i = lane; i < D; i += 32) v[i] = mx4_to_f32(q[i]);
            } else {
                for (int i = lane; i < D; i += 32) v[i] = 0.0f;
            }
            __syncwarp();
            for (int st = 1; st < a.group; st *= 4) {
                for (int i = lane; i < D / 4; i += 32) {
                    float* p = v + (i / st) * 4 * st + i % st;
                    h4(p[0], p[st], p[2 * st], p[3 * st]);
                }
                __syncwarp();
            }
            const float f = a.group == 16 ? 0.25f : a.group == 64 ? 0.125f : a.group == 256 ? 0.0625f : 1.0f;
            float top = 0.0f;
            for (int i = lane; i < D; i += 32) top = fmaxf(top, fabsf(v[i]));
            #pragma unroll
            for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
            // 2^(8 - exponent of the row's largest value), within fp32's normal range
            const int e = static_cast<int>(__float_as_uint(top) >> 23);
            const int up = top > 0.0f ? min(max(135 - e, -120), 120) : 0;
            const float to_f16 = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
            if (lane == 0) row_scale[r] = a.scale * f * __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
            __half* dst = reinterpret_cast<__half*>(q_smem + r * Cfg::kQStride);
            for (int i = lane; i < D; i += 32) dst[i] = __float2half_rn(v[i] * to_f16);
            __syncwarp();
        }
    }
    __syncthreads();

    float o[MT][D / 8][4];
    float m[MT][2], mn[MT][2], l[MT][2], rs[MT][2];
    int vis[MT][2];                                               // tokens a row sees
    #pragma unroll
    for (int i = 0; i < MT; ++i) {
        #pragma unroll
        for (int j = 0; j < D / 8; ++j)
            #pragma unroll
            for (int e = 0; e < 4; ++e) o[i][j][e] = 0.0f;
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = 16 * i + 8 * h + g;
            m[i][h] = mn[i][h] = -INFINITY;
            l[i][h] = 0.0f;
            rs[i][h] = row_scale[r];
            vis[i][h] = r < rows ? n - a.tq + (row0 + r) / per_head + 1 : 0;
        }
    }
    const int sees_all = n - a.tq + row0 / per_head + 1;          // tokens that every row of the tile sees

    for (int it = 0; ci < c_end; ci += kMx4AttnWarps, ++it) {
        if (ahead < c_end) issue((it + Cfg::kStages - 1) % Cfg::kStages, ahead, page);
        cp_async_commit();
        ahead += kMx4AttnWarps;
        page = page_of(ahead);
        cp_async_wait<Cfg::kStages - 1>();
        __syncwarp();
        const unsigned char* st = ring + (it % Cfg::kStages) * Cfg::kStageBytes;
        const unsigned char* vcodes = st + Cfg::kCodeBytes;
        // this lane's token: factors of its keys and values
        {
            const unsigned char* sc = st + 2 * Cfg::kCodeBytes + lane * Cfg::kScaleSlot;
            const uint32_t place = reinterpret_cast<const uint32_t*>(st + 2 * Cfg::kCodeBytes + 2 * Cfg::kScaleBytes)[lane];
            uint32_t ks[2], vs[2];
            ks[0] = *reinterpret_cast<const uint32_t*>(sc);
            vs[0] = *reinterpret_cast<const uint32_t*>(sc + Cfg::kScaleBytes);
            if constexpr (D == 64) {
                ks[0] >>= 16 * (place & 1);
                vs[0] >>= 16 * ((place + v_off) & 1);
            }
            if constexpr (D == 256) {
                ks[1] = *reinterpret_cast<const uint32_t*>(sc + 4);
                vs[1] = *reinterpret_cast<const uint32_t*>(sc + Cfg::kScaleBytes + 4);
            }
            int top = 0;
            #pragma unroll
            for (int i = 0; i < kB; ++i) {
                const uint32_t ek = (ks[i / 4] >> (8 * (i % 4))) & 255u;
                const int ev = (vs[i / 4] >> (8 * (i % 4))) & 255u;
                kf[i * 32 + my_pos] = mx4_scale_value(ek);
                if (ev != 255) top = max(top, ev);
            }
            #pragma unroll
            for (int i = 0; i < kB; ++i) {
                const int ev = (vs[i / 4] >> (8 * (i % 4))) & 255u;
                const int d = max(ev - top, -126);
                vf[i * 32 + my_pos] = ev == 255 ? __ushort_as_half(0x7FFF) : __float2half_rn(__uint_as_float(static_cast<uint32_t>(127 + d) << 23));
            }
            info[my_pos] = place != 0xFFFFFFFFu ? make_float2(0.0f, static_cast<float>(top - 127)) : make_float2(-INFINITY, 0.0f);
        }
        __syncwarp();

        // ---------------- scores
        float s[MT][4][4];
        #pragma unroll
        for (int i = 0; i < MT; ++i)
            #pragma unroll
            for (int c = 0; c < 4; ++c)
                #pragma unroll
                for (int e = 0; e < 4; ++e) s[i][c][e] = 0.0f;
        const int ktok = (g >> 1) + 4 * (g & 1);
        #pragma unroll
        for (int blk = 0; blk < kB; ++blk) {
            uint4 qa[MT][2];
            #pragma unroll
            for (int i = 0; i < MT; ++i)
                #pragma unroll
                for (int h = 0; h < 2; ++h)
                    qa[i][h] = *reinterpret_cast<const uint4*>(q_smem + (16 * i + 8 * h + g) * Cfg::kQStride + blk * 64 + t4 * 16);
            #pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int tok = 8 * c + ktok;
                const uint32_t w = *reinterpret_cast<const uint32_t*>(st + tok * (D / 2) + mx4_chunk_pos<D>(tok, blk) * 16 + t4 * 4);
                uint32_t h[4];
                codes_to_f16(w, h);
                const float2 f = *reinterpret_cast<const float2*>(kf + blk * 32 + 8 * c + 2 * t4);
                #pragma unroll
                for (int i = 0; i < MT; ++i) {
                    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    mma_f16(acc, qa[i][0].x, qa[i][1].x, qa[i][0].y, qa[i][1].y, h[0], h[1]);
                    mma_f16(acc, qa[i][0].z, qa[i][1].z, qa[i][0].w, qa[i][1].w, h[2], h[3]);
                    s[i][c][0] = fmaf(acc[0], f.x, s[i][c][0]);
                    s[i][c][1] = fmaf(acc[1], f.y, s[i][c][1]);
                    s[i][c][2] = fmaf(acc[2], f.x, s[i][c][2]);
                    s[i][c][3] = fmaf(acc[3], f.y, s[i][c][3]);
                }
            }
        }

        // ---------------- weights
        float4 tk[4];                                             // {0 or -inf, E} of tokens t and t + 4 of each tile
        #pragma unroll
        for (int c = 0; c < 4; ++c) tk[c] = *reinterpret_cast<const float4*>(info + 8 * c + 2 * t4);
        uint32_t p[MT][4][2];                                     // numerator weights, f16 pairs: tile, row half
        const bool cut = (ci + 1) * kMx4AttnChunk > sees_all;
        bool moved = false;
        float fn[MT][2];
        #pragma unroll
        for (int i = 0; i < MT; ++i)
            #pragma unroll
            for (int h = 0; h < 2; ++h) {
                float x[8], top = -INFINITY, topn = -INFINITY;
                #pragma unroll
                for (int c = 0; c < 4; ++c) {
                    x[2 * c] = fmaf(s[i][c][2 * h], rs[i][h], tk[c].x);
                    x[2 * c + 1] = fmaf(s[i][c][2 * h + 1], rs[i][h], tk[c].z);
                    if (cut) {
                        const int j = ci * kMx4AttnChunk + 8 * c + t4;
                        if (j >= vis[i][h]) x[2 * c] = -INFINITY;
                        if (j + 4 >= vis[i][h]) x[2 * c + 1] = -INFINITY;
                    }
                    top = fmaxf(top, fmaxf(x[2 * c], x[2 * c + 1]));
                    topn = fmaxf(topn, fmaxf(x[2 * c] + tk[c].y, x[2 * c + 1] + tk[c].w));
                }
                #pragma unroll
                for (int w = 1; w < 4; w *= 2) {
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, w));
                    topn = fmaxf(topn, __shfl_xor_sync(0xFFFFFFFFu, topn, w));
                }
                const float m2 = fmaxf(m[i][h], top), mn2 = fmaxf(mn[i][h], topn);
                const float base = m2 == -INFINITY ? 0.0f : m2, basen = mn2 == -INFINITY ? 0.0f : mn2;
                l[i][h] *= ex2(m[i][h] - base);
                fn[i][h] = ex2(mn[i][h] - basen);
                moved |= mn2 != mn[i][h];
                m[i][h] = m2;
                mn[i][h] = mn2;
                #pragma unroll
                for (int c = 0; c < 4; ++c) {
                    l[i][h] += ex2(x[2 * c] - base) + ex2(x[2 * c + 1] - base);
                    p[i][c][h] = f16x2_bits(ex2(x[2 * c] + (tk[c].y - basen)), ex2(x[2 * c + 1] + (tk[c].w - basen)));
                }
            }
        if (__any_sync(0xFFFFFFFFu, moved)) {
            #pragma unroll
            for (int i = 0; i < MT; ++i)
                #pragma unroll
                for (int j = 0; j < D / 8; ++j) {
                    o[i][j][0] *= fn[i][0];
                    o[i][j][1] *= fn[i][0];
                    o[i][j][2] *= fn[i][1];
                    o[i][j][3] *= fn[i][1];
                }
        }

        // ---------------- values
        #pragma unroll
        for (int u = 0; u < 2; ++u) {
            #pragma unroll
            for (int hf = 0; hf < D / 64; ++hf) {
                const int blk = 2 * hf + (g >> 2);
                uint32_t lo[2], hi[2], f[2];
                #pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int tok = 8 * (2 * u + x) + t4;
                    const uint32_t wa = *reinterpret_cast<const uint32_t*>(vcodes + tok * (D / 2) + mx4_chunk_pos<D>(tok, blk) * 16 + (g & 3) * 4);
                    const uint32_t wb = *reinterpret_cast<const uint32_t*>(vcodes + (tok + 4) * (D / 2) + mx4_chunk_pos<D>(tok + 4, blk) * 16 + (g & 3) * 4);
                    lo[x] = (wa & 0x0F0F0F0Fu) | ((wb << 4) & 0xF0F0F0F0u);
                    hi[x] = ((wa >> 4) & 0x0F0F0F0Fu) | (wb & 0xF0F0F0F0u);
                    f[x] = *reinterpret_cast<const uint32_t*>(vf + blk * 32 + 8 * (2 * u + x) + 2 * t4);
                }
                uint32_t e0[4], e1[4], d0[4], d1[4];
                codes_to_f16(lo[0], e0);
                codes_to_f16(lo[1], e1);
                codes_to_f16(hi[0], d0);
                codes_to_f16(hi[1], d1);
                #pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t b0 = hmul2_bits(e0[k], f[0]), b1 = hmul2_bits(e1[k], f[1]);
                    const uint32_t c0 = hmul2_bits(d0[k], f[0]), c1 = hmul2_bits(d1[k], f[1]);
                    #pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        mma_f16(o[i][8 * hf + 2 * k], p[i][2 * u][0], p[i][2 * u][1], p[i][2 * u + 1][0], p[i][2 * u + 1][1], b0, b1);
                        mma_f16(o[i][8 * hf + 2 * k + 1], p[i][2 * u][0], p[i][2 * u][1], p[i][2 * u + 1][0], p[i][2 * u + 1][1], c0, c1);
                    }
                }
            }
        }
        __syncwarp();
    }
    cp_async_wait<0>();
    __syncthreads();

    // ---------------- join the warps
    float* part = reinterpret_cast<float*>(mx4att + Cfg::kQBytes);
    #pragma unroll
    for (int i = 0; i < MT; ++i)
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = 16 * i + 8 * h + g;
            float sum = l[i][h];
            sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
            sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
            const float f = m[i][h] == -INFINITY ? 0.0f : ex2(mn[i][h] - m[i][h]);
            if (t4 == 0) {
                pm[warp][r] = m[i][h];
                pl[warp][r] = sum;
            }
            float* dst = part + (warp * Cfg::kRows + r) * Cfg::kPartStride;
            #pragma unroll
            for (int j = 0; j < D / 8; ++j)
                #pragma unroll
                for (int e = 0; e < 2; ++e)
                    dst[64 * (j / 8) + 8 * (2 * t4 + e) + (j % 8)] = o[i][j][2 * h + e] * f;
        }
    __syncthreads();
    float* joined = part;                                          // warp 0's rows become the block's
    for (int i = tid; i < rows * D; i += kMx4AttnWarps * 32) {
        const int r = i / D, c = i % D;
        float top = -INFINITY;
        #pragma unroll
        for (int w = 0; w < kMx4AttnWarps; ++w) top = fmaxf(top, pm[w][r]);
        float sum = 0.0f, acc = 0.0f;
        #pragma unroll
        for (int w = 0; w < kMx4AttnWarps; ++w) {
            const float f = pm[w][r] == -INFINITY ? 0.0f : ex2(pm[w][r] - top);
            sum += f * pl[w][r];
            acc += f * part[(w * Cfg::kRows + r) * Cfg::kPartStride + c];
        }
        if (a.splits > 1) {
            const size_t at = (static_cast<size_t>(tile) * a.splits + split) * Cfg::kRows + r;
            a.part[at * D + c] = acc;
            if (c == 0) a.part_ml[at] = make_float2(top, sum);
        } else {
            joined[r * Cfg::kPartStride + c] = sum == 0.0f ? 0.0f : acc / sum;
        }
    }
    if (a.splits > 1) return;
    __syncthreads();
    for (int r = warp; r < rows; r += kMx4AttnWarps) {
        float* v = joined + r * Cfg::kPartStride;
        for (int st = 1; st < a.group; st *= 4) {
            for (int i = lane; i < D / 4; i += 32) {
                float* p = v + (i / st) * 4 * st + i % st;
                h4(p[0], p[st], p[2 * st], p[3 * st]);
            }
            __syncwarp();
        }
        const float f = a.group == 16 ? 0.25f : a.group == 64 ? 0.125f : a.group == 256 ? 0.0625f : 1.0f;
        const int row = row0 + r;
        T* out = static_cast<T*>(a.out) + ((static_cast<size_t>(b) * a.tq + row / per_head) * a.hq + hk * per_head + row % per_head) * D;
        for (int i = lane; i < D; i += 32) out[i] = mx4_from_f32<T>(v[i] * f);
    }
}

// Joins a row's splits, rotates back and rounds. One block a row, a thread a channel.
template <typename T, int D>
__global__ void __launch_bounds__(D) mx4_attn_join_kernel(Mx4AttnArgs a, int tile_rows) {
    __shared__ float v[D];
    griddep_wait();
    griddep_launch_dependents();
    const int per_head = a.hq / a.hkv, rows_all = a.tq * per_head;
    const int row = blockIdx.x % rows_all, hk = blockIdx.x / rows_all % a.hkv, b = blockIdx.x / rows_all / a.hkv;
    const int n = max(0, static_cast<int>(min(static_cast<long long>(a.lens[b]), a.cap)));
    const int per_split = mx4_split_groups(n, a.splits) * kMx4AttnGroup;
    const int held = per_split ? (n + per_split - 1) / per_split : 0;          // splits that hold tokens
    const size_t at = ((static_cast<size_t>(b) * a.hkv + hk) * a.row_tiles + row / tile_rows) * a.splits * tile_rows + row % tile_rows;
    float top = -INFINITY;
    for (int s = 0; s < held; ++s) top = fmaxf(top, a.part_ml[at + static_cast<size_t>(s) * tile_rows].x);
    float sum = 0.0f, acc = 0.0f;
    for (int s = 0; s < held; ++s) {
        const size_t i = at + static_cast<size_t>(s) * tile_rows;
        const float2 ml = a.part_ml[i];
        const float f = ml.x == -INFINITY ? 0.0f : ex2(ml.x - top);
        sum += f * ml.y;
        acc += f * a.part[i * D + threadIdx.x];
    }
    v[threadIdx.x] = sum == 0.0f ? 0.0f : acc / sum;
    __syncthreads();
    mx4_rotate_shared(v, D, a.group, threadIdx.x, D);
    T* out = static_cast<T*>(a.out) + ((static_cast<size_t>(b) * a.tq + row / per_head) * a.hq + hk * per_head + row % per_head) * D;
    out[threadIdx.x] = mx4_from_f32<T>(v[threadIdx.x]);
}

}  // namespace convrot
