// Attention of the newest tokens' queries over the paged MX4 cache.
//
// Included by mx4.cu. For one sequence and cache head, the tq * (hq / hkv) query
// rows that read it are taken together (8, 16 or 32 a block), so the cache is read
// once for all of them; the sequence is split over blocks, and each warp of a
// block walks its own chunks of 32 tokens with a running maximum and sum. Warps
// are joined through shared memory; up to 8 splits of a sequence are a cluster and
// join over distributed shared memory where all blocks are resident at once, others
// by mx4_attn_join_kernel.
//
// Rotated cache: q k = (H q) (H k), so the query rows are rotated once, and the
// output, a mean of rotated values, is rotated back at the end.
//
// Products run on mma.m16n8k16 (f16 operands, fp32 sums) with the cache on the
// side of 16 and the query rows on the side of 8: S^T = K Q^T and O^T = V^T P^T.
// Few rows then waste nothing, and tcgen05 (128 rows at least) would. A code is an
// f16 value exactly.
//   Scores: two pairs of MMAs per block of 32 channels, their result times the
//   block's scale in fp32. Query rows are times a power of two that brings the row's
//   largest value to 2^8.
//   Values: a token's codes times 2^(E_b - E), E the token's largest scale
//   exponent, are f16 values exactly; the rest, 2^E, goes to the probabilities: the
//   numerator's weights are 2^((s - m) + (E - dn)), with a reference dn of their own, so
//   that they are f16 values whatever the values' range. The denominator keeps the
//   usual weights 2^(s - m) in fp32. (dn is relative to m: large scores would take the
//   bits of an E added to them.)
//   A weight is off by 2^-25 at most where the row's largest is 2^8 to 2^15. That is
//   relative to the token with the largest values: a channel block whose values are far
//   smaller would lose its own precision, so chunks with a block more than 2^8 below the
//   largest seen so far take fp32 products instead (three to four times as long).
// Rotated queries and numerator weights are the sum of two f16 values each (22 bits):
// with one, a seventh of the bf16 outputs and half of the f16 ones were rounded to
// a neighbour of the nearest value.
//
// Columns. The contraction's order is free, so a thread's operands are whole
// words of codes: in a tile of 8 tokens row r is token (r >> 1) + 4 (r & 1); a
// thread (g = lane / 4, t = lane % 4) takes word t of each block of its tokens for
// the scores, and word g (8 channels) of tokens t and t + 4 for the values, whose
// nibbles are interleaved so that one conversion gives both tokens' value of a
// channel. 16-byte chunks of a token are XORed so that neither read meets a bank
// conflict.
//
// Bound by issue: some 910 instructions a warp for 32 tokens of 128, 2.5 a cycle, half of
// them on the ALU pipe that converts codes (busy 51 %; tensor pipe 35 %). 16 sequences of
// 32768, 64 heads on 8 of 128: 181 us (3.2 TB/s of the cache; 146 us with one f16 term an
// operand); 64 of 4096, 32 heads on 32: 320 us (3.6 TB/s); 128 x 2048: 104 us (2.7 TB/s); one of
// 777: 7.8 us.
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
    float* part;                   // per (tile, split, row): the mean of the split's values, D floats ...
    float2* part_ml;               // ... and {reference, sum of weights}; in a tree's first split below zero: the row is written
    int B, tq, hq, hkv, page_bits, pages, group, row_tiles, splits;
    int clustered;                 // a sequence's splits are one cluster and join themselves
    float scale;                   // softmax scale times log2(e)
    // a tree of drafted tokens (TREE): node t of a sequence, one of its last nodes[b] tokens
    // (null: tq), sees those before them and the nodes that mask[b][t] names
    const uint8_t* mask;
    const int* nodes;
    long long mask_seq, mask_row;  // strides in bytes
};

// A sequence's nodes and the tokens before them (negative: nodes -context .. 0 do not exist).
struct Mx4Tree {
    int nodes, context;
    const uint8_t* mask;
    long long row;
    Mx4Tree() = default;
    __device__ __forceinline__ Mx4Tree(const Mx4AttnArgs& a, int b, int n) {
        nodes = a.nodes ? max(0, min(a.nodes[b], a.tq)) : a.tq;
        context = n - nodes;
        mask = a.mask + b * a.mask_seq;
        row = a.mask_row;
    }
    // Whether node t, one of the tree's, sees token j, one of the cache's.
    __device__ __forceinline__ bool sees(int t, int j) const { return j < context || mask[t * row + (j - context)] != 0; }
    // The same for any t and j, without a branch: several loads are then on their way at once.
    __device__ __forceinline__ bool sees_any(int t, int j) const {
        const int last = nodes - 1, from = j - context;
        if (last < 0) return false;
        const uint8_t named = __ldg(mask + min(t, last) * row + min(max(from, 0), last));
        return (t <= last) & ((from < 0) | ((from <= last) & (named != 0)));
    }
};

constexpr int kMx4AttnWarps = 4;
constexpr int kMx4MostSplits = 256;            // of one sequence
constexpr long long kMx4MostTokens = 0x7FFFFFFFll - 1023;      // of one sequence: positions, and the chunks and groups
                                                               // looked at beyond the last, fit 32 bits
constexpr float kMx4NoScore = -3.402823466e38f;        // a row's reference before its first score: the lowest finite
                                                       // value (-inf less it is -inf)
constexpr int kMx4NarrowBits = 8;              // blocks of values this many powers of two apart share f16 weights
constexpr int kMx4AttnChunk = 32;              // tokens a warp takes at a time
constexpr int kMx4AttnGroup = kMx4AttnWarps * kMx4AttnChunk;   // tokens a block takes at a time

// Blocks a multiprocessor holds, for the launch bound (registers) and the plan alike; `size`
// is rows / 8 * D. Two leave a thread 255 registers, four 128. Heads of 128, 8 rows: 180 us
// with four, 183 with three, 199 with five (16 x 32768); heads of 64, 8 rows: 119.5 with four,
// 121.8 with five (64 x 8192), 16 rows: 61 with four, 66 with three (37 up to 4096), 32 rows: 187
// with two, 197 with three, which spill (64 x 4096, 8 tokens); heads of 128, 16 rows: 154 with two, 156 with
// three (32 x 8192, 4 tokens); heads of 256, 8 rows: 176 with two, which is what shared memory
// holds, 195 planned for three (32 x 8192).
__host__ __device__ constexpr int mx4_attn_resident(int size) { return size <= 128 ? 4 : 2; }

template <int D, int NT>
struct Mx4AttnCfg {
    static constexpr int kRows = 8 * NT;
    static constexpr int kCodeBytes = kMx4AttnChunk * D / 2;
    static constexpr int kScaleSlot = D == 256 ? 8 : 4;           // bytes kept of a token's scales
    static constexpr int kScaleBytes = kMx4AttnChunk * kScaleSlot;
    static constexpr int kStageBytes = 2 * kCodeBytes + 2 * kScaleBytes + kMx4AttnChunk * 4;   // + the tokens' places
    static constexpr int kStages = 2;
    static constexpr int kBlocks = D / 32;
    static constexpr int kTableBytes = kMx4AttnChunk * (kBlocks * 4 + kBlocks * 2 + 8);
    static constexpr int kWarpBytes = kStages * kStageBytes + kTableBytes;
    static constexpr int kQStride = D * 2 + 64;                   // bytes; + 64: two rows in distinct banks
    static constexpr int kQBytes = 2 * kRows * kQStride;          // rows, then what their rounding to f16 left (first in fp32)
    static constexpr int kPartStride = D + 4;                     // floats of a joined row
    static constexpr int kPartBytes = kMx4AttnWarps * kRows * kPartStride * 4;
    static constexpr int kRing = kMx4AttnWarps * kWarpBytes;
    static constexpr int kSmemBytes = kQBytes + (kRing > kPartBytes ? kRing : kPartBytes);
    static constexpr int kResident = mx4_attn_resident(NT * D);
    // (with up to 2 KB of static memory and the 1 KB that the system takes a block)
    static_assert(kResident * (kSmemBytes + 3072) <= 228 * 1024, "the blocks that are planned for fit");
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

// 1 / x to about 2^-23, x a sum of weights (1 at least, unless none).
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same from a zero accumulator.
__device__ __forceinline__ void mma_f16_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
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

__device__ __forceinline__ float2 ld_shared_cluster_f2(uint32_t cluster_addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(cluster_addr) : "memory");
    return v;
}

template <int BYTES>
__device__ __forceinline__ void cp_async_small(void* dst, const void* src, bool held) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;"
                 :: "r"(smem_u32(dst)), "l"(src), "n"(BYTES), "r"(held ? BYTES : 0) : "memory");
}

// Groups of tokens of a sequence of `n` tokens, and those that each of `splits` takes.
__device__ __forceinline__ int mx4_groups(int n) { return (n + kMx4AttnGroup - 1) / kMx4AttnGroup; }
__device__ __forceinline__ int mx4_split_groups(int n, int splits) { return (mx4_groups(n) + splits - 1) / splits; }

// Transposes an 8 x 8 tile of 16-bit values held as an MMA fragment.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

template <typename T, int D, int NT, bool TREE = false>
__global__ void __launch_bounds__(kMx4AttnWarps * 32, Mx4AttnCfg<D, NT>::kResident)
mx4_attn_kernel(Mx4AttnArgs a) {
    using Cfg = Mx4AttnCfg<D, NT>;
    constexpr int kB = Cfg::kBlocks, kR16 = D / 32;               // blocks; 16-byte chunks of a token
    extern __shared__ __align__(128) unsigned char mx4att[];
    __shared__ float row_scale[Cfg::kRows], pm[kMx4AttnWarps][Cfg::kRows], pl[kMx4AttnWarps][Cfg::kRows];
    __shared__ float2 block_ml[Cfg::kRows];                       // {m, sum} of the block's rows
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int tile = blockIdx.x, split = blockIdx.y;
    const int rt = tile % a.row_tiles, hk = tile / a.row_tiles % a.hkv, b = tile / a.row_tiles / a.hkv;
    const int per_head = a.hq / a.hkv, rows_all = a.tq * per_head, row0 = rt * Cfg::kRows;
    const int rows = min(Cfg::kRows, rows_all - row0);
    griddep_wait();
    griddep_launch_dependents();
    // this warp's query rows (used after the first chunks' loads are on their way)
    constexpr int kRw = Cfg::kRows / kMx4AttnWarps;
    float qv[kRw][D / 32];
    #pragma unroll
    for (int k = 0; k < kRw; ++k) {
        const int r = warp * kRw + k, row = row0 + r;
        const T* q = static_cast<const T*>(a.q) + b * a.qsb + (row / per_head) * a.qst + (hk * per_head + row % per_head) * a.qsh;
        #pragma unroll
        for (int i = 0; i < D / 32; ++i) qv[k][i] = r < rows ? mx4_to_f32(q[lane + 32 * i]) : 0.0f;
    }
    const int n = max(0, static_cast<int>(min(static_cast<long long>(a.lens[b]), a.cap)));
    const int per_split = mx4_split_groups(n, a.splits) * kMx4AttnWarps;      // chunks
    const int chunks = (n + kMx4AttnChunk - 1) / kMx4AttnChunk;
    const int c_begin = split * per_split, c_end = min(chunks, c_begin + per_split);
    if (a.splits > 1 && !a.clustered && c_begin >= c_end) return; // (the join knows how many splits hold tokens)

    unsigned char* q_smem = mx4att;
    unsigned char* ring = mx4att + Cfg::kQBytes + warp * Cfg::kWarpBytes;
    float* kf = reinterpret_cast<float*>(ring + Cfg::kStages * Cfg::kStageBytes);          // [32][blocks]
    float2* info = reinterpret_cast<float2*>(kf + kB * kMx4AttnChunk);                     // [32] {0 or -inf, E}
    __half* vf = reinterpret_cast<__half*>(info + kMx4AttnChunk);                          // [blocks][32]
    // a token's place in the value factors: tokens t and t + 4 next to each other
    const int my_pos = (lane & ~7) + 2 * (lane & 3) + ((lane >> 2) & 1);

    // ---------------- the pipeline of this warp's chunks
    const int* table = a.table + b * a.table_ld;
    auto page_of = [&](int chunk) -> int {                        // page of this lane's token, -1: none
        const int j = chunk * kMx4AttnChunk + lane;
        return chunk < c_end && j < n ? __ldg(table + (j >> a.page_bits)) : -1;
    };
    const uint32_t v_off = static_cast<uint32_t>(a.hkv) << a.page_bits;       // from a key's place to its value's
    const size_t v_bytes = static_cast<size_t>(v_off) * (D / 2);
    // where this lane's 16 bytes of 512-byte step i go: the swizzle repeats every 8
    // tokens, in heads of 256 every second step
    const int copy_at = lane / kR16 * (D / 2) + mx4_chunk_pos<D>(lane / kR16, lane % kR16) * 16;
    auto copy_dst = [&](int i) { return (D == 256 && (i & 1) ? copy_at ^ 16 : copy_at) + i * 512; };
    auto issue = [&](int stage, int chunk, int page) {
        unsigned char* st = ring + stage * Cfg::kStageBytes;
        const bool held = page >= 0 && page < a.pages;
        const uint32_t off = (chunk * kMx4AttnChunk + lane) & ((1 << a.page_bits) - 1);
        const uint32_t place = held ? (((static_cast<uint32_t>(page) * 2) * a.hkv + hk) << a.page_bits) + off : 0xFFFFFFFFu;
        if (a.page_bits >= 5) {
            // the chunk lies in one page: its rows are contiguous, and the tokens that
            // exist come first
            const int count = __popc(__ballot_sync(0xFFFFFFFFu, held));
            const uint32_t first = __shfl_sync(0xFFFFFFFFu, place, 0);
            const uint8_t* src = a.codes + (count ? static_cast<size_t>(first) * (D / 2) + lane * 16 : 0);
            const uint8_t* vsrc = src + (count ? v_bytes : 0);
            unsigned char* dst = st;
            if (count == kMx4AttnChunk) {
                #pragma unroll
                for (int i = 0; i < kR16; ++i) {
                    cp_async16(dst + copy_dst(i), src + i * 512);
                    cp_async16(dst + copy_dst(i) + Cfg::kCodeBytes, vsrc + i * 512);
                }
            } else {
                #pragma unroll
                for (int i = 0; i < kR16; ++i) {
                    const bool h = (i * 32 + lane) / kR16 < count;
                    cp_async16(dst + copy_dst(i), h ? src + i * 512 : a.codes, h);
                    cp_async16(dst + copy_dst(i) + Cfg::kCodeBytes, h ? vsrc + i * 512 : a.codes, h);
                }
            }
        } else {
            #pragma unroll
            for (int i = 0; i < kR16; ++i) {
                const int tok = (i * 32 + lane) / kR16, c = (i * 32 + lane) % kR16;
                const uint32_t p = __shfl_sync(0xFFFFFFFFu, place, tok);
                const bool h = p != 0xFFFFFFFFu;
                const uint8_t* src = a.codes + (h ? static_cast<size_t>(p) * (D / 2) + c * 16 : 0);
                unsigned char* dst = st + copy_dst(i);
                cp_async16(dst, src, h);
                cp_async16(dst + Cfg::kCodeBytes, src + (h ? v_bytes : 0), h);
            }
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

    // ---------------- query rows: rotated in fp32, then f16 times a power of two
    {
        float* v = reinterpret_cast<float*>(q_smem) + warp * kRw * D;
        #pragma unroll
        for (int k = 0; k < kRw; ++k)
            #pragma unroll
            for (int i = 0; i < D / 32; ++i) v[k * D + lane + 32 * i] = qv[k][i];
        __syncwarp();
        for (int st = 1; st < a.group; st *= 4) {
            #pragma unroll
            for (int j = 0; j < kRw * D / 128 || j == 0; ++j) {
                const int i = lane + 32 * j;
                if (kRw * D < 128 && i >= kRw * D / 4) break;
                float* p = v + (i / st) * 4 * st + i % st;
                h4(p[0], p[st], p[2 * st], p[3 * st]);
            }
            __syncwarp();
        }
        const float f = a.group == 16 ? 0.25f : a.group == 64 ? 0.125f : a.group == 256 ? 0.0625f : 1.0f;
        float to_f16[kRw];
        #pragma unroll
        for (int k = 0; k < kRw; ++k) {
            float top = 0.0f;
            #pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                qv[k][i] = v[k * D + lane + 32 * i];
                top = fmaxf(top, fabsf(qv[k][i]));
            }
            #pragma unroll
            for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
            // 2^(8 - exponent of the row's largest value), within fp32's normal range
            const int e = static_cast<int>(__float_as_uint(top) >> 23);
            const int up = top > 0.0f ? min(max(135 - e, -120), 120) : 0;
            to_f16[k] = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
            if (lane == 0) row_scale[warp * kRw + k] = a.scale * f * __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
        }
        __syncthreads();                                          // the f16 rows take the place of every warp's fp32 rows
        #pragma unroll
        for (int k = 0; k < kRw; ++k) {
            __half* dst = reinterpret_cast<__half*>(q_smem + (warp * kRw + k) * Cfg::kQStride);
            #pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                const float x = qv[k][i] * to_f16[k];
                const __half hi = __float2half_rn(x);
                dst[lane + 32 * i] = hi;
                dst[Cfg::kRows * Cfg::kQStride / 2 + lane + 32 * i] = __float2half_rn(x - __half2float(hi));
            }
        }
    }
    __syncthreads();

    float o[NT][D / 16][4];                                       // channels g, g + 8 of each 16; rows 2t, 2t + 1
    float m[NT][2], dn[NT][2], l[NT][2], rs[NT][2];               // rows 2t, 2t + 1 of each 8
    #pragma unroll
    for (int i = 0; i < NT; ++i) {
        #pragma unroll
        for (int j = 0; j < D / 16; ++j)
            #pragma unroll
            for (int e = 0; e < 4; ++e) o[i][j][e] = 0.0f;
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = 8 * i + 2 * t4 + h;
            m[i][h] = kMx4NoScore;
            dn[i][h] = 0.0f;
            l[i][h] = 0.0f;
            rs[i][h] = row_scale[r];
        }
    }
    int sees_all = n - a.tq + row0 / per_head + 1;                // tokens that every row of the tile sees
    const Mx4Tree tree = TREE ? Mx4Tree(a, b, n) : Mx4Tree{};
    if constexpr (TREE) sees_all = (row0 + rows - 1) / per_head < tree.nodes ? tree.context : 0;   // (padding sees nothing)
    const int ktok = (g >> 1) + 4 * (g & 1);                      // this thread's token of each tile of 8
    int most_seen = 0;                                            // largest scale byte of the warp's values so far

    for (int it = 0; ci < c_end; ci += kMx4AttnWarps, ++it) {
        if (ahead < c_end) issue((it + Cfg::kStages - 1) % Cfg::kStages, ahead, page);
        cp_async_commit();
        ahead += kMx4AttnWarps;
        page = page_of(ahead);
        cp_async_wait<Cfg::kStages - 1>();
        __syncwarp();
        const unsigned char* st = ring + (it % Cfg::kStages) * Cfg::kStageBytes;
        const unsigned char* vcodes = st + Cfg::kCodeBytes;
        bool narrow = true;                                       // the chunk's blocks of values are near the largest
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
            int top = 0, low = 255;                               // (blocks of zeros have 0)
            float kv[kB];
            __half vv[kB];
            bool bad = false;                                     // a block of NaN
            #pragma unroll
            for (int i = 0; i < kB; ++i) {
                const uint32_t ek = (ks[i / 4] >> (8 * (i % 4))) & 255u;
                kv[i] = __uint_as_float(max(ek << 23, 0x00400000u));          // (0: the subnormal 2^-127)
                const int ev = (vs[i / 4] >> (8 * (i % 4))) & 255u;
                top = max(top, ev);
                low = min(low, ev ? ev : 255);
                bad |= ek == 255u;
            }
            bad |= top == 255;
            #pragma unroll
            for (int i = 0; i < kB; ++i) {
                const int ev = (vs[i / 4] >> (8 * (i % 4))) & 255u;
                vv[i] = __float2half_rn(__uint_as_float(static_cast<uint32_t>(max(ev - top + 127, 0)) << 23));
            }
            if (__any_sync(0xFFFFFFFFu, bad || top > most_seen || low < most_seen - kMx4NarrowBits)) {
                top = 0;
                #pragma unroll
                for (int i = 0; i < kB; ++i) {
                    const int ev = (vs[i / 4] >> (8 * (i % 4))) & 255u;
                    if (ev != 255) top = max(top, ev);
                    if (kv[i] == INFINITY) kv[i] = NAN;
                }
                #pragma unroll
                for (int i = 0; i < kB; ++i) {
                    const int ev = (vs[i / 4] >> (8 * (i % 4))) & 255u;
                    vv[i] = ev == 255 ? __ushort_as_half(0x7FFF) : __float2half_rn(__uint_as_float(static_cast<uint32_t>(max(ev - top + 127, 0)) << 23));
                }
                most_seen = max(most_seen, __reduce_max_sync(0xFFFFFFFFu, top));
                narrow = __reduce_min_sync(0xFFFFFFFFu, low) >= most_seen - kMx4NarrowBits;
            }
            #pragma unroll
            for (int i = 0; i < kB; i += 2) *reinterpret_cast<float2*>(kf + lane * kB + i) = make_float2(kv[i], kv[i + 1]);
            #pragma unroll
            for (int i = 0; i < kB; ++i) vf[i * 32 + my_pos] = vv[i];
            info[lane] = place != 0xFFFFFFFFu ? make_float2(0.0f, static_cast<float>(top - 127)) : make_float2(-INFINITY, 0.0f);
        }
        __syncwarp();

        // ---------------- scores: tiles of 16 tokens (rows g, g + 8) by 8 query rows
        float s[NT][2][4];
        #pragma unroll
        for (int i = 0; i < NT; ++i)
            #pragma unroll
            for (int c = 0; c < 2; ++c)
                #pragma unroll
                for (int e = 0; e < 4; ++e) s[i][c][e] = 0.0f;
        float fk[4][kB];                                          // the scales of this thread's four tokens
        #pragma unroll
        for (int c = 0; c < 4; ++c)
            #pragma unroll
            for (int i = 0; i < kB; i += (kB < 4 ? 2 : 4)) {
                if constexpr (kB < 4) {
                    const float2 x = *reinterpret_cast<const float2*>(kf + (8 * c + ktok) * kB + i);
                    fk[c][i] = x.x; fk[c][i + 1] = x.y;
                } else {
                    const float4 x = *reinterpret_cast<const float4*>(kf + (8 * c + ktok) * kB + i);
                    fk[c][i] = x.x; fk[c][i + 1] = x.y; fk[c][i + 2] = x.z; fk[c][i + 3] = x.w;
                }
            }
        #pragma unroll
        for (int blk = 0; blk < kB; ++blk) {
            const unsigned char* kc = st + ktok * (D / 2) + mx4_chunk_pos<D>(ktok, blk) * 16 + t4 * 4;
            uint4 qb[NT], ql[NT];
            #pragma unroll
            for (int i = 0; i < NT; ++i) {
                const unsigned char* at = q_smem + (8 * i + g) * Cfg::kQStride + blk * 64 + t4 * 16;
                qb[i] = *reinterpret_cast<const uint4*>(at);
                ql[i] = *reinterpret_cast<const uint4*>(at + Cfg::kRows * Cfg::kQStride);
            }
            #pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t h0[4], h1[4];                            // (a token's swizzle is that of the token 8 on)
                codes_to_f16(*reinterpret_cast<const uint32_t*>(kc + 16 * c * (D / 2)), h0);
                codes_to_f16(*reinterpret_cast<const uint32_t*>(kc + (16 * c + 8) * (D / 2)), h1);
                const float f0 = fk[2 * c][blk], f1 = fk[2 * c + 1][blk];
                #pragma unroll
                for (int i = 0; i < NT; ++i) {
                    float acc[4];
                    mma_f16_zero(acc, h0[0], h1[0], h0[1], h1[1], qb[i].x, qb[i].y);
                    mma_f16(acc, h0[2], h1[2], h0[3], h1[3], qb[i].z, qb[i].w);
                    mma_f16(acc, h0[0], h1[0], h0[1], h1[1], ql[i].x, ql[i].y);
                    mma_f16(acc, h0[2], h1[2], h0[3], h1[3], ql[i].z, ql[i].w);
                    s[i][c][0] = fmaf(acc[0], f0, s[i][c][0]);
                    s[i][c][1] = fmaf(acc[1], f0, s[i][c][1]);
                    s[i][c][2] = fmaf(acc[2], f1, s[i][c][2]);
                    s[i][c][3] = fmaf(acc[3], f1, s[i][c][3]);
                }
            }
        }

        // ---------------- weights
        float2 tk[4];                                             // {0 or -inf, E} of this thread's tokens
        #pragma unroll
        for (int c = 0; c < 4; ++c) tk[c] = info[8 * c + ktok];
        #pragma unroll
        for (int i = 0; i < NT; ++i)
            #pragma unroll
            for (int c = 0; c < 4; ++c)
                #pragma unroll
                for (int h = 0; h < 2; ++h) s[i][c >> 1][2 * (c & 1) + h] = fmaf(s[i][c >> 1][2 * (c & 1) + h], rs[i][h], tk[c].x);
        if ((ci + 1) * kMx4AttnChunk > sees_all) {                // some row's last tokens: hide what a row does not see
            #pragma unroll
            for (int i = 0; i < NT; ++i)
                #pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = 8 * i + 2 * t4 + h;
                    const int t = (row0 + r) / per_head;
                    const int sees = r >= rows ? 0 : !TREE ? n - a.tq + t + 1 : n;
                    #pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int j = ci * kMx4AttnChunk + 8 * c + ktok;
                        bool seen = j < sees;
                        if constexpr (TREE) seen &= tree.sees_any(t, j);
                        if (!seen) s[i][c >> 1][2 * (c & 1) + h] = -INFINITY;
                    }
                }
            // a value's block of NaN: straight to the accumulators of the rows that see its
            // token, which are those that see the first such (a product with the weight 0 would
            // give it to all)
            #pragma unroll
            for (int hf = 0; hf < D / 64; ++hf) {
                __half* mine = vf + 64 * hf + my_pos;
                const uint32_t nan0 = __ballot_sync(0xFFFFFFFFu, __hisnan(mine[0])), nan1 = __ballot_sync(0xFFFFFFFFu, __hisnan(mine[32]));
                if ((nan0 | nan1) == 0) continue;
                const uint32_t nan = g >> 2 ? nan1 : nan0;        // of this thread's channels
                const int first = nan ? ci * kMx4AttnChunk + __ffs(nan) - 1 : n;
                #pragma unroll
                for (int i = 0; i < NT; ++i)
                    #pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int r = 8 * i + 2 * t4 + h, t = (row0 + r) / per_head;
                        bool seen = first <= n - a.tq + t;
                        if constexpr (TREE) {                     // any of them, not the first alone
                            seen = false;
                            if (r < rows && t < tree.nodes)
                                for (uint32_t left = nan; left; left &= left - 1) {
                                    const int j = ci * kMx4AttnChunk + __ffs(left) - 1;
                                    seen |= j < n && tree.sees(t, j);
                                }
                        }
                        if (seen) {
                            #pragma unroll
                            for (int j = 4 * hf; j < 4 * hf + 4; ++j) o[i][j][h] = o[i][j][2 + h] = NAN;
                        }
                    }
                if (nan0 >> lane & 1) mine[0] = __ushort_as_half(0);
                if (nan1 >> lane & 1) mine[32] = __ushort_as_half(0);
                __syncwarp();
            }
        }
        // The references m and dn need not be the maxima, only near them: they move when
        // some weight is above 2^8 in the denominator or 2^15 in the numerator (f16 holds it),
        // which is rare, and only then do lanes compare and accumulators get a new scale. dn
        // moves to 2^8 below the maximum, so that f16 holds small weights too (2^12 below moves
        // more often: 37 sequences up to 4096 of heads of 64, 4 tokens: 62.6 against 60.2 us).
        bool above = false;
        const float most = fmaxf(fmaxf(tk[0].y, tk[1].y), fmaxf(tk[2].y, tk[3].y));   // (s + E is at most max s + max E)
        #pragma unroll
        for (int i = 0; i < NT; ++i)
            #pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float top = fmaxf(fmaxf(s[i][0][h], s[i][0][2 + h]), fmaxf(s[i][1][h], s[i][1][2 + h]));
                above |= top > m[i][h] + 8.0f || (top - m[i][h]) + most > dn[i][h] + 15.0f;
            }
        if (__any_sync(0xFFFFFFFFu, above)) {
            #pragma unroll
            for (int i = 0; i < NT; ++i)
                #pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float top = m[i][h], topn = -INFINITY;
                    #pragma unroll
                    for (int c = 0; c < 4; ++c) top = fmaxf(top, s[i][c >> 1][2 * (c & 1) + h]);
                    #pragma unroll
                    for (int z = 4; z < 32; z *= 2) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, z));
                    #pragma unroll
                    for (int c = 0; c < 4; ++c) topn = fmaxf(topn, (s[i][c >> 1][2 * (c & 1) + h] - top) + tk[c].y);
                    #pragma unroll
                    for (int z = 4; z < 32; z *= 2) topn = fmaxf(topn, __shfl_xor_sync(0xFFFFFFFFu, topn, z));
                    const float down = m[i][h] - top, was = dn[i][h] + down;
                    l[i][h] *= ex2(down);
                    m[i][h] = top;
                    dn[i][h] = fmaxf(was, topn - 8.0f);
                    const float fn = ex2(was - dn[i][h]);
                    #pragma unroll
                    for (int j = 0; j < D / 16; ++j) {
                        o[i][j][h] *= fn;
                        o[i][j][2 + h] *= fn;
                    }
                }
        }
        if (!narrow) {
            #pragma unroll
            for (int i = 0; i < NT; ++i)
                #pragma unroll
                for (int h = 0; h < 2; ++h)
                    #pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        float& x = s[i][c >> 1][2 * (c & 1) + h];
                        l[i][h] += ex2(x - m[i][h]);
                        x = ex2((x - m[i][h]) + (tk[c].y - dn[i][h]));
                    }
            // blocks of values far apart: fp32 products, token by token, with the block's own
            // scale (NaN and its masking as in the table of factors)
            #pragma unroll
            for (int c = 0; c < 4; ++c)
                #pragma unroll 1
                for (int j = 0; j < 8; ++j) {
                    const int tok = 8 * c + j, from = (2 * (j & 3) + (j >> 2)) * 4 + t4;
                    float x[NT][2];
                    #pragma unroll
                    for (int i = 0; i < NT; ++i)
                        #pragma unroll
                        for (int h = 0; h < 2; ++h) x[i][h] = __shfl_sync(0xFFFFFFFFu, s[i][c >> 1][2 * (c & 1) + h], from);
                    const uint32_t place = reinterpret_cast<const uint32_t*>(st + 2 * Cfg::kCodeBytes + 2 * Cfg::kScaleBytes)[tok];
                    const unsigned char* sc = st + 2 * Cfg::kCodeBytes + Cfg::kScaleBytes + tok * Cfg::kScaleSlot + (D == 64 ? 2 * ((place + v_off) & 1) : 0);
                    const int top = static_cast<int>(info[tok].y) + 127;
                    #pragma unroll
                    for (int hf = 0; hf < D / 64; ++hf) {
                        const int blk = 2 * hf + (g >> 2), ev = sc[blk];
                        const float f = ev == 255 ? __half2float(vf[blk * 32 + (tok & ~7) + 2 * (tok & 3) + ((tok >> 2) & 1)])
                                                  : __uint_as_float(static_cast<uint32_t>(max(ev - top + 127, 0)) << 23);
                        float v[8];
                        mx4_decode8(*reinterpret_cast<const uint32_t*>(vcodes + tok * (D / 2) + mx4_chunk_pos<D>(tok, blk) * 16 + (g & 3) * 4), v);
                        #pragma unroll
                        for (int k = 0; k < 4; ++k)
                            #pragma unroll
                            for (int i = 0; i < NT; ++i)
                                #pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    o[i][4 * hf + k][h] = fmaf(x[i][h], v[2 * k] * f, o[i][4 * hf + k][h]);
                                    o[i][4 * hf + k][2 + h] = fmaf(x[i][h], v[2 * k + 1] * f, o[i][4 * hf + k][2 + h]);
                                }
                    }
                }
            __syncwarp();
            continue;
        }
        uint32_t p[NT][4], pr[NT][4];                             // numerator weights as MMA operands, tile by tile of 8 tokens
        #pragma unroll
        for (int i = 0; i < NT; ++i) {
            float w[2][4];
            #pragma unroll
            for (int h = 0; h < 2; ++h) {
                #pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float x = s[i][c >> 1][2 * (c & 1) + h];
                    l[i][h] += ex2(x - m[i][h]);
                    w[h][c] = ex2((x - m[i][h]) + (tk[c].y - dn[i][h]));
                }
            }
            #pragma unroll
            for (int c = 0; c < 4; ++c) {
                const uint32_t hi = f16x2_bits(w[0][c], w[1][c]);
                p[i][c] = movmatrix_trans(hi);
                __half2 r;
                memcpy(&r, &hi, 4);
                const float2 back = __half22float2(r);
                pr[i][c] = movmatrix_trans(f16x2_bits(w[0][c] - back.x, w[1][c] - back.y));
            }
        }

        // ---------------- values: tiles of 16 channels by 8 query rows over 16 tokens
        const unsigned char *va[D / 64], *vb[D / 64];             // this thread's word of tokens t and t + 4
        #pragma unroll
        for (int hf = 0; hf < D / 64; ++hf) {
            const int blk = 2 * hf + (g >> 2);
            va[hf] = vcodes + t4 * (D / 2) + mx4_chunk_pos<D>(t4, blk) * 16 + (g & 3) * 4;
            vb[hf] = vcodes + (t4 + 4) * (D / 2) + mx4_chunk_pos<D>(t4 + 4, blk) * 16 + (g & 3) * 4;
        }
        const __half* vfac = vf + (g >> 2) * 32 + 2 * t4;
        #pragma unroll
        for (int u = 0; u < 2; ++u) {
            #pragma unroll
            for (int hf = 0; hf < D / 64; ++hf) {
                uint32_t lo[2], hi[2], f[2];
                #pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const uint32_t wa = *reinterpret_cast<const uint32_t*>(va[hf] + 8 * (2 * u + x) * (D / 2));
                    const uint32_t wb = *reinterpret_cast<const uint32_t*>(vb[hf] + 8 * (2 * u + x) * (D / 2));
                    lo[x] = (wa & 0x0F0F0F0Fu) | ((wb << 4) & 0xF0F0F0F0u);
                    hi[x] = ((wa >> 4) & 0x0F0F0F0Fu) | (wb & 0xF0F0F0F0u);
                    f[x] = *reinterpret_cast<const uint32_t*>(vfac + 64 * hf + 8 * (2 * u + x));
                }
                uint32_t e0[4], e1[4], d0[4], d1[4];
                codes_to_f16(lo[0], e0);
                codes_to_f16(hi[0], d0);
                codes_to_f16(lo[1], e1);
                codes_to_f16(hi[1], d1);
                #pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t a0 = hmul2_bits(e0[k], f[0]), a1 = hmul2_bits(d0[k], f[0]);
                    const uint32_t a2 = hmul2_bits(e1[k], f[1]), a3 = hmul2_bits(d1[k], f[1]);
                    #pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        mma_f16(o[i][4 * hf + k], a0, a1, a2, a3, p[i][2 * u], p[i][2 * u + 1]);
                        mma_f16(o[i][4 * hf + k], a0, a1, a2, a3, pr[i][2 * u], pr[i][2 * u + 1]);
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
    for (int i = 0; i < NT; ++i)
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = 8 * i + 2 * t4 + h;
            float sum = l[i][h];
            #pragma unroll
            for (int z = 4; z < 32; z *= 2) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, z);
            const bool none = m[i][h] == kMx4NoScore && sum == 0.0f;      // (scores that are all NaN move no reference)
            // the mean of the warp's values (their sum could leave fp32's range), by two factors:
            // 2^dn alone could be below it
            const float half = none ? 0.0f : ex2(0.5f * dn[i][h]), f = none ? 0.0f : half * rcp(sum);
            if (g == 0) {
                pm[warp][r] = none ? -INFINITY : m[i][h];
                pl[warp][r] = sum;
            }
            float* dst = part + (warp * Cfg::kRows + r) * Cfg::kPartStride;
            #pragma unroll
            for (int j = 0; j < D / 16; ++j)                      // channels 8 g + 2 k and the next of each 64
                *reinterpret_cast<float2*>(dst + 64 * (j / 4) + 8 * g + 2 * (j % 4)) = make_float2(o[i][j][h] * half * f, o[i][j][2 + h] * half * f);
        }
    __syncthreads();
    float* joined = part;                                          // warp 0's rows become the block's
    for (int i = tid; i < rows * D / 4; i += kMx4AttnWarps * 32) {
        const int r = i / (D / 4), c = i % (D / 4) * 4;
        float top = -INFINITY;
        #pragma unroll
        for (int w = 0; w < kMx4AttnWarps; ++w) top = fmaxf(top, pm[w][r]);
        float sum = 0.0f, f[kMx4AttnWarps];
        #pragma unroll
        for (int w = 0; w < kMx4AttnWarps; ++w) {
            f[w] = pm[w][r] == -INFINITY ? 0.0f : ex2(pm[w][r] - top) * pl[w][r];
            sum += f[w];
        }
        const float inv = sum == 0.0f ? 0.0f : rcp(sum);
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        #pragma unroll
        for (int w = 0; w < kMx4AttnWarps; ++w) {
            const float share = f[w] * inv;
            const float4 x = *reinterpret_cast<const float4*>(part + (w * Cfg::kRows + r) * Cfg::kPartStride + c);
            acc.x += share * x.x;
            acc.y += share * x.y;
            acc.z += share * x.z;
            acc.w += share * x.w;
        }
        if (a.clustered || a.splits == 1) {
            *reinterpret_cast<float4*>(joined + r * Cfg::kPartStride + c) = acc;
            if (c == 0) block_ml[r] = make_float2(top, sum);
        } else {
            const size_t at = (static_cast<size_t>(tile) * a.splits + split) * Cfg::kRows + r;
            *reinterpret_cast<float4*>(a.part + at * D + c) = acc;
            if (c == 0) a.part_ml[at] = make_float2(top, sum);
        }
    }
    if (a.splits > 1 && !a.clustered) return;
    if (a.clustered) cluster_sync(); else __syncthreads();
    // rows in turn over the warps, and over the cluster's blocks
    const int first = a.clustered ? split + a.splits * warp : warp, step = a.clustered ? a.splits * kMx4AttnWarps : kMx4AttnWarps;
    for (int r = first; r < rows; r += step) {
        float* v = joined + r * Cfg::kPartStride;
        if (a.clustered) {
            // the splits' sums of this row, each from its block's memory
            constexpr int kPer = D / 32;
            float2 ml[8];
            float x[8][kPer];
            const uint32_t ml_at = smem_u32(&block_ml[r]), row_at = smem_u32(v + lane * kPer);
            #pragma unroll
            for (int k = 0; k < 8; ++k) {
                ml[k] = make_float2(-INFINITY, 0.0f);
                if (k >= a.splits) continue;
                const uint32_t from = mapa_shared(row_at, k);
                ml[k] = ld_shared_cluster_f2(mapa_shared(ml_at, k));
                #pragma unroll
                for (int i = 0; i < kPer; i += 2) {
                    const float2 y = ld_shared_cluster_f2(from + i * 4);
                    x[k][i] = y.x;
                    x[k][i + 1] = y.y;
                }
            }
            float top = -INFINITY, sum = 0.0f, acc[kPer] = {};
            #pragma unroll
            for (int k = 0; k < 8; ++k) top = fmaxf(top, ml[k].x);
            #pragma unroll
            for (int k = 0; k < 8; ++k) {
                ml[k].y = ml[k].x == -INFINITY ? 0.0f : ex2(ml[k].x - top) * ml[k].y;
                sum += ml[k].y;
            }
            const float inv = sum == 0.0f ? 0.0f : rcp(sum);
            #pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (ml[k].x == -INFINITY) continue;
                const float share = ml[k].y * inv;
                #pragma unroll
                for (int i = 0; i < kPer; ++i) acc[i] += share * x[k][i];
            }
            v = reinterpret_cast<float*>(q_smem) + warp * D;      // (the joined rows are still read by other blocks)
            #pragma unroll
            for (int i = 0; i < kPer; ++i) v[lane * kPer + i] = acc[i];
            __syncwarp();
        }
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
        __syncwarp();
    }
    if (a.clustered) cluster_sync();                              // no block leaves while others read its memory
}

// Joins a row's splits, rotates back and rounds. `wide`: a block (eight warps) a
// row, for many splits of few rows; otherwise a warp a row.
template <typename T, int D>
__global__ void __launch_bounds__(256) mx4_attn_join_kernel(Mx4AttnArgs a, int tile_rows, int wide) {
    constexpr int kPer = D / 32;
    __shared__ float v[8][D], weight[kMx4MostSplits];
    griddep_wait();
    griddep_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per_head = a.hq / a.hkv, rows_all = a.tq * per_head;
    const int index = wide ? blockIdx.x : blockIdx.x * 8 + warp;
    if (index >= a.B * a.hkv * rows_all) return;                   // (not wide: whole warps leave, no barrier below)
    const int row = index % rows_all, hk = index / rows_all % a.hkv, b = index / rows_all / a.hkv;
    const int n = max(0, static_cast<int>(min(static_cast<long long>(a.lens[b]), a.cap)));
    const int per_split = mx4_split_groups(n, a.splits);
    const int held = per_split ? (mx4_groups(n) + per_split - 1) / per_split : 0;          // splits that hold tokens
    const size_t at = ((static_cast<size_t>(b) * a.hkv + hk) * a.row_tiles + row / tile_rows) * a.splits * tile_rows + row % tile_rows;
    const float2* ml = a.part_ml + at;
    if (a.mask && held && ml->y < 0.0f) return;                   // (the row is written)
    float top = -INFINITY, sum = 0.0f;
    for (int s = lane; s < held; s += 32) top = fmaxf(top, ml[static_cast<size_t>(s) * tile_rows].x);
    #pragma unroll
    for (int z = 16; z; z >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, z));
    float f = 0.0f;                                                // not wide: at most 32 splits, lane s has split s's
    for (int s = lane; s < held; s += 32) {
        const float2 x = ml[static_cast<size_t>(s) * tile_rows];
        f = x.x == -INFINITY ? 0.0f : ex2(x.x - top) * x.y;
        sum += f;
        if (wide && warp == 0) weight[s] = f;
    }
    #pragma unroll
    for (int z = 16; z; z >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, z);
    const float inv = sum == 0.0f ? 0.0f : rcp(sum);
    if (wide) __syncthreads();
    float acc[kPer] = {};
    const float* src = a.part + at * D + lane;
    #pragma unroll 4
    for (int s = wide ? warp : 0; s < held; s += wide ? 8 : 1) {
        const float w = (wide ? weight[s] : __shfl_sync(0xFFFFFFFFu, f, s)) * inv;
        #pragma unroll
        for (int i = 0; i < kPer; ++i) acc[i] += w * src[static_cast<size_t>(s) * tile_rows * D + 32 * i];
    }
    #pragma unroll
    for (int i = 0; i < kPer; ++i) v[warp][lane + 32 * i] = acc[i];
    if (wide) {
        __syncthreads();
        if (warp != 0) return;
        #pragma unroll
        for (int i = 0; i < kPer; ++i) {
            for (int w = 1; w < 8; ++w) acc[i] += v[w][lane + 32 * i];
            v[0][lane + 32 * i] = acc[i];
        }
    }
    float* r = v[wide ? 0 : warp];
    __syncwarp();
    for (int st = 1; st < a.group; st *= 4) {
        for (int i = lane; i < D / 4; i += 32) {
            float* p = r + (i / st) * 4 * st + i % st;
            h4(p[0], p[st], p[2 * st], p[3 * st]);
        }
        __syncwarp();
    }
    const float g = a.group == 16 ? 0.25f : a.group == 64 ? 0.125f : a.group == 256 ? 0.0625f : 1.0f;
    T* out = static_cast<T*>(a.out) + ((static_cast<size_t>(b) * a.tq + row / per_head) * a.hq + hk * per_head + row % per_head) * D;
    for (int i = lane; i < D; i += 32) out[i] = mx4_from_f32<T>(r[i] * g);
}

}  // namespace convrot
