// Attention of a tree of drafted tokens over the paged MX4 cache, many query rows
// of a cache head: both products on tcgen05 (mx4_attn.cuh has the kernel for few rows).
//
// A block takes two streams of 128 query rows each. Where a cache head has more than 128 rows
// (nodes times query heads), the streams are two row tiles that share each tile of 128
// tokens; otherwise they are the same rows over two halves of the block's tokens, joined at
// the end. Warps 0 - 3 and 4 - 7 are the streams' softmax (a thread a row), 8 - 11 turn the
// values' codes into operands, 12 and 13 the keys', 14 issues the MMAs.
//
//   S = Q K^T   queries rotated in fp32, then two f16 terms (22 bits) of the row times a power of two;
//               a key's codes times 2^(E_b - E), E its largest scale exponent, are f16 values, and
//               2^E goes to its column of S in fp32; blocks more than 2^23 below it are left out there and
//               added to the scores by fp32 products (tree_far_scores)
//   O = P V     values are bf16 exactly, whatever their scale; weights two bf16 terms (16 bits)
//
// S lies in tensor memory, the weights take its place (16 columns of S: 8 of the first terms, 8 of
// the second), O beside it. The order of the MMAs is P_A V, Q_A K, P_B V, Q_B K, ..., so that
// one stream's softmax runs under the other's products, and K and V (32 KB a tile at heads of 128)
// are refilled under the products that do not read them.
//
// Weights are 2^(s - m - 24). m lags the row's maximum by 2^10 at most: a chunk of 16 columns whose weights sum to
// more than 2^-14 moves it, where scores go column by column a score 2^6 above it. A stream's sum is then below one up to
// 2^18 tokens, below 2^13 at the longest table, so that O stays in fp32's range for values up to 2^114; and
// values below 2^-102 give products below its normal numbers: means lose bits from some 2^-115 down.
// 16 bits a weight (the kernel for few rows has 22): what they leave out is 2^-16 of the mean of the
// magnitudes at most, and by its random sign far less of the mean; a third term has no room in tensor memory.
//
// What bounds it: a stream's softmax (load, exp2, split, store: some 3500 cycles a tile, by the
// latency of its 128 threads) takes turns with its own two products, and two streams a block
// are what registers and tensor memory hold; a block starts in 3 to 9 us and ends in 6. 8 x 16384 tokens, 64
// nodes of 64 query heads on 8 of 128: 464 to 484 us (1.16 PFLOP/s with both terms counted, 0.58 of the formula's;
// tensor pipe 44 to 53 % of the active time, exp2's 22 to 27 %); 37 x 4096, 24 nodes of 24 on 8 of 64: 72 to 79 us.
// Registers are full: heads of 128 spill 32 to 40 bytes, heads of 64 none.
// The kernel for few rows took 1820 and 277. Tiles in halves of 64 tokens: 541 and 103.
#pragma once

namespace convrot {

constexpr int kTreeTile = 128;                 // tokens of a tile, rows of a stream
constexpr int kTreeThreads = 15 * 32;
constexpr float kTreeDown = 24.0f;
constexpr float kTreeMost = 6.1035156e-5f;     // 2^-14: weights of a chunk above this move the reference
constexpr int kTreeBits = 23;                  // a code times 2^-23 is an f16 value exactly
constexpr float kTreeHuge = 268435456.0f;      // 2^28: scores whose own step is 16 and more
constexpr uint32_t kTreeApart = 1, kTreeFar = 2;          // of a tile: keys, or blocks of one key, lie further apart

template <int D, bool PAIR>
struct Mx4TreeCfg {
    static constexpr int kOperand = kTreeTile * D * 2;            // a term of a stream's queries, a tile of K or V
    static constexpr int kAtom = kTreeTile * 128;                 // 128 rows of 64 16-bit columns, 128-byte swizzle
    static constexpr int kVAtom = D * 128;                        // D rows (channels) of 64 tokens
    static constexpr int kBlocks = D / 32;
    // a pair: four terms of queries, K, two tiles of V; otherwise two terms, then K and V of each stream
    static constexpr int kFacOffset = (PAIR ? 7 : 6) * kOperand;  // [buffer][parity][128] fp32: factors of a tile's keys
    static constexpr int kBufs = PAIR ? 1 : 2;                    // buffers of K
    static constexpr int kHidOffset = kFacOffset + kBufs * 1024;  // [buffer][parity][8]: hidden tokens' bits, kTreeApart | kTreeFar
    static constexpr int kRangeOffset = kHidOffset + kBufs * 64;  // [2][2] largest and least exponents of a tile's keys, [2][2] of a closer look
    static constexpr int kOneOffset = kRangeOffset + 32;          // [16] fp32 ones: factors of columns that have theirs already
    static constexpr int kRowOffset = kOneOffset + 64;            // [256] fp32: the rows' scales (both streams' the same rows)
    static constexpr int kBarOffset = kRowOffset + (PAIR ? 0 : 1024);
    static constexpr int kBars = 2 * 4 + 2 * 2 + 2 * 3 + 2;
    static constexpr int kEnd = kBarOffset + kBars * 8 + 16;
    // (all of the tensor memory is taken: one block a multiprocessor, by shared memory too)
    static constexpr int kSmemBytes = (kEnd > 116 * 1024 ? kEnd : 116 * 1024) + 1024;
    static_assert(kSmemBytes <= 227 * 1024, "fits a multiprocessor");
    static constexpr uint32_t kIdescS = idesc_f16(kTreeTile, kTreeTile), kIdescO = idesc_bf16(kTreeTile, D);
};

// 32 lanes x 16 consecutive 32-bit columns from and to tensor memory.
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr));
}

__device__ __forceinline__ void tmem_ld_wait_regs16(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}

// D (+)= A B^T, kind::f16, A from tensor memory.
__device__ __forceinline__ void mma_f16kind_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        :: "r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

__device__ __forceinline__ uint32_t bf16x2_bits(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ float2 half2_bits(uint32_t x) {
    __half2 h;
    memcpy(&h, &x, 4);
    return __half22float2(h);
}

// Two weights as the sum of two bf16 terms each: the upper halves as they are, and what they leave out.
__device__ __forceinline__ void split_bf16(float2 w, uint32_t& hi, uint32_t& lo) {
    const uint32_t x = __float_as_uint(w.x), y = __float_as_uint(w.y);
    hi = __byte_perm(x, y, 0x7632);
    const float2 left = ffma2_rn(make_float2(__uint_as_float(x & 0xFFFF0000u), __uint_as_float(y & 0xFFFF0000u)), make_float2(-1.0f, -1.0f), w);
    lo = bf16x2_bits(left.x, left.y);
}

// Eight codes as bf16, in pairs of neighbours: the two bytes of a value are looked up by its
// three low bits, the sign byte comes from bit 3.
__device__ __forceinline__ void codes_to_bf16(uint32_t x, uint32_t (&h)[4]) {
    const uint32_t mag = x & 0x77777777u, low = x << 4;           // low: bit 3 of the even nibbles at their byte's end
    #pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t sel = i ? mag >> 16 : mag;
        const uint32_t lb = __byte_perm(0xC0800000u, 0xC0804000u, sel);           // 0, .5, 1, 1.5, 2, 3, 4, 6: low bytes
        uint32_t hb = __byte_perm(0x3F3F3F00u, 0x40404040u, sel);                 // and high bytes
        hb |= __byte_perm(low, x, i ? 0xFBEAu : 0xD9C8u) & 0x80808080u;
        h[2 * i] = __byte_perm(lb, hb, 0x5140);
        h[2 * i + 1] = __byte_perm(lb, hb, 0x7362);
    }
}

// The rotation of 64 channels of a row without its factor (groups of 16 or 64), in the order of the
// other kernels.
__device__ __forceinline__ void tree_rotate(float (&v)[64], int group) {
    constexpr int D = 64;
    if (group >= 16) {
        #pragma unroll
        for (int i = 0; i < D; i += 4) h4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        #pragma unroll
        for (int i = 0; i < D; i += 16)
            #pragma unroll
            for (int j = 0; j < 4; ++j) h4(v[i + j], v[i + j + 4], v[i + j + 8], v[i + j + 12]);
    }
    if (group >= 64) {
        #pragma unroll
        for (int i = 0; i < D; i += 64)
            #pragma unroll
            for (int j = 0; j < 16; ++j) h4(v[i + j], v[i + j + 16], v[i + j + 32], v[i + j + 48]);
    }
}

__device__ __forceinline__ float tree_factor(int group) { return group == 16 ? 0.25f : group == 64 ? 0.125f : 1.0f; }

// A tile's scores in tensor memory times its keys' factors, with what the products left out: the blocks of a key more
// than 2^kTreeBits below its largest, times their own scales. All lanes of a warp take the same tokens, each its row r
// of those that begin at `q`. Not inlined: few tiles need it, and the loop that calls it has no register to give. (8 x 4096 tokens
// of 64 nodes, 64 query heads on 8 of 128: 133 us, with one such key among 64 387, with every key 3150.)
template <int D>
__device__ __noinline__ void tree_far_scores(uint32_t ts, const unsigned char* q, int r, const uint8_t* codes, const uint8_t* scales, const int* table,
                                             int page_bits, int pages, int hkv, int hk, int j0, int n, const float* f) {
    constexpr int kB = D / 32, kAtom = kTreeTile * 128, kOperand = kTreeTile * D * 2;
    auto place_of = [&](int j) -> long long {
        const int page = j < n ? table[j >> page_bits] : -1;
        if (page < 0 || page >= pages) return -1;
        return (((static_cast<long long>(page) * 2 * hkv + hk) << page_bits) + (j & ((1 << page_bits) - 1)));
    };
    auto exps_of = [&](long long place) -> uint32_t {
        return D == 128 ? reinterpret_cast<const uint32_t*>(scales)[place] : static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(scales)[place]);
    };
    auto exp_at = [](uint32_t exps, int c) { return static_cast<int>((exps >> (8 * c)) & 255u); };
    auto top_of = [&](uint32_t exps) {
        int top = 0;
        #pragma unroll
        for (int c = 0; c < kB; ++c)
            if (exp_at(exps, c) != 255) top = max(top, exp_at(exps, c));
        return top;
    };
    #pragma unroll 1
    for (int at = 0; at < kTreeTile; at += 16) {
        const long long mine = place_of(j0 + at + (threadIdx.x & 15));
        const uint32_t own = mine < 0 ? 0u : exps_of(mine);
        bool far = false;
        #pragma unroll
        for (int c = 0; c < kB; ++c) far |= exp_at(own, c) != 255 && top_of(own) - exp_at(own, c) > kTreeBits;
        uint32_t left = __ballot_sync(0xFFFFFFFFu, far) & 0xFFFFu;
        float more[16];
        #pragma unroll
        for (int k = 0; k < 16; ++k) more[k] = 0.0f;
        #pragma unroll 1
        for (; left; left &= left - 1) {
            const int k = __ffs(left) - 1;
            const long long place = __shfl_sync(0xFFFFFFFFu, mine, k);
            const uint32_t exps = __shfl_sync(0xFFFFFFFFu, own, k);
            const int top = top_of(exps);
            float all = 0.0f;
            #pragma unroll 1
            for (int c = 0; c < kB; ++c) {
                const int e = exp_at(exps, c);
                if (e == 255 || top - e <= kTreeBits) continue;
                const uint4 x = *reinterpret_cast<const uint4*>(codes + place * (D / 2) + c * 16);
                const uint32_t words[4] = {x.x, x.y, x.z, x.w};
                float sum = 0.0f;
                #pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t h[4];
                    codes_to_f16(words[w], h);
                    const unsigned char* row = q + (c / 2) * kAtom + r * 128 + ((((c & 1) * 4 + w) ^ (r & 7)) << 4);
                    const uint4 hi = *reinterpret_cast<const uint4*>(row), lo = *reinterpret_cast<const uint4*>(row + kOperand);
                    const uint32_t a[4] = {hi.x, hi.y, hi.z, hi.w}, b[4] = {lo.x, lo.y, lo.z, lo.w};
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 u = half2_bits(a[i]), v = half2_bits(b[i]), z = half2_bits(h[i]);
                        sum = fmaf(u.x + v.x, z.x, fmaf(u.y + v.y, z.y, sum));
                    }
                }
                all = fmaf(sum, __uint_as_float(max(static_cast<uint32_t>(e) << 23, 0x00400000u)), all);
            }
            #pragma unroll
            for (int i = 0; i < 16; ++i)
                if (i == k) more[i] = all;
        }
        uint32_t x[16];
        __syncwarp();
        tmem_ld_32x32b_x16(ts + at, x);
        tmem_ld_wait_regs16(x);
        #pragma unroll
        for (int k = 0; k < 16; ++k) x[k] = __float_as_uint(fmaf(__uint_as_float(x[k]), f[at + k], more[k]));
        tmem_st_32x32b_x16(ts + at, x);
    }
    tmem_st_wait();
}

template <typename T, int D, bool PAIR>
__global__ void __launch_bounds__(kTreeThreads, 1) mx4_tree_kernel(Mx4AttnArgs a, int vec_q, int by_length) {
    using Cfg = Mx4TreeCfg<D, PAIR>;
    constexpr int kB = Cfg::kBlocks;
    extern __shared__ __align__(1024) unsigned char tree_smem_raw[];
    unsigned char* smem = tree_smem_raw + ((1024u - (smem_u32(tree_smem_raw) & 1023u)) & 1023u);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kBarOffset);
    uint64_t *k_full = bars, *k_empty = bars + 2, *v_full = bars + 4, *v_empty = bars + 6;       // [buffer]
    uint64_t* f_full = bars + 8;                                  // [buffer][parity]: the columns' factors
    uint64_t *s_full = bars + 12, *p_full = bars + 14, *o_done = bars + 16;                      // [stream]
    uint64_t *q_full = bars + 18, *drain = bars + 19;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::kBars);
    int* nan_nodes = reinterpret_cast<int*>(tmem_slot + 1);       // a node's values hold a block of NaN
    float* row_scale = reinterpret_cast<float*>(smem + Cfg::kRowOffset);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = blockIdx.y;
    int splits = a.splits;                                        // of the sequence
    const int rt = blockIdx.x % a.row_tiles, hk = blockIdx.x / a.row_tiles % a.hkv;
    int b = blockIdx.x / a.row_tiles / a.hkv;
    const int per_head = a.hq / a.hkv, rows_all = a.tq * per_head;
    constexpr int kTileRows = PAIR ? 2 * kTreeTile : kTreeTile;
    const int row0 = rt * kTileRows, rows = min(kTileRows, rows_all - row0);
    griddep_wait();
    griddep_launch_dependents();
    auto tokens_of = [&](int i) { return max(0, static_cast<int>(min(static_cast<long long>(a.lens[i]), a.cap))); };
    if (by_length) {
        // More blocks than multiprocessors: long sequences first, so that what is left at the end is short (37 sequences
        // of up to 4096 tokens, 296 blocks: 74 against 93 to 99 us). A sequence's place is the number of longer ones,
        // of the same length those before it. Splits are cut by the table's width; a sequence that is no
        // more than a quarter above a multiprocessor's share of all tiles stays whole.
        int* held = reinterpret_cast<int*>(smem);                 // [threads] lengths, behind them the block's sequence, whether it stays whole
        const int mine = tid < a.B ? tokens_of(tid) : -1;
        held[tid] = mine;
        __syncthreads();
        if (tid < a.B) {
            int place = 0;
            for (int i = 0; i < a.B; ++i) place += held[i] > mine || (held[i] == mine && i < tid);
            if (place == b) {
                float tiles = 0.0f;
                for (int i = 0; splits > 1 && i < a.B; ++i) tiles += mx4_groups(held[i]);
                held[kTreeThreads] = tid;
                held[kTreeThreads + 1] = mx4_groups(mine) * static_cast<float>(by_length) <= 1.25f * tiles * (a.hkv * a.row_tiles);
            }
        }
        __syncthreads();
        b = held[kTreeThreads];
        if (held[kTreeThreads + 1]) splits = 1;
    }
    if (split >= splits) return;
    const int tile = (b * a.hkv + hk) * a.row_tiles + rt;
    const int n = tokens_of(b);
    const Mx4Tree tree(a, b, n);
    const int per_split = mx4_split_groups(n, splits), groups = mx4_groups(n);
    const int c0 = min(groups, split * per_split), count = min(groups, c0 + per_split) - c0;
    if (splits > 1 && count == 0) return;                         // (the join knows how many splits hold tokens)
    // tiles of each stream, and where the second starts
    const int n0 = PAIR ? count : (count + 1) / 2, n1 = PAIR ? (rows > kTreeTile ? count : 0) : count - n0;
    const int c1 = PAIR ? c0 : c0 + n0;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], 64);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], 128);
            mbar_init(&v_empty[i], 1);
            mbar_init(&f_full[2 * i], 64);
            mbar_init(&f_full[2 * i + 1], 64);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 128);
            mbar_init(&o_done[i], 1);
        }
        mbar_init(q_full, PAIR || D == 128 ? 256 : 128);
        mbar_init(drain, 1);
        *nan_nodes = 0;
        fence_mbar_init();
    }
    if (tid < 16) reinterpret_cast<float*>(smem + Cfg::kOneOffset)[tid] = 1.0f;
    if (warp == 14) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    auto tmem_s = [&](int s) { return tmem + s * kTreeTile; };
    auto tmem_o = [&](int s) { return tmem + 2 * kTreeTile + s * D; };
    auto k_buf = [&](int i) { return smem + (PAIR || i == 0 ? 4 : 2) * Cfg::kOperand; };
    auto v_buf = [&](int i) { return smem + (PAIR ? 5 + i : i == 0 ? 5 : 3) * Cfg::kOperand; };
    // a tile's place among the values: a pair's tiles take turns, otherwise each stream has one
    auto v_at = [](int s, int i) { return PAIR ? i & 1 : s; };
    auto v_use = [](int i) { return PAIR ? i >> 1 : i; };
    float* fac = reinterpret_cast<float*>(smem + Cfg::kFacOffset);
    uint32_t* hid = reinterpret_cast<uint32_t*>(smem + Cfg::kHidOffset);

    if (warp == 14) {
        // ---------------- MMAs
        const int streams = PAIR ? (n1 ? 2 : 1) : 2;
        bool ok = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(q_full, 0));
        for (int i = 0; ok && i <= n0; ++i) {
            for (int s = 0; ok && s < streams; ++s) {
                const int ns = s ? n1 : n0, buf = PAIR ? 0 : s;
                const bool last = !PAIR || s == streams - 1;      // of those that read the buffers
                if (i > 0 && i - 1 < ns) {
                    const int t = i - 1, vb = v_at(s, t);
                    ok = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(&v_full[vb], v_use(t) & 1) && mbar_wait_bounded(&p_full[s], t & 1));
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t vd = smem_desc_kmajor(smem_u32(v_buf(vb)), 1024, 2);
                    if (elect_one()) {
                        #pragma unroll
                        for (int j = 0; j < kTreeTile / 16; ++j)
                            #pragma unroll
                            for (int term = 0; term < 2; ++term)
                                mma_f16kind_ts(tmem_o(s), tmem_s(s) + 16 * j + 8 * term,
                                               vd + (j / 4) * (Cfg::kVAtom / 16) + 2 * (j % 4), Cfg::kIdescO, t > 0 || j > 0 || term > 0);
                        if (last) mma_commit(&v_empty[vb]);
                        if (t == ns - 1) mma_commit(&o_done[s]);
                    }
                    __syncwarp();
                }
                if (i < ns) {
                    ok = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(&k_full[buf], i & 1));
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t kd = smem_desc_kmajor(smem_u32(k_buf(buf)), 1024, 2);
                    const uint64_t qd = smem_desc_kmajor(smem_u32(smem + (PAIR ? 2 * s : 0) * Cfg::kOperand), 1024, 2);
                    if (elect_one()) {
                        #pragma unroll
                        for (int term = 0; term < 2; ++term)
                            #pragma unroll
                            for (int j = 0; j < D / 16; ++j) {
                                const int at = (j / 4) * (Cfg::kAtom / 16) + 2 * (j % 4);
                                mma_f16kind_ss(tmem_s(s), qd + term * (Cfg::kOperand / 16) + at, kd + at, Cfg::kIdescS, term > 0 || j > 0);
                            }
                        mma_commit(&s_full[s]);
                        if (last) mma_commit(&k_empty[buf]);
                    }
                    __syncwarp();
                }
            }
        }
        if (!ok && lane == 0) tree_record_status(kMx4TimeoutMma);
        if (elect_one()) mma_commit(drain);
        __syncwarp();
        if (!__all_sync(0xFFFFFFFFu, mbar_wait_bounded(drain, 0)) && lane == 0) tree_record_status(kMx4TimeoutMma);
    } else if (warp >= 8) {
        // ---------------- codes to operands. The next tile's codes are loaded into registers when this
        // one's are laid down, and are there when its place gets free; page numbers a tile earlier.
        const int* table = a.table + b * a.table_ld;
        const uint32_t in_page = (1u << a.page_bits) - 1;
        const int streams = PAIR ? 1 : 2;
        // tiles in the order of the MMAs: stream after stream (the second may have one less)
        const int units = PAIR ? n0 : n0 + n1;
        auto first_of = [&](int u) { return ((PAIR || u % 2 == 0 ? c0 : c1) + u / streams) * kTreeTile; };
        auto page_at = [&](int j) { return j < n ? __ldg(table + (j >> a.page_bits)) : -1; };
        auto place_of = [&](int page, int j, int value) {         // in tokens of a head, the highest number: none
            return page >= 0 && page < a.pages ? (((static_cast<uint32_t>(page) * 2 + value) * a.hkv + hk) << a.page_bits) + (static_cast<uint32_t>(j) & in_page)
                                               : 0xFFFFFFFFu;
        };
        bool ok = true;
        if (warp < 12) {
            // values: groups of 8 tokens by 8 channels, word w of the tokens' codes
            constexpr int kItems = kTreeTile / 8 * (D / 8) / 128;
            const int id = tid - 256, g = id & 7, w = (id >> 3) % (D / 8);
            uint32_t words[kItems][8], exps[kItems][8];           // exps: the words that hold the scale bytes
            int pages[kItems];
            auto group_at = [&](int u, int k) { return first_of(u) + 64 * (D == 128 ? k : id >> 6) + 8 * g; };
            auto look = [&](int u) {
                #pragma unroll
                for (int k = 0; k < kItems; ++k) pages[k] = u < units ? page_at(group_at(u, k)) : -1;
            };
            auto load = [&](int u) {
                #pragma unroll
                for (int k = 0; k < kItems; ++k) {
                    const int j = group_at(u, k);
                    #pragma unroll
                    for (int e = 0; e < 8; ++e) words[k][e] = exps[k][e] = 0u;
                    if (a.page_bits >= 3) {                       // a group lies in one page
                        const uint32_t place = place_of(pages[k], j, 1);
                        if (place == 0xFFFFFFFFu) continue;
                        const uint32_t* from = reinterpret_cast<const uint32_t*>(a.codes + static_cast<size_t>(place) * (D / 2)) + w;
                        const uint8_t* scales = a.scales + static_cast<size_t>(place) * kB;
                        if (j + 8 <= n) {
                            #pragma unroll
                            for (int e = 0; e < 8; ++e) words[k][e] = __ldg(from + e * (D / 8));
                            if constexpr (D == 128) {
                                const uint4 lo = __ldg(reinterpret_cast<const uint4*>(scales)), hi = __ldg(reinterpret_cast<const uint4*>(scales) + 1);
                                exps[k][0] = lo.x; exps[k][1] = lo.y; exps[k][2] = lo.z; exps[k][3] = lo.w;
                                exps[k][4] = hi.x; exps[k][5] = hi.y; exps[k][6] = hi.z; exps[k][7] = hi.w;
                            } else {
                                const uint4 x = __ldg(reinterpret_cast<const uint4*>(scales));
                                exps[k][0] = x.x; exps[k][2] = x.y; exps[k][4] = x.z; exps[k][6] = x.w;
                                #pragma unroll
                                for (int e = 1; e < 8; e += 2) exps[k][e] = exps[k][e - 1] >> 16;
                            }
                        } else {
                            #pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                if (j + e >= n) continue;
                                words[k][e] = __ldg(from + e * (D / 8));
                                exps[k][e] = D == 128 ? __ldg(reinterpret_cast<const uint32_t*>(scales) + e)
                                                      : static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(scales) + e));
                            }
                        }
                    } else {
                        #pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const uint32_t place = place_of(page_at(j + e), j + e, 1);
                            if (place == 0xFFFFFFFFu) continue;
                            words[k][e] = __ldg(reinterpret_cast<const uint32_t*>(a.codes + static_cast<size_t>(place) * (D / 2)) + w);
                            exps[k][e] = D == 128 ? __ldg(reinterpret_cast<const uint32_t*>(a.scales) + place)
                                                  : static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(a.scales) + place));
                        }
                    }
                }
            };
            look(0);
            load(0);
            look(1);
            for (int u = 0; u < units; ++u) {
                const int buf = v_at(u % streams, u / streams), use = v_use(u / streams);
                ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait_bounded(&v_empty[buf], (use & 1) ^ 1));
                if (!ok) break;
                #pragma unroll 1
                for (int k = 0; k < kItems; ++k) {
                    const int half = D == 128 ? k : id >> 6;
                    uint32_t (&word)[8] = words[0], (&exp)[8] = exps[0];          // (the second item's move up below)
                    uint32_t f[4];                                // scales of pairs of tokens as bf16
                    bool odd_scale = false;
                    #pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        const uint32_t x = exp[2 * p] >> (8 * (w >> 2)) & 255u, y = exp[2 * p + 1] >> (8 * (w >> 2)) & 255u;
                        f[p] = x << 7 | y << 23;
                        odd_scale |= x - 1u >= 254u || y - 1u >= 254u;
                    }
                    if (odd_scale) {
                        // 0 is a subnormal. NaN goes straight to the weighted sums where every row sees the token, at
                        // the end to those rows that do where it is a node (a product with the weight 0 would give it to all)
                        #pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const uint32_t x = exp[e] >> (8 * (w >> 2)) & 255u;
                            const bool context = group_at(u, k) + e < tree.context;
                            if (x == 255u && !context) *nan_nodes = 1;
                            const uint32_t bits = x == 0u ? 0x0040u : x < 255u ? x << 7 : context ? 0x7FC0u : 0u;
                            f[e / 2] = e % 2 ? (f[e / 2] & 0xFFFFu) | bits << 16 : bits;
                        }
                    }
                    uint32_t out[8][4];                           // [channel][pair of tokens]
                    #pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        const uint32_t x = word[2 * p], y = word[2 * p + 1];
                        uint32_t even[4], odd[4];
                        codes_to_bf16((x & 0x0F0F0F0Fu) | ((y << 4) & 0xF0F0F0F0u), even);
                        codes_to_bf16(((x >> 4) & 0x0F0F0F0Fu) | (y & 0xF0F0F0F0u), odd);
                        #pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            out[2 * c][p] = mul_bf16x2(even[c], f[p]);
                            out[2 * c + 1][p] = mul_bf16x2(odd[c], f[p]);
                        }
                    }
                    // (rows are channels, 128 bytes of 64 tokens each: lanes of eight groups in distinct banks)
                    unsigned char* to = v_buf(buf) + half * Cfg::kVAtom + w * 1024;
                    #pragma unroll
                    for (int c = 0; c < 8; ++c)
                        *reinterpret_cast<uint4*>(to + c * 128 + ((g ^ c) << 4)) = make_uint4(out[c][0], out[c][1], out[c][2], out[c][3]);
                    #pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        word[e] = words[kItems - 1][e];
                        exp[e] = exps[kItems - 1][e];
                    }
                }
                fence_proxy_async_smem();
                mbar_arrive(&v_full[buf]);
                if (u + 1 < units) {
                    load(u + 1);
                    look(u + 2);
                }
            }
        } else {
            // keys: a thread has tokens t and t + 64
            const int id = tid - 384;
            uint4 codes[2][kB];
            uint32_t exps[2];
            int pages[2];
            bool held[2];
            short2* range = reinterpret_cast<short2*>(smem + Cfg::kRangeOffset);
            auto look = [&](int u) {
                #pragma unroll
                for (int k = 0; k < 2; ++k) pages[k] = u < units ? page_at(first_of(u) + id + 64 * k) : -1;
            };
            auto load = [&](int u) {
                #pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t place = place_of(pages[k], first_of(u) + id + 64 * k, 0);
                    held[k] = place != 0xFFFFFFFFu;
                    exps[k] = 0u;
                    #pragma unroll
                    for (int c = 0; c < kB; ++c) codes[k][c] = make_uint4(0, 0, 0, 0);
                    if (!held[k]) continue;
                    const uint4* from = reinterpret_cast<const uint4*>(a.codes + static_cast<size_t>(place) * (D / 2));
                    #pragma unroll
                    for (int c = 0; c < kB; ++c) codes[k][c] = __ldg(from + c);
                    exps[k] = D == 128 ? __ldg(reinterpret_cast<const uint32_t*>(a.scales) + place)
                                       : static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(a.scales) + place));
                }
            };
            look(0);
            load(0);
            look(1);
            for (int u = 0; u < units; ++u) {
                const int buf = u % streams, i = u / streams, at = buf * 2 + (i & 1);
                int top[2] = {0, 0}, low = 255;                   // scale exponents of the tokens
                #pragma unroll
                for (int k = 0; k < 2; ++k) {
                    #pragma unroll
                    for (int c = 0; c < kB; ++c) {
                        const int e = static_cast<int>((exps[k] >> (8 * c)) & 255u);
                        if (e != 255) top[k] = max(top[k], e);
                        if (e != 255 && held[k]) low = min(low, e);
                    }
                }
                const uint32_t gone0 = __ballot_sync(0xFFFFFFFFu, !held[0]), gone1 = __ballot_sync(0xFFFFFFFFu, !held[1]);
                int most = __reduce_max_sync(0xFFFFFFFFu, max(top[0], top[1])), least = __reduce_min_sync(0xFFFFFFFFu, low);
                if (lane == 0) range[(u & 1) * 2 + warp - 12] = make_short2(static_cast<short>(most), static_cast<short>(least));
                named_barrier_sync(1, 64);
                // Where the tile's exponents lie no further apart than kTreeBits one factor serves all columns.
                const short2 other = range[(u & 1) * 2 + (warp & 1 ^ 1)];
                most = max(most, static_cast<int>(other.x));
                least = min(least, static_cast<int>(other.y));
                uint32_t spread = 0;
                if (__builtin_expect(most - least > kTreeBits, 0)) {          // (the same in both warps)
                    // Once more without blocks of zeros, whose exponent is 0, and for each token by itself.
                    int own[2] = {255, 255};
                    #pragma unroll
                    for (int k = 0; k < 2; ++k)
                        #pragma unroll
                        for (int c = 0; c < kB; ++c) {
                            const int e = static_cast<int>((exps[k] >> (8 * c)) & 255u);
                            const uint4 x = codes[k][c];
                            if (e != 255 && (e != 0 || ((x.x | x.y | x.z | x.w) & 0x77777777u) != 0u)) own[k] = min(own[k], e);
                        }
                    const bool far = __any_sync(0xFFFFFFFFu, max(top[0] - own[0], top[1] - own[1]) > kTreeBits);
                    least = __reduce_min_sync(0xFFFFFFFFu, min(own[0], own[1]));
                    if (lane == 0) range[4 + (u & 1) * 2 + warp - 12] = make_short2(far, static_cast<short>(least));
                    named_barrier_sync(1, 64);
                    const short2 there = range[4 + (u & 1) * 2 + (warp & 1 ^ 1)];
                    spread = (most - min(least, static_cast<int>(there.y)) > kTreeBits ? kTreeApart : 0u) | (far || there.x ? kTreeFar : 0u);
                    #pragma unroll
                    for (int k = 0; k < 2; ++k)
                        #pragma unroll
                        for (int c = 0; c < kB; ++c) {
                            const int e = static_cast<int>((exps[k] >> (8 * c)) & 255u);
                            if (e != 255 && top[k] - e > kTreeBits) codes[k][c] = make_uint4(0, 0, 0, 0);      // (tree_far_scores takes it)
                        }
                }
                const bool apart = spread != 0u;
                // (the barriers of the two warps go on: neither waits for one that left)
                ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait_bounded(&k_empty[buf], (i & 1) ^ 1));
                if (!ok) continue;
                // the products of the tile before are done: the softmax of the tile that had these factors is, too
                if (lane == 0) {
                    hid[at * 8 + warp - 12] = gone0;
                    hid[at * 8 + warp - 10] = gone1;
                }
                #pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (!apart) top[k] = most;
                    fac[at * 128 + id + 64 * k] = __uint_as_float(max(static_cast<uint32_t>(top[k]) << 23, 0x00400000u));
                }
                if (id == 0) hid[at * 8 + 4] = spread;
                mbar_arrive(&f_full[at]);
                #pragma unroll 1
                for (int k = 0; k < 2; ++k) {
                    const int t = id + 64 * k;
                    #pragma unroll
                    for (int c = 0; c < kB; ++c) {
                        const int e = static_cast<int>((exps[0] >> (8 * c)) & 255u);
                        const float x = e == 255 ? NAN : __uint_as_float(static_cast<uint32_t>(max(e - top[0] + 127, 0)) << 23);
                        const uint32_t f = f16x2_bits(x, x);
                        const uint32_t words[4] = {codes[0][c].x, codes[0][c].y, codes[0][c].z, codes[0][c].w};
                        unsigned char* to = k_buf(buf) + (c / 2) * Cfg::kAtom + t * 128;
                        #pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            uint32_t h[4];
                            codes_to_f16(words[y], h);
                            *reinterpret_cast<uint4*>(to + ((((c & 1) * 4 + y) ^ (t & 7)) << 4)) =
                                make_uint4(hmul2_bits(h[0], f), hmul2_bits(h[1], f), hmul2_bits(h[2], f), hmul2_bits(h[3], f));
                        }
                        codes[0][c] = codes[1][c];                // (the second token's, for the second round)
                    }
                    exps[0] = exps[1];
                    top[0] = top[1];
                }
                fence_proxy_async_smem();
                mbar_arrive(&k_full[buf]);
                if (u + 1 < units) {
                    load(u + 1);
                    look(u + 2);
                }
            }
        }
        if (!ok && lane == 0) tree_record_status(kMx4TimeoutProducer);
    } else {
        // ---------------- a stream's softmax, a thread a row
        const int s = warp >> 2, r = tid & 127;
        const int row = row0 + (PAIR ? s * kTreeTile : 0) + r, t = row / per_head;
        const bool real = row < rows_all && (PAIR || r < rows);
        float rs = 0.0f;                                          // the row's scale
        {
            // the row's queries: rotated, then two f16 terms of the row times a power of two. 64 channels at a
            // time: where both streams have the same rows of 128, the second's threads take the second
            // half; a pair's threads load their rows twice, for the largest value and as operands.
            constexpr bool kSplit = !PAIR && D == 128;
            const T* q = static_cast<const T*>(a.q) + b * a.qsb + t * a.qst + (hk * per_head + row % per_head) * a.qsh;
            float v[64], top = 0.0f;
            auto channels = [&](int from) {
                #pragma unroll
                for (int i = 0; i < 64; ++i) v[i] = 0.0f;
                if (real && vec_q) {
                    #pragma unroll
                    for (int i = 0; i < 64; i += 8) {
                        const uint4 x = __ldg(reinterpret_cast<const uint4*>(q + from + i));
                        T e[8];
                        memcpy(e, &x, 16);
                        #pragma unroll
                        for (int k = 0; k < 8; ++k) v[i + k] = mx4_to_f32(e[k]);
                    }
                } else if (real) {
                    #pragma unroll
                    for (int i = 0; i < 64; ++i) v[i] = mx4_to_f32(q[from + i]);
                }
                tree_rotate(v, a.group);
            };
            const bool mine = PAIR || kSplit || s == 0;
            #pragma unroll 1
            for (int from = kSplit ? 64 * s : 0; mine && from < D; from += 64) {
                channels(from);
                #pragma unroll
                for (int i = 0; i < 64; ++i) top = fmaxf(top, fabsf(v[i]));
                if (kSplit) break;
            }
            if constexpr (kSplit) {
                row_scale[s * 128 + r] = top;
                named_barrier_sync(2, 256);
                top = fmaxf(top, row_scale[(s ^ 1) * 128 + r]);
                named_barrier_sync(2, 256);
            }
            // 2^(8 - exponent of the row's largest value), within fp32's normal range
            const int e = static_cast<int>(__float_as_uint(top) >> 23);
            const int up = top > 0.0f ? min(max(135 - e, -120), 120) : 0;
            // (the scale's sign goes to the queries, and 0 to the smallest number: a hidden score stays -inf)
            const float to_f16 = copysignf(__uint_as_float(static_cast<uint32_t>(127 + up) << 23), a.scale);
            rs = fmaxf(fabsf(a.scale) * tree_factor(a.group) * __uint_as_float(static_cast<uint32_t>(127 - up) << 23), 1.4e-45f);
            if (!PAIR && D == 64 && mine) row_scale[r] = rs;
            #pragma unroll 1
            for (int from = kSplit ? 64 * s : 0; mine && from < D; from += 64) {
                if (PAIR && D == 128) channels(from);
                unsigned char* base = smem + (PAIR ? 2 * s : 0) * Cfg::kOperand + from / 64 * Cfg::kAtom + r * 128;
                #pragma unroll
                for (int c = 0; c < 8; ++c) {
                    uint32_t hi[4], lo[4];
                    #pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float x = v[8 * c + 2 * k] * to_f16, y = v[8 * c + 2 * k + 1] * to_f16;
                        hi[k] = f16x2_bits(x, y);
                        __half2 h;
                        memcpy(&h, &hi[k], 4);
                        const float2 back = __half22float2(h);
                        lo[k] = f16x2_bits(x - back.x, y - back.y);
                    }
                    unsigned char* to = base + ((c ^ (r & 7)) << 4);
                    *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *reinterpret_cast<uint4*>(to + Cfg::kOperand) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
                if (kSplit) break;
            }
            if (mine) {
                fence_proxy_async_smem();
                mbar_arrive(q_full);
            }
        }
        const int ns = s ? n1 : n0, first = s ? c1 : c0, buf = PAIR ? 0 : s;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem_s(s) + lanes, to = tmem_o(s) + lanes;
        float m = kMx4NoScore, l = 0.0f;
        bool ok = true;
        if (!PAIR && D == 64 && s == 1 && ns) {                   // (the first stream's threads have scaled the rows)
            ok = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(q_full, 0));
            rs = row_scale[r];
        }
        const bool node = real && t < tree.nodes;                 // (what other rows compute is not kept)
        bool huge = false;                                        // some row's reference is beyond kTreeHuge (one without a score has none)
        for (int i = 0; ok && i < ns; ++i) {
            ok = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(&s_full[s], i & 1) && mbar_wait_bounded(&f_full[buf * 2 + (i & 1)], (i >> 1) & 1));
            if (!ok) break;
            tc_fence_after();
            const float* f = fac + (buf * 2 + (i & 1)) * 128;
            const uint32_t* gone = hid + (buf * 2 + (i & 1)) * 8;
            const int j0 = (first + i) * kTreeTile;
            const bool hides = !__all_sync(0xFFFFFFFFu, !node || (j0 + kTreeTile <= tree.context && (gone[0] | gone[1] | gone[2] | gone[3]) == 0));
            // Scores to m's scale: what the products gave times the tile's own factor, or with columns that are
            // hidden or keys far apart, column by column.
            const bool slow = hides || gone[4] != 0u || huge;
            const float sc = slow ? rs : rs * f[0];
            float sum = 0.0f;
            auto weights = [&](const uint32_t (&x)[16], float2 (&w)[8], float scale) {
                const float2 less = make_float2(-(m + kTreeDown), -(m + kTreeDown)), by = make_float2(scale, scale);
                float2 part[2] = {};
                #pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float2 y = ffma2_rn(make_float2(__uint_as_float(x[2 * k]), __uint_as_float(x[2 * k + 1])), by, less);
                    w[k] = make_float2(ex2(y.x), ex2(y.y));
                    part[k & 1] = fadd2_rn(part[k & 1], w[k]);
                }
                const float2 both = fadd2_rn(part[0], part[1]);
                return both.x + both.y;
            };
            auto store = [&](int c, const float2 (&w)[8]) {
                uint32_t p[16];
                #pragma unroll
                for (int k = 0; k < 8; ++k) split_bf16(w[k], p[k], p[8 + k]);
                tmem_st_32x32b_x16(ts + 16 * c, p);
            };
            // The reference is one of earlier tiles, as long as the weights stay below 2^-14 (their sum tells).
            // Chunks of 16 columns in three stages: scores on their way, weights of the next chunk, terms of
            // this one, so that the unit of exp2 works while others do. (Two chunks a round and no more:
            // with all roles' loops unrolled, warps waited for instructions a fifth of the time.)
            int c = 0;
            if (!slow) {
                uint32_t sr[16];
                float2 w[2][8];
                float here[2];
                tmem_ld_32x32b_x16(ts, sr);
                tmem_ld_wait_regs16(sr);
                here[0] = weights(sr, w[0], sc);
                tmem_ld_32x32b_x16(ts + 16, sr);
                #pragma unroll 1
                for (; c < 6; c += 2) {
                    tmem_ld_wait_regs16(sr);
                    here[1] = weights(sr, w[1], sc);
                    tmem_ld_32x32b_x16(ts + 16 * (c + 2), sr);
                    if (__any_sync(0xFFFFFFFFu, here[0] > kTreeMost)) break;
                    sum += here[0];
                    store(c, w[0]);
                    tmem_ld_wait_regs16(sr);
                    here[0] = weights(sr, w[0], sc);
                    tmem_ld_32x32b_x16(ts + 16 * (c + 3), sr);
                    if (__any_sync(0xFFFFFFFFu, here[1] > kTreeMost)) { ++c; break; }
                    sum += here[1];
                    store(c + 1, w[1]);
                }
                tmem_ld_wait_regs16(sr);
                if (c == 6) {
                    here[1] = weights(sr, w[1], sc);
                    if (!__any_sync(0xFFFFFFFFu, here[0] > kTreeMost)) {
                        sum += here[0];
                        store(6, w[0]);
                        c = 7;
                        if (!__any_sync(0xFFFFFFFFu, here[1] > kTreeMost)) {
                            sum += here[1];
                            store(7, w[1]);
                            c = 8;
                        }
                    }
                }
            }
            if (c < 8) {
                // From chunk c on: the reference moves to the largest score, what was summed and laid down
                // gets the new scale.
                const bool far = slow && (gone[4] & kTreeFar);
                if (__builtin_expect(far, 0)) tree_far_scores<D>(ts, smem + (PAIR ? 2 * s : 0) * Cfg::kOperand, r, a.codes, a.scales, a.table + b * a.table_ld, a.page_bits, a.pages,
                                            a.hkv, hk, j0, n, f);
                unsigned long long seen[2] = {~0ull, ~0ull};      // columns that this row sees
                if (hides) {
                    #pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        unsigned long long bits = 0;
                        #pragma unroll 1
                        for (int k = 0; k < 64; k += 16) {
                            const int from = j0 + 64 * half + k;
                            uint32_t some = 0;
                            if (from + 16 <= tree.context) {
                                some = 0xFFFFu;
                            } else if (from < n) {
                                #pragma unroll
                                for (int e = 0; e < 16; ++e) some |= static_cast<uint32_t>(tree.sees_any(t, from + e)) << e;
                            }
                            bits |= static_cast<unsigned long long>(some) << k;
                        }
                        seen[half] = bits & ~(static_cast<unsigned long long>(gone[2 * half]) | static_cast<unsigned long long>(gone[2 * half + 1]) << 32);
                    }
                }
                auto columns = [&](int at, uint32_t (&x)[16]) {
                    if (!slow) return;
                    const uint32_t bits = static_cast<uint32_t>((at < 4 ? seen[0] : seen[1]) >> (16 * (at & 3)));
                    const float* by = far ? reinterpret_cast<const float*>(smem + Cfg::kOneOffset) : f + 16 * at;
                    #pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const float y = __uint_as_float(x[k]) * by[k];
                        x[k] = bits >> k & 1u ? __float_as_uint(y) : 0xFF800000u;
                    }
                };
                float top = -INFINITY;
                #pragma unroll 1
                for (int at = c; at < 8; ++at) {
                    uint32_t x[16];
                    tmem_ld_32x32b_x16(ts + 16 * at, x);
                    tmem_ld_wait_regs16(x);
                    columns(at, x);
                    #pragma unroll
                    for (int k = 0; k < 16; ++k) top = fmaxf(top, __uint_as_float(x[k]));
                }
                top *= sc;
                if (__any_sync(0xFFFFFFFFu, top > m + 6.0f)) {
                    const float was = m;
                    m = fmaxf(m, top);
                    huge = __any_sync(0xFFFFFFFFu, fabsf(m) >= kTreeHuge && m > kMx4NoScore);
                    const float down = ex2(was - m);
                    l *= down;
                    sum *= down;
                    #pragma unroll 1
                    for (int at = 0; i > 0 && at < D / 16; ++at) {
                        uint32_t o[16];
                        tmem_ld_32x32b_x16(to + 16 * at, o);
                        tmem_ld_wait_regs16(o);
                        #pragma unroll
                        for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * down);
                        tmem_st_32x32b_x16(to + 16 * at, o);
                    }
                    if (c > 0) tmem_st_wait();                    // (what was laid down is read back)
                    #pragma unroll 1
                    for (int at = 0; at < c; ++at) {
                        uint32_t p[16];
                        tmem_ld_32x32b_x16(ts + 16 * at, p);
                        tmem_ld_wait_regs16(p);
                        #pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float x = (__uint_as_float(p[k] << 16) + __uint_as_float(p[8 + k] << 16)) * down;
                            const float y = (__uint_as_float(p[k] & 0xFFFF0000u) + __uint_as_float(p[8 + k] & 0xFFFF0000u)) * down;
                            split_bf16(make_float2(x, y), p[k], p[8 + k]);
                        }
                        tmem_st_32x32b_x16(ts + 16 * at, p);
                    }
                }
                #pragma unroll 1
                for (; c < 8; ++c) {
                    uint32_t x[16];
                    float2 w[8];
                    tmem_ld_32x32b_x16(ts + 16 * c, x);
                    tmem_ld_wait_regs16(x);
                    columns(c, x);
                    if (__builtin_expect(huge, 0)) {
                        // (rounded like the reference: half a step between the two would be more than an exponent holds)
                        #pragma unroll
                        for (int k = 0; k < 16; ++k) x[k] = __float_as_uint(__fmul_rn(__uint_as_float(x[k]), sc));
                    }
                    sum += weights(x, w, huge ? 1.0f : sc);
                    store(c, w);
                }
            }
            l += sum;
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(&p_full[s]);
        }
        // ---------------- the row's mean
        if (ok && ns) ok = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(&o_done[s], 0));
        if (!ok && lane == 0) tree_record_status(kMx4TimeoutEpilogue);
        tc_fence_after();
        const bool none = !ok || !node || (m == kMx4NoScore && l == 0.0f);        // (scores that are all NaN move no reference)
        if (none) { m = -INFINITY; l = 0.0f; }
        float* part = reinterpret_cast<float*>(smem);             // the operands' place, which nothing reads any more
        constexpr int kLd = 64 + 4;                               // floats of a row: rows in distinct banks
        float2* ml = reinterpret_cast<float2*>(smem + 128 * kLd * 4);
        static_assert(128 * (kLd * 4 + 8) <= 4 * Cfg::kOperand, "fits the first operands");
        float2 other = make_float2(-INFINITY, 0.0f);              // of the same rows in the second stream
        float mine_share = 1.0f, other_share = 0.0f;
        if constexpr (!PAIR) {
            named_barrier_sync(2, 256);                           // both streams' products are done
            if (s == 1) ml[r] = make_float2(m, l);
            named_barrier_sync(2, 256);
            other = ml[r];
        }
        const float own_m = m, own_l = l;
        if (!PAIR && s == 0) {
            m = fmaxf(own_m, other.x);
            const float w0 = own_m == -INFINITY ? 0.0f : ex2(own_m - m) * own_l, w1 = other.x == -INFINITY ? 0.0f : ex2(other.x - m) * other.y;
            l = w0 + w1;
            mine_share = w0 == 0.0f ? 0.0f : w0 / l;
            other_share = w1 == 0.0f ? 0.0f : w1 / l;
        }
        #pragma unroll 1
        for (int from = 0; from < D; from += 64) {
            float v[64];
            #pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t o[32];
                if (ns) {                                         // (of the whole warp)
                    tmem_ld_32x32b_x32(to + from + 32 * c, o);
                    tmem_ld_wait_regs(o);
                }
                const float inv = none ? 0.0f : 1.0f / own_l;
                #pragma unroll
                for (int k = 0; k < 32; ++k) v[32 * c + k] = none ? 0.0f : __uint_as_float(o[k]) * inv;
            }
            if constexpr (!PAIR) {
                named_barrier_sync(2, 256);
                if (s == 1) {
                    #pragma unroll
                    for (int i = 0; i < 64; i += 4) *reinterpret_cast<float4*>(part + r * kLd + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                }
                named_barrier_sync(2, 256);
                if (s == 0) {
                    #pragma unroll
                    for (int i = 0; i < 64; i += 4) {
                        const float4 x = *reinterpret_cast<const float4*>(part + r * kLd + i);
                        v[i] = mine_share * v[i] + other_share * x.x;
                        v[i + 1] = mine_share * v[i + 1] + other_share * x.y;
                        v[i + 2] = mine_share * v[i + 2] + other_share * x.z;
                        v[i + 3] = mine_share * v[i + 3] + other_share * x.w;
                    }
                }
            }
            if (!real || (!PAIR && s == 1)) continue;
            if (*nan_nodes && node) {
                for (int j = max(tree.context, c0 * kTreeTile); j < min(n, (c0 + count) * kTreeTile); ++j) {
                    const int page = a.table[b * a.table_ld + (j >> a.page_bits)];
                    if (page < 0 || page >= a.pages || !tree.sees(t, j)) continue;
                    const size_t place = (((static_cast<size_t>(page) * 2 + 1) * a.hkv + hk) << a.page_bits) + (j & ((1 << a.page_bits) - 1));
                    #pragma unroll
                    for (int k = 0; k < 2; ++k)
                        if (a.scales[place * kB + from / 32 + k] == 255) {
                            #pragma unroll
                            for (int i = 0; i < 32; ++i) v[32 * k + i] = NAN;
                        }
                }
            }
            const size_t at = (static_cast<size_t>(tile) * a.splits + split) * kTileRows + (row - row0);
            // (a whole sequence's rows need no join, which the sum below zero tells it)
            if (from == 0 && a.splits > 1) a.part_ml[at] = splits > 1 ? make_float2(m, l) : make_float2(0.0f, -1.0f);
            if (splits > 1) {
                #pragma unroll
                for (int i = 0; i < 64; i += 4) *reinterpret_cast<float4*>(a.part + at * D + from + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
            } else {
                tree_rotate(v, a.group);
                const float f = tree_factor(a.group);
                T* out = static_cast<T*>(a.out) + ((static_cast<size_t>(b) * a.tq + t) * a.hq + hk * per_head + row % per_head) * D + from;
                #pragma unroll
                for (int i = 0; i < 64; i += 8) {
                    T e[8];
                    #pragma unroll
                    for (int k = 0; k < 8; ++k) e[k] = mx4_from_f32<T>(v[i + k] * f);
                    uint4 x;
                    memcpy(&x, e, 16);
                    *reinterpret_cast<uint4*>(out + i) = x;
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 14) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace convrot
