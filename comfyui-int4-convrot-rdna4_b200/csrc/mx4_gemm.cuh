// out[m, n] = sum_k x[m, k] w[n, k] + bias[n] on MX4 operands: tcgen05 block-scaled
// MMAs on CTA pairs (kind::mxf4, cta_group::2), persistent over output tiles.
//
// Included by mx4.cu. The codes go by TMA from global memory to shared memory and
// from there to the tensor cores as they are stored; the scale tiles take the
// same way through tcgen05.cp into tensor memory. A tile is 256 rows of x times
// BN rows of w; each CTA of the pair holds half of both operands, the scales of
// its own rows of x and those of all BN rows of w.
//
// A stage of the ring is 256 values of K: [x 128 rows x 128 B | w BN/2 rows x
// 128 B | x scales: two tiles | w scales: two tiles for each 128 rows].
//
// Warp roles (8 warps, both CTAs alike):
//   w0, w2   TMA producers: codes, scales
//   w1       TMEM allocation; in the even CTA the MMA issuer
//   w4..w7   epilogue (TMEM lanes 32 * (w % 4) ..): fp32 + bias, one rounding, a
//            warp's 32 rows x 128 bytes at a time through shared memory and TMA
//            (direct stores where the output's pitch is no multiple of 16 bytes)
//
// Tensor memory, 512 columns. BN = 256: two accumulators of 256 columns that
// share 64 (columns 192..255), and 64 columns of scales (two stages of 24). The
// epilogue reads the shared columns first and hands them over, so the next
// tile's MMAs wait for those 64 columns only and run beside the rest of the
// epilogue. BN = 128: two separate accumulators.
//
// Bound by the tensor cores: 4096 x 16384 x 8192 takes 173 us (6.4 PFLOP/s, tensor pipe
// busy 85 % of the launch), 4096 x 15360 x 3840 86 us (5.6 PFLOP/s, 73 %: 15 stages a
// tile, and 500 cycles from a tile's last MMA to the next one's first). A stage of a
// 256-wide tile is 502 cycles of MMAs and 35 KB a CTA, at the 64 bytes a cycle that L2
// gives a multiprocessor 560; of a 128-wide tile 250 and 27 KB, 400. In long runs the
// power limit holds the clock near 1.3 GHz: 16384 x 15360 x 3840 in 345 to 385 us.
// Two pairs a tile with half of K each were slower or equal at every size tried: only 33
// clusters of four fit the machine, and the exchange costs what half the stages save.
#pragma once

namespace convrot {

constexpr int kMx4PairThreads = 256;
constexpr int kMx4StageK = 256;               // values of K a stage
constexpr int kMx4TmemCols = 512;

// A slot of a ring of N and the parity of its current use.
template <int N>
struct Mx4Ring {
    int slot = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next() {
        if (++slot == N) {
            slot = 0;
            phase ^= 1;
        }
    }
};

// Whole-warp wait: one look (often taken ahead, by the caller) and a vote when the
// phase is complete, else the bounded wait.
__device__ __forceinline__ bool mx4_wait_warp(uint64_t* bar, uint32_t parity, bool seen) {
    if (__all_sync(0xFFFFFFFFu, seen)) return true;
    return __all_sync(0xFFFFFFFFu, mbar_wait_bounded(bar, parity));
}

template <int BN>
struct Mx4PairCfg {
    static constexpr int kABytes = 128 * kMx4StageK / 2;
    static constexpr int kBBytes = BN / 2 * kMx4StageK / 2;
    static constexpr int kSaBytes = 2 * kMx4TileBytes;
    static constexpr int kSbBytes = BN / 128 * 2 * kMx4TileBytes;
    static constexpr int kStageBytes = kABytes + kBBytes + kSaBytes + kSbBytes;
    static constexpr int kStagingBytes = 4 * 2 * 32 * 128;        // four warps, two buffers of 32 rows x 128 B
    static constexpr int kStages0 = (227 * 1024 - 1024 - 512 - 2 * BN * 4 - kStagingBytes) / kStageBytes;
    static constexpr int kStages = kStages0 > 8 ? 8 : kStages0;
    static constexpr int kStagingOffset = kStages * kStageBytes;
    static constexpr int kBiasOffset = kStagingOffset + kStagingBytes;
    static constexpr int kBarOffset = kBiasOffset + 2 * BN * 4;
    static constexpr int kSmemBytes = kBarOffset + 512 + 1024;
    static constexpr int kAcc1 = BN == 256 ? 192 : BN;            // column of the second accumulator
    static constexpr int kShared = BN == 256 ? 64 : 0;            // columns both accumulators use
    static constexpr int kScaleCol = 448;
    static constexpr int kScaleCols = 8 + BN / 128 * 8;           // one stage: x 2 x 4, w 2 x 4 x (BN / 128)
    static_assert(kStages >= 4 && kSmemBytes <= 227 * 1024, "shared memory budget");
    static_assert(kAcc1 + BN <= kScaleCol && kScaleCol + 2 * kScaleCols <= kMx4TmemCols, "TMEM budget");
};

// One row's 128 bytes of output (32 f32 or 64 16-bit values) from accumulator
// columns and bias, packed for the store.
template <typename T>
__device__ __forceinline__ void mx4_pack_row(const uint32_t* acc, const float* bias, uint32_t (&w)[32]) {
    if constexpr (sizeof(T) == 4) {
        #pragma unroll
        for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(__uint_as_float(acc[i]) + bias[i]);
    } else {
        #pragma unroll
        for (int i = 0; i < 32; ++i) {
            const float a = __uint_as_float(acc[2 * i]) + bias[2 * i], b = __uint_as_float(acc[2 * i + 1]) + bias[2 * i + 1];
            if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
                memcpy(&w[i], &p, 4);
            } else {
                const __half2 p = __floats2half2_rn(a, b);
                memcpy(&w[i], &p, 4);
            }
        }
    }
}

template <int BN, typename T>
__global__ void __launch_bounds__(kMx4PairThreads, 1)
mx4_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
                     const __grid_constant__ CUtensorMap tmap_xs, const __grid_constant__ CUtensorMap tmap_ws,
                     const __grid_constant__ CUtensorMap tmap_out, BiasRef bias, T* __restrict__ out, int M, int N, int K,
                     int tiles_m, int num_tiles, int staged) {
    using Cfg = Mx4PairCfg<BN>;
    constexpr int kCols = 128 / static_cast<int>(sizeof(T));      // output columns of one store box
    extern __shared__ __align__(1024) unsigned char mx4smem_raw[];
    unsigned char* smem = mx4smem_raw + ((1024u - (smem_u32(mx4smem_raw) & 1023u)) & 1023u);
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + Cfg::kBarOffset);
    uint64_t* empty_bar = full_bar + Cfg::kStages;
    uint64_t* acc_full = empty_bar + Cfg::kStages;                // [2]
    uint64_t* acc_free = acc_full + 2;                            // [2] what the waiting tile's MMAs overwrite is read
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_free + 2);
    float* bias_cols = reinterpret_cast<float*>(smem + Cfg::kBiasOffset);    // [2][BN]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t cta = cluster_ctarank();
    const int cluster_id = blockIdx.x >> 1, num_clusters = gridDim.x >> 1;
    const int num_kt = (K + kMx4StageK - 1) / kMx4StageK;
    const int my_tiles = (num_tiles - cluster_id + num_clusters - 1) / num_clusters;

    if (threadIdx.x == 0) {
        for (int s = 0; s < Cfg::kStages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_free[b], 8);                           // four epilogue warps of each CTA
        }
        fence_mbar_init();
        tma_prefetch_desc(&tmap_x);
        tma_prefetch_desc(&tmap_w);
        tma_prefetch_desc(&tmap_xs);
        tma_prefetch_desc(&tmap_ws);
        if (staged) tma_prefetch_desc(&tmap_out);
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, kMx4TmemCols);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0 || warp == 2) {
        // ---------------- TMA producers: w0 codes, w2 scales; both CTAs' tiles complete on
        // the even CTA's barrier. The warp runs the loop (uniform addresses), one elected
        // lane issues: a lane on its own took 600 cycles a stage for its four copies.
        const uint32_t full0 = mapa_shared(smem_u32(full_bar), 0);
        Mx4Ring<Cfg::kStages> ring;
        bool ok = true;
        for (int t = cluster_id; t < num_tiles && ok; t += num_clusters) {
            const int m0 = t % tiles_m * 256 + static_cast<int>(cta) * 128;
            const int n0 = t / tiles_m * BN;
            for (int kt = 0; kt < num_kt; ++kt, ring.next()) {
                const int s = ring.slot;
                if (!mx4_wait_warp(&empty_bar[s], ring.phase ^ 1, mbar_test_wait(&empty_bar[s], ring.phase ^ 1))) {
                    if (lane == 0) mx4_record_status(kMx4TimeoutProducer);
                    ok = false;
                    break;
                }
                unsigned char* st = smem + s * Cfg::kStageBytes;
                const uint32_t full = full0 + s * 8;
                if (elect_one()) {
                    if (warp == 0) {
                        if (cta == 0) mbar_arrive_expect_tx(&full_bar[s], 2 * Cfg::kStageBytes);
                        tma_load_2d_pair(st, &tmap_x, full, kt * (kMx4StageK / 2), m0);
                        tma_load_2d_pair(st + Cfg::kABytes, &tmap_w, full, kt * (kMx4StageK / 2),
                                         n0 + static_cast<int>(cta) * (BN / 2));
                    } else {
                        unsigned char* sf = st + Cfg::kABytes + Cfg::kBBytes;
                        tma_load_2d_pair(sf, &tmap_xs, full, kt * 256, m0 / 128);
                        tma_load_2d_pair(sf + Cfg::kSaBytes, &tmap_ws, full, kt * 256, n0 / 128);
                    }
                }
                __syncwarp();
            }
        }
    } else if (warp == 1) {
        if (cta == 0) {
            // ---------------- MMA issuer: the warp runs the loop, one elected lane issues.
            // The loop has to take less than a stage's MMAs (500 cycles at BN = 256): the
            // next stage's barrier is looked at before this stage's MMAs are issued, and
            // descriptors are a base and a multiple of the slot.
            const uint32_t base = smem_u32(smem);
            const uint64_t da0 = smem_desc_kmajor(base, 1024, 2), db0 = smem_desc_kmajor(base + Cfg::kABytes, 1024, 2);
            // scale tiles: 512 bytes each, 32 in descriptor units
            const uint64_t dsa0 = smem_desc_kmajor(base + Cfg::kABytes + Cfg::kBBytes, 128, 0);
            const uint64_t dsb0 = smem_desc_kmajor(base + Cfg::kABytes + Cfg::kBBytes + Cfg::kSaBytes, 128, 0);
            const int odd_tail = (K + 127) / 128 & 1;              // the last stage has one 128-value half
            Mx4Ring<Cfg::kStages> ring;
            uint32_t sf = tmem + Cfg::kScaleCol;
            const uint32_t sf_flip = sf ^ (sf + Cfg::kScaleCols);
            bool ok = true, seen = mbar_test_wait(&full_bar[0], 0);
            for (int lt = 0; lt < my_tiles && ok; ++lt) {
                // the tile before this one shares columns with it (kShared), else the
                // one before that used this accumulator
                const int before = Cfg::kShared ? lt - 1 : lt - 2;
                if (before >= 0 && !__all_sync(0xFFFFFFFFu, mbar_wait_bounded(&acc_free[before & 1], (before >> 1) & 1))) {
                    if (lane == 0) mx4_record_status(kMx4TimeoutMma);
                    break;
                }
                tc_fence_after();
                const uint32_t acc = tmem + ((lt & 1) ? Cfg::kAcc1 : 0);
                for (int kt = 0; kt < num_kt; ++kt) {
                    const int s = ring.slot;
                    if (!mx4_wait_warp(&full_bar[s], ring.phase, seen)) {
                        if (lane == 0) mx4_record_status(kMx4TimeoutMma);
                        ok = false;
                        break;
                    }
                    ring.next();
                    seen = mbar_test_wait(&full_bar[ring.slot], ring.phase);
                    tc_fence_after();
                    const uint64_t at = static_cast<uint64_t>(s * (Cfg::kStageBytes / 16));
                    const bool both = !(odd_tail && kt == num_kt - 1);
                    if (elect_one()) {
                        const uint64_t da = da0 + at, db = db0 + at, dsa = dsa0 + at, dsb = dsb0 + at;
                        auto half = [&](int h) {
                            tmem_cp_scales<true>(sf + 4 * h, dsa + 32 * h);
                            #pragma unroll
                            for (int j = 0; j < BN / 128; ++j)
                                tmem_cp_scales<true>(sf + 8 + (BN / 32) * h + 4 * j, dsb + 64 * j + 32 * h);
                        };
                        auto product = [&](int j) {
                            mma_mxf4<true>(acc, da + 2 * j, db + 2 * j, idesc_mxf4(256, BN, (j & 1) * 2), sf + 4 * (j >> 1),
                                           sf + 8 + (BN / 32) * (j >> 1), (kt | j) != 0);
                        };
                        half(0);
                        if (both) half(1);
                        product(0);
                        product(1);
                        if (both) {
                            product(2);
                            product(3);
                        }
                        mma_commit_pair_multicast(&empty_bar[s], 0x3);
                    }
                    sf ^= sf_flip;
                    __syncwarp();
                }
                if (ok && elect_one()) mma_commit_pair_multicast(&acc_full[lt & 1], 0x3);
                __syncwarp();
            }
        }
    } else if (warp >= 4) {
        // ---------------- epilogue
        const int quarter = warp & 3, et = threadIdx.x - 128;
        unsigned char* staging = smem + Cfg::kStagingOffset + quarter * 2 * 4096;
        const uint32_t free_leader = mapa_shared(smem_u32(acc_free), 0);
        int box = 0;                                              // store boxes so far (buffer = box % 2)
        for (int lt = 0; lt < my_tiles; ++lt) {
            const int t = cluster_id + lt * num_clusters;
            const int row0 = t % tiles_m * 256 + static_cast<int>(cta) * 128 + quarter * 32;
            const int n0 = t / tiles_m * BN;
            float* bc = bias_cols + (lt & 1) * BN;
            for (int c = et; c < BN; c += 128) bc[c] = bias.ptr != nullptr && n0 + c < N ? bias.at(n0 + c) : 0.0f;
            named_barrier_sync(1, 128);
            if (!__all_sync(0xFFFFFFFFu, mbar_wait_bounded(&acc_full[lt & 1], (lt >> 1) & 1))) {
                if (lane == 0) mx4_record_status(kMx4TimeoutEpilogue);
                break;
            }
            tc_fence_after();
            const uint32_t acc = tmem + ((lt & 1) ? Cfg::kAcc1 : 0) + (static_cast<uint32_t>(quarter * 32) << 16);
            // columns in steps of one store box, the shared ones (the end of the
            // first accumulator, the start of the second) first
            constexpr int kSteps = BN / kCols;
            constexpr int kSharedSteps = Cfg::kShared / kCols;
            #pragma unroll 1
            for (int i = 0; i < kSteps; ++i) {
                const int step = (lt & 1) ? i : (i + kSteps - kSharedSteps) % kSteps;
                const int col = step * kCols;
                uint32_t v[64];
                tmem_ld_32x32b_x32(acc + col, *reinterpret_cast<uint32_t (*)[32]>(v));
                if constexpr (kCols == 64) tmem_ld_32x32b_x32(acc + col + 32, *reinterpret_cast<uint32_t (*)[32]>(v + 32));
                tmem_ld_wait_regs(*reinterpret_cast<uint32_t (*)[32]>(v));
                if constexpr (kCols == 64) tmem_ld_wait_regs(*reinterpret_cast<uint32_t (*)[32]>(v + 32));
                if (i == (kSharedSteps ? kSharedSteps : kSteps) - 1) {
                    // read: hand the shared columns (BN = 128: the accumulator) over. The values are
                    // in registers, so the arrival orders nothing in memory: CTA scope, as a
                    // cluster-scope release waits for the stores under way
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if (cta == 0) mbar_arrive(&acc_free[lt & 1]);
                        else mbar_arrive_remote_cta(free_leader + (lt & 1) * 8);
                    }
                }
                const int n = n0 + col;
                if (n >= N) continue;
                uint32_t w[32];
                mx4_pack_row<T>(v, bc + col, w);
                if (staged) {
                    unsigned char* buf = staging + (box & 1) * 4096;
                    if (lane == 0) bulk_wait_group_read1();       // the store two boxes ago has read this buffer
                    __syncwarp();
                    #pragma unroll
                    for (int q = 0; q < 8; ++q)
                        *reinterpret_cast<uint4*>(buf + lane * 128 + ((q ^ (lane & 7)) << 4)) =
                            make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        if (row0 < M) tma_store_2d(&tmap_out, buf, n, row0);
                        bulk_commit_group();
                    }
                    ++box;
                } else if (row0 + lane < M) {
                    T* o = out + static_cast<size_t>(row0 + lane) * N + n;
                    #pragma unroll
                    for (int e = 0; e < kCols; ++e) {
                        if (n + e >= N) break;
                        if constexpr (sizeof(T) == 4) o[e] = __uint_as_float(w[e]);
                        else reinterpret_cast<uint16_t*>(o)[e] = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
                    }
                }
            }
        }
        if (staged && lane == 0) bulk_wait_group0();
    }
    tc_fence_before();
    cluster_sync();                       // no CTA leaves while its pair may still touch its TMEM
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, kMx4TmemCols);
    }
}

}  // namespace convrot
