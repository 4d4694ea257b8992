// The MX4 linear for few rows (M <= 128): bound by the weight's bytes.
//
// Included by mx4.cu. The weight takes the tensor core's side of 128 rows and the
// tokens the other (BT = 16, 32, 64 or 128 columns), so a block streams 128 weight
// rows and multiplies them with all tokens. The blocks of a cluster take slices of
// K of one tile (few weight rows then still fill the machine) and add their fp32
// accumulators over distributed shared memory, in rank order.
//
// FUSED (up to 16 rows): the activations are rotated and quantized here, by the
// epilogue's warps while the weight is on its way, a stage (256 columns of 16
// rows: 32 units, a lane each) by one warp. Every block quantizes its slice of K
// again, which for 16 rows costs less than a launch and a pass through memory.
//
// Warp roles (6 warps, so that two blocks' registers fit a multiprocessor): w0 TMA
// producer (one lane), w1 tensor memory and MMA issue, w2..w5 quantizers (FUSED) and
// epilogue (TMEM lanes 32 * (w % 4) ..).
#pragma once

namespace convrot {

constexpr int kMx4FewThreads = 192;
constexpr int kMx4FusedRows = 16;              // rows up to which the kernel quantizes them itself

template <typename T, int BT, bool FUSED>
struct Mx4FewCfg {
    static constexpr int kABytes = 128 * kMx4StageK / 2;
    static constexpr int kBBytes = BT * kMx4StageK / 2;
    static constexpr int kScaleBytes = 2 * kMx4TileBytes;         // of each operand
    static constexpr int kStageBytes = (kABytes + kBBytes + 2 * kScaleBytes + 1023) / 1024 * 1024;
    static constexpr int kStages = BT == 128 || FUSED ? 3 : 4;    // two blocks a multiprocessor (fp32 rows: one)
    static constexpr int kSlabBytes = FUSED ? 4 * Mx4Slab<T>::kBytes : 0;
    static constexpr int kSlabOffset = kStages * kStageBytes;
    static constexpr int kBarOffset = kSlabOffset + kSlabBytes;
    static constexpr int kSmemBytes = kBarOffset + 256 + 1024;
    static constexpr int kScaleCol = BT;                          // two buffers of 8 + 8 columns after the accumulator
    static constexpr int kTmemCols = BT == 16 ? 64 : BT == 32 ? 64 : BT == 64 ? 128 : 256;
    static_assert(kScaleCol + 32 <= kTmemCols, "tensor memory");
    static_assert(BT * 128 * 4 <= kStages * kStageBytes, "the accumulators fit the ring");
};

__device__ __forceinline__ void tmem_ld_32x32b_x16_wait(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                   "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(taddr) : "memory");
}

// Adds the S ranks' accumulators [token][128] of this rank's tokens (rank, rank + S,
// ..), in rank order. A warp a token, a lane four outputs; eight loads are under way
// before the first is used.
template <typename T, int S>
__device__ __forceinline__ void few_reduce(unsigned char* smem, int rank, const BiasRef& bias, T* out, int n0, int M, int N) {
    constexpr int kBatch = 8 / S;                                 // tokens of a batch
    const int t = static_cast<int>(threadIdx.x) - 64, n = n0 + (t & 31) * 4;
    const uint32_t red = smem_u32(smem) + (t & 31) * 16;
    uint32_t at[S];
    #pragma unroll
    for (int r = 0; r < S; ++r) at[r] = mapa_shared(red, r);
    float b[4];
    #pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = bias.ptr != nullptr && n + e < N ? bias.at(n + e) : 0.0f;
    for (int m0 = rank + (t >> 5) * S; m0 < M; m0 += 4 * S * kBatch) {
        float4 v[kBatch][S];
        #pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int m = min(m0 + 4 * S * i, M - 1);             // (a token beyond the last: read, not written)
            #pragma unroll
            for (int r = 0; r < S; ++r) v[i][r] = ld_shared_cluster_f4(at[r] + m * 512);
        }
        #pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int m = m0 + 4 * S * i;
            float4 sum = v[i][0];
            #pragma unroll
            for (int r = 1; r < S; ++r) {
                sum.x += v[i][r].x;
                sum.y += v[i][r].y;
                sum.z += v[i][r].z;
                sum.w += v[i][r].w;
            }
            const T o[4] = {mx4_from_f32<T>(sum.x + b[0]), mx4_from_f32<T>(sum.y + b[1]), mx4_from_f32<T>(sum.z + b[2]), mx4_from_f32<T>(sum.w + b[3])};
            if (m >= M) break;
            T* dst = out + static_cast<size_t>(m) * N + n;
            if (N % 4 == 0 && n < N) {
                memcpy(__builtin_assume_aligned(dst, 4 * sizeof(T)), o, 4 * sizeof(T));
            } else {
                #pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n + e < N) dst[e] = o[e];
            }
        }
    }
}

template <typename T, int G, int BT, bool FUSED>
__global__ void __launch_bounds__(kMx4FewThreads, 2)
mx4_gemm_few_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_ws,
                    const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_xs,
                    const T* __restrict__ x, long long ldx, bool vec, BiasRef bias,
                    T* __restrict__ out, int M, int N, int K) {
    using Cfg = Mx4FewCfg<T, BT, FUSED>;
    constexpr int kLd = BT < 32 ? 16 : 32;                        // accumulator columns read at a time
    extern __shared__ __align__(1024) unsigned char mx4few_raw[];
    unsigned char* smem = mx4few_raw + ((1024u - (smem_u32(mx4few_raw) & 1023u)) & 1023u);
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + Cfg::kBarOffset);
    uint64_t* ready_bar = full_bar + Cfg::kStages;                // FUSED: the stage's tokens are quantized
    uint64_t* empty_bar = ready_bar + Cfg::kStages;
    uint64_t* acc_bar = empty_bar + Cfg::kStages;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_bar + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n0 = blockIdx.x * 128, splits = gridDim.y, rank = blockIdx.y;
    const int num_kt = (K + kMx4StageK - 1) / kMx4StageK, per = (num_kt + splits - 1) / splits;
    const int kt0 = min(rank * per, num_kt), kts = min(per, num_kt - kt0);     // this block's stages (some, or none)

    if (threadIdx.x == 0) {
        for (int s = 0; s < Cfg::kStages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&ready_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        mbar_init(acc_bar, 1);
        fence_mbar_init();
        tma_prefetch_desc(&tmap_w);
        tma_prefetch_desc(&tmap_ws);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, Cfg::kTmemCols);
        tmem_relinquish();
    }
    // the first weight boxes into L2 (a hint: safe whatever the previous kernel wrote)
    if (warp == 2 && lane < Cfg::kStages && lane < kts) tma_prefetch_l2_2d(&tmap_w, (kt0 + lane) * (kMx4StageK / 2), n0);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            // ---------------- TMA producer
            for (int it = 0; it < kts; ++it) {
                const int s = it % Cfg::kStages;
                if (!mbar_wait_bounded(&empty_bar[s], ((it / Cfg::kStages) & 1) ^ 1)) {
                    mx4_record_status(kMx4TimeoutProducer);
                    break;
                }
                unsigned char* st = smem + s * Cfg::kStageBytes;
                unsigned char* sf = st + Cfg::kABytes + Cfg::kBBytes;
                const int kt = kt0 + it;
                mbar_arrive_expect_tx(&full_bar[s], Cfg::kABytes + Cfg::kScaleBytes + (FUSED ? 0 : Cfg::kBBytes + Cfg::kScaleBytes));
                tma_load_2d(st, &tmap_w, &full_bar[s], kt * (kMx4StageK / 2), n0);
                tma_load_2d(sf, &tmap_ws, &full_bar[s], kt * 256, n0 / 128);
                if constexpr (!FUSED) {
                    tma_load_2d(st + Cfg::kABytes, &tmap_x, &full_bar[s], kt * (kMx4StageK / 2), 0);
                    tma_load_2d(sf + Cfg::kScaleBytes, &tmap_xs, &full_bar[s], kt * 256, 0);
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer: the warp runs the loop, one elected lane issues
        bool ok = true;
        for (int it = 0; it < kts && ok; ++it) {
            const int s = it % Cfg::kStages;
            const uint32_t ph = (it / Cfg::kStages) & 1;
            bool in = mbar_wait_bounded(&full_bar[s], ph);
            if (FUSED && in) in = mbar_wait_bounded(&ready_bar[s], ph);
            if (!__all_sync(0xFFFFFFFFu, in)) {
                if (lane == 0) mx4_record_status(kMx4TimeoutMma);
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t a = smem_u32(smem + s * Cfg::kStageBytes), sf = a + Cfg::kABytes + Cfg::kBBytes;
            const uint64_t da = smem_desc_kmajor(a, 1024, 2), db = smem_desc_kmajor(a + Cfg::kABytes, 1024, 2);
            const uint64_t dsa = smem_desc_kmajor(sf, 128, 0), dsb = smem_desc_kmajor(sf + Cfg::kScaleBytes, 128, 0);
            const uint32_t col = tmem + Cfg::kScaleCol + (it & 1) * 16;
            const int halves = K - (kt0 + it) * kMx4StageK > 128 ? 2 : 1;
            if (elect_one()) {
                #pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (h >= halves) break;
                    tmem_cp_scales<false>(col + 4 * h, dsa + 32 * h);
                    tmem_cp_scales<false>(col + 8 + 4 * h, dsb + 32 * h);
                }
                #pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (j >= 2 * halves) break;
                    mma_mxf4<false>(tmem, da + 2 * j, db + 2 * j, idesc_mxf4(128, BT, (j & 1) * 2), col + 4 * (j >> 1),
                                    col + 8 + 4 * (j >> 1), (it | j) != 0);
                }
                mma_commit(&empty_bar[s]);
            }
            __syncwarp();
        }
        if (ok && kts > 0 && elect_one()) mma_commit(acc_bar);
        __syncwarp();
    } else if (FUSED && warp >= 2) {
        // ---------------- quantizers: stages in turn, a lane a unit (row lane / 2, half lane & 1)
        unsigned char* slab = smem + Cfg::kSlabOffset + (warp - 2) * Mx4Slab<T>::kBytes;
        auto load = [&](int it) {
            const int row = lane >> 1, k = (kt0 + it) * kMx4StageK + (lane & 1) * kMx4Unit;
            const int cols = row < M ? max(0, min(kMx4Unit, K - k)) : 0;
            slab_load<false>(slab, Mx4UnitAt<T>{reinterpret_cast<const unsigned char*>(cols ? x + row * ldx + k : x), cols / Mx4Slab<T>::kPer}, 0, vec);
            cp_async_commit();
        };
        if (warp - 2 < kts) load(warp - 2);
        for (int it = warp - 2; it < kts; it += 4) {
            const int s = it % Cfg::kStages;
            cp_async_wait<0>();
            __syncwarp();
            float2 v[64];
            slab_to_unit<T>(slab, v);
            __syncwarp();
            if (it + 4 < kts) load(it + 4);
            unit_rotate<G>(v);
            uint4 q[4];
            const uint32_t word = unit_quantize(v, unit_factor<G>(), q);
            if (!__all_sync(0xFFFFFFFFu, mbar_wait_bounded(&empty_bar[s], ((it / Cfg::kStages) & 1) ^ 1))) {
                if (lane == 0) mx4_record_status(kMx4TimeoutProducer);
                break;
            }
            const int u = lane ^ (G == 256 ? 1 : 0), row = u >> 1, half = u & 1;
            unsigned char* b = smem + s * Cfg::kStageBytes + Cfg::kABytes;
            #pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(b + row * 128 + (((4 * half + i) ^ (row & 7)) << 4)) = q[i];
            *reinterpret_cast<uint32_t*>(b + Cfg::kBBytes + Cfg::kScaleBytes + half * kMx4TileBytes + row * 16) = word;
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ready_bar[s]);
        }
        cp_async_wait<0>();
    }
    if (warp >= 2) {
        // ---------------- epilogue: lane n0 + 32 q + lane, a column a token
        const int quarter = warp & 3, n = n0 + quarter * 32 + lane;
        float* red = reinterpret_cast<float*>(smem);              // [BT][128], in the ring's place
        const bool ok = kts == 0 || __all_sync(0xFFFFFFFFu, mbar_wait_bounded(acc_bar, 0));
        if (!ok && lane == 0) mx4_record_status(kMx4TimeoutEpilogue);
        tc_fence_after();
        const float b = bias.ptr != nullptr && n < N ? bias.at(n) : 0.0f;
        #pragma unroll 1
        for (int c = 0; c < BT && c < M; c += kLd) {
            uint32_t v[kLd];
            if (kts > 0) {
                const uint32_t at = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + c;
                if constexpr (kLd == 32) {
                    tmem_ld_32x32b_x32(at, v);
                    tmem_ld_wait_regs(v);
                } else {
                    tmem_ld_32x32b_x16_wait(at, v);
                }
            } else {
                #pragma unroll
                for (int e = 0; e < kLd; ++e) v[e] = 0u;
            }
            if (splits > 1) {
                // (columns beyond M too: the ring holds all BT)
                #pragma unroll
                for (int e = 0; e < kLd; ++e) red[(c + e) * 128 + quarter * 32 + lane] = __uint_as_float(v[e]);
            } else if (n < N) {
                T* dst = out + static_cast<size_t>(c) * N + n;
                #pragma unroll
                for (int e = 0; e < kLd; ++e)
                    if (c + e < M) dst[static_cast<size_t>(e) * N] = mx4_from_f32<T>(__uint_as_float(v[e]) + b);
            }
        }
        tc_fence_before();
    }
    if (splits > 1) {
        cluster_sync();                                           // every block's accumulators are in its shared memory
        if (warp >= 2) {
            if (splits == 2) few_reduce<T, 2>(smem, rank, bias, out, n0, M, N);
            else if (splits == 4) few_reduce<T, 4>(smem, rank, bias, out, n0, M, N);
            else few_reduce<T, 8>(smem, rank, bias, out, n0, M, N);
        }
        cluster_sync();                                           // no block leaves while others read its memory
    } else {
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, Cfg::kTmemCols);
    }
}

}  // namespace convrot
