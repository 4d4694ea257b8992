// The MX4 linear for few rows (M <= 128): bound by the weight's bytes.
//
// Included by mx4.cu. The weight takes the tensor core's side of 128 rows and the
// tokens the other (BT = 16, 32, 64 or 128 columns), so a block streams 128 weight
// rows and multiplies them with all tokens. The blocks of a cluster take slices of
// K of one tile (few weight rows then still fill the machine) and send each other
// their fp32 accumulators over distributed shared memory: each rank adds those of
// its own tokens, in rank order.
//
// FUSED (up to 8 rows): the activations are rotated and quantized here, by the
// epilogue's warps while the weight is on its way, a stage (256 columns) by one
// warp. Every block quantizes its slice of K again, which for few rows costs less
// than a launch and a pass through memory (15360 x 3840: 1 row 7.7 us, 8 rows 9.4 us;
// 16 rows would take 14.3 us, with a kernel of its own 10.5 us). A lane takes 16
// columns of two rows: short code and a short wait (128 columns a lane, as in
// mx4_unit.cuh, took 2.8 us to the first stage, most of it the first run through its
// instructions).
//
// Measured, weights beyond what L2 keeps: 1 x 15360 x 3840 7.7 us (31 MB, 4.1 TB/s), of
// it about 2 us to the first MMA and 2 us from the last one to the end of the output; with
// the quantizer's launch, 64 x 4096 x 4096 9.1 us and 128 x 15360 x 3840 13.8 us.
//
// Warp roles (6 warps, so that two blocks fit a multiprocessor): w0 TMA producer
// (one lane), w1 tensor memory and MMA issue, w2..w5 quantizers (FUSED) and epilogue
// (TMEM lanes 32 * (w % 4) ..).
#pragma once

namespace convrot {

constexpr int kMx4FewThreads = 192;
constexpr int kMx4FusedRows = 8;               // rows up to which the kernel quantizes them itself

template <int BT, bool FUSED>
struct Mx4FewCfg {
    static constexpr int kABytes = 128 * kMx4StageK / 2;
    static constexpr int kBBytes = BT * kMx4StageK / 2;
    static constexpr int kScaleBytes = 2 * kMx4TileBytes;         // of each operand
    static constexpr int kStageBytes = kABytes + kBBytes + 2 * kScaleBytes;
    // the ranks' accumulators of this rank's tokens: memory of its own where it is
    // small (after a barrier that says every rank has started), else the ring's (after one
    // that says the ring is free everywhere)
    static constexpr bool kOwnInbox = BT <= 32;
    static constexpr int kInboxBytes = BT * 128 * 4;
    static constexpr int kStages = BT == 128 ? 3 : 4;             // two blocks a multiprocessor
    static constexpr int kInboxOffset = kOwnInbox ? kStages * kStageBytes : 0;
    static constexpr int kBarOffset = kStages * kStageBytes + (kOwnInbox ? kInboxBytes : 0);
    static constexpr int kSmemBytes = kBarOffset + 256 + 1024;
    static constexpr int kScaleCol = BT;                          // two buffers of 8 + 8 columns after the accumulator
    static constexpr int kTmemCols = BT <= 32 ? 64 : BT == 64 ? 128 : 256;
    static_assert(kStageBytes % 1024 == 0, "operand tiles are 1024-byte aligned");
    static_assert(kScaleCol + 32 <= kTmemCols, "tensor memory");
    static_assert(kInboxBytes <= kStages * kStageBytes, "the accumulators fit the ring");
};

__device__ __forceinline__ void st_shared_cluster_f32(uint32_t cluster_addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" :: "r"(cluster_addr), "f"(v) : "memory");
}

__device__ __forceinline__ void tmem_ld_32x32b_x16_wait(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                   "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(taddr) : "memory");
}

// 16 accumulator columns from c on (zeros without any stage).
__device__ __forceinline__ void few_load(uint32_t tmem, int quarter, int c, bool held, uint32_t (&v)[16]) {
    if (held) {
        tmem_ld_32x32b_x16_wait(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + c, v);
    } else {
        #pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = 0u;
    }
}

// Sends this rank's accumulators to the tokens' owners (token m: rank m % S), into
// their inboxes [rank][token of the owner][128].
template <int S, int BT>
__device__ __forceinline__ void few_send(uint32_t inbox, uint32_t tmem, int rank, int M, bool held) {
    const int quarter = (threadIdx.x >> 5) & 3, i = quarter * 32 + (threadIdx.x & 31);
    uint32_t at[S];
    #pragma unroll
    for (int r = 0; r < S; ++r) at[r] = mapa_shared(inbox + (rank * (BT / S) * 128 + i) * 4, r);
    #pragma unroll 1
    for (int c = 0; c < M; c += 16) {
        uint32_t v[16];
        few_load(tmem, quarter, c, held, v);
        #pragma unroll
        for (int e = 0; e < 16; ++e)                              // (columns beyond M too: the inbox holds all BT)
            st_shared_cluster_f32(at[e % S] + (c / S + e / S) * 512, __uint_as_float(v[e]));
    }
}

// Adds the ranks' accumulators of this rank's tokens. A warp a token, a lane four
// outputs.
template <typename T, int S, int BT>
__device__ __forceinline__ void few_reduce(const unsigned char* inbox, int rank, const BiasRef& bias, T* out, int n0, int M, int N) {
    const int t = static_cast<int>(threadIdx.x) - 64, n = n0 + (t & 31) * 4;
    float b[4];
    #pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = bias.ptr != nullptr && n + e < N ? bias.at(n + e) : 0.0f;
    #pragma unroll 2
    for (int j = t >> 5; j * S + rank < M; j += 4) {
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        #pragma unroll
        for (int r = 0; r < S; ++r) {
            const float4 v = *reinterpret_cast<const float4*>(inbox + (r * (BT / S) + j) * 512 + (t & 31) * 16);
            sum.x += v.x;
            sum.y += v.y;
            sum.z += v.z;
            sum.w += v.w;
        }
        const T o[4] = {mx4_from_f32<T>(sum.x + b[0]), mx4_from_f32<T>(sum.y + b[1]), mx4_from_f32<T>(sum.z + b[2]), mx4_from_f32<T>(sum.w + b[3])};
        T* dst = out + static_cast<size_t>(j * S + rank) * N + n;
        if (N % 4 == 0 && n < N) {
            memcpy(__builtin_assume_aligned(dst, 4 * sizeof(T)), o, 4 * sizeof(T));
        } else {
            #pragma unroll
            for (int e = 0; e < 4; ++e)
                if (n + e < N) dst[e] = o[e];
        }
    }
}

// 16 columns of x as loaded, and as floats.
template <typename T> struct Few16 { uint4 v[sizeof(T)]; };

template <typename T>
__device__ __forceinline__ Few16<T> load16(const T* src, bool held, bool vec) {
    Few16<T> w;
    #pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) w.v[i] = make_uint4(0u, 0u, 0u, 0u);
    if (held && vec) {
        #pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) w.v[i] = __ldg(reinterpret_cast<const uint4*>(src) + i);
    } else if (held) {
        T e[16];
        #pragma unroll
        for (int i = 0; i < 16; ++i) e[i] = src[i];
        memcpy(&w, e, sizeof(w));
    }
    return w;
}

template <typename T>
__device__ __forceinline__ void to_floats(const Few16<T>& w, float (&f)[16]) {
    T e[16];
    memcpy(e, &w, sizeof(w));
    #pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = mx4_to_f32(e[i]);
}

// One radix-4 step over lanes whose bits `bit` and 2 * bit number the four values:
// (v0 + v1) + (v2 + v3) - 2 v_(3-i) in every lane.
__device__ __forceinline__ float2 h4_lanes(float2 v, int bit) {
    const float2 o = make_float2(__shfl_xor_sync(0xFFFFFFFFu, v.x, bit), __shfl_xor_sync(0xFFFFFFFFu, v.y, bit));
    const float2 p = fadd2_rn(v, o);
    const float2 q = make_float2(__shfl_xor_sync(0xFFFFFFFFu, p.x, 2 * bit), __shfl_xor_sync(0xFFFFFFFFu, p.y, 2 * bit));
    const float2 w = make_float2(__shfl_xor_sync(0xFFFFFFFFu, v.x, 3 * bit), __shfl_xor_sync(0xFFFFFFFFu, v.y, 3 * bit));
    return ffma2_rn(make_float2(-2.0f, -2.0f), w, fadd2_rn(p, q));
}

// Rotates and quantizes rows r and r + 1 (component x and y) of a stage; lane % 16
// has columns 16 (lane % 16) ... Writes codes (128-byte swizzle) and scale bytes.
template <int G>
__device__ __forceinline__ void few_quantize(float2 (&v)[16], int r, unsigned char* codes, unsigned char* scales) {
    const int a = threadIdx.x & 15;
    if constexpr (G >= 16) {
        #pragma unroll
        for (int i = 0; i < 16; i += 4) h4_pair(v[i], v[i + 1], v[i + 2], v[i + 3]);
        #pragma unroll
        for (int i = 0; i < 4; ++i) h4_pair(v[i], v[i + 4], v[i + 8], v[i + 12]);
    }
    if constexpr (G >= 64) {
        #pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = h4_lanes(v[i], 1);
    }
    if constexpr (G == 256) {
        #pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = h4_lanes(v[i], 4);
    }
    float mx = 0.0f, my = 0.0f;
    #pragma unroll
    for (int i = 0; i < 16; i += 2) {
        mx = max3_abs_nan(mx, v[i].x, v[i + 1].x);
        my = max3_abs_nan(my, v[i].y, v[i + 1].y);
    }
    // a block is two lanes
    mx = max3_abs_nan(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1), 0.0f) * unit_factor<G>();
    my = max3_abs_nan(my, __shfl_xor_sync(0xFFFFFFFFu, my, 1), 0.0f) * unit_factor<G>();
    const uint32_t ex = mx4_scale_byte(mx), ey = mx4_scale_byte(my);
    const float2 inv = make_float2(mx4_inv_scale(ex) * unit_factor<G>(), mx4_inv_scale(ey) * unit_factor<G>());
    #pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = fmul2_rn(v[i], inv);
    #pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = r + h;
        uint2 w;
        if (h == 0) {
            w.x = mx4_encode8(v[0].x, v[1].x, v[2].x, v[3].x, v[4].x, v[5].x, v[6].x, v[7].x);
            w.y = mx4_encode8(v[8].x, v[9].x, v[10].x, v[11].x, v[12].x, v[13].x, v[14].x, v[15].x);
        } else {
            w.x = mx4_encode8(v[0].y, v[1].y, v[2].y, v[3].y, v[4].y, v[5].y, v[6].y, v[7].y);
            w.y = mx4_encode8(v[8].y, v[9].y, v[10].y, v[11].y, v[12].y, v[13].y, v[14].y, v[15].y);
        }
        *reinterpret_cast<uint2*>(codes + row * 128 + (((a >> 1) ^ (row & 7)) << 4) + (a & 1) * 8) = w;
        if (!(a & 1)) scales[(a >> 3) * kMx4TileBytes + row * 16 + ((a >> 1) & 3)] = static_cast<uint8_t>(h ? ey : ex);
    }
}

template <typename T, int G, int BT, bool FUSED>
__global__ void __launch_bounds__(kMx4FewThreads, 2)
mx4_gemm_few_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_ws,
                    const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_xs,
                    const T* __restrict__ x, long long ldx, bool vec, BiasRef bias, T* __restrict__ out, int M, int N, int K) {
    using Cfg = Mx4FewCfg<BT, FUSED>;
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
    // this block's weights into L2 (a hint: safe whatever the previous kernel wrote), so
    // that what the ring does not hold yet is nearer when the first tokens are ready
    if (warp == 2)
        for (int it = lane; it < kts; it += 32) tma_prefetch_l2_2d(&tmap_w, (kt0 + it) * (kMx4StageK / 2), n0);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // (waited for ahead of the first store to another rank: its block has to have started,
    // and a rank without any stage would be there at once)
    if (Cfg::kOwnInbox && splits > 1) cluster_arrive_started();
    griddep_wait();
    griddep_launch_dependents();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        // ---------------- TMA producer: the warp runs the loop, one elected lane issues
        Mx4Ring<Cfg::kStages> ring;
        for (int it = 0; it < kts; ++it, ring.next()) {
            const int s = ring.slot;
            if (!mx4_wait_warp(&empty_bar[s], ring.phase ^ 1, mbar_test_wait(&empty_bar[s], ring.phase ^ 1))) {
                if (lane == 0) mx4_record_status(kMx4TimeoutProducer);
                break;
            }
            unsigned char* st = smem + s * Cfg::kStageBytes;
            unsigned char* sf = st + Cfg::kABytes + Cfg::kBBytes;
            const int kt = kt0 + it;
            if (elect_one()) {
                mbar_arrive_expect_tx(&full_bar[s], Cfg::kABytes + Cfg::kScaleBytes + (FUSED ? 0 : Cfg::kBBytes + Cfg::kScaleBytes));
                tma_load_2d(st, &tmap_w, &full_bar[s], kt * (kMx4StageK / 2), n0);
                tma_load_2d(sf, &tmap_ws, &full_bar[s], kt * 256, n0 / 128);
                if constexpr (!FUSED) {
                    tma_load_2d(st + Cfg::kABytes, &tmap_x, &full_bar[s], kt * (kMx4StageK / 2), 0);
                    tma_load_2d(sf + Cfg::kScaleBytes, &tmap_xs, &full_bar[s], kt * 256, 0);
                }
            }
            __syncwarp();
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer: the warp runs the loop, one elected lane issues
        const uint32_t base = smem_u32(smem);
        const uint64_t da0 = smem_desc_kmajor(base, 1024, 2), db0 = smem_desc_kmajor(base + Cfg::kABytes, 1024, 2);
        const uint64_t dsa0 = smem_desc_kmajor(base + Cfg::kABytes + Cfg::kBBytes, 128, 0);
        const uint64_t dsb0 = smem_desc_kmajor(base + Cfg::kABytes + Cfg::kBBytes + Cfg::kScaleBytes, 128, 0);
        const int odd_tail = (K + 127) / 128 & 1;                 // the last stage of K has one 128-value half
        Mx4Ring<Cfg::kStages> ring;
        bool ok = true;
        for (int it = 0; it < kts && ok; ++it, ring.next()) {
            const int s = ring.slot;
            ok = mx4_wait_warp(&full_bar[s], ring.phase, mbar_test_wait(&full_bar[s], ring.phase));
            if (FUSED && ok) ok = mx4_wait_warp(&ready_bar[s], ring.phase, mbar_test_wait(&ready_bar[s], ring.phase));
            if (!ok) {
                if (lane == 0) mx4_record_status(kMx4TimeoutMma);
                break;
            }
            tc_fence_after();
            const uint64_t at = static_cast<uint64_t>(s * (Cfg::kStageBytes / 16));
            const uint32_t col = tmem + Cfg::kScaleCol + (it & 1) * 16;
            const bool both = !(odd_tail && kt0 + it == num_kt - 1);
            if (elect_one()) {
                const uint64_t da = da0 + at, db = db0 + at, dsa = dsa0 + at, dsb = dsb0 + at;
                auto half = [&](int h) {
                    tmem_cp_scales<false>(col + 4 * h, dsa + 32 * h);
                    tmem_cp_scales<false>(col + 8 + 4 * h, dsb + 32 * h);
                };
                auto product = [&](int j) {
                    mma_mxf4<false>(tmem, da + 2 * j, db + 2 * j, idesc_mxf4(128, BT, (j & 1) * 2), col + 4 * (j >> 1),
                                    col + 8 + 4 * (j >> 1), (it | j) != 0);
                };
                half(0);
                if (both) half(1);
                product(0);
                product(1);
                if (both) {
                    product(2);
                    product(3);
                }
                mma_commit(&empty_bar[s]);
            }
            __syncwarp();
        }
        if (ok && kts > 0 && elect_one()) mma_commit(acc_bar);
        __syncwarp();
    } else {
        if constexpr (FUSED) {
            // ---------------- quantizers: stages in turn, four rows a pass; the next pass's
            // columns are on their way meanwhile
            const int r0 = 2 * (lane >> 4), col = (lane & 15) * 16;
            Few16<T> nx, ny;
            auto fetch = [&](int it, int p) {
                const int r = p + r0, k = (kt0 + it) * kMx4StageK + col;
                nx = load16(x + r * ldx + k, it < kts && r < M && k < K, vec);
                ny = load16(x + (r + 1) * ldx + k, it < kts && r + 1 < M && k < K, vec);
            };
            fetch(warp - 2, 0);
            for (int it = warp - 2; it < kts; it += 4) {
                const int s = it % Cfg::kStages;
                unsigned char* b = smem + s * Cfg::kStageBytes + Cfg::kABytes;
                bool ok = true;
                #pragma unroll 1
                for (int p = 0; p < M; p += 4) {
                    float fx[16], fy[16];
                    to_floats(nx, fx);
                    to_floats(ny, fy);
                    if (p + 4 < M) fetch(it, p + 4);
                    else fetch(it + 4, 0);
                    float2 v[16];
                    #pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = make_float2(fx[i], fy[i]);
                    // (the slot is free once the MMAs of its last stage are done)
                    if (p == 0) ok = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(&empty_bar[s], ((it / Cfg::kStages) & 1) ^ 1));
                    if (!ok) break;
                    few_quantize<G>(v, p + r0, b, b + Cfg::kBBytes + Cfg::kScaleBytes);
                }
                if (!ok) {
                    if (lane == 0) mx4_record_status(kMx4TimeoutProducer);
                    break;
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ready_bar[s]);
            }
        }
        // ---------------- accumulators: lane n0 + 32 q + lane, a column a token
        const bool ok = kts == 0 || __all_sync(0xFFFFFFFFu, mbar_wait_bounded(acc_bar, 0));
        if (!ok && lane == 0) mx4_record_status(kMx4TimeoutEpilogue);
        tc_fence_after();
        if (splits == 1) {
            const int quarter = warp & 3, n = n0 + quarter * 32 + lane;
            const float b = bias.ptr != nullptr && n < N ? bias.at(n) : 0.0f;
            #pragma unroll 1
            for (int c = 0; c < M; c += 16) {
                uint32_t v[16];
                few_load(tmem, quarter, c, kts > 0, v);
                T* dst = out + static_cast<size_t>(c) * N + n;
                #pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (c + e < M && n < N) dst[static_cast<size_t>(e) * N] = mx4_from_f32<T>(__uint_as_float(v[e]) + b);
            }
        }
    }
    if (splits > 1) {
        unsigned char* inbox = smem + Cfg::kInboxOffset;
        if constexpr (Cfg::kOwnInbox) cluster_wait_started();
        else cluster_sync();                                      // every rank's ring is free
        if (warp >= 2) {
            const uint32_t to = smem_u32(inbox);
            if (splits == 2) few_send<2, BT>(to, tmem, rank, M, kts > 0);
            else if (splits == 4) few_send<4, BT>(to, tmem, rank, M, kts > 0);
            else few_send<8, BT>(to, tmem, rank, M, kts > 0);
        }
        cluster_sync();                                           // all inboxes are filled
        if (warp >= 2) {
            if (splits == 2) few_reduce<T, 2, BT>(inbox, rank, bias, out, n0, M, N);
            else if (splits == 4) few_reduce<T, 4, BT>(inbox, rank, bias, out, n0, M, N);
            else few_reduce<T, 8, BT>(inbox, rank, bias, out, n0, M, N);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, Cfg::kTmemCols);
    }
}

}  // namespace convrot
