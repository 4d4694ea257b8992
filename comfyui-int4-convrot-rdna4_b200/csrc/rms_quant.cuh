// The int8 quantizer behind a root-mean-square norm: h = x + r, y = R(h g / rms(h)),
// s = max |y| / 127, codes = y / s to nearest, ties to even. R is the ConvRot rotation,
// which is linear, so 1 / rms goes to the scale alone: the codes are those of
// R(h g), and a row needs one pass and one exchange (sum of squares and largest
// magnitude together). All in fp32, without an intermediate rounding.
//
// A thread has 128 columns (a unit, mx4_unit.cuh), a row one to four warps; a block
// goes through rows of the matrix and keeps g in shared memory.
#pragma once

namespace convrot {

constexpr int kRmsMostK = 16384;              // four warps a row, with g and two slabs of it in shared memory

struct RmsQuantArgs {
    const void *x, *r, *g;                    // r null: no residual; g null: ones
    long long ldx, ldr;
    void* h;                                  // [M, K] where there is a residual
    int8_t* codes;                            // [M, K]
    float* scales;                            // [M]
    int M, K, g_type;
    int row_warps, rows;                      // warps of a row, rows of a block at a time
    int vec_x, vec_r;                         // 16-byte aligned rows
    float eps;
};

template <typename T>
__host__ __device__ constexpr int rms_quant_smem(int warps, int row_warps) {
    return warps * 2 * Mx4Slab<T>::kBytes + row_warps * Mx4Slab<float>::kBytes;
}

template <typename T, int G>
__global__ void __launch_bounds__(128, 3) rms_quant_int8_kernel(RmsQuantArgs a) {
    using S = Mx4Slab<T>;
    extern __shared__ __align__(128) unsigned char mx4slabs[];
    __shared__ float2 part[4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    unsigned char* slab = mx4slabs + warp * 2 * S::kBytes;
    unsigned char* gains = mx4slabs + warps * 2 * S::kBytes;
    const int in_row = warp % a.row_warps, col = (in_row * 32 + lane) * kMx4Unit;       // this thread's first column
    auto start = [&](int row) {
        const bool held = row < a.M && col < a.K;
        const int chunks = held ? min(S::kChunks, (a.K - col) / S::kPer) : 0;
        const T* x = static_cast<const T*>(a.x);
        slab_load<false>(slab, Mx4UnitAt<T>{reinterpret_cast<const unsigned char*>(held ? x + row * a.ldx + col : x), chunks}, 0, a.vec_x);
        if (a.r) {
            const T* r = static_cast<const T*>(a.r);
            slab_load<false>(slab + S::kBytes, Mx4UnitAt<T>{reinterpret_cast<const unsigned char*>(held ? r + row * a.ldr + col : r), chunks}, 0, a.vec_r);
        }
    };
    griddep_wait();
    griddep_launch_dependents();
    const int first = static_cast<int>(blockIdx.x) * a.rows + warp / a.row_warps;
    start(first);
    cp_async_commit();
    for (int i = threadIdx.x; i < a.row_warps * 4096; i += blockDim.x) {
        float g = 0.0f;
        if (i < a.K)
            g = !a.g ? 1.0f : a.g_type == 0 ? static_cast<const float*>(a.g)[i] : a.g_type == 1 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.g)[i])
                                                                                             : __half2float(static_cast<const __half*>(a.g)[i]);
        *reinterpret_cast<float*>(gains + i / 4096 * Mx4Slab<float>::kBytes + Mx4Slab<float>::offset(i % 4096 / kMx4Unit, i % kMx4Unit / 4) + i % 4 * 4) = g;
    }
    __syncthreads();
    for (int row0 = static_cast<int>(blockIdx.x) * a.rows; row0 < a.M; row0 += static_cast<int>(gridDim.x) * a.rows) {
        const int row = row0 + warp / a.row_warps;
        const bool held = row < a.M && col < a.K;
        cp_async_wait<0>();
        __syncwarp();
        float2 v[64];
        slab_to_unit<T>(slab, v);
        if (a.r) {
            float2 w[64];
            slab_to_unit<T>(slab + S::kBytes, w);
            #pragma unroll
            for (int i = 0; i < 64; ++i) v[i] = fadd2_rn(v[i], w[i]);
            __syncwarp();
            unit_to_slab<T>(slab, lane, v, 1.0f);
            __syncwarp();
            T* h = static_cast<T*>(a.h);
            slab_store<T>(slab, Mx4UnitAt<T>{reinterpret_cast<const unsigned char*>(held ? h + static_cast<size_t>(row) * a.K + col : h),
                                             held ? min(S::kChunks, (a.K - col) / S::kPer) : 0});
        }
        __syncwarp();
        float2 sum[4] = {};
        #pragma unroll
        for (int i = 0; i < 64; ++i) sum[i & 3] = ffma2_rn(v[i], v[i], sum[i & 3]);
        float ss = ((sum[0].x + sum[1].x) + (sum[2].x + sum[3].x)) + ((sum[0].y + sum[1].y) + (sum[2].y + sum[3].y));
        {
            const unsigned char* gs = gains + in_row * Mx4Slab<float>::kBytes;
            #pragma unroll
            for (int c = 0; c < 16; ++c) {
                const float4 lo = *reinterpret_cast<const float4*>(gs + Mx4Slab<float>::offset(lane, c));
                const float4 hi = *reinterpret_cast<const float4*>(gs + Mx4Slab<float>::offset(lane, c + 16));
                v[4 * c] = fmul2_rn(v[4 * c], make_float2(lo.x, hi.x));
                v[4 * c + 1] = fmul2_rn(v[4 * c + 1], make_float2(lo.y, hi.y));
                v[4 * c + 2] = fmul2_rn(v[4 * c + 2], make_float2(lo.z, hi.z));
                v[4 * c + 3] = fmul2_rn(v[4 * c + 3], make_float2(lo.w, hi.w));
            }
        }
        unit_rotate<G>(v);
        float top[4] = {};
        #pragma unroll
        for (int i = 0; i < 64; ++i) top[i & 3] = max3_abs_nan(top[i & 3], v[i].x, v[i].y);
        float amax = max3_abs_nan(max3_abs_nan(top[0], top[1], top[2]), top[3], 0.0f);
        #pragma unroll
        for (int z = 16; z; z >>= 1) {
            ss += __shfl_xor_sync(0xFFFFFFFFu, ss, z);
            amax = max3_abs_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, z), 0.0f);
        }
        if (a.row_warps > 1) {                                    // (every warp of the block passes the same barriers)
            if (lane == 0) part[warp] = make_float2(ss, amax);
            __syncthreads();
            ss = amax = 0.0f;
            for (int w = warp - in_row; w < warp - in_row + a.row_warps; ++w) {
                ss += part[w].x;
                amax = max3_abs_nan(amax, part[w].y, 0.0f);
            }
            __syncthreads();
        }
        const float rstd = 1.0f / sqrtf(ss / static_cast<float>(a.K) + a.eps);
        const float y = amax * unit_factor<G>() * rstd;
        const float s = (y < 1e-10f ? 1e-10f : y) / 127.0f;       // (NaN stays)
        const float f = unit_factor<G>() * rstd / s;
        const int mine = lane ^ (G == 256 ? 1 : 0);               // whose columns this lane has after the rotation
        #pragma unroll
        for (int c = 0; c < 4; ++c) {                             // 16 columns of each half of the unit
            uint32_t wx[4], wy[4];
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
                wx[j] = wy[j] = 0;
                #pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 z = fmul2_rn(v[16 * c + 4 * j + e], make_float2(f, f));
                    const int ix = max(-127, min(127, __float2int_rn(z.x))), iy = max(-127, min(127, __float2int_rn(z.y)));
                    wx[j] |= static_cast<uint32_t>(ix & 255) << (8 * e);
                    wy[j] |= static_cast<uint32_t>(iy & 255) << (8 * e);
                }
            }
            *reinterpret_cast<uint4*>(slab + mine * 128 + ((c ^ (mine & 7)) << 4)) = make_uint4(wx[0], wx[1], wx[2], wx[3]);
            *reinterpret_cast<uint4*>(slab + mine * 128 + (((c + 4) ^ (mine & 7)) << 4)) = make_uint4(wy[0], wy[1], wy[2], wy[3]);
        }
        __syncwarp();
        if (row < a.M) {
            int8_t* to = a.codes + static_cast<size_t>(row) * a.K + in_row * 4096;
            #pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int unit = (i * 32 + lane) >> 3, c = lane & 7;
                if (in_row * 4096 + unit * 128 + c * 16 < a.K)
                    *reinterpret_cast<uint4*>(to + unit * 128 + c * 16) = *reinterpret_cast<const uint4*>(slab + unit * 128 + ((c ^ (unit & 7)) << 4));
            }
            if (in_row == 0 && lane == 0) a.scales[row] = s;
        }
        __syncwarp();
        start(row + static_cast<int>(gridDim.x) * a.rows);
        cp_async_commit();
    }
    cp_async_wait<0>();
}

}  // namespace convrot
