// The int8 quantizer behind a root-mean-square norm: h = x + r, y = R(h g / rms(h)),
// s = max |y| / 127, codes = y / s to nearest, ties to even. R is the ConvRot rotation,
// which is linear, so 1 / rms goes to the scale alone: the codes are those of
// R(h g), and a row needs one pass and one exchange (sum of squares and largest
// magnitude together). All in fp32, without an intermediate rounding. Rows that leave its range on the
// way (squares from 1.8 10^19, h g beyond 3.4 10^38, squares that vanish) are left to a second loop
// of the block, which takes them times powers of two.
//
// A thread has 16 neighbouring columns, a warp 512 (two groups of 256). The steps of the
// rotation at strides 1 and 4 stay in the thread; for those at 16 and 64 the 16 x 16 values
// of a group are transposed through shared memory, codes go back the same way. A block
// goes through rows, keeps its columns' g in registers and loads the next row's
// values under the current one's work.
//
// 16384 x 3840 in bf16, caches cold: 72 us, 2.6 TB/s (a copy of the rows 41); the fp32 pipe, shared memory and issue
// are each busy half to two thirds of the time, and a row's exchange and divisions leave 24 warps a
// multiprocessor waiting in turns. With a residual 86 us (5.1 TB/s); 8192 x 8192 with one 108 (4.3), 4096 x 15360 113 (3.9; fp32
// 246, 3.3). Above 4096 columns a row's warps are a block of 64 registers a thread: 52 to 64 bytes spill (fp32 304; below,
// fp32 24 to 52). The second loop inside the first, instead of behind it, took 80 us; single operations instead of pairs, and codes
// by conversions, 78 against 64 without that loop; four blocks a multiprocessor (64 registers) 73. The product behind it is the
// int8 GEMM of the other linears.
#pragma once

namespace convrot {

constexpr int kRmsMostK = 16384;              // 32 warps a row
constexpr float kRmsLeast = 0x1p-100f;        // a mean of squares below it has lost some of them
constexpr int kRmsWarpFloats = 512 + 16;      // a warp's values; the second group 16 floats on: other banks

struct RmsQuantArgs {
    const void *x, *r, *g;                    // r null: no residual; g null: ones
    long long ldx, ldr;
    void* h;                                  // [M, K] where there is a residual
    int8_t* codes;                            // [M, K]
    float* scales;                            // [M]
    int M, K, g_type;
    int row_warps, rows;                      // warps of a row, rows of a block at a time
    int vec_x, vec_r, vec_g;                  // 16-byte aligned rows
    float eps;
};

// 16 values of a row from memory as they are.
template <typename T>
struct RmsRaw {
    static constexpr int kChunks = sizeof(T);                     // of 16 bytes: 16 values are as many as a value's bytes
    uint4 v[kChunks];
    __device__ __forceinline__ void load(const T* p, bool held, bool vec) {
        #pragma unroll
        for (int c = 0; c < kChunks; ++c) v[c] = make_uint4(0, 0, 0, 0);
        if (!held) return;
        if (vec) {
            #pragma unroll
            for (int c = 0; c < kChunks; ++c) v[c] = __ldg(reinterpret_cast<const uint4*>(p) + c);
        } else {
            T e[16];
            #pragma unroll
            for (int i = 0; i < 16; ++i) e[i] = p[i];
            memcpy(v, e, sizeof(e));
        }
    }
    __device__ __forceinline__ void get(float2 (&f)[8]) const {
        T e[16];
        memcpy(e, v, sizeof(e));
        #pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = make_float2(mx4_to_f32(e[2 * i]), mx4_to_f32(e[2 * i + 1]));
    }
    __device__ __forceinline__ void put(const float2 (&f)[8]) {
        T e[16];
        #pragma unroll
        for (int i = 0; i < 8; ++i) {
            e[2 * i] = mx4_from_f32<T>(f[i].x);
            e[2 * i + 1] = mx4_from_f32<T>(f[i].y);
        }
        memcpy(v, e, sizeof(e));
    }
};

// Steps at strides 1 and 4 of 16 values in pairs (two fp32 operations an instruction). Value e is then
// in place e ^ 3: a step at stride 1 gives its sums in reverse where it need not swap halves.
__device__ __forceinline__ void rms_rotate16(float2 (&v)[8], bool second) {
    const float2 less = make_float2(-2.0f, -2.0f);
    #pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float2 t = fadd2_rn(v[i], v[i + 1]);
        const float2 sum = make_float2(t.x + t.y, t.x + t.y);
        v[i] = ffma2_rn(less, v[i], sum);
        v[i + 1] = ffma2_rn(less, v[i + 1], sum);
    }
    if (second) {
        #pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 sum = fadd2_rn(fadd2_rn(v[i], v[i + 2]), fadd2_rn(v[i + 4], v[i + 6]));
            const float2 w0 = ffma2_rn(less, v[i + 6], sum), w1 = ffma2_rn(less, v[i + 4], sum), w2 = ffma2_rn(less, v[i + 2], sum);
            v[i + 6] = ffma2_rn(less, v[i], sum);
            v[i] = w0;
            v[i + 2] = w1;
            v[i + 4] = w2;
        }
    }
}

// The sum of `ss` and the largest `amax` (NaN above all; neither is negative) over the lanes
// that differ in the bits below WIDTH, and of `amax` over the warp.
template <int WIDTH>
__device__ __forceinline__ void rms_reduce(float& ss, float& amax) {
    amax = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(amax)));
    #pragma unroll
    for (int z = WIDTH / 2; z; z >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, z);
}

// THREADS: 256 (rows up to 4096 columns) or 1024.
template <typename T, int G, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 3 : 1) rms_quant_int8_kernel(const __grid_constant__ RmsQuantArgs a) {
    extern __shared__ __align__(128) unsigned char rms_smem[];
    __shared__ float2 part[2][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* mine = reinterpret_cast<float*>(rms_smem) + warp * kRmsWarpFloats;
    const int in_row = warp % a.row_warps, col = in_row * 512 + lane * 16;
    const bool column = col < a.K;
    const int group = lane >> 4, j = lane & 15;
    griddep_wait();
    griddep_launch_dependents();
    int row = static_cast<int>(blockIdx.x) * a.rows + warp / a.row_warps;
    RmsRaw<T> x, r;
    auto load = [&](int at) {
        const bool held = column && at < a.M;
        x.load(static_cast<const T*>(a.x) + (held ? at * a.ldx + col : 0), held, a.vec_x);
        if (a.r) r.load(static_cast<const T*>(a.r) + (held ? at * a.ldr + col : 0), held, a.vec_r);
    };
    load(row);
    float2 g[8];
    #pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = make_float2(1.0f, 1.0f);
    if (a.g) {
        auto gains = [&](auto* p) {
            RmsRaw<std::remove_const_t<std::remove_pointer_t<decltype(p)>>> raw;
            raw.load(p + (column ? col : 0), column, a.vec_g);
            raw.get(g);
        };
        if (a.g_type == 0) gains(static_cast<const float*>(a.g));
        else if (a.g_type == 1) gains(static_cast<const __nv_bfloat16*>(a.g));
        else gains(static_cast<const __half*>(a.g));
    }
    const float per_k = 1.0f / static_cast<float>(a.K);
    // The row's codes and scale from its h times a power of two up_h, and v, h g times up_v; the sum of squares and the
    // largest magnitude meet in p. In the first loop (both powers 1) a row that left fp32's range gets instead
    // of a scale -(1 + 3 i + j), with which powers it has to be taken; whether it did is returned.
    auto quantize = [&](auto first, float2 (&v)[8], float ss, int now, bool kept, float2* p, float up_h, float up_v) -> bool {
        constexpr bool kFirst = decltype(first)::value;
        float amax = 0.0f;
        rms_rotate16(v, true);
        if constexpr (G >= 64) {
            // value 16 l + i of a group (of its thread l) lies in row l, its chunks of four XORed: neither
            // side meets a bank conflict
            float* base = mine + group * (256 + 16);
            #pragma unroll
            for (int c = 0; c < 4; ++c)
                *reinterpret_cast<float4*>(base + j * 16 + ((c ^ (j >> 1 & 3)) << 2)) = make_float4(v[2 * c].x, v[2 * c].y, v[2 * c + 1].x, v[2 * c + 1].y);
            __syncwarp();
            const float* from = base + (j & 3 ^ 3);
            #pragma unroll
            for (int i = 0; i < 8; ++i)
                v[i] = make_float2(from[2 * i * 16 + (((j >> 2) ^ (i & 3)) << 2)], from[(2 * i + 1) * 16 + (((j >> 2) ^ (i & 3)) << 2)]);
            rms_rotate16(v, G == 256);
        }
        #pragma unroll
        for (int i = 0; i < 8; ++i) amax = max3_abs_nan(amax, v[i].x, v[i].y);
        rms_reduce<32>(ss, amax);
        if (a.row_warps > 1) {
            constexpr int kMost = THREADS / 32;                   // warps of a row
            if (lane == 0) p[warp] = make_float2(ss, amax);
            __syncthreads();
            const float2 y = lane % kMost < a.row_warps ? p[warp - in_row + lane % kMost] : make_float2(0.0f, 0.0f);
            ss = y.x;
            amax = y.y;
            rms_reduce<kMost>(ss, amax);
        }
        const float mean = fmaf(ss, per_k, kFirst ? a.eps : a.eps * up_h * up_h);
        float rstd = 1.0f / sqrtf(mean);
        if (!kFirst) rstd *= up_h / up_v;                          // (for h g as it is scaled)
        const float y = amax * unit_factor<G>() * rstd;
        float s = (y < 1e-10f ? 1e-10f : y) / 127.0f;             // (NaN stays)
        // |v f| is 127 and roundings at most: a sum with 1.5 * 2^23 has the code in its last byte. (f finite: 0 stays 0)
        const float f = fminf(unit_factor<G>() * rstd / s, 3.4e38f);
        const float2 by = make_float2(f, f), shift = make_float2(12582912.0f, 12582912.0f);
        #pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = ffma2_rn(v[i], by, shift);
        const bool odd = kFirst && !(mean >= kRmsLeast && mean < INFINITY && amax < INFINITY);
        if (odd) {
            // What 2^-100 takes below the range is less than 2^-60 of the row's largest; 2^100 is for rows below 2^-43.
            const bool small = mean < kRmsLeast, large = !(mean < INFINITY), wide = !(amax < INFINITY);
            s = -1.0f - (small ? 3.0f : large ? 6.0f : 0.0f) - (wide || (large && amax >= 1.0f) ? 2.0f : small && amax < 0x1p-60f ? 1.0f : 0.0f);
        }
        uint32_t out[4];
        if constexpr (G >= 64) {
            __syncwarp();
            unsigned char* bytes = reinterpret_cast<unsigned char*>(mine) + group * (256 + 16);
            #pragma unroll
            for (int i = 0; i < 8; ++i) {                         // (places 2i and 2i + 1: values 2i ^ 3 and 2i ^ 2)
                bytes[(2 * i ^ 3) * 16 + j] = static_cast<unsigned char>(__float_as_uint(v[i].x));
                bytes[(2 * i ^ 2) * 16 + j] = static_cast<unsigned char>(__float_as_uint(v[i].y));
            }
            __syncwarp();
            const uint4 o = *reinterpret_cast<const uint4*>(bytes + j * 16);
            out[0] = o.x; out[1] = o.y; out[2] = o.z; out[3] = o.w;
            __syncwarp();
        } else {
            #pragma unroll
            for (int c = 0; c < 4; ++c) {
                const uint32_t hi = __byte_perm(__float_as_uint(v[2 * c].x), __float_as_uint(v[2 * c].y), 0x0004);      // values 2, 3
                const uint32_t lo = __byte_perm(__float_as_uint(v[2 * c + 1].x), __float_as_uint(v[2 * c + 1].y), 0x0004);
                out[c] = __byte_perm(lo, hi, 0x5410);
            }
        }
        if (kept) {
            if (column) *reinterpret_cast<uint4*>(a.codes + static_cast<size_t>(now) * a.K + col) = make_uint4(out[0], out[1], out[2], out[3]);
            if (in_row == 0 && lane == 0) a.scales[now] = s;
        }
        return odd && kept;
    };
    auto sum_of = [&](float2 (&v)[8]) {                           // x + r
        x.get(v);
        if (!a.r) return;
        float2 w[8];
        r.get(w);
        #pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fadd2_rn(v[i], w[i]);
    };
    // (every warp of the block makes as many rounds: they meet at barriers)
    const int stride = static_cast<int>(gridDim.x) * a.rows;
    bool odd = false;
    for (int row0 = static_cast<int>(blockIdx.x) * a.rows, round = 0; row0 < a.M; row0 += stride, ++round) {
        float2 v[8];
        sum_of(v);
        if (a.r && column && row < a.M) {
            RmsRaw<T> o;
            o.put(v);
            uint4* h = reinterpret_cast<uint4*>(static_cast<T*>(a.h) + static_cast<size_t>(row) * a.K + col);
            #pragma unroll
            for (int c = 0; c < RmsRaw<T>::kChunks; ++c) h[c] = o.v[c];
        }
        const int now = row;
        row += stride;
        load(row);
        float2 squares = make_float2(0.0f, 0.0f);
        #pragma unroll
        for (int i = 0; i < 8; ++i) {
            squares = ffma2_rn(v[i], v[i], squares);
            v[i] = fmul2_rn(v[i], g[i]);
        }
        odd |= quantize(std::true_type{}, v, squares.x + squares.y, now, now < a.M, part[round & 1], 1.0f, 1.0f);
    }
    if (!__syncthreads_or(odd)) return;
    row = static_cast<int>(blockIdx.x) * a.rows + warp / a.row_warps;
    #pragma unroll 1
    for (int row0 = static_cast<int>(blockIdx.x) * a.rows; row0 < a.M; row0 += stride, row += stride) {
        const float mark = row < a.M ? __ldcg(a.scales + row) : 0.0f;
        if (!__syncthreads_or(mark < 0.0f)) continue;             // (a round's exchange is over, too, before the next)
        const int code = mark < 0.0f ? static_cast<int>(-mark) - 1 : 0;
        const float up_h = code >= 6 ? 0x1p-100f : code >= 3 ? 0x1p100f : 1.0f, up_v = code % 3 == 2 ? 0x1p-100f : code % 3 == 1 ? 0x1p100f : 1.0f;
        load(row);
        float2 v[8];
        sum_of(v);
        float2 squares = make_float2(0.0f, 0.0f);
        #pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 h = fmul2_rn(v[i], make_float2(up_h, up_h));
            squares = ffma2_rn(h, h, squares);
            v[i] = fmul2_rn(fmul2_rn(v[i], make_float2(up_v, up_v)), g[i]);
        }
        quantize(std::false_type{}, v, squares.x + squares.y, row, mark < 0.0f, part[0], up_h, up_v);
    }
}

// ---------------------------------------------------------------- few rows times the int8 weight

// out[m, n] = ((float(D) xs[m]) ws[n]) + bias[n], D the exact product, for up to 8 NT rows (NT 1 or 2): bound by the
// weight's bytes. A block takes 16 outputs, its warps a share of K each; products run on
// mma.m16n8k32 with the weight on the side of 16 (tcgen05 wants 128 rows of it a tile,
// and the tiles of a weight of some thousand rows do not fill the multiprocessors). The order of
// the contraction is free, so a thread's operands are 16 bytes of a row as they lie. The weight
// is not written by the kernel before (this library's quantizer), so its first loads
// start under that kernel. A thread has 32 neighbouring bytes of each of two rows, so that four threads
// ask for a whole line: 1 x 15360 x 3840 takes 14.8 us with the quantizer, against 16.2 in
// pieces of 16 bytes (9.0 by the weight's bytes; a start of two kernels is some 4).
// (16 rows here and 17 in tiles of 256 rows, us with the quantizer: 15360 x 3840 14.3 and 19.8, 4096 x 4096 8.1 and 12.8,
// 3840 x 15360 17.0 and 27.5. 32 rows of 15360 x 3840 took 33 here, and 20 in tiles.)
constexpr int kFewI8Rows = 16;

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int NT, typename T>
__global__ void __launch_bounds__(512)
few_i8_kernel(const int8_t* x, const int8_t* __restrict__ w, const float* xs, const float* __restrict__ ws, BiasRef bias, T* out, int M, int N, int K) {
    constexpr int kAhead = 2;                                     // segments of 128 columns on their way
    extern __shared__ int few_sums[];                             // [warp][row][17]
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = static_cast<int>(blockIdx.x) * 16;
    const int segs = (K + 127) / 128, per = (segs + warps - 1) / warps;
    const int s0 = min(segs, warp * per), s1 = min(segs, s0 + per);
    // (a thread's 32 bytes of a segment, so that four threads ask for a whole line of a row)
    const int8_t* row0 = w + static_cast<size_t>(min(n0 + g, N - 1)) * K + 32 * t;
    const int8_t* row1 = w + static_cast<size_t>(min(n0 + g + 8, N - 1)) * K + 32 * t;
    uint4 a[kAhead][2][2];
    const uint4 zero = make_uint4(0, 0, 0, 0);
    auto load_w = [&](int s, uint4 (&to)[2][2]) {
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = 128 * s + 16 * h;
            const bool held = s < s1 && at + 32 * t < K;
            to[h][0] = held ? __ldg(reinterpret_cast<const uint4*>(row0 + at)) : zero;
            to[h][1] = held ? __ldg(reinterpret_cast<const uint4*>(row1 + at)) : zero;
        }
    };
    #pragma unroll
    for (int i = 0; i < kAhead; ++i) load_w(s0 + i, a[i]);
    griddep_wait();
    griddep_launch_dependents();
    int d[NT][4] = {};
    const int8_t* xr[NT];
    #pragma unroll
    for (int k = 0; k < NT; ++k) xr[k] = x + static_cast<size_t>(min(8 * k + g, M - 1)) * K + 32 * t;
    #pragma unroll 1
    for (int s = s0; s < s1; s += kAhead) {
        #pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (s + i < s1) {
                #pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint4 lo = a[i][h][0], hi = a[i][h][1];
                    const int at = 128 * (s + i) + 16 * h;
                    #pragma unroll
                    for (int k = 0; k < NT; ++k) {
                        // (the rows' codes come from the kernel before, which may still write: no read-only loads)
                        const uint4 b = at + 32 * t < K ? *reinterpret_cast<const uint4*>(xr[k] + at) : zero;
                        mma_s8(d[k], lo.x, hi.x, lo.y, hi.y, b.x, b.y);
                        mma_s8(d[k], lo.z, hi.z, lo.w, hi.w, b.z, b.w);
                    }
                }
                load_w(s + i + kAhead, a[i]);
            }
        }
    }
    #pragma unroll
    for (int k = 0; k < NT; ++k) {
        int* to = few_sums + (warp * 8 * NT + 8 * k + 2 * t) * 17 + g;
        to[0] = d[k][0];
        to[17] = d[k][1];
        to[8] = d[k][2];
        to[25] = d[k][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * 8 * NT; i += blockDim.x) {
        const int m = i >> 4, n = n0 + (i & 15);
        if (m >= M || n >= N) continue;
        int sum = 0;
        for (int k = 0; k < warps; ++k) sum += few_sums[(k * 8 * NT + m) * 17 + (i & 15)];
        float y = __fmul_rn(__fmul_rn(static_cast<float>(sum), xs[m]), ws[n]);
        if (bias.ptr) y = __fadd_rn(y, bias.at(n));
        out[static_cast<size_t>(m) * N + n] = mx4_from_f32<T>(y);
    }
}

}  // namespace convrot
