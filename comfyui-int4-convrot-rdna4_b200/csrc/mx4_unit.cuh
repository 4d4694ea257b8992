// The work unit of the MX4 quantizers and readers: 128 consecutive values of a
// row held by one thread, in registers from the load to the codes (or back).
//
// Value i of the unit (i < 64) is v[i].x and value 64 + i is v[i].y: the radix-4
// steps of the rotation at strides 1, 4 and 16 then act on whole pairs with the
// packed fp32 instructions, and the step at stride 64 (groups of 256: two units,
// neighbouring lanes) needs one exchanged sum a pair. A unit is four blocks of
// 32, so amplitudes, scales and codes need no other thread; its four scale bytes
// are one 32-bit word of a scale tile.
//
// 128 values a thread would make global accesses of a warp 256 bytes apart, so
// units pass through shared memory: a warp's 32 units come in by 16-byte
// asynchronous copies whose lanes run along the rows, and the chunk index is
// XORed with the unit's number so that neither side meets a bank conflict.
#pragma once

namespace convrot {

constexpr int kMx4Unit = 128;                 // values of a thread

__device__ __forceinline__ float2 ffma2_rn(float2 a, float2 b, float2 c) {
    uint64_t ua, ub, uc, r;
    memcpy(&ua, &a, 8);
    memcpy(&ub, &b, 8);
    memcpy(&uc, &c, 8);
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(ua), "l"(ub), "l"(uc));
    float2 o;
    memcpy(&o, &r, 8);
    return o;
}

// h4 (hadamard.cuh) on pairs: the same sums, component by component.
__device__ __forceinline__ void h4_pair(float2& v0, float2& v1, float2& v2, float2& v3) {
    const float2 s = fadd2_rn(fadd2_rn(v0, v1), fadd2_rn(v2, v3));
    const float2 m = make_float2(-2.0f, -2.0f);
    const float2 o0 = ffma2_rn(m, v3, s), o1 = ffma2_rn(m, v2, s), o2 = ffma2_rn(m, v1, s), o3 = ffma2_rn(m, v0, s);
    v0 = o0; v1 = o1; v2 = o2; v3 = o3;
}

// Rotates the unit in groups of G without the factor 1 / sqrt(G). With G = 256
// lanes 2j and 2j + 1 hold the two halves of a group, and each ends with the half
// that the other began with (out_i of the last step needs v_(3-i) only, which is
// in the lane of the other half).
template <int G>
__device__ __forceinline__ void unit_rotate(float2 (&v)[64]) {
    if constexpr (G >= 16) {
        #pragma unroll
        for (int i = 0; i < 64; i += 4) h4_pair(v[i], v[i + 1], v[i + 2], v[i + 3]);
        #pragma unroll
        for (int i = 0; i < 64; i += 16)
            #pragma unroll
            for (int j = 0; j < 4; ++j) h4_pair(v[i + j], v[i + j + 4], v[i + j + 8], v[i + j + 12]);
    }
    if constexpr (G >= 64) {
        #pragma unroll
        for (int j = 0; j < 16; ++j) h4_pair(v[j], v[j + 16], v[j + 32], v[j + 48]);
    }
    if constexpr (G == 256) {
        #pragma unroll
        for (int i = 0; i < 64; ++i) {
            const float p = __fadd_rn(v[i].x, v[i].y);
            const float s = __fadd_rn(p, __shfl_xor_sync(0xFFFFFFFFu, p, 1));
            v[i] = make_float2(__fmaf_rn(-2.0f, v[i].y, s), __fmaf_rn(-2.0f, v[i].x, s));
        }
    }
}

template <int G>
__host__ __device__ constexpr float unit_factor() { return G == 16 ? 0.25f : G == 64 ? 0.125f : G == 256 ? 0.0625f : 1.0f; }

__device__ __forceinline__ float max3_abs_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Eight values to one word of codes, value 0 in the low nibble.
__device__ __forceinline__ uint32_t mx4_encode8(float a0, float a1, float a2, float a3, float a4, float a5, float a6, float a7) {
    uint32_t r;
    asm("{\n\t.reg .b8 c0, c1, c2, c3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c3, %8, %7;\n\t"
        "mov.b32 %0, {c0, c1, c2, c3};\n\t}"
        : "=r"(r) : "f"(a0), "f"(a1), "f"(a2), "f"(a3), "f"(a4), "f"(a5), "f"(a6), "f"(a7));
    return r;
}

// Codes (16 bytes a block) and the word of scale bytes of a unit whose values are
// v * factor (a power of two). The factor goes into the amplitude and into the
// inverse scale, both exact.
__device__ __forceinline__ uint32_t unit_quantize(float2 (&v)[64], float factor, uint4 (&codes)[4]) {
    uint32_t word = 0;
    #pragma unroll
    for (int half = 0; half < 2; ++half) {                      // blocks half (x) and half + 2 (y)
        float ax[4] = {}, ay[4] = {};                            // four chains: a step waits for nothing
        #pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float2 a = v[32 * half + 2 * i], b = v[32 * half + 2 * i + 1];
            ax[i & 3] = max3_abs_nan(ax[i & 3], a.x, b.x);
            ay[i & 3] = max3_abs_nan(ay[i & 3], a.y, b.y);
        }
        const float mx = max3_abs_nan(max3_abs_nan(ax[0], ax[1], ax[2]), ax[3], 0.0f) * factor;
        const float my = max3_abs_nan(max3_abs_nan(ay[0], ay[1], ay[2]), ay[3], 0.0f) * factor;
        const uint32_t ex = mx4_scale_byte(mx), ey = mx4_scale_byte(my);
        const float2 inv = make_float2(mx4_inv_scale(ex) * factor, mx4_inv_scale(ey) * factor);
        word |= (ex << (8 * half)) | (ey << (8 * half + 16));
        uint32_t wx[4], wy[4];
        #pragma unroll
        for (int q = 0; q < 4; ++q) {
            float2 y[8];
            #pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = fmul2_rn(v[32 * half + 8 * q + e], inv);
            wx[q] = mx4_encode8(y[0].x, y[1].x, y[2].x, y[3].x, y[4].x, y[5].x, y[6].x, y[7].x);
            wy[q] = mx4_encode8(y[0].y, y[1].y, y[2].y, y[3].y, y[4].y, y[5].y, y[6].y, y[7].y);
        }
        codes[half] = make_uint4(wx[0], wx[1], wx[2], wx[3]);
        codes[half + 2] = make_uint4(wy[0], wy[1], wy[2], wy[3]);
    }
    return word;
}

// Eight codes as floats without their block's scale.
__device__ __forceinline__ void mx4_decode8(uint32_t w, float (&f)[8]) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 c0, c1, c2, c3;\n\t"
        "mov.b32 {c0, c1, c2, c3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, c0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, c1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, c3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        __half2 p;
        memcpy(&p, &h[i], 4);
        const float2 q = __half22float2(p);
        f[2 * i] = q.x;
        f[2 * i + 1] = q.y;
    }
}

// The values that codes and scale bytes stand for.
__device__ __forceinline__ void unit_decode(const uint4 (&codes)[4], uint32_t word, float2 (&v)[64]) {
    #pragma unroll
    for (int half = 0; half < 2; ++half) {
        const float2 s = make_float2(mx4_scale_value((word >> (8 * half)) & 255u), mx4_scale_value((word >> (8 * half + 16)) & 255u));
        const uint32_t wx[4] = {codes[half].x, codes[half].y, codes[half].z, codes[half].w};
        const uint32_t wy[4] = {codes[half + 2].x, codes[half + 2].y, codes[half + 2].z, codes[half + 2].w};
        #pragma unroll
        for (int q = 0; q < 4; ++q) {
            float fx[8], fy[8];
            mx4_decode8(wx[q], fx);
            mx4_decode8(wy[q], fy);
            #pragma unroll
            for (int e = 0; e < 8; ++e) v[32 * half + 8 * q + e] = fmul2_rn(make_float2(fx[e], fy[e]), s);
        }
    }
}

// ---------------------------------------------------------------- a warp's slab of 32 units

template <typename T>
struct Mx4Slab {
    static constexpr int kPer = 16 / static_cast<int>(sizeof(T));       // values of a 16-byte chunk
    static constexpr int kChunks = kMx4Unit / kPer;                     // chunks of a unit: 16, or 32 in fp32
    static constexpr int kUnitBytes = kMx4Unit * static_cast<int>(sizeof(T));
    static constexpr int kBytes = 32 * kUnitBytes;
    __device__ static __forceinline__ uint32_t offset(int unit, int chunk) {
        return static_cast<uint32_t>(unit * kUnitBytes + ((chunk ^ (unit & 7)) << 4));
    }
};

__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool held) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                 :: "r"(smem_u32(dst)), "l"(src), "r"(held ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }

// Where a unit lies: `ptr` its first value (a readable address even when nothing
// of the unit exists), `chunks` of it exist: the rest reads as zero and is not
// written.
template <typename T>
struct Mx4UnitAt {
    const unsigned char* ptr;
    int chunks;
};

// Starts the copies of the warp's 32 units into its slab (lane l gives unit l's
// place). SPLIT: chunks from kChunks / 2 on lie `skip` bytes further than their
// place in the unit (two heads of 64). `vec`: every place is 16-byte aligned;
// otherwise plain loads.
template <bool SPLIT, typename T>
__device__ __forceinline__ void slab_load(unsigned char* slab, const Mx4UnitAt<T>& at, long long skip, bool vec) {
    using S = Mx4Slab<T>;
    const int lane = threadIdx.x & 31;
    #pragma unroll 4
    for (int i = 0; i < S::kChunks; ++i) {                              // 32 chunks an instruction
        const int unit = (i * 32 + lane) / S::kChunks, c = (i * 32 + lane) % S::kChunks;
        const auto p = reinterpret_cast<const unsigned char*>(
            __shfl_sync(0xFFFFFFFFu, reinterpret_cast<unsigned long long>(at.ptr), unit));
        const bool held = c < __shfl_sync(0xFFFFFFFFu, at.chunks, unit);
        const unsigned char* src = held ? p + c * 16 : p;
        if constexpr (SPLIT) {
            const long long more = __shfl_sync(0xFFFFFFFFu, skip, unit);
            if (held && c >= S::kChunks / 2) src += more;
        }
        unsigned char* dst = slab + S::offset(unit, c);
        if (vec) {
            cp_async16(dst, src, held);
        } else {
            T e[S::kPer];
            #pragma unroll
            for (int j = 0; j < S::kPer; ++j) e[j] = held ? reinterpret_cast<const T*>(src)[j] : mx4_from_f32<T>(0.0f);
            memcpy(dst, e, 16);
        }
    }
}

// The same for 32 whole units that lie one after the other, 16-byte aligned: no
// places to hand around (128 values a lane cost 2 instructions a copy instead of 15).
template <typename T>
__device__ __forceinline__ void slab_load_linear(unsigned char* slab, const void* src) {
    using S = Mx4Slab<T>;
    const int lane = threadIdx.x & 31;
    const unsigned char* p = static_cast<const unsigned char*>(src) + lane * 16;
    #pragma unroll
    for (int i = 0; i < S::kChunks; ++i)
        cp_async16(slab + S::offset((i * 32 + lane) / S::kChunks, (i * 32 + lane) % S::kChunks), p + i * 512);
}

template <typename T>
__device__ __forceinline__ void slab_store_linear(const unsigned char* slab, void* dst) {
    using S = Mx4Slab<T>;
    const int lane = threadIdx.x & 31;
    unsigned char* p = static_cast<unsigned char*>(dst) + lane * 16;
    #pragma unroll
    for (int i = 0; i < S::kChunks; ++i)
        *reinterpret_cast<uint4*>(p + i * 512) =
            *reinterpret_cast<const uint4*>(slab + S::offset((i * 32 + lane) / S::kChunks, (i * 32 + lane) % S::kChunks));
}

// Lane l's unit from the slab to registers, in fp32.
template <typename T>
__device__ __forceinline__ void slab_to_unit(const unsigned char* slab, float2 (&v)[64]) {
    using S = Mx4Slab<T>;
    const int lane = threadIdx.x & 31;
    #pragma unroll
    for (int c = 0; c < S::kChunks / 2; ++c) {
        const uint4 lo = *reinterpret_cast<const uint4*>(slab + S::offset(lane, c));
        const uint4 hi = *reinterpret_cast<const uint4*>(slab + S::offset(lane, c + S::kChunks / 2));
        const uint32_t a[4] = {lo.x, lo.y, lo.z, lo.w}, b[4] = {hi.x, hi.y, hi.z, hi.w};
        #pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (std::is_same_v<T, float>) {
                v[4 * c + e] = make_float2(__uint_as_float(a[e]), __uint_as_float(b[e]));
            } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                v[8 * c + 2 * e] = make_float2(__uint_as_float(a[e] << 16), __uint_as_float(b[e] << 16));
                v[8 * c + 2 * e + 1] = make_float2(__uint_as_float(a[e] & 0xFFFF0000u), __uint_as_float(b[e] & 0xFFFF0000u));
            } else {
                __half2 x, y;
                memcpy(&x, &a[e], 4);
                memcpy(&y, &b[e], 4);
                const float2 fx = __half22float2(x), fy = __half22float2(y);
                v[8 * c + 2 * e] = make_float2(fx.x, fy.x);
                v[8 * c + 2 * e + 1] = make_float2(fx.y, fy.y);
            }
        }
    }
}

// Lane l's unit, times a factor, rounded once to T, to the slab.
template <typename T>
__device__ __forceinline__ void unit_to_slab(unsigned char* slab, int unit, const float2 (&v)[64], float factor) {
    using S = Mx4Slab<T>;
    const float2 f = make_float2(factor, factor);
    #pragma unroll
    for (int c = 0; c < S::kChunks / 2; ++c) {
        uint32_t a[4], b[4];
        #pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (std::is_same_v<T, float>) {
                const float2 y = fmul2_rn(v[4 * c + e], f);
                a[e] = __float_as_uint(y.x);
                b[e] = __float_as_uint(y.y);
            } else {
                const float2 y0 = fmul2_rn(v[8 * c + 2 * e], f), y1 = fmul2_rn(v[8 * c + 2 * e + 1], f);
                if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                    const __nv_bfloat162 p = __floats2bfloat162_rn(y0.x, y1.x), q = __floats2bfloat162_rn(y0.y, y1.y);
                    memcpy(&a[e], &p, 4);
                    memcpy(&b[e], &q, 4);
                } else {
                    const __half2 p = __floats2half2_rn(y0.x, y1.x), q = __floats2half2_rn(y0.y, y1.y);
                    memcpy(&a[e], &p, 4);
                    memcpy(&b[e], &q, 4);
                }
            }
        }
        *reinterpret_cast<uint4*>(slab + S::offset(unit, c)) = make_uint4(a[0], a[1], a[2], a[3]);
        *reinterpret_cast<uint4*>(slab + S::offset(unit, c + S::kChunks / 2)) = make_uint4(b[0], b[1], b[2], b[3]);
    }
}

// Writes the slab's units to their places (16-byte aligned, contiguous units).
template <typename T>
__device__ __forceinline__ void slab_store(const unsigned char* slab, const Mx4UnitAt<T>& at) {
    using S = Mx4Slab<T>;
    const int lane = threadIdx.x & 31;
    #pragma unroll 4
    for (int i = 0; i < S::kChunks; ++i) {
        const int unit = (i * 32 + lane) / S::kChunks, c = (i * 32 + lane) % S::kChunks;
        const auto p = reinterpret_cast<unsigned char*>(
            __shfl_sync(0xFFFFFFFFu, reinterpret_cast<unsigned long long>(at.ptr), unit));
        const bool held = c < __shfl_sync(0xFFFFFFFFu, at.chunks, unit);
        if (held) *reinterpret_cast<uint4*>(p + c * 16) = *reinterpret_cast<const uint4*>(slab + S::offset(unit, c));
    }
}

}  // namespace convrot
