// Rotary positions: pair i of a head is turned by the angle p f_i, p the token's
// position on the pair's axis.
//
// Pairs are channels (2i, 2i + 1) (interleaved) or (i, i + P) of P pairs; the
// channels behind the 2P first stay as they are. The pairs are cut into sections, one an
// axis (text: one; images and video: index, height, width).
//
// The angle p f and its sine and cosine are taken in 64 bits and rounded once: at position 10^6 an
// fp32 product would be 0.06 radians off. (64-bit products run at half the fp32 rate here, some 25 a
// pair, and a token's angles serve all of its heads.) Products and sums of the turn are fp32 operations
// each of its own: the values are those of the formula computed step by step in fp32, which matters
// where they are quantized to 4 bits afterwards.
//
// Bound by its bytes where it is large: 4608 tokens of 60 heads of 128 in bf16 take 27.9 us, 5.1 TB/s
// (a copy of the tensor 28.7). A thread keeps a token's angles for as many heads as leave one wave of
// blocks, four heads' loads ahead; one head a thread took 37.5 us, most of it for angles. One token
// of 40 heads is a launch (2.9 us in a graph).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>
#include <type_traits>

#include "mx4_common.cuh"
#include "sm100_ptx.cuh"

namespace convrot {

constexpr int kRopeMostAxes = 8;

struct RopeArgs {
    const void* pos;               // [B, T, axes] by strides
    const double* freqs;           // [pairs], radians a position
    long long pb, pt, pa;
    int pos_type;                  // 0 int32, 1 int64, 2 f32
    int pairs, axes, interleaved;
    float sign;                    // -1: the rotation back
    int ends[kRopeMostAxes];       // where each axis's section ends

    __device__ __forceinline__ double position(long long b, long long t, int axis) const {
        const long long at = b * pb + t * pt + axis * pa;
        if (pos_type == 0) return static_cast<double>(static_cast<const int*>(pos)[at]);
        if (pos_type == 1) return static_cast<double>(static_cast<const long long*>(pos)[at]);
        return static_cast<double>(static_cast<const float*>(pos)[at]);
    }
};

// Where a thread's 2 VP channels lie: VP from a and VP from b, so that neighbours' chunks are
// neighbours in memory. In halves a pair has one channel in each; interleaved, each chunk holds VP / 2 pairs.
// `pair`, `pair_b`: the first pair of each chunk; -1: none, the chunk is copied as it is (b if a is: it lies behind).
template <int VP>
struct RopePlace {
    int a, b, pair, pair_b;
    __device__ __forceinline__ RopePlace(const RopeArgs& r, int D, int u, bool turned) {
        const int whole = r.pairs / VP;                           // chunks of pairs in halves
        pair = pair_b = -1;
        if (r.interleaved && VP > 1) {
            a = VP * u;
            b = D / 2 + a;
            if (turned && a < 2 * r.pairs) pair = a / 2;
            if (turned && b < 2 * r.pairs) pair_b = b / 2;
        } else if (r.interleaved) {
            a = 2 * u;
            b = a + 1;
            if (turned && u < r.pairs) pair = pair_b = u;
        } else if (u < whole) {
            a = VP * u;
            b = r.pairs + a;
            if (turned) pair = pair_b = a;
        } else {
            a = 2 * r.pairs + VP * (u - whole);
            b = a + (D / 2 - r.pairs);
        }
    }
    __device__ __forceinline__ bool any() const { return pair >= 0; }
};

// Sine and cosine of a (radians, finite and below some 2^50 in magnitude), rounded to fp32: reduced to
// |x| <= pi / 4 around a quarter turn with 1 / (2 pi) in two terms, then the Taylor polynomials of degree 13
// and 14, whose remainders are below 2 * 10^-14.
__device__ __forceinline__ void rope_sincos(double a, float& s, float& c) {
    const double hi = a * 0.15915494309189535, lo = fma(a, 0.15915494309189535, -hi) + a * -9.839338337591243e-18;
    const double r = (hi - rint(hi)) + lo, q = rint(4.0 * r), x = fma(-0.25, q, r) * 6.283185307179586, y = x * x;
    double u = fma(y, 1.0 / 6227020800.0, -1.0 / 39916800.0), v = fma(y, -1.0 / 87178291200.0, 1.0 / 479001600.0);
    u = fma(u, y, 1.0 / 362880.0);
    v = fma(v, y, -1.0 / 3628800.0);
    u = fma(u, y, -1.0 / 5040.0);
    v = fma(v, y, 1.0 / 40320.0);
    u = fma(u, y, 1.0 / 120.0);
    v = fma(v, y, -1.0 / 720.0);
    u = fma(u, y, -1.0 / 6.0);
    v = fma(v, y, 1.0 / 24.0);
    v = fma(v, y, -0.5);
    const float sx = static_cast<float>(fma(u * y, x, x)), cx = static_cast<float>(fma(v, y, 1.0));
    const int quarter = static_cast<int>(q);                      // -2 .. 2
    s = quarter & 1 ? cx : sx;
    c = quarter & 1 ? sx : cx;
    if (quarter & 2) s = -s;
    if ((quarter + 1) & 2) c = -c;
}

// Cosine and sine of a thread's pairs, those of chunk a's first where they are interleaved.
template <int VP>
struct RopeCoef {
    float c[VP], s[VP];
    // N pairs in a row to the places from FROM on.
    template <int FROM, int N>
    __device__ __forceinline__ void group(const RopeArgs& r, long long b, long long t, int pair) {
        int axis = 0;
        while (axis < r.axes - 1 && pair >= r.ends[axis]) ++axis;
        int end = axis < r.axes - 1 ? r.ends[axis] : 0x7FFFFFFF;
        double p = r.position(b, t, axis);
        #pragma unroll
        for (int i = 0; i < N; ++i) {
            if (pair + i >= end) {
                do ++axis; while (axis < r.axes - 1 && pair + i >= r.ends[axis]);
                end = axis < r.axes - 1 ? r.ends[axis] : 0x7FFFFFFF;
                p = r.position(b, t, axis);
            }
            rope_sincos(p * r.freqs[pair + i], s[FROM + i], c[FROM + i]);
            s[FROM + i] *= r.sign;
        }
    }
    __device__ __forceinline__ void load(const RopeArgs& r, long long b, long long t, const RopePlace<VP>& at) {
        if (VP == 1 || !r.interleaved) {
            group<0, VP>(r, b, t, at.pair);
            return;
        }
        constexpr int kHalf = VP > 1 ? VP / 2 : 1;
        group<0, kHalf>(r, b, t, at.pair);
        if constexpr (VP > 1)
            if (at.pair_b >= 0) group<kHalf, VP - kHalf>(r, b, t, at.pair_b);
    }
};

// (A chunk of interleaved channels without pairs stays: a turn by 0 would give a neighbour's infinity or NaN to it.)
template <int VP>
__device__ __forceinline__ void rope_turn(float (&a)[VP], float (&b)[VP], const RopeCoef<VP>& w, const RopePlace<VP>& at, bool interleaved) {
    auto turn = [](float& x, float& y, float c, float s) {
        const float z = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
        y = __fadd_rn(__fmul_rn(x, s), __fmul_rn(y, c));
        x = z;
    };
    if (VP > 1 && interleaved) {
        #pragma unroll
        for (int i = 0; i + 1 < VP; i += 2) {
            turn(a[i], a[i + 1], w.c[i / 2], w.s[i / 2]);
            if (at.pair_b >= 0) turn(b[i], b[i + 1], w.c[(VP + i) / 2], w.s[(VP + i) / 2]);
        }
    } else {
        #pragma unroll
        for (int i = 0; i < VP; ++i) turn(a[i], b[i], w.c[i], w.s[i]);
    }
}

// VP values from memory as they are: 16 bytes where VP is more than one.
template <typename T, int VP>
struct RopeRaw {
    static_assert(VP == 1 || VP * sizeof(T) == 16, "a chunk is 16 bytes or one value");
    std::conditional_t<VP == 1, T, uint4> v;
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (VP == 1) v = *p;
        else v = __ldg(reinterpret_cast<const uint4*>(p));
    }
    __device__ __forceinline__ void zero() {
        if constexpr (VP == 1) v = mx4_from_f32<T>(0.0f);
        else v = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void get(float (&f)[VP]) const {
        if constexpr (VP == 1) {
            f[0] = mx4_to_f32(v);
        } else {
            T e[VP];
            memcpy(e, &v, 16);
            #pragma unroll
            for (int i = 0; i < VP; ++i) f[i] = mx4_to_f32(e[i]);
        }
    }
    __device__ __forceinline__ void put(const float (&f)[VP]) {
        if constexpr (VP == 1) {
            v = mx4_from_f32<T>(f[0]);
        } else {
            T e[VP];
            #pragma unroll
            for (int i = 0; i < VP; ++i) e[i] = mx4_from_f32<T>(f[i]);
            memcpy(&v, e, 16);
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (VP == 1) *p = v;
        else *reinterpret_cast<uint4*>(p) = v;
    }
};

struct RopeShape {
    long long xb, xt, xh;          // strides of the input in elements: batch, token, head
    long long tokens;
    int T, H, D;
    int heads, runs;               // heads a thread takes, threads that a chunk of a token needs
    int slice;                     // tokens of a row of blocks
};

constexpr int kRopeThreads = 256;
constexpr int kRopeResident = 2;   // blocks a multiprocessor holds

// x [B, T, H, D] by strides -> out [B, T, H, D] without gaps. A thread has 2 VP channels
// of one token and goes through its heads.
template <typename T, int VP>
__global__ void __launch_bounds__(kRopeThreads, kRopeResident) rope_kernel(const T* __restrict__ x, T* __restrict__ out, RopeShape s,
                                                                         const __grid_constant__ RopeArgs r) {
    constexpr int kAhead = 4;
    const int chunks = s.D / (2 * VP);
    const unsigned id = blockIdx.x * static_cast<unsigned>(kRopeThreads) + threadIdx.x;
    const unsigned rest = id / chunks, in_slice = rest / s.runs;
    const int u = static_cast<int>(id - rest * chunks), run = static_cast<int>(rest - in_slice * s.runs);
    const long long token = static_cast<long long>(blockIdx.y) * s.slice + in_slice;
    griddep_wait();
    griddep_launch_dependents();
    if (in_slice >= static_cast<unsigned>(s.slice) || token >= s.tokens) return;
    const int h0 = run * s.heads, h1 = min(s.H, h0 + s.heads);
    long long b = 0, t = token;
    if (token >= s.T) {
        b = s.tokens <= 0x7FFFFFFF ? static_cast<int>(token) / s.T : token / s.T;
        t = token - b * s.T;
    }
    const RopePlace<VP> at(r, s.D, u, true);
    const T* src = x + b * s.xb + t * s.xt;
    T* dst = out + token * s.H * s.D;
    RopeCoef<VP> w;
    bool known = false;
    #pragma unroll 1
    for (int h = h0; h < h1; h += kAhead) {
        RopeRaw<T, VP> ra[kAhead], rb[kAhead];
        #pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (h + i < h1) {
                ra[i].load(src + (h + i) * s.xh + at.a);
                rb[i].load(src + (h + i) * s.xh + at.b);
            }
        if (!known) {                                             // (the first loads are on their way)
            if (at.any()) w.load(r, b, t, at);
            known = true;
        }
        #pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (h + i < h1) {
                T* to = dst + static_cast<long long>(h + i) * s.D;
                if (at.any()) {
                    float fa[VP], fb[VP];
                    ra[i].get(fa);
                    rb[i].get(fb);
                    rope_turn<VP>(fa, fb, w, at, r.interleaved);
                    ra[i].put(fa);
                    if (at.pair_b >= 0) rb[i].put(fb);
                }
                ra[i].store(to + at.a);
                rb[i].store(to + at.b);
            }
    }
}

}  // namespace convrot
