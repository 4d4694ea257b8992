// MX4 quantization of matrix rows (with the ConvRot rotation) and back.
//
// Included by mx4.cu. A unit (mx4_unit.cuh) is 128 columns of one row, and the
// units of the matrix are numbered row after row; a warp takes 32 of them at a
// time, copying the next 32 while it works on these. Missing columns of a row's
// last unit read as zeros, which leaves their scale bytes 0. The first `linear_units`
// units lie one after the other in memory (rows without a gap, whole units).
//
// Bound by memory, in groups of 256 as much by issue (10 instructions a value, the
// exchanged step alone 2.5). 4608 x 15360 bf16: 37 us in groups of 256 (4.8 TB/s), 33 us
// in groups of 64, 31 us not rotated (5.8 TB/s); fp32 56 us (5.8 TB/s). Back: 30 us not
// rotated (5.9 TB/s), 44 / 36 / 34 us in groups of 256 / 64 / 16.
#pragma once

namespace convrot {

constexpr int kMx4QuantWarps = 4;

template <typename T> constexpr int mx4_quant_smem() { return kMx4QuantWarps * 2 * Mx4Slab<T>::kBytes; }

template <typename T, int G>
__global__ void __launch_bounds__(kMx4QuantWarps * 32, 3)
mx4_quant_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                 int M, int K, int units, bool vec, int linear_units) {
    using S = Mx4Slab<T>;
    extern __shared__ __align__(128) unsigned char mx4slabs[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned char* slab = mx4slabs + warp * 2 * S::kBytes;
    const int kt = (K + 127) / 128;
    const int step = static_cast<int>(gridDim.x) * kMx4QuantWarps * 32;
    int base = (static_cast<int>(blockIdx.x) * kMx4QuantWarps + warp) * 32;
    auto place = [&](int u) {
        const int row = u / kt, c = u - row * kt;
        const bool held = u < units && row < M;
        return Mx4UnitAt<T>{reinterpret_cast<const unsigned char*>(held ? x + row * ldx + c * kMx4Unit : x),
                            held ? min(S::kChunks, (K - c * kMx4Unit) / S::kPer) : 0};
    };
    auto load = [&](unsigned char* to, int first) {
        if (first + 32 <= linear_units) slab_load_linear<T>(to, x + static_cast<size_t>(first) * kMx4Unit);
        else slab_load<false>(to, place(first + lane), 0, vec);
    };
    griddep_wait();
    griddep_launch_dependents();
    if (base < units) load(slab, base);
    cp_async_commit();
    for (int it = 0; base < units; base += step, ++it) {
        const unsigned char* cur = slab + (it & 1) * S::kBytes;
        if (base + step < units) load(slab + ((it + 1) & 1) * S::kBytes, base + step);
        cp_async_commit();
        cp_async_wait<1>();
        __syncwarp();
        float2 v[64];
        slab_to_unit<T>(cur, v);
        unit_rotate<G>(v);
        uint4 q[4];
        const uint32_t word = unit_quantize(v, unit_factor<G>(), q);
        const int u = (base + lane) ^ (G == 256 ? 1 : 0);
        const int row = u / kt, c = u - row * kt;
        if (u < units) {
            *reinterpret_cast<uint32_t*>(scales + mx4_scale_pos(row, 4 * c, kt)) = word;
            if (row < M) {
                uint4* dst = reinterpret_cast<uint4*>(codes + (static_cast<size_t>(row) * K + c * kMx4Unit) / 2);
                const int blocks = min(4, (K - c * kMx4Unit) / kMx4Block);
                #pragma unroll
                for (int b = 0; b < 4; ++b)
                    if (b < blocks) dst[b] = q[b];
            }
        }
        __syncwarp();
    }
}

// Back, with the rotation: values go out through the warp's slab.
template <typename T, int G>
__global__ void __launch_bounds__(kMx4QuantWarps * 32, 3)
mx4_dequant_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ out, int K,
                   int units) {
    using S = Mx4Slab<T>;
    extern __shared__ __align__(128) unsigned char mx4slabs[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned char* slab = mx4slabs + warp * S::kBytes;
    const int kt = (K + 127) / 128;
    const int step = static_cast<int>(gridDim.x) * kMx4QuantWarps * 32;
    const bool linear = K % kMx4Unit == 0;
    griddep_wait();
    griddep_launch_dependents();
    for (int base = (static_cast<int>(blockIdx.x) * kMx4QuantWarps + warp) * 32; base < units; base += step) {
        const int u = base + lane;
        const int row = u / kt, c = u - row * kt;
        const int blocks = u < units ? min(4, (K - c * kMx4Unit) / kMx4Block) : 0;
        const uint4* src = reinterpret_cast<const uint4*>(codes + (static_cast<size_t>(row) * K + c * kMx4Unit) / 2);
        uint4 q[4];
        #pragma unroll
        for (int b = 0; b < 4; ++b) q[b] = b < blocks ? src[b] : make_uint4(0, 0, 0, 0);
        const uint32_t word = blocks ? *reinterpret_cast<const uint32_t*>(scales + mx4_scale_pos(row, 4 * c, kt)) : 0;
        float2 v[64];
        unit_decode(q, word, v);
        unit_rotate<G>(v);
        unit_to_slab<T>(slab, lane ^ (G == 256 ? 1 : 0), v, unit_factor<G>());
        __syncwarp();
        if (linear && base + 32 <= units) {
            slab_store_linear<T>(slab, out + static_cast<size_t>(base) * kMx4Unit);
        } else {
            slab_store<T>(slab, Mx4UnitAt<T>{reinterpret_cast<const unsigned char*>(out + static_cast<size_t>(row) * K + c * kMx4Unit),
                                             blocks * (kMx4Block / S::kPer)});
        }
        __syncwarp();
    }
}

// Back, without a rotation: a thread takes words of eight codes, neighbouring
// threads neighbouring words.
constexpr int kMx4DecodeThreads = 256, kMx4DecodeWords = 8;

template <typename T>
__global__ void __launch_bounds__(kMx4DecodeThreads)
mx4_decode_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ out, int K, long long words) {
    const int row_words = K / 8, kt = (K + 127) / 128;
    griddep_wait();
    griddep_launch_dependents();
    const long long first = static_cast<long long>(blockIdx.x) * (kMx4DecodeThreads * kMx4DecodeWords) + threadIdx.x;
    int row = static_cast<int>(first / row_words), col = static_cast<int>(first - static_cast<long long>(row) * row_words);
    uint32_t w[kMx4DecodeWords], e[kMx4DecodeWords];
    #pragma unroll
    for (int i = 0; i < kMx4DecodeWords; ++i) {
        const long long at = first + i * kMx4DecodeThreads;
        w[i] = 0;
        e[i] = 0;
        if (at < words) {
            w[i] = __ldg(codes + at);
            e[i] = __ldg(scales + mx4_scale_pos(row, col >> 2, kt));
        }
        row += kMx4DecodeThreads / row_words;
        col += kMx4DecodeThreads % row_words;
        if (col >= row_words) {
            col -= row_words;
            ++row;
        }
    }
    #pragma unroll
    for (int i = 0; i < kMx4DecodeWords; ++i) {
        const long long at = first + i * kMx4DecodeThreads;
        if (at >= words) break;
        float f[8];
        mx4_decode8(w[i], f);
        const float s = mx4_scale_value(e[i]);
        T v[8];
        #pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = mx4_from_f32<T>(f[j] * s);
        uint4 p[sizeof(T) / 2];
        memcpy(p, v, sizeof(v));
        #pragma unroll
        for (int j = 0; j < static_cast<int>(sizeof(T)) / 2; ++j) *(reinterpret_cast<uint4*>(out + at * 8) + j) = p[j];
    }
}

}  // namespace convrot
