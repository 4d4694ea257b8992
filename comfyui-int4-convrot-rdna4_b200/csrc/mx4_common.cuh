// The MX4 format (OCP microscaling MXFP4) on the device: blocks of 32 values,
// each block one power-of-two scale E8M0 (byte E stands for 2^(E - 127), 255 for
// NaN), each value a 4-bit float e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6, sign in bit 3).
// Two codes a byte, the even column in the low nibble.
//
// A block of amplitude a gets E = floor(log2 a) - 2 + 127 (at least 0), so its
// largest value lands in [4, 8) and saturates at 6; codes are rounded to
// nearest, ties to even. A block that holds an infinity or a NaN gets E = 255
// and stands for NaN as a whole.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "hadamard.cuh"

namespace convrot {

constexpr int kMx4Block = 32;                 // values per scale
constexpr int kMx4TileBytes = 512;            // one scale tile: 128 rows x 4 blocks

// Scale byte of a block whose largest magnitude is `amax` (>= 0, inf or NaN).
__device__ __forceinline__ uint32_t mx4_scale_byte(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    if (bits >= 0x7F800000u) return 255u;
    const uint32_t e = bits >> 23;
    return e > 2u ? e - 2u : 0u;
}

// 2^(127 - E), the factor that brings a block onto the code grid; exact and
// normal for every E that mx4_scale_byte gives a finite block (0 .. 252).
__device__ __forceinline__ float mx4_inv_scale(uint32_t e) {
    return e == 255u ? 0.0f : __uint_as_float((254u - e) << 23);
}

// 2^(E - 127) (E = 0 is the subnormal 2^-127), NaN for 255.
__device__ __forceinline__ float mx4_scale_value(uint32_t e) {
    const uint32_t bits = e == 0u ? 0x00400000u : e == 255u ? 0x7FC00000u : e << 23;
    return __uint_as_float(bits);
}

__device__ __forceinline__ float mx4_to_f32(float v) { return v; }
__device__ __forceinline__ float mx4_to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float mx4_to_f32(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T mx4_from_f32(float v);
template <> __device__ __forceinline__ float mx4_from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 mx4_from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half mx4_from_f32<__half>(float v) { return __float2half_rn(v); }

// Position of the scale byte of (row, block) in the tiled scale matrix
// [ceil(R / 128), kt, 512]: the layout in which the tensor cores take scales
// (32 lanes of 16 bytes: four row groups of four blocks).
__device__ __forceinline__ size_t mx4_scale_pos(int row, int block, int kt) {
    return (static_cast<size_t>(row >> 7) * kt + (block >> 2)) * kMx4TileBytes +
           (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

}  // namespace convrot
