// MX4 quantization of matrix rows (with the ConvRot rotation) and back.
//
// Included by mx4.cu. One block takes 1024 columns of one row: the values go
// to shared memory in fp32, the radix-4 steps of the rotation run there, then
// each warp quantizes blocks of 32, a lane a value.
#pragma once

namespace convrot {

constexpr int kMx4QuantCols = 1024;           // columns of a block's piece of a row (holds whole groups)
constexpr int kMx4QuantThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kMx4QuantThreads)
mx4_quant_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                 int M, int K, int group) {
    __shared__ float v[kMx4QuantCols];
    const int pieces = (K + kMx4QuantCols - 1) / kMx4QuantCols;
    const int row = blockIdx.x / pieces, k0 = (blockIdx.x % pieces) * kMx4QuantCols;
    const int n = min(kMx4QuantCols, K - k0);
    const int kt = (K + 127) / 128;
    griddep_wait();
    griddep_launch_dependents();
    const T* src = x + row * ldx + k0;
    for (int i = threadIdx.x; i < n; i += kMx4QuantThreads) v[i] = mx4_to_f32(src[i]);
    __syncthreads();
    mx4_rotate_shared(v, n, group, threadIdx.x, kMx4QuantThreads);
    const int lane = threadIdx.x & 31;
    const int blocks = n / kMx4Block;
    for (int b = threadIdx.x >> 5; b < blocks; b += kMx4QuantThreads / 32) {
        const float a = v[b * 32 + lane];
        uint32_t amax = __float_as_uint(a) & 0x7FFFFFFFu;      // as integers: NaN above inf above every number
        amax = __reduce_max_sync(0xFFFFFFFFu, amax);
        const uint32_t e = mx4_scale_byte(__uint_as_float(amax));
        const float y = a * mx4_inv_scale(e);
        const float hi = __shfl_down_sync(0xFFFFFFFFu, y, 1);
        const size_t at = static_cast<size_t>(row) * K + k0 + b * 32 + lane;
        if (!(lane & 1)) codes[at >> 1] = e == 255u ? 0 : static_cast<uint8_t>(mx4_encode2(y, hi));
        if (lane == 0) scales[mx4_scale_pos(row, k0 / 32 + b, kt)] = static_cast<uint8_t>(e);
    }
    // the last tile's missing blocks and rows stand for 2^-127 (their codes are never read)
    const int block_end = k0 + n == K ? kt * 4 : (k0 + n) / 32;
    if (k0 + n == K && static_cast<int>(threadIdx.x) < kt * 4 - K / 32)
        scales[mx4_scale_pos(row, K / 32 + threadIdx.x, kt)] = 0;
    if (row == M - 1)
        for (int r = M + (threadIdx.x >> 5); r < (M + 127) / 128 * 128; r += kMx4QuantThreads / 32)
            for (int b = k0 / 32 + lane; b < block_end; b += 32) scales[mx4_scale_pos(r, b, kt)] = 0;
}

template <typename T>
__global__ void __launch_bounds__(kMx4QuantThreads)
mx4_dequant_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ out, int K,
                   int group) {
    __shared__ float v[kMx4QuantCols];
    const int pieces = (K + kMx4QuantCols - 1) / kMx4QuantCols;
    const int row = blockIdx.x / pieces, k0 = (blockIdx.x % pieces) * kMx4QuantCols;
    const int n = min(kMx4QuantCols, K - k0);
    const int kt = (K + 127) / 128;
    griddep_wait();
    griddep_launch_dependents();
    const size_t at = static_cast<size_t>(row) * K + k0;
    for (int i = threadIdx.x; i < n; i += kMx4QuantThreads) {
        const uint32_t c = (codes[(at + i) >> 1] >> (4 * (i & 1))) & 15u;
        v[i] = mx4_code_value(c) * mx4_scale_value(scales[mx4_scale_pos(row, (k0 + i) / 32, kt)]);
    }
    __syncthreads();
    mx4_rotate_shared(v, n, group, threadIdx.x, kMx4QuantThreads);
    for (int i = threadIdx.x; i < n; i += kMx4QuantThreads) out[at + i] = mx4_from_f32<T>(v[i]);
}

}  // namespace convrot
