// out[m, n] = sum_k x[m, k] w[n, k] + bias[n] on MX4 operands.
//
// Included by mx4.cu. One thread an output, fp32 products and sums.
#pragma once

namespace convrot {

template <typename T>
__global__ void __launch_bounds__(256)
mx4_gemm_kernel(const uint8_t* __restrict__ xc, const uint8_t* __restrict__ xs, const uint8_t* __restrict__ wc,
                const uint8_t* __restrict__ ws, BiasRef bias, T* __restrict__ out, int M, int N, int K) {
    griddep_wait();
    griddep_launch_dependents();
    const int n = blockIdx.x * 32 + (threadIdx.x & 31);
    const int m = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (n >= N || m >= M) return;
    const int kt = (K + 127) / 128;
    float acc = 0.0f;
    for (int b = 0; b < K / 32; ++b) {
        const uint8_t* xr = xc + (static_cast<size_t>(m) * K + b * 32) / 2;
        const uint8_t* wr = wc + (static_cast<size_t>(n) * K + b * 32) / 2;
        float part = 0.0f;                               // exact: 32 products of at most 36, in quarters
        for (int i = 0; i < 16; ++i)
            part += mx4_code_value(xr[i] & 15u) * mx4_code_value(wr[i] & 15u) +
                    mx4_code_value(xr[i] >> 4) * mx4_code_value(wr[i] >> 4);
        acc += part * mx4_scale_value(xs[mx4_scale_pos(m, b, kt)]) * mx4_scale_value(ws[mx4_scale_pos(n, b, kt)]);
    }
    if (bias.ptr != nullptr) acc += bias.at(n);
    out[static_cast<size_t>(m) * N + n] = mx4_from_f32<T>(acc);
}

}  // namespace convrot
