// C entry of the W8A8 linear behind a root-mean-square norm with residual.
// Conventions of include/convrot_b200.h.
#include <algorithm>

#include "mx4_host.cuh"
#include "rms_quant.cuh"

#define CONVROT_API extern "C" __attribute__((visibility("default")))

using namespace convrot;

namespace {

template <typename T, int G>
int launch_rms_quant(const RmsQuantArgs& a, cudaStream_t stream) {
    const int warps = a.rows * a.row_warps, blocks = std::min((a.M + a.rows - 1) / a.rows, 8 * sm_count());
    auto launch = [&](auto kernel, int most) {
        cudaError_t e = ensure_smem(kernel, most * kRmsWarpFloats * 4);
        if (e != cudaSuccess) return static_cast<int>(e);
        return static_cast<int>(launch_pdl(kernel, dim3(blocks), dim3(warps * 32), warps * kRmsWarpFloats * 4, stream, a));
    };
    if (warps <= 8) return launch(rms_quant_int8_kernel<T, G, 256>, 8);
    return launch(rms_quant_int8_kernel<T, G, 1024>, 32);
}

// Four warps a block, as many blocks as there are outputs by 16, or sixteen where those would
// leave places empty (1 x 15360 x 3840: one wave of blocks, with eight warps it were two and a bit).
template <int NT, typename T>
int launch_few(const RmsQuantArgs& a, const void* W, const float* ws, BiasRef bias, void* out, int N, cudaStream_t stream) {
    const int blocks = (N + 15) / 16, warps = blocks >= 2 * sm_count() ? 4 : 16;
    return static_cast<int>(launch_pdl(few_i8_kernel<NT, T>, dim3(blocks), dim3(warps * 32), warps * 8 * NT * 17 * 4, stream, static_cast<const int8_t*>(a.codes),
                                       static_cast<const int8_t*>(W), static_cast<const float*>(a.scales), ws, bias, static_cast<T*>(out), a.M, N, a.K));
}

template <typename T>
int run_few(const RmsQuantArgs& a, const void* W, const float* ws, BiasRef bias, void* out, int N, cudaStream_t stream) {
    if (a.M <= 8) return launch_few<1, T>(a, W, ws, bias, out, N, stream);
    return launch_few<2, T>(a, W, ws, bias, out, N, stream);
}

}  // namespace

CONVROT_API size_t ck_convrot_w8a8_linear_rmsnorm_workspace_size(int M, int K) {
    if (M <= 0 || K <= 0) return 0;
    return align256(static_cast<size_t>(M) * K) + align256(static_cast<size_t>(M) * 4);
}

CONVROT_API int ck_convrot_w8a8_linear_rmsnorm(const void* x, const void* residual, int dtype, long long ldx, long long ldr,
                                               const void* norm_weight, int norm_dtype, float eps, const void* W, const void* wscale,
                                               const void* bias, int bias_dtype, void* hidden, void* out, int out_dtype, int M, int N, int K,
                                               int G, void* workspace, size_t workspace_bytes, void* stream) {
    if (M < 0 || N < 0 || K <= 0) return fail("M, N must be >= 0 and K > 0");
    if (dtype < 0 || dtype > 2) return fail("dtype must be 0 (f32), 1 (bf16) or 2 (f16)");
    if (G != 16 && G != 64 && G != 256) return fail("G must be 16, 64 or 256");
    if (K % G) return fail("K must be a multiple of G");
    if (K > kRmsMostK) return fail("K must be at most 16384");
    if (out_dtype != 0 && out_dtype != 1) return fail("out_dtype must be 0 (f32) or 1 (bf16)");
    if (norm_weight && (norm_dtype < 0 || norm_dtype > 2)) return fail("norm_dtype must be 0 (f32), 1 (bf16) or 2 (f16)");
    if (bias && (bias_dtype < 0 || bias_dtype > 2)) return fail("bias_dtype must be 0 (f32), 1 (bf16) or 2 (f16)");
    if (M == 0) return 0;
    if (M > 0x7FFFFFFF - (1 << 20)) return fail("too many rows");
    if (ldx < 0 || ldr < 0 || (M > 1 && (ldx < K || (residual && ldr < K)))) return fail("row strides must be at least K");
    if (!x || (residual && !hidden) || (N && (!W || !wscale || !out))) return fail("null pointer");
    const size_t size = type_size(dtype);
    if (!aligned_to(x, size) || !aligned_to(residual, size)) return fail("rows are not aligned to their type");
    if ((residual && !aligned16(hidden)) || !aligned16(W) || !aligned16(out)) return fail("the hidden rows, the weight and out must be 16-byte aligned");
    if ((norm_weight && !aligned_to(norm_weight, type_size(norm_dtype))) || (bias && !aligned_to(bias, type_size(bias_dtype))) || !aligned_to(wscale, 4))
        return fail("vectors are not aligned to their types");
    const size_t need = ck_convrot_w8a8_linear_rmsnorm_workspace_size(M, K);
    if (!workspace || !aligned_to(workspace, 256)) return fail("the workspace must be 256-byte aligned");
    if (workspace_bytes < need) return fail("workspace smaller than ck_convrot_w8a8_linear_rmsnorm_workspace_size");
    RmsQuantArgs a{};
    a.x = x;
    a.r = residual;
    a.g = norm_weight;
    a.ldx = ldx;
    a.ldr = ldr;
    a.h = hidden;
    a.codes = static_cast<int8_t*>(workspace);
    a.scales = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + align256(static_cast<size_t>(M) * K));
    a.M = M;
    a.K = K;
    a.g_type = norm_dtype;
    a.row_warps = (K + 511) / 512;
    a.rows = std::max(1, 8 / a.row_warps);
    a.vec_x = aligned16(x) && ldx * static_cast<long long>(size) % 16 == 0;
    a.vec_g = aligned16(norm_weight);
    a.vec_r = aligned16(residual) && ldr * static_cast<long long>(size) % 16 == 0;
    a.eps = eps;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (int rc = with_type(dtype, [&](auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            if (G == 16) return launch_rms_quant<T, 16>(a, st);
            if (G == 64) return launch_rms_quant<T, 64>(a, st);
            return launch_rms_quant<T, 256>(a, st);
        }))
        return rc;
    if (N == 0) return 0;
    const float* s = static_cast<const float*>(wscale);
    const BiasRef b{bias, bias_dtype};
    if (M <= kFewI8Rows) return out_dtype == 1 ? run_few<__nv_bfloat16>(a, W, s, b, out, N, st) : run_few<float>(a, W, s, b, out, N, st);
    return run_gemm_i8(a.codes, W, a.scales, s, b, out, out_dtype, M, N, K, st);
}
