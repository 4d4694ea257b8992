// C entries of the MX4 (microscaled 4-bit float) operators: quantization of
// rows, the linear on MX4 weights, the paged key/value cache and attention over
// it. Conventions of include/convrot_b200.h: device pointers, caller-allocated
// outputs, nothing synchronises; 0, -1 with a message, or a CUDA error.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <type_traits>

#include "sm100_ptx.cuh"
#include "linear_api.cuh"
#include "host_launch.cuh"
#include "mx4_common.cuh"

#define CONVROT_API extern "C" __attribute__((visibility("default")))

namespace convrot {

// Status word of this translation unit's kernels (a bounded wait that gave up);
// ck_convrot_device_status reads and clears it.
static __device__ int g_mx4_status;

enum : int { kMx4TimeoutProducer = 1, kMx4TimeoutMma = 2, kMx4TimeoutEpilogue = 4 };

__device__ __forceinline__ void mx4_record_status(int code) { atomicCAS(&g_mx4_status, 0, code); }

cudaError_t mx4_take_status(cudaStream_t stream, int* status) {
    cudaError_t e = cudaMemcpyFromSymbolAsync(status, g_mx4_status, sizeof(int), 0, cudaMemcpyDeviceToHost, stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
    const int zero = 0;
    if (e == cudaSuccess) e = cudaMemcpyToSymbolAsync(g_mx4_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
    return e;
}

}  // namespace convrot

#include "mx4_unit.cuh"
#include "mx4_quant.cuh"
#include "mx4_gemm.cuh"
#include "mx4_few.cuh"
#include "mx4_cache.cuh"
#include "mx4_attn.cuh"

namespace convrot {

// Units (128 values each) of one call: their numbers, and one grid's step beyond,
// fit 32 bits.
constexpr long long kMx4MostUnits = 0x7FFFFFFFll - (1 << 20);

static size_t align256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

static size_t scales_bytes(int rows, int K) {
    return static_cast<size_t>((rows + 127) / 128) * ((K + 127) / 128) * kMx4TileBytes;
}

static int check_group(int K, int G) {
    if (G != 0 && G != 16 && G != 64 && G != 256) return fail("G must be 0, 16, 64 or 256");
    if (K <= 0 || K % kMx4Block) return fail("K must be a positive multiple of 32");
    if (G != 0 && K % G) return fail("K must be a multiple of G");
    return 0;
}

// Calls f with a null pointer of the C type of dtype code 0 f32, 1 bf16, 2 f16.
template <typename F>
static int with_type(int code, F f) {
    if (code == 0) return f(static_cast<float*>(nullptr));
    if (code == 1) return f(static_cast<__nv_bfloat16*>(nullptr));
    return f(static_cast<__half*>(nullptr));
}

static size_t type_size(int code) { return code == 0 ? 4 : 2; }

static bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

static int check_matrix(const void* x, int dtype, const void* codes, const void* scales, int M, int K, int G) {
    if (M < 0) return fail("M must not be negative");
    if (dtype < 0 || dtype > 2) return fail("dtype must be 0 (f32), 1 (bf16) or 2 (f16)");
    if (int rc = check_group(K, G)) return rc;
    if (M == 0) return 0;
    if (!x || !codes || !scales) return fail("null pointer");
    if (!aligned_to(x, type_size(dtype))) return fail("values are not aligned to their type");
    if (!aligned16(codes) || !aligned16(scales)) return fail("codes and scales must be 16-byte aligned");
    if (static_cast<long long>(M + 127LL) / 128 * 128 * ((K + 127) / 128) > kMx4MostUnits) return fail("matrix too large");
    return 0;
}

// Calls f with an integral constant for the rotation group.
template <typename F>
static int with_group(int G, F f) {
    if (G == 16) return f(std::integral_constant<int, 16>{});
    if (G == 64) return f(std::integral_constant<int, 64>{});
    if (G == 256) return f(std::integral_constant<int, 256>{});
    return f(std::integral_constant<int, 0>{});
}

// Blocks of the unit kernels: one wave of three a multiprocessor, a warp's 32
// units at a time.
static int unit_blocks(long long units) {
    const long long want = (units + kMx4QuantWarps * 32 - 1) / (kMx4QuantWarps * 32), most = 3LL * sm_count();
    return static_cast<int>(want < most ? want : most);
}

static int run_quant(const void* x, int dtype, long long ldx, void* codes, void* scales, int M, int K, int G, cudaStream_t st) {
    const long long units = static_cast<long long>((M + 127) / 128 * 128) * ((K + 127) / 128);
    return with_type(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return with_group(G, [&](auto g) {
            auto kernel = mx4_quant_kernel<T, decltype(g)::value>;
            cudaError_t e = ensure_smem(kernel, mx4_quant_smem<T>());
            if (e != cudaSuccess) return static_cast<int>(e);
            const bool vec = aligned16(x) && ldx * sizeof(T) % 16 == 0;
            const int linear = vec && (ldx == K || M == 1) && K % kMx4Unit == 0 ? static_cast<int>(static_cast<long long>(M) * K / kMx4Unit) : 0;
            return static_cast<int>(launch_pdl(kernel, dim3(unit_blocks(units)), dim3(kMx4QuantWarps * 32), mx4_quant_smem<T>(), st,
                                               static_cast<const T*>(x), ldx, static_cast<uint8_t*>(codes),
                                               static_cast<uint8_t*>(scales), M, K, static_cast<int>(units), vec, linear));
        });
    });
}

// 2D tensor map of `rows` rows of `cols` elements at a pitch in bytes.
static bool make_tmap(CUtensorMap* map, CUtensorMapDataType type, const void* base, long long rows, long long cols,
                      long long pitch, int box_rows, int box_cols, CUtensorMapSwizzle swizzle) {
    auto enc = get_encode_fn();
    if (!enc) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch)};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t estr[2] = {1, 1};
    return enc(map, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Codes [rows, K/2] in boxes of 256 values x box_rows; scale tiles as rows of
// 32-bit words in boxes of two K tiles x box_tiles.
static bool make_mx4_tmaps(CUtensorMap* codes_map, CUtensorMap* scales_map, const void* codes, const void* scales, int rows,
                           int K, int box_rows, int box_tiles) {
    const long long kt = (K + 127) / 128, rt = (rows + 127) / 128;
    return make_tmap(codes_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, rows, K / 2, K / 2, box_rows, kMx4StageK / 2,
                     CU_TENSOR_MAP_SWIZZLE_128B) &&
           make_tmap(scales_map, CU_TENSOR_MAP_DATA_TYPE_UINT32, scales, rt, kt * 128, kt * kMx4TileBytes, box_tiles, 256,
                     CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <int BN, typename T>
static int launch_gemm_pair(const void* xc, const void* xs, const void* wc, const void* ws, BiasRef bias, T* out, int M, int N,
                            int K, cudaStream_t stream) {
    using Cfg = Mx4PairCfg<BN>;
    CUtensorMap tx, tw, txs, tws, to;
    memset(&to, 0, sizeof(to));
    if (!make_mx4_tmaps(&tx, &txs, xc, xs, M, K, 128, 1) || !make_mx4_tmaps(&tw, &tws, wc, ws, N, K, BN / 2, BN / 128))
        return fail("cuTensorMapEncodeTiled failed (operand size out of range or driver entry point missing)");
    const int staged = (static_cast<size_t>(N) * sizeof(T)) % 16 == 0;
    if (staged && !make_tmap(&to, sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, out, M, N,
                             static_cast<long long>(N) * sizeof(T), 32, 128 / sizeof(T), CU_TENSOR_MAP_SWIZZLE_128B))
        return fail("cuTensorMapEncodeTiled failed for the output");
    auto kernel = mx4_gemm_pair_kernel<BN, T>;
    cudaError_t e = ensure_smem(kernel, Cfg::kSmemBytes);
    if (e != cudaSuccess) return static_cast<int>(e);
    const int tiles_m = (M + 255) / 256;
    const long long num_tiles = static_cast<long long>(tiles_m) * ((N + BN - 1) / BN);
    if (num_tiles > 0x7FFFFFFF) return fail("too many output tiles");
    const int clusters = static_cast<int>(num_tiles < sm_count() / 2 ? num_tiles : sm_count() / 2);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * clusters, 1, 1);
    cfg.blockDim = dim3(kMx4PairThreads, 1, 1);
    cfg.dynamicSmemBytes = Cfg::kSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, tx, tw, txs, tws, to, bias, out, M, N, K, tiles_m,
                                               static_cast<int>(num_tiles), staged));
}

// The few-row kernel: 1, 2, 4 or 8 slices of K (a cluster), as many as leave the
// blocks two a multiprocessor and each slice four stages (4 x 4096 x 4096: 4.5 us in four
// slices, 5.3 in eight, 7.9 in one; 1 x 15360 x 3840: 7.7 us in two, 9.4 in one; weights beyond L2).
template <typename T, int G, int BT, bool FUSED>
static int launch_gemm_few(const void* x, long long ldx, const void* xc, const void* xs, const void* wc, const void* ws,
                           BiasRef bias, T* out, int M, int N, int K, cudaStream_t stream) {
    using Cfg = Mx4FewCfg<BT, FUSED>;
    CUtensorMap tx, tw, txs, tws;
    memset(&tx, 0, sizeof(tx));
    memset(&txs, 0, sizeof(txs));
    if (!make_mx4_tmaps(&tw, &tws, wc, ws, N, K, 128, 1) || (!FUSED && !make_mx4_tmaps(&tx, &txs, xc, xs, M, K, BT, 1)))
        return fail("cuTensorMapEncodeTiled failed (operand size out of range or driver entry point missing)");
    auto kernel = mx4_gemm_few_kernel<T, G, BT, FUSED>;
    cudaError_t e = ensure_smem(kernel, Cfg::kSmemBytes);
    if (e != cudaSuccess) return static_cast<int>(e);
    const int tiles = (N + 127) / 128, num_kt = (K + kMx4StageK - 1) / kMx4StageK;
    int splits = 1;
    while (splits < 8 && 2 * splits * tiles <= 2 * sm_count() && 8 * splits <= num_kt) splits *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles, splits, 1);
    cfg.blockDim = dim3(kMx4FewThreads, 1, 1);
    cfg.dynamicSmemBytes = Cfg::kSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = splits;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = splits > 1 ? 2 : 1;
    const bool vec = aligned16(x) && ldx * sizeof(T) % 16 == 0;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, tw, tws, tx, txs, static_cast<const T*>(x), ldx, vec,
                                               bias, out, M, N, K));
}

// x [M, K] quantized (xc, xs) times the weight; few rows go through the kernel
// that is bound by the weight's bytes.
template <typename T>
static int run_gemm(const void* xc, const void* xs, const void* wc, const void* ws, BiasRef bias, T* out, int M, int N, int K,
                    cudaStream_t stream) {
    if (M <= 32) return launch_gemm_few<T, 0, 32, false>(nullptr, 0, xc, xs, wc, ws, bias, out, M, N, K, stream);
    if (M <= 64) return launch_gemm_few<T, 0, 64, false>(nullptr, 0, xc, xs, wc, ws, bias, out, M, N, K, stream);
    if (M <= 128) return launch_gemm_few<T, 0, 128, false>(nullptr, 0, xc, xs, wc, ws, bias, out, M, N, K, stream);
    // Tile width by the waves of tiles over the SM pairs: a stage of 256 values of K
    // takes 560 cycles in a 256-wide tile and 400 in a 128-wide one (measured), a tile's
    // start about 500.
    const long long tiles_m = (M + 255) / 256, pairs = sm_count() / 2, stages = (K + kMx4StageK - 1) / kMx4StageK;
    auto cost = [&](int width, int cycles) {
        const long long tiles = tiles_m * ((N + width - 1) / width);
        return (tiles + pairs - 1) / pairs * (stages * cycles + 500);
    };
    if (cost(256, 560) <= cost(128, 400)) return launch_gemm_pair<256>(xc, xs, wc, ws, bias, out, M, N, K, stream);
    return launch_gemm_pair<128>(xc, xs, wc, ws, bias, out, M, N, K, stream);
}

}  // namespace convrot

using namespace convrot;

CONVROT_API size_t ck_mx4_scales_size(int rows, int K) {
    if (rows <= 0 || K <= 0) return 0;
    return scales_bytes(rows, K);
}

CONVROT_API int ck_mx4_quant(const void* x, int in_dtype, long long ldx, void* codes, void* scales, int M, int K, int G,
                             void* stream) {
    if (int rc = check_matrix(x, in_dtype, codes, scales, M, K, G)) return rc;
    if (M == 0) return 0;
    if (ldx < 0 || (M > 1 && ldx < K)) return fail("ldx must be at least K");
    return run_quant(x, in_dtype, ldx, codes, scales, M, K, G, static_cast<cudaStream_t>(stream));
}

CONVROT_API int ck_mx4_dequant(const void* codes, const void* scales, void* out, int out_dtype, int M, int K, int G,
                               void* stream) {
    if (int rc = check_matrix(out, out_dtype, codes, scales, M, K, G)) return rc;
    if (M == 0) return 0;
    if (!aligned16(out)) return fail("out must be 16-byte aligned");
    const long long units = static_cast<long long>(M) * ((K + 127) / 128), words = static_cast<long long>(M) * K / 8;
    return with_type(out_dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (G == 0) {
            const long long per = kMx4DecodeThreads * kMx4DecodeWords;
            return static_cast<int>(launch_pdl(mx4_decode_kernel<T>, dim3(static_cast<unsigned>((words + per - 1) / per)), dim3(kMx4DecodeThreads),
                                               0, static_cast<cudaStream_t>(stream), static_cast<const uint32_t*>(codes),
                                               static_cast<const uint8_t*>(scales), static_cast<T*>(out), K, words));
        }
        return with_group(G, [&](auto g) {
            constexpr int g0 = decltype(g)::value == 0 ? 16 : decltype(g)::value;
            auto kernel = mx4_dequant_kernel<T, g0>;
            cudaError_t e = ensure_smem(kernel, mx4_quant_smem<T>() / 2);
            if (e != cudaSuccess) return static_cast<int>(e);
            return static_cast<int>(launch_pdl(kernel, dim3(unit_blocks(units)), dim3(kMx4QuantWarps * 32), mx4_quant_smem<T>() / 2,
                                               static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(codes),
                                               static_cast<const uint8_t*>(scales), static_cast<T*>(out), K, static_cast<int>(units)));
        });
    });
}

CONVROT_API size_t ck_mx4_linear_workspace_size(int M, int K) {
    if (M <= kMx4FusedRows || K <= 0) return 0;
    return align256(static_cast<size_t>(M) * K / 2) + align256(scales_bytes(M, K));
}

CONVROT_API int ck_mx4_linear(const void* x, int dtype, long long ldx, const void* Wcodes, const void* Wscales,
                              const void* bias, int bias_dtype, void* out, int M, int N, int K, int G, void* workspace, size_t workspace_bytes, void* stream) {
    if (N < 0) return fail("N must not be negative");
    if (N == 0) return 0;
    if (int rc = check_matrix(x, dtype, Wcodes, Wscales, M, K, G)) return rc;
    if (M == 0) return 0;
    if (ldx < 0 || (M > 1 && ldx < K)) return fail("ldx must be at least K");
    if (bias && (bias_dtype < 0 || bias_dtype > 2)) return fail("bias_dtype must be 0 (f32), 1 (bf16) or 2 (f16)");
    if (bias && !aligned_to(bias, type_size(bias_dtype))) return fail("bias is not aligned to its type");
    if (!out || !aligned16(out)) return fail("out must be 16-byte aligned");
    const size_t need = ck_mx4_linear_workspace_size(M, K);
    if (need && (!workspace || !aligned_to(workspace, 256))) return fail("the workspace must be 256-byte aligned");
    if (workspace_bytes < need) return fail("workspace smaller than ck_mx4_linear_workspace_size");
    uint8_t* xc = static_cast<uint8_t*>(workspace);
    uint8_t* xs = xc + align256(static_cast<size_t>(M) * K / 2);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const BiasRef b{bias, bias_dtype};
    if (M > kMx4FusedRows)
        if (int rc = run_quant(x, dtype, ldx, xc, xs, M, K, G, st)) return rc;
    return with_type(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (M > kMx4FusedRows) return run_gemm(xc, xs, Wcodes, Wscales, b, static_cast<T*>(out), M, N, K, st);
        return with_group(G, [&](auto g) {
            return launch_gemm_few<T, decltype(g)::value, 16, true>(x, ldx, nullptr, nullptr, Wcodes, Wscales, b,
                                                                               static_cast<T*>(out), M, N, K, st);
        });
    });
}

// Calls f with integral constants for the head dimension and the rotation group.
template <typename F>
static int with_head(int d, int G, F f) {
    return with_group(G, [&](auto g) {
        constexpr int g0 = decltype(g)::value;
        if (d == 64) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, g0 == 256 ? 0 : g0>{});
        if (d == 128) return f(std::integral_constant<int, 128>{}, std::integral_constant<int, g0 == 256 ? 0 : g0>{});
        return f(std::integral_constant<int, 256>{}, g);
    });
}

static int page_bits(int page) {
    int b = 0;
    while ((1 << b) < page) ++b;
    return b;
}

// How an attention call is cut: tiles of query rows (one sequence and cache head
// each) and splits of the sequences.
struct AttnPlan {
    long long tiles;
    int tile_rows, row_tiles, splits;
    bool clustered;                // a sequence's splits are one cluster and join themselves
    size_t partials() const { return splits > 1 && !clustered ? static_cast<size_t>(tiles) * splits * tile_rows : 0; }
};

static AttnPlan attn_plan(int B, int tq, int hq, int hkv, int d, long long longest) {
    AttnPlan p;
    const long long rows = static_cast<long long>(tq) * (hq / hkv);
    p.tile_rows = rows <= 8 ? 8 : rows <= 16 || d == 256 ? 16 : 32;
    p.row_tiles = static_cast<int>((rows + p.tile_rows - 1) / p.tile_rows);
    p.tiles = static_cast<long long>(B) * hkv * p.row_tiles;
    // splits: one full wave of blocks always, as far as every split has a group of
    // tokens; up to four waves, which even the tail out, while each split keeps eight
    // groups (a block's start and end cost about as much as three). Waves counted by the
    // blocks a multiprocessor really holds, and whole ones: 64 x 4096 tokens of 32 heads 320 us,
    // 355 with a part of a wave; 64 x 1024 of 32 heads on 8: 30.4 against 35.5
    const long long groups = (longest + kMx4AttnGroup - 1) / kMx4AttnGroup, tiles = p.tiles > 0 ? p.tiles : 1;
    const long long places = static_cast<long long>(mx4_attn_resident(p.tile_rows / 8 * d)) * sm_count();
    long long waves = 4;
    while (waves > 1 && waves * places / tiles > groups / 8) --waves;
    const long long want = waves * places / tiles;
    p.splits = static_cast<int>(std::max(1LL, std::min({want, groups, static_cast<long long>(kMx4MostSplits)})));
    // one launch instead of two (1 x 777 tokens: 7.8 against 9.9 us), where every block is
    // resident at once; with more, a cluster's blocks wait for each other and for places
    // (64 x 4096 tokens, 4 splits: 106 against 99 us)
    p.clustered = p.splits > 1 && p.splits <= 8 && tiles * p.splits <= 2LL * sm_count();
    return p;
}

template <typename T, int D, int NT>
static int launch_attention(const Mx4AttnArgs& a, const AttnPlan& p, cudaStream_t stream) {
    using Cfg = Mx4AttnCfg<D, NT>;
    auto kernel = mx4_attn_kernel<T, D, NT>;
    cudaError_t e = ensure_smem(kernel, Cfg::kSmemBytes);
    if (e != cudaSuccess) return static_cast<int>(e);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.tiles), p.splits, 1);
    cfg.blockDim = dim3(kMx4AttnWarps * 32, 1, 1);
    cfg.dynamicSmemBytes = Cfg::kSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = p.splits;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.clustered ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, kernel, a);
    if (e == cudaSuccess && p.splits > 1 && !p.clustered) {
        const unsigned rows = static_cast<unsigned>(a.B * a.tq * a.hq);
        const int wide = p.splits > 16;
        e = launch_pdl(mx4_attn_join_kernel<T, D>, dim3(wide ? rows : (rows + 7) / 8), dim3(256), 0, stream, a, p.tile_rows, wide);
    }
    return static_cast<int>(e);
}

template <typename T, int D>
static int launch_attention_rows(const Mx4AttnArgs& a, const AttnPlan& p, cudaStream_t stream) {
    if (p.tile_rows == 8) return launch_attention<T, D, 1>(a, p, stream);
    if constexpr (D < 256)
        if (p.tile_rows == 32) return launch_attention<T, D, 4>(a, p, stream);
    return launch_attention<T, D, 2>(a, p, stream);
}

template <typename T>
static int run_attention(const Mx4AttnArgs& a, int d, const AttnPlan& p, cudaStream_t stream) {
    if (d == 256) return launch_attention_rows<T, 256>(a, p, stream);
    if (d == 128) return launch_attention_rows<T, 128>(a, p, stream);
    return launch_attention_rows<T, 64>(a, p, stream);
}

static int check_cache(const void* codes, const void* scales, long long pages, int heads, int d, int page, int G) {
    if (d != 64 && d != 128 && d != 256) return fail("the head dimension must be 64, 128 or 256");
    if (int rc = check_group(d, G)) return rc;
    if (heads <= 0 || page <= 0 || pages < 0) return fail("heads and page must be positive, pages not negative");
    if (page & (page - 1) || page > 65536) return fail("the page size must be a power of two up to 65536");
    if (pages > 0x7FFFFFFFll) return fail("too many pages");
    if (pages && (!codes || !scales)) return fail("null cache pointer");
    if (!aligned16(codes) || !aligned16(scales)) return fail("the cache must be 16-byte aligned");
    return 0;
}

CONVROT_API int ck_mx4_cache_append(void* codes, void* scales, long long pages, int heads, int d, int page, int G,
                                    const void* k, const void* v, int in_dtype, long long k_token, long long k_head,
                                    long long v_token, long long v_head, const void* slots, int T, void* stream) {
    if (int rc = check_cache(codes, scales, pages, heads, d, page, G)) return rc;
    if (T < 0) return fail("T must not be negative");
    if (in_dtype < 0 || in_dtype > 2) return fail("dtype must be 0 (f32), 1 (bf16) or 2 (f16)");
    if (T == 0) return 0;
    if (!k || !v || !slots) return fail("null pointer");
    if (!aligned_to(k, type_size(in_dtype)) || !aligned_to(v, type_size(in_dtype)) || !aligned_to(slots, 8))
        return fail("keys, values or slots are not aligned to their type");
    const Mx4CacheShape c{pages * page, heads, d, page_bits(page)};
    return with_type(in_dtype, [&](auto* t) {
        using E = std::remove_pointer_t<decltype(t)>;
        return with_head(d, G, [&](auto dim, auto g) {
            auto kernel = mx4_cache_append_kernel<E, decltype(dim)::value, decltype(g)::value>;
            cudaError_t e = ensure_smem(kernel, mx4_quant_smem<E>());
            if (e != cudaSuccess) return static_cast<int>(e);
            const long long units = static_cast<long long>(T) * 2 * mx4_cache_units<decltype(dim)::value>(heads);
            if (units > kMx4MostUnits) return fail("too many tokens in one call");
            const long long strides = k_token | k_head | v_token | v_head;
            const bool vec = aligned16(k) && aligned16(v) && strides * static_cast<long long>(sizeof(E)) % 16 == 0;
            const bool linear = vec && k_head == d && v_head == d && k_token == static_cast<long long>(heads) * d &&
                                v_token == k_token && (d != 64 || heads % 2 == 0);
            return static_cast<int>(launch_pdl(kernel, dim3(unit_blocks(units)), dim3(kMx4QuantWarps * 32), mx4_quant_smem<E>(),
                                               static_cast<cudaStream_t>(stream), static_cast<uint8_t*>(codes),
                                               static_cast<uint8_t*>(scales), static_cast<const E*>(k), static_cast<const E*>(v),
                                               k_token, k_head, v_token, v_head, static_cast<const long long*>(slots), static_cast<int>(units), c, vec, linear));
        });
    });
}

CONVROT_API int ck_mx4_cache_read(const void* codes, const void* scales, long long pages, int heads, int d, int page, int G,
                                  const void* slots, int T, void* k, void* v, int out_dtype, void* stream) {
    if (int rc = check_cache(codes, scales, pages, heads, d, page, G)) return rc;
    if (T < 0) return fail("T must not be negative");
    if (out_dtype < 0 || out_dtype > 2) return fail("dtype must be 0 (f32), 1 (bf16) or 2 (f16)");
    if (T == 0) return 0;
    if (!k || !v || !slots) return fail("null pointer");
    if (!aligned16(k) || !aligned16(v) || !aligned_to(slots, 8)) return fail("outputs must be 16-byte, slots 8-byte aligned");
    const Mx4CacheShape c{pages * page, heads, d, page_bits(page)};
    return with_type(out_dtype, [&](auto* t) {
        using E = std::remove_pointer_t<decltype(t)>;
        return with_head(d, G, [&](auto dim, auto g) {
            auto kernel = mx4_cache_read_kernel<E, decltype(dim)::value, decltype(g)::value>;
            const int smem = kMx4QuantWarps * (Mx4Slab<E>::kBytes + kMx4ReadWarpBytes);
            cudaError_t e = ensure_smem(kernel, smem);
            if (e != cudaSuccess) return static_cast<int>(e);
            const long long units = static_cast<long long>(T) * 2 * mx4_cache_units<decltype(dim)::value>(heads);
            if (units > kMx4MostUnits) return fail("too many tokens in one call");
            return static_cast<int>(launch_pdl(kernel, dim3(unit_blocks(units)), dim3(kMx4QuantWarps * 32), smem,
                                               static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(codes),
                                               static_cast<const uint8_t*>(scales), static_cast<const long long*>(slots),
                                               static_cast<E*>(k), static_cast<E*>(v), static_cast<int>(units), c));
        });
    });
}

CONVROT_API size_t ck_mx4_attention_workspace_size(int B, int tq, int hq, int hkv, int d, long long longest) {
    if (B <= 0 || tq <= 0 || hkv <= 0 || hq <= 0 || hq % hkv || d <= 0) return 0;
    const AttnPlan p = attn_plan(B, tq, hq, hkv, d, longest);
    return align256(p.partials() * d * 4) + align256(p.partials() * 8);
}

CONVROT_API int ck_mx4_attention(const void* q, int dtype, long long q_seq, long long q_token, long long q_head,
                                 const void* codes, const void* scales, long long pages, int page, const void* table,
                                 long long table_ld, int table_pages, const void* lens, void* out, int B, int tq, int hq,
                                 int hkv, int d, int G, float softmax_scale, void* workspace, size_t workspace_bytes,
                                 void* stream) {
    if (int rc = check_cache(codes, scales, pages, hkv, d, page, G)) return rc;
    if (dtype != 1 && dtype != 2) return fail("queries must be bf16 (1) or f16 (2)");
    if (B < 0 || tq <= 0 || hq <= 0 || hq % hkv) return fail("query heads must be a positive multiple of the cache's heads");
    if (table_pages < 0 || table_ld < table_pages) return fail("bad block table shape");
    if (static_cast<long long>(table_pages) * page > kMx4MostTokens) return fail("block table longer than 2^31 - 1024 tokens");
    if (B == 0) return 0;
    if (static_cast<long long>(B) * tq * hq > 0x7FFFFFFFll) return fail("too many query rows");
    if (!q || !lens || !out || (table_pages && !table)) return fail("null pointer");
    if (!aligned_to(q, 2) || !aligned_to(table, 4) || !aligned_to(lens, 4) || !aligned16(out))
        return fail("queries, table or lengths not aligned to their type, or out not to 16 bytes");
    if (pages * 2 * hkv * page > 0xFFFFFFFEll) return fail("the cache holds more than 2^32 - 2 rows");
    const long long longest = static_cast<long long>(table_pages) * page;
    const AttnPlan p = attn_plan(B, tq, hq, hkv, d, longest);
    if (static_cast<long long>(p.tiles) > 0x7FFFFFFF || static_cast<long long>(B) * tq * hq > 0x7FFFFFFFll) return fail("too many query rows");
    const size_t need = ck_mx4_attention_workspace_size(B, tq, hq, hkv, d, longest);
    if (need && (!workspace || !aligned_to(workspace, 256))) return fail("the workspace must be 256-byte aligned");
    if (workspace_bytes < need) return fail("workspace smaller than ck_mx4_attention_workspace_size");
    Mx4AttnArgs a{q, q_seq, q_token, q_head, static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales),
                  static_cast<const int*>(table), table_ld, longest, static_cast<const int*>(lens), out,
                  static_cast<float*>(workspace),
                  need ? reinterpret_cast<float2*>(static_cast<unsigned char*>(workspace) + align256(p.partials() * d * 4)) : nullptr,
                  B, tq, hq, hkv, page_bits(page), static_cast<int>(pages), G, p.row_tiles, p.splits, p.clustered,
                  softmax_scale * 1.4426950408889634f};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == 1) return run_attention<__nv_bfloat16>(a, d, p, st);
    return run_attention<__half>(a, d, p, st);
}
