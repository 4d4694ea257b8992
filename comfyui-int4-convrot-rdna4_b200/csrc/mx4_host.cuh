// Host-side checks and dispatch shared by the translation units of the MX4 operators.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>
#include <type_traits>

#include "host_launch.cuh"
#include "linear_api.cuh"
#include "sm100_ptx.cuh"
#include "mx4_common.cuh"
#include "mx4_unit.cuh"
#include "mx4_quant.cuh"

namespace convrot {

// Units (128 values each) of one call: their numbers, and one grid's step beyond,
// fit 32 bits.
constexpr long long kMx4MostUnits = 0x7FFFFFFFll - (1 << 20);

inline size_t align256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

inline int check_group(int K, int G) {
    if (G != 0 && G != 16 && G != 64 && G != 256) return fail("G must be 0, 16, 64 or 256");
    if (K <= 0 || K % kMx4Block) return fail("K must be a positive multiple of 32");
    if (G != 0 && K % G) return fail("K must be a multiple of G");
    return 0;
}

// Calls f with a null pointer of the C type of dtype code 0 f32, 1 bf16, 2 f16.
template <typename F>
inline int with_type(int code, F f) {
    if (code == 0) return f(static_cast<float*>(nullptr));
    if (code == 1) return f(static_cast<__nv_bfloat16*>(nullptr));
    return f(static_cast<__half*>(nullptr));
}

inline size_t type_size(int code) { return code == 0 ? 4 : 2; }

inline bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Calls f with an integral constant for the rotation group.
template <typename F>
inline int with_group(int G, F f) {
    if (G == 16) return f(std::integral_constant<int, 16>{});
    if (G == 64) return f(std::integral_constant<int, 64>{});
    if (G == 256) return f(std::integral_constant<int, 256>{});
    return f(std::integral_constant<int, 0>{});
}

// Blocks of the unit kernels: one wave of three a multiprocessor, a warp's 32
// units at a time.
inline int unit_blocks(long long units) {
    const long long want = (units + kMx4QuantWarps * 32 - 1) / (kMx4QuantWarps * 32), most = 3LL * sm_count();
    return static_cast<int>(want < most ? want : most);
}

// Calls f with integral constants for the head dimension and the rotation group.
template <typename F>
inline int with_head(int d, int G, F f) {
    return with_group(G, [&](auto g) {
        constexpr int g0 = decltype(g)::value;
        if (d == 64) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, g0 == 256 ? 0 : g0>{});
        if (d == 128) return f(std::integral_constant<int, 128>{}, std::integral_constant<int, g0 == 256 ? 0 : g0>{});
        return f(std::integral_constant<int, 256>{}, g);
    });
}

inline int page_bits(int page) {
    int b = 0;
    while ((1 << b) < page) ++b;
    return b;
}

inline int check_cache(const void* codes, const void* scales, long long pages, int heads, int d, int page, int G) {
    if (d != 64 && d != 128 && d != 256) return fail("the head dimension must be 64, 128 or 256");
    if (int rc = check_group(d, G)) return rc;
    if (heads <= 0 || page <= 0 || pages < 0) return fail("heads and page must be positive, pages not negative");
    if (page & (page - 1) || page > 65536) return fail("the page size must be a power of two up to 65536");
    if (pages > 0x7FFFFFFFll) return fail("too many pages");
    if (pages && (!codes || !scales)) return fail("null cache pointer");
    if (!aligned16(codes) || !aligned16(scales)) return fail("the cache must be 16-byte aligned");
    return 0;
}

// Keys and values [T, heads, d] to their slots (mx4.cu), or the values alone; arguments checked by the caller.
int run_cache_append(void* codes, void* scales, long long pages, int heads, int d, int page, int G, const void* k, const void* v, int in_dtype,
                     long long k_token, long long k_head, long long v_token, long long v_head, const void* slots, int T, bool values_only,
                     cudaStream_t stream);

}  // namespace convrot
