// The paged MX4 key/value cache: writing new tokens, reading slots back.
//
// Included by mx4.cu. Codes [pages, 2, heads, page, D/2], scales [pages, 2,
// heads, page, D/32]; keys at index 0, values at 1, both rotated along D. Slot
// s is token s % page of page s / page; a slot outside [0, pages * page) is
// skipped on writing and reads as zeros.
//
// A unit (mx4_unit.cuh) is 128 values of one token's key or value: one head of
// 128, half a head of 256 or two heads of 64 (the second may be missing). Units
// are numbered token, key or value, position, so a warp's rows are neighbours on
// the side of the [T, heads, D] tensors.
#pragma once

namespace convrot {

struct Mx4CacheShape {
    long long slots;       // pages * page
    int heads, d, page_bits;
    // index of (slot, key or value, head) in units of tokens of one head
    __device__ __forceinline__ size_t token(long long slot, int kv, int head) const {
        const long long p = slot >> page_bits;
        return ((static_cast<size_t>(p * 2 + kv) * heads + head) << page_bits) + static_cast<size_t>(slot & ((1 << page_bits) - 1));
    }
};

// What a unit's number stands for.
template <int D>
struct Mx4CacheUnit {
    int t, kv, head, part;           // part: which half of a head of 256
    int halves;                      // 64-value halves of the unit that exist
    __device__ __forceinline__ Mx4CacheUnit(int u, int per, int heads) {
        t = u / (2 * per);
        const int r = u - t * 2 * per;
        kv = r >= per;
        const int p = r - kv * per;
        head = D == 64 ? 2 * p : D == 128 ? p : p >> 1;
        part = D == 256 ? p & 1 : 0;
        halves = D == 64 && head + 1 >= heads ? 1 : 2;
    }
};

// Units of one token's keys (or values).
template <int D>
__host__ __device__ constexpr int mx4_cache_units(int heads) { return D == 64 ? (heads + 1) / 2 : D == 128 ? heads : 2 * heads; }

template <typename T, int D, int G>
__global__ void __launch_bounds__(kMx4QuantWarps * 32, 3)
mx4_cache_append_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, const T* __restrict__ k,
                        const T* __restrict__ v, long long kst, long long ksh, long long vst, long long vsh,
                        const long long* __restrict__ slots, int units, Mx4CacheShape c, bool vec) {
    using S = Mx4Slab<T>;
    extern __shared__ __align__(128) unsigned char mx4slabs[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned char* slab = mx4slabs + warp * 2 * S::kBytes;
    const int per = mx4_cache_units<D>(c.heads);
    const int step = static_cast<int>(gridDim.x) * kMx4QuantWarps * 32;
    int base = (static_cast<int>(blockIdx.x) * kMx4QuantWarps + warp) * 32;
    auto load = [&](unsigned char* to, int u) {
        const Mx4CacheUnit<D> at(u, per, c.heads);
        const T* src = at.kv ? v + at.t * vst + at.head * vsh : k + at.t * kst + at.head * ksh;
        // (two heads of 64: the second lies a head stride from the first)
        const long long skip = D == 64 ? (at.kv ? vsh : ksh) - 64 : 0;
        const Mx4UnitAt<T> place{reinterpret_cast<const unsigned char*>(u < units ? src + at.part * 128 : k),
                                 u < units ? at.halves * (S::kChunks / 2) : 0};
        slab_load<D == 64>(to, place, skip * static_cast<long long>(sizeof(T)), vec);
    };
    griddep_wait();
    griddep_launch_dependents();
    if (base < units) load(slab, base + lane);
    cp_async_commit();
    for (int it = 0; base < units; base += step, ++it) {
        const unsigned char* cur = slab + (it & 1) * S::kBytes;
        if (base + step < units) load(slab + ((it + 1) & 1) * S::kBytes, base + step + lane);
        cp_async_commit();
        cp_async_wait<1>();
        __syncwarp();
        float2 val[64];
        slab_to_unit<T>(cur, val);
        unit_rotate<G>(val);
        uint4 q[4];
        const uint32_t word = unit_quantize(val, unit_factor<G>(), q);
        const int u = (base + lane) ^ (G == 256 ? 1 : 0);
        const Mx4CacheUnit<D> at(u, per, c.heads);
        const long long slot = u < units ? slots[at.t] : -1;
        if (slot >= 0 && slot < c.slots) {
            const size_t tok = c.token(slot, at.kv, at.head);
            if constexpr (D == 64) {
                #pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (h >= at.halves) break;
                    const size_t to = tok + (static_cast<size_t>(h) << c.page_bits);
                    uint4* dst = reinterpret_cast<uint4*>(codes + to * 32);
                    dst[0] = q[2 * h];
                    dst[1] = q[2 * h + 1];
                    *reinterpret_cast<uint16_t*>(scales + to * 2) = static_cast<uint16_t>(word >> (16 * h));
                }
            } else {
                uint4* dst = reinterpret_cast<uint4*>(codes + tok * (D / 2) + at.part * 64);
                #pragma unroll
                for (int b = 0; b < 4; ++b) dst[b] = q[b];
                *reinterpret_cast<uint32_t*>(scales + tok * (D / 32) + at.part * 4) = word;
            }
        }
        __syncwarp();
    }
}

template <typename T, int D, int G>
__global__ void __launch_bounds__(kMx4QuantWarps * 32, 3)
mx4_cache_read_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                      const long long* __restrict__ slots, T* __restrict__ k, T* __restrict__ v, int units, Mx4CacheShape c) {
    using S = Mx4Slab<T>;
    extern __shared__ __align__(128) unsigned char mx4slabs[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned char* slab = mx4slabs + warp * S::kBytes;
    const int per = mx4_cache_units<D>(c.heads);
    const int step = static_cast<int>(gridDim.x) * kMx4QuantWarps * 32;
    griddep_wait();
    griddep_launch_dependents();
    for (int base = (static_cast<int>(blockIdx.x) * kMx4QuantWarps + warp) * 32; base < units; base += step) {
        const int u = base + lane;
        const Mx4CacheUnit<D> at(u, per, c.heads);
        const long long slot = u < units ? slots[at.t] : -1;
        uint4 q[4];
        uint32_t word = 0;
        #pragma unroll
        for (int b = 0; b < 4; ++b) q[b] = make_uint4(0, 0, 0, 0);
        if (slot >= 0 && slot < c.slots) {
            const size_t tok = c.token(slot, at.kv, at.head);
            if constexpr (D == 64) {
                #pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (h >= at.halves) break;
                    const size_t from = tok + (static_cast<size_t>(h) << c.page_bits);
                    const uint4* src = reinterpret_cast<const uint4*>(codes + from * 32);
                    q[2 * h] = src[0];
                    q[2 * h + 1] = src[1];
                    word |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(scales + from * 2)) << (16 * h);
                }
            } else {
                const uint4* src = reinterpret_cast<const uint4*>(codes + tok * (D / 2) + at.part * 64);
                #pragma unroll
                for (int b = 0; b < 4; ++b) q[b] = src[b];
                word = *reinterpret_cast<const uint32_t*>(scales + tok * (D / 32) + at.part * 4);
            }
        }
        float2 val[64];
        unit_decode(q, word, val);
        unit_rotate<G>(val);
        unit_to_slab<T>(slab, lane ^ (G == 256 ? 1 : 0), val, unit_factor<G>());
        __syncwarp();
        T* dst = (at.kv ? v : k) + (static_cast<size_t>(at.t) * c.heads + at.head) * D + at.part * 128;
        slab_store<T>(slab, Mx4UnitAt<T>{reinterpret_cast<const unsigned char*>(dst), u < units ? at.halves * (S::kChunks / 2) : 0});
        __syncwarp();
    }
}

}  // namespace convrot
