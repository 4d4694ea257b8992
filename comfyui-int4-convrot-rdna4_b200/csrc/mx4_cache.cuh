// The paged MX4 key/value cache: writing new tokens, reading slots back.
//
// Included by mx4.cu. Codes [pages, 2, heads, page, D/2], scales [pages, 2,
// heads, page, D/32]; keys at index 0, values at 1, both rotated along D. Slot
// s is token s % page of page s / page; a slot outside [0, pages * page) is
// skipped on writing and reads as zeros.
//
// A unit (mx4_unit.cuh) is 128 values of one token's key or value: one head of
// 128, half a head of 256 or two heads of 64 (the second may be missing). Units
// are numbered key or value, token, position, so a warp's units are neighbours on
// the side of the [T, heads, D] tensors (`linear`: without a gap).
//
// Bound by memory. 8 heads of 128, pages of 64, groups of 64: 32768 tokens written in
// 40 us from a view of a QKV projection (4.2 TB/s), 32 us from contiguous tensors;
// 65536 tokens read back in 66 us (5.2 TB/s, four fifths of it writing bf16).
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
    __device__ __forceinline__ Mx4CacheUnit(int u, int per, int heads, int units) {
        kv = u >= units / 2;         // (units is even)
        const int r = kv ? u - units / 2 : u;
        t = r / per;
        const int p = r - t * per;
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
                        const long long* __restrict__ slots, int units, Mx4CacheShape c, bool vec, bool linear) {
    using S = Mx4Slab<T>;
    extern __shared__ __align__(128) unsigned char mx4slabs[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned char* slab = mx4slabs + warp * 2 * S::kBytes;
    const int per = mx4_cache_units<D>(c.heads);
    const int step = static_cast<int>(gridDim.x) * kMx4QuantWarps * 32;
    int base = (static_cast<int>(blockIdx.x) * kMx4QuantWarps + warp) * 32;
    auto load = [&](unsigned char* to, int first) {
        const int u = first + lane;
        if (linear && first + 32 <= units && (first + 32 <= units / 2 || first >= units / 2)) {
            const int half = first >= units / 2;
            slab_load_linear<T>(to, (half ? v : k) + static_cast<size_t>(first - half * (units / 2)) * kMx4Unit);
            return;
        }
        const Mx4CacheUnit<D> at(u, per, c.heads, units);
        const T* src = at.kv ? v + at.t * vst + at.head * vsh : k + at.t * kst + at.head * ksh;
        // (two heads of 64: the second lies a head stride from the first)
        const long long skip = D == 64 ? (at.kv ? vsh : ksh) - 64 : 0;
        const Mx4UnitAt<T> place{reinterpret_cast<const unsigned char*>(u < units ? src + at.part * 128 : k),
                                 u < units ? at.halves * (S::kChunks / 2) : 0};
        slab_load<D == 64>(to, place, skip * static_cast<long long>(sizeof(T)), vec);
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
        float2 val[64];
        slab_to_unit<T>(cur, val);
        unit_rotate<G>(val);
        uint4 q[4];
        const uint32_t word = unit_quantize(val, unit_factor<G>(), q);
        const int u = (base + lane) ^ (G == 256 ? 1 : 0);
        const Mx4CacheUnit<D> at(u, per, c.heads, units);
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

// Reading: a lane copies its next unit's codes into its own 64 bytes of shared memory
// while the warp works on the current ones; the slot after that is on its way too.
constexpr int kMx4ReadWarpBytes = 2 * 32 * 64;

template <typename T, int D, int G>
__global__ void __launch_bounds__(kMx4QuantWarps * 32, 3)
mx4_cache_read_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                      const long long* __restrict__ slots, T* __restrict__ k, T* __restrict__ v, int units, Mx4CacheShape c) {
    using S = Mx4Slab<T>;
    extern __shared__ __align__(128) unsigned char mx4slabs[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned char* slab = mx4slabs + warp * (S::kBytes + kMx4ReadWarpBytes);
    unsigned char* ahead = slab + S::kBytes;                      // [2][block][lane][16]
    const int per = mx4_cache_units<D>(c.heads);
    const int step = static_cast<int>(gridDim.x) * kMx4QuantWarps * 32;
    const bool linear = D != 64 || c.heads % 2 == 0;
    auto slot_of = [&](int u) -> long long { return u < units ? __ldg(slots + Mx4CacheUnit<D>(u, per, c.heads, units).t) : -1; };
    uint32_t word = 0;                                            // scale bytes of the unit copied last
    auto fetch = [&](int buf, int u, long long slot) {
        const Mx4CacheUnit<D> at(u, per, c.heads, units);
        const bool held = u < units && slot >= 0 && slot < c.slots;
        const size_t tok = held ? c.token(slot, at.kv, at.head) : 0;
        unsigned char* dst = ahead + buf * 2048 + lane * 16;
        word = 0;
        #pragma unroll
        for (int b = 0; b < 4; ++b) {
            // (heads of 64: blocks 2 and 3 are the next head's)
            const bool here = held && (D != 64 || b < 2 * at.halves);
            const size_t row = D == 64 ? tok + (b >= 2 ? static_cast<size_t>(1) << c.page_bits : 0) : tok;
            const size_t byte = D == 64 ? row * 32 + (b & 1) * 16 : row * (D / 2) + at.part * 64 + b * 16;
            cp_async16(dst + b * 512, codes + (here ? byte : 0), here);
        }
        if constexpr (D == 64) {
            if (held) word = __ldg(reinterpret_cast<const uint16_t*>(scales + tok * 2));
            if (held && at.halves == 2)
                word |= static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(scales + (tok + (static_cast<size_t>(1) << c.page_bits)) * 2))) << 16;
        } else if (held) {
            word = __ldg(reinterpret_cast<const uint32_t*>(scales + tok * (D / 32) + at.part * 4));
        }
    };
    griddep_wait();
    griddep_launch_dependents();
    int base = (static_cast<int>(blockIdx.x) * kMx4QuantWarps + warp) * 32;
    if (base < units) fetch(0, base + lane, slot_of(base + lane));
    cp_async_commit();
    long long slot = slot_of(base + step + lane);
    for (int it = 0; base < units; base += step, ++it) {
        const uint32_t cur = word;
        if (base + step < units) fetch((it + 1) & 1, base + step + lane, slot);
        cp_async_commit();
        slot = slot_of(base + 2 * step + lane);
        cp_async_wait<1>();
        uint4 q[4];
        #pragma unroll
        for (int b = 0; b < 4; ++b) q[b] = *reinterpret_cast<const uint4*>(ahead + (it & 1) * 2048 + lane * 16 + b * 512);
        float2 val[64];
        unit_decode(q, cur, val);
        unit_rotate<G>(val);
        unit_to_slab<T>(slab, lane ^ (G == 256 ? 1 : 0), val, unit_factor<G>());
        __syncwarp();
        const int half = base >= units / 2;
        if (linear && base + 32 <= units && (half || base + 32 <= units / 2)) {
            slab_store_linear<T>(slab, (half ? v : k) + static_cast<size_t>(base - half * (units / 2)) * kMx4Unit);
        } else {
            const int u = base + lane;
            const Mx4CacheUnit<D> at(u, per, c.heads, units);
            T* dst = (at.kv ? v : k) + (static_cast<size_t>(at.t) * c.heads + at.head) * D + at.part * 128;
            slab_store<T>(slab, Mx4UnitAt<T>{reinterpret_cast<const unsigned char*>(dst), u < units ? at.halves * (S::kChunks / 2) : 0});
        }
        __syncwarp();
    }
}

}  // namespace convrot
