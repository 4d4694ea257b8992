// The paged MX4 key/value cache: writing new tokens, reading slots back.
//
// Included by mx4.cu. Codes [pages, 2, heads, page, D/2], scales [pages, 2,
// heads, page, D/32]; keys at index 0, values at 1, both rotated along D. Slot
// s is token s % page of page s / page; a slot outside [0, pages * page) is
// skipped on writing and reads as zeros.
#pragma once

namespace convrot {

struct Mx4CacheShape {
    long long slots;       // pages * page
    int heads, d, page, group;
    // index of (slot, key or value, head) in units of tokens of one head
    __device__ __forceinline__ size_t token(long long slot, int kv, int head) const {
        const long long p = slot / page;
        return (static_cast<size_t>(p * 2 + kv) * heads + head) * page + static_cast<size_t>(slot - p * page);
    }
};

// One block: one token's key or value rows of all heads.
template <typename T>
__global__ void __launch_bounds__(256)
mx4_cache_append_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, const T* __restrict__ k,
                        const T* __restrict__ v, long long kst, long long ksh, long long vst, long long vsh,
                        const long long* __restrict__ slots, Mx4CacheShape c) {
    __shared__ float buf[256];
    griddep_wait();
    griddep_launch_dependents();
    const int t = blockIdx.x, kv = blockIdx.y;
    const long long slot = slots[t];
    if (slot < 0 || slot >= c.slots) return;
    const int lane = threadIdx.x & 31;
    for (int h = 0; h < c.heads; ++h) {
        const T* src = kv ? v + t * vst + h * vsh : k + t * kst + h * ksh;
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < c.d) buf[threadIdx.x] = mx4_to_f32(src[threadIdx.x]);
        __syncthreads();
        mx4_rotate_shared(buf, c.d, c.group, threadIdx.x, 256);
        const int b = threadIdx.x >> 5;
        if (b < c.d / 32) {
            const float a = buf[threadIdx.x];
            const uint32_t amax = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(a) & 0x7FFFFFFFu);
            const uint32_t e = mx4_scale_byte(__uint_as_float(amax));
            const float y = a * mx4_inv_scale(e);
            const float hi = __shfl_down_sync(0xFFFFFFFFu, y, 1);
            const size_t tok = c.token(slot, kv, h);
            if (!(lane & 1)) codes[tok * (c.d / 2) + threadIdx.x / 2] = e == 255u ? 0 : static_cast<uint8_t>(mx4_encode2(y, hi));
            if (lane == 0) scales[tok * (c.d / 32) + b] = static_cast<uint8_t>(e);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256)
mx4_cache_read_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                      const long long* __restrict__ slots, T* __restrict__ k, T* __restrict__ v, Mx4CacheShape c) {
    __shared__ float buf[256];
    griddep_wait();
    griddep_launch_dependents();
    const int t = blockIdx.x, kv = blockIdx.y, i = threadIdx.x;
    const long long slot = slots[t];
    const bool held = slot >= 0 && slot < c.slots;
    for (int h = 0; h < c.heads; ++h) {
        __syncthreads();
        if (i < c.d) {
            float val = 0.0f;
            if (held) {
                const size_t tok = c.token(slot, kv, h);
                const uint32_t code = (codes[tok * (c.d / 2) + i / 2] >> (4 * (i & 1))) & 15u;
                val = mx4_code_value(code) * mx4_scale_value(scales[tok * (c.d / 32) + i / 32]);
            }
            buf[i] = val;
        }
        __syncthreads();
        mx4_rotate_shared(buf, c.d, c.group, i, 256);
        if (i < c.d) (kv ? v : k)[(static_cast<size_t>(t) * c.heads + h) * c.d + i] = mx4_from_f32<T>(buf[i]);
    }
}

}  // namespace convrot
