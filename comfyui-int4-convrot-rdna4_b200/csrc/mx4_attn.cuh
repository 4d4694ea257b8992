// Attention of the newest tokens' queries over the paged MX4 cache.
//
// Included by mx4.cu. One block a query row: the row is rotated like the cached
// keys, each warp walks every eighth token with a running maximum and sum (a
// lane holds D / 32 channels), the warps' partial results are joined and the
// output is rotated back.
#pragma once

namespace convrot {

struct Mx4AttnArgs {
    const void* q;
    long long qsb, qst, qsh;       // strides of the query in elements: sequence, token, head
    const uint8_t* codes;
    const uint8_t* scales;
    const int* table;              // [B, table_ld] page numbers
    long long table_ld;
    int table_pages;               // pages a table row holds
    const int* lens;
    void* out;
    int B, tq, hq, hkv, d, page, pages, group;
    float scale;
};

template <typename T>
__global__ void __launch_bounds__(256) mx4_attn_kernel(Mx4AttnArgs a) {
    __shared__ float buf[256];
    __shared__ float part[8][256];
    __shared__ float pm[8], pl[8];
    griddep_wait();
    griddep_launch_dependents();
    const int row = blockIdx.x;
    const int h = row % a.hq, t = row / a.hq % a.tq, b = row / a.hq / a.tq;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int hk = h / (a.hq / a.hkv);
    const T* q = static_cast<const T*>(a.q) + b * a.qsb + t * a.qst + h * a.qsh;
    if (tid < a.d) buf[tid] = mx4_to_f32(q[tid]);
    __syncthreads();
    mx4_rotate_shared(buf, a.d, a.group, tid, 256);
    const int cap = static_cast<int>(min(static_cast<long long>(a.table_pages) * a.page, 0x7FFFFFFFll));
    const int n = min(a.lens[b], cap) - a.tq + t + 1;     // tokens this row sees
    const int per = a.d / 32;
    float m = -INFINITY, l = 0.0f, o[8] = {};
    for (int j = warp; j < n; j += 8) {
        const int page = a.table[b * a.table_ld + j / a.page];
        if (page < 0 || page >= a.pages) continue;
        const size_t kt = ((static_cast<size_t>(page) * 2) * a.hkv + hk) * a.page + j % a.page;
        const size_t vt = kt + static_cast<size_t>(a.hkv) * a.page;
        float s = 0.0f;
        for (int i = 0; i < per; ++i) {
            const int c = lane * per + i;
            const uint32_t code = (a.codes[kt * (a.d / 2) + c / 2] >> (4 * (c & 1))) & 15u;
            s += buf[c] * mx4_code_value(code) * mx4_scale_value(a.scales[kt * per + c / 32]);
        }
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, x);
        s *= a.scale;
        const float mn = fmaxf(m, s);
        const float f = __expf(m - mn), p = __expf(s - mn);
        m = mn;
        l = l * f + p;
        for (int i = 0; i < per; ++i) {
            const int c = lane * per + i;
            const uint32_t code = (a.codes[vt * (a.d / 2) + c / 2] >> (4 * (c & 1))) & 15u;
            o[i] = o[i] * f + p * mx4_code_value(code) * mx4_scale_value(a.scales[vt * per + c / 32]);
        }
    }
    for (int i = 0; i < per; ++i) part[warp][lane * per + i] = o[i];
    if (lane == 0) { pm[warp] = m; pl[warp] = l; }
    __syncthreads();
    if (tid < a.d) {
        float top = -INFINITY;
        for (int w = 0; w < 8; ++w) top = fmaxf(top, pm[w]);
        float sum = 0.0f, acc = 0.0f;
        for (int w = 0; w < 8; ++w) {
            const float f = pl[w] > 0.0f ? __expf(pm[w] - top) : 0.0f;
            sum += f * pl[w];
            acc += f * part[w][tid];
        }
        buf[tid] = sum > 0.0f ? acc / sum : 0.0f;
    }
    __syncthreads();
    mx4_rotate_shared(buf, a.d, a.group, tid, 256);
    if (tid < a.d)
        static_cast<T*>(a.out)[((static_cast<size_t>(b) * a.tq + t) * a.hq + h) * a.d + tid] = mx4_from_f32<T>(buf[tid]);
}

}  // namespace convrot
