// Writing new tokens to the paged MX4 cache with their positions: queries and keys are
// turned (rope.cuh), keys and values rotated and quantized (mx4_cache.cuh).
//
// Included by rope.cu. A warp's task is 32 units of keys, 32 units of values or as many
// values of queries. Keys and values: the lanes read 16-byte chunks, pairs in one lane,
// turn the keys in fp32 and lay 32 units down in shared memory as fp32; then a lane has a
// unit, as in the append without positions, and gives the same codes for the same fp32
// values. A lane's chunk stays the same from head to head, so a token's angles are
// computed once for all of its heads.
#pragma once

namespace convrot {

struct Mx4AppendRope {
    const void *q, *k, *v;
    void* q_out;
    long long qst, qsh, kst, ksh, vst, vsh;        // token and head strides in elements
    const long long* slots;
    uint8_t *codes, *scales;
    int tokens, hq, units;                         // units of the keys
    int kv_tasks, tasks;                           // tasks of the keys (and of the values), of all
    int wide;                                      // 16-byte chunks (rows aligned, sections of whole chunks)
};

// Items (heads of D channels, token by token) first .. first + kItems of a task, `heads` a
// token of which `held` exist; `sink(item, place, raw a, raw b)` or, for turned keys, floats.
template <typename T, int D, int VP, typename Sink>
__device__ __forceinline__ void rope_items(const T* src, long long st, long long sh, int tokens, int heads, int held, long long first,
                                           bool turn, const RopeArgs& r, Sink sink) {
    constexpr int kItems = 32 * 128 / D, kChunks = D / (2 * VP), kRuns = kChunks < 32 ? 32 / kChunks : 1, kPer = kItems / kRuns;
    constexpr int kAhead = 4;
    const int lane = threadIdx.x & 31;
    #pragma unroll 1
    for (int u = lane % kChunks; u < kChunks; u += 32) {
        RopePlace<VP> at(r, u);
        if (!turn && !r.interleaved) {                            // (values lie in a row of chunks: no pairs)
            at.a = 2 * VP * u;
            at.b = at.a + VP;
        }
        if (!turn) at.pair = -1;
        const int from = lane / kChunks * kPer;
        int t = static_cast<int>((first + from) / heads), h = static_cast<int>((first + from) % heads), known = -1;
        RopeCoef<VP> w;
        #pragma unroll 1
        for (int i0 = 0; i0 < kPer; i0 += kAhead) {
            RopeRaw<T, VP> ra[kAhead], rb[kAhead];
            int it[kAhead], ih[kAhead];
            #pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                it[i] = t;
                ih[i] = h;
                if (t < tokens && h < held) {
                    const T* p = src + t * st + h * sh;
                    ra[i].load(p + at.a);
                    rb[i].load(p + at.b);
                } else {
                    ra[i].zero();
                    rb[i].zero();
                }
                if (++h == heads) { h = 0; ++t; }
            }
            #pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                float fa[VP], fb[VP];
                ra[i].get(fa);
                rb[i].get(fb);
                if (at.pair >= 0 && it[i] < tokens) {
                    if (it[i] != known) {
                        w.load(r, 0, it[i], at.pair);
                        known = it[i];
                    }
                    rope_turn<VP>(fa, fb, w, r.interleaved);
                }
                sink(from + i0 + i, it[i], ih[i], at, fa, fb);
            }
        }
    }
}

// Lays item `item`'s channels [c, c + VP) into the slab of 32 fp32 units.
template <int D, int VP>
__device__ __forceinline__ void slab_put(unsigned char* slab, int item, int c, const float (&f)[VP]) {
    const int value = item * D + c, unit = value / kMx4Unit, in = value % kMx4Unit;
    if constexpr (VP == 1) {
        *reinterpret_cast<float*>(slab + Mx4Slab<float>::offset(unit, in / 4) + in % 4 * 4) = f[0];
    } else {
        #pragma unroll
        for (int j = 0; j < VP; j += 4)
            *reinterpret_cast<float4*>(slab + Mx4Slab<float>::offset(unit, in / 4 + j / 4)) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
    }
}

template <typename T, int D, int G>
__global__ void __launch_bounds__(kMx4QuantWarps * 32, 3)
mx4_cache_append_rope_kernel(Mx4AppendRope a, Mx4CacheShape c, RopeArgs r) {
    constexpr int kWide = 16 / static_cast<int>(sizeof(T));
    extern __shared__ __align__(128) unsigned char mx4slabs[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned char* slab = mx4slabs + warp * Mx4Slab<float>::kBytes;
    const int per = mx4_cache_units<D>(c.heads);                  // units of a token
    const int padded = D == 64 ? 2 * per : c.heads;               // heads of a token with the missing one of its last unit
    griddep_wait();
    griddep_launch_dependents();
    #pragma unroll 1
    for (int task = static_cast<int>(blockIdx.x) * kMx4QuantWarps + warp; task < a.tasks; task += static_cast<int>(gridDim.x) * kMx4QuantWarps) {
        if (task >= 2 * a.kv_tasks) {                             // queries
            const long long first = static_cast<long long>(task - 2 * a.kv_tasks) * (32 * 128 / D);
            auto sink = [&](auto vp, int t, int h, auto& at, auto& fa, auto& fb) {
                constexpr int VP = decltype(vp)::value;
                if (t >= a.tokens) return;
                T* to = static_cast<T*>(a.q_out) + (static_cast<long long>(t) * a.hq + h) * D;
                RopeRaw<T, VP> o;
                o.put(fa);
                o.store(to + at.a);
                o.put(fb);
                o.store(to + at.b);
            };
            const T* q = static_cast<const T*>(a.q);
            if (a.wide) rope_items<T, D, kWide>(q, a.qst, a.qsh, a.tokens, a.hq, a.hq, first, true, r,
                [&](int, int t, int h, auto& at, auto& fa, auto& fb) { sink(std::integral_constant<int, kWide>{}, t, h, at, fa, fb); });
            else rope_items<T, D, 1>(q, a.qst, a.qsh, a.tokens, a.hq, a.hq, first, true, r,
                [&](int, int t, int h, auto& at, auto& fa, auto& fb) { sink(std::integral_constant<int, 1>{}, t, h, at, fa, fb); });
            continue;
        }
        const bool value = task >= a.kv_tasks;
        const int base = (value ? task - a.kv_tasks : task) * 32;
        const T* src = static_cast<const T*>(value ? a.v : a.k);
        const long long st = value ? a.vst : a.kst, sh = value ? a.vsh : a.ksh, first = static_cast<long long>(base) * 128 / D;
        if (a.wide) rope_items<T, D, kWide>(src, st, sh, a.tokens, padded, c.heads, first, !value, r,
            [&](int item, int, int, auto& at, auto& fa, auto& fb) {
                slab_put<D, kWide>(slab, item, at.a, fa);
                slab_put<D, kWide>(slab, item, at.b, fb);
            });
        else rope_items<T, D, 1>(src, st, sh, a.tokens, padded, c.heads, first, !value, r,
            [&](int item, int, int, auto& at, auto& fa, auto& fb) {
                slab_put<D, 1>(slab, item, at.a, fa);
                slab_put<D, 1>(slab, item, at.b, fb);
            });
        __syncwarp();
        float2 val[64];
        slab_to_unit<float>(slab, val);
        unit_rotate<G>(val);
        uint4 codes[4];
        const uint32_t word = unit_quantize(val, unit_factor<G>(), codes);
        const int u = (base + lane) ^ (G == 256 ? 1 : 0);
        const Mx4CacheUnit<D> at(value ? u + a.units : u, per, c.heads, 2 * a.units);
        cache_store_unit<D>(a.codes, a.scales, c, u < a.units ? a.slots[at.t] : -1, at, codes, word);
        __syncwarp();
    }
}

}  // namespace convrot
