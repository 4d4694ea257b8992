// Writing new tokens to the paged MX4 cache with their positions: queries and keys are
// turned (rope.cuh), keys and values rotated and quantized (mx4_cache.cuh).
//
// Included by rope.cu. A warp's task is up to 32 units of keys, as many of values or as many
// values of queries. The lanes read 16-byte chunks, pairs in one lane, and turn them in
// fp32; queries go out, keys and values are laid down in shared memory as fp32 units, of which
// each lane then has one, as in the append without positions: the same codes for the same
// fp32 values. A lane's chunk stays the same from head to head, so a token's angles are
// computed once for all of its heads.
//
// 32768 tokens of 8 heads of 128 in bf16, keys alone: 52 us (2.9 TB/s; issue 54 % of the cycles: angles,
// the turn, the rotation and the codes); 7 tokens of 32 query heads on 8: 5.5 us in a graph, one
// task's latency. Blocks are not kept for several tasks: a wave that counts on three blocks a
// multiprocessor has fewer where it starts under the kernel before it.
#pragma once

namespace convrot {

struct Mx4AppendRope {
    const void *q, *k, *v;
    void* q_out;
    long long qst, qsh, kst, ksh, vst, vsh;        // token and head strides in elements
    const long long* slots;
    uint8_t *codes, *scales;
    int tokens, hq, units;                         // units of the keys
    int size, k_tasks, v_tasks, tasks;             // units of a task, tasks of the keys, of the values, of all
};

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

template <typename T, int D, int G, int VP>
__global__ void __launch_bounds__(kMx4QuantWarps * 32, 3)
mx4_cache_append_rope_kernel(const __grid_constant__ Mx4AppendRope a, Mx4CacheShape c, const __grid_constant__ RopeArgs r) {
    constexpr int kChunks = D / (2 * VP), kRuns = kChunks < 32 ? 32 / kChunks : 1, kAhead = 4;
    extern __shared__ __align__(128) unsigned char mx4slabs[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned char* slab = mx4slabs + warp * Mx4Slab<float>::kBytes;
    const int per = mx4_cache_units<D>(c.heads);                  // units of a token
    const int task = static_cast<int>(blockIdx.x) * kMx4QuantWarps + warp;
    griddep_wait();
    griddep_launch_dependents();
    if (task >= a.tasks) return;
    const int kind = task < a.k_tasks ? 0 : task < a.k_tasks + a.v_tasks ? 1 : 2;  // keys, values, queries
    const int base = (task - (kind > 0 ? a.k_tasks : 0) - (kind > 1 ? a.v_tasks : 0)) * a.size;      // the first unit
    const T* src = static_cast<const T*>(kind == 0 ? a.k : kind == 1 ? a.v : a.q);
    const long long st = kind == 0 ? a.kst : kind == 1 ? a.vst : a.qst, sh = kind == 0 ? a.ksh : kind == 1 ? a.vsh : a.qsh;
    // heads of a token, and with the missing one of heads of 64 whose last unit is half
    const int held = kind == 2 ? a.hq : c.heads, heads = kind != 2 && D == 64 ? 2 * per : held;
    const int items = a.size * 128 / D, share = (items + kRuns - 1) / kRuns;      // heads of the task, of a lane
    const int first = static_cast<int>(static_cast<long long>(base) * 128 / D);
    #pragma unroll 1
    for (int u = lane % kChunks; u < kChunks; u += 32) {
        const RopePlace<VP> at(r, D, u, kind != 1);               // (values are not turned)
        const int from = lane / kChunks * share, count = min(share, items - from);
        int t = (first + from) / heads, h = first + from - t * heads, known = -1;
        RopeCoef<VP> w;
        #pragma unroll 1
        for (int i0 = 0; i0 < count; i0 += kAhead) {
            RopeRaw<T, VP> ra[kAhead], rb[kAhead];
            const int t0 = t, h_first = h;
            #pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                if (i0 + i < count && t < a.tokens && h < held) {
                    const T* p = src + t * st + h * sh;
                    ra[i].load(p + at.a);
                    rb[i].load(p + at.b);
                } else {
                    ra[i].zero();
                    rb[i].zero();
                }
                if (++h == heads) { h = 0; ++t; }
            }
            int ti = t0, hi = h_first;
            #pragma unroll 1
            for (int i = 0; i < kAhead; ++i) {
                // (rolled, the next item moved up: a short program, which a small call has to fetch)
                if (i0 + i < count && ti < a.tokens && at.any() && ti != known) {
                    w.load(r, 0, ti, at);
                    known = ti;
                }
                float fa[VP], fb[VP];
                ra[0].get(fa);
                rb[0].get(fb);
                if (at.any()) rope_turn<VP>(fa, fb, w, at, r.interleaved);
                if (i0 + i < count) {
                    if (kind == 2) {
                        if (ti < a.tokens) {
                            T* to = static_cast<T*>(a.q_out) + (static_cast<long long>(ti) * a.hq + hi) * D;
                            if (at.any()) ra[0].put(fa);
                            if (at.pair_b >= 0) rb[0].put(fb);
                            ra[0].store(to + at.a);
                            rb[0].store(to + at.b);
                        }
                    } else {
                        slab_put<D, VP>(slab, from + i0 + i, at.a, fa);
                        slab_put<D, VP>(slab, from + i0 + i, at.b, fb);
                    }
                }
                #pragma unroll
                for (int k = 0; k + 1 < kAhead; ++k) {
                    ra[k] = ra[k + 1];
                    rb[k] = rb[k + 1];
                }
                if (++hi == heads) { hi = 0; ++ti; }
            }
        }
    }
    if (kind == 2) return;
    __syncwarp();
    // (lanes beyond a small task's units have what the slab happens to hold, and store nothing)
    float2 val[64];
    slab_to_unit<float>(slab, val);
    unit_rotate<G>(val);
    uint4 codes[4];
    const uint32_t word = unit_quantize(val, unit_factor<G>(), codes);
    const int mine = lane ^ (G == 256 ? 1 : 0), u = base + mine;
    const Mx4CacheUnit<D> at(kind ? u + a.units : u, per, c.heads, 2 * a.units);
    cache_store_unit<D>(a.codes, a.scales, c, mine < a.size && u < a.units ? a.slots[at.t] : -1, at, codes, word);
}

}  // namespace convrot
