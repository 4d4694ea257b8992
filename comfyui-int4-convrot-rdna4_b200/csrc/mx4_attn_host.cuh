// Host side of the attention over the MX4 cache: how a call is cut, and its launches.
#pragma once

#include <algorithm>

#include "mx4_attn.cuh"
#include "mx4_host.cuh"

namespace convrot {

// How an attention call is cut: tiles of query rows (one sequence and cache head
// each) and splits of the sequences.
struct AttnPlan {
    long long tiles;
    int tile_rows, row_tiles, splits;
    bool clustered;                // a sequence's splits are one cluster and join themselves
    size_t partials() const { return splits > 1 && !clustered ? static_cast<size_t>(tiles) * splits * tile_rows : 0; }
};

// With tiles of `tile_rows` of a cache head's `rows`.
inline AttnPlan attn_plan_rows(int B, long long rows, int tile_rows, int hkv, int d, long long longest) {
    AttnPlan p;
    p.tile_rows = tile_rows;
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

inline AttnPlan attn_plan(int B, int tq, int hq, int hkv, int d, long long longest) {
    const long long rows = static_cast<long long>(tq) * (hq / hkv);
    return attn_plan_rows(B, rows, rows <= 8 ? 8 : rows <= 16 || d == 256 ? 16 : 32, hkv, d, longest);
}

template <typename T, int D, int NT, bool TREE>
int launch_attention(const Mx4AttnArgs& a, const AttnPlan& p, cudaStream_t stream) {
    using Cfg = Mx4AttnCfg<D, NT>;
    auto kernel = mx4_attn_kernel<T, D, NT, TREE>;
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

template <typename T, int D, bool TREE>
int launch_attention_rows(const Mx4AttnArgs& a, const AttnPlan& p, cudaStream_t stream) {
    if (p.tile_rows == 8) return launch_attention<T, D, 1, TREE>(a, p, stream);
    if constexpr (D < 256 && !TREE)
        if (p.tile_rows == 32) return launch_attention<T, D, 4, TREE>(a, p, stream);
    return launch_attention<T, D, 2, TREE>(a, p, stream);
}

template <typename T, bool TREE>
int run_attention(const Mx4AttnArgs& a, int d, const AttnPlan& p, cudaStream_t stream) {
    if (d == 256) return launch_attention_rows<T, 256, TREE>(a, p, stream);
    if (d == 128) return launch_attention_rows<T, 128, TREE>(a, p, stream);
    return launch_attention_rows<T, 64, TREE>(a, p, stream);
}

}  // namespace convrot
