"""GPU tests of the attention of a tree of drafted tokens over the MX4 cache, against 64 bits.

Tolerance. Rotated queries are held to 2^-22 (two terms) after the rotation's 2^-21 in fp32: scores move
by `reach` 2^-20 at most, reach = scale * sum |q||k|, and a weight relatively by twice that. Weights are
held to 2^-16, exp2 and the sums lose 2^-16 more, so the mean of rotated values is off by
sum p |v| (reach 2^-18 + 2^-15); the rotation back sums a group's errors over sqrt(G); then half a step.
"""
import numpy as np
import pytest
import torch

from oracle import mx4_oracle as orc

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def mx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import _int4
    assert _int4.is_available()
    return _int4


def make_cache(mx, lens, page, hkv, d, group, seed, spread=1.0):
    """(codes, scales, table): the sequences' tokens on pages anywhere; values of mixed magnitudes with `spread`."""
    each = max(1, -(-max(max(lens), 1) // page))
    pages = len(lens) * each + 1
    g = torch.Generator().manual_seed(seed)
    codes, scales = mx.mx4_cache_empty(pages, page, hkv, d)
    k = torch.randn(pages * page, hkv, d, generator=g)
    k[..., 3] *= 8
    v = torch.randn(pages * page, hkv, d, generator=g) * spread ** torch.randn(pages * page, 1, 1, generator=g)
    mx.convrot_mx4_cache_append(codes, scales, k.cuda(), v.cuda(), torch.arange(pages * page, device="cuda"), group)
    table = torch.randperm(pages, generator=g)[: len(lens) * each].reshape(len(lens), each).int().cuda()
    return codes, scales, table


def trees(b, t, seed):
    g = torch.Generator().manual_seed(seed)
    parents = [[int(torch.randint(-1, j, (), generator=g)) if j else -1 for j in range(t)] for _ in range(b)]
    return torch.tensor(parents).reshape(b, t)


def reference(q, codes, scales, table, lens, nodes, mask, scale, group):
    """(out, slack) in 64 bits: per sequence, node and head."""
    c, e = orc.unpack(codes.cpu().numpy()), scales.cpu().numpy()
    page, hkv, d = c.shape[3], c.shape[2], c.shape[4]
    qn = orc.rotate64(q.double().cpu().numpy(), group)
    b, t, hq, _ = qn.shape
    out, err = np.zeros(qn.shape), np.zeros(qn.shape)
    per = hq // hkv
    tab, mk = table.cpu().numpy(), mask.cpu().numpy()
    for i in range(b):
        n = max(0, min(int(lens[i]), tab.shape[1] * page))
        m = max(0, min(int(nodes[i]), t))
        at = tab[i, np.arange(n) // page]
        held = (at >= 0) & (at < c.shape[0])
        at = np.where(held, at, 0)
        k = orc.decode(c[at, 0, :, np.arange(n) % page], e[at, 0, :, np.arange(n) % page])
        v = orc.decode(c[at, 1, :, np.arange(n) % page], e[at, 1, :, np.arange(n) % page])
        for x in range(m):
            node = np.arange(n) - (n - m)
            row = mk[i, x] if mk.ndim == 3 else mk[x]
            seen = held & ((node < 0) | row[np.clip(node, 0, t - 1)])
            if not seen.any():
                continue
            kk, vv = k[seen], v[seen]
            s = np.einsum("hgd,nhd->hgn", qn[i, x].reshape(hkv, per, d), kk) * scale
            reach = np.einsum("hgd,nhd->hgn", np.abs(qn[i, x]).reshape(hkv, per, d), np.abs(kk)).max(-1) * abs(scale)
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            out[i, x] = np.einsum("hgn,nhd->hgd", p, vv).reshape(hq, d)
            err[i, x] = (np.einsum("hgn,nhd->hgd", p, np.abs(vv)) * (reach * 2.0 ** -18 + 2.0 ** -15)[..., None]).reshape(hq, d)
    if group:
        err = np.repeat(err.reshape(-1, group).sum(-1), group).reshape(err.shape) / group ** 0.5
    return orc.rotate64(out, group), err


def check(out, ref, q):
    want, err = ref
    step = torch.finfo(q.dtype)
    assert out.shape == q.shape and out.dtype == q.dtype
    got = out.double().cpu().numpy()
    slack = err + np.abs(want) * step.eps / 2 * 1.001 + step.smallest_normal * step.eps
    assert (np.abs(got - want) <= slack).all(), float((np.abs(got - want) - slack).max())


CASES = [  # lens, nodes (None: all), t, hq, hkv, D, page, group
    ([5], None, 1, 1, 1, 64, 16, 64), ([1], None, 1, 8, 2, 128, 16, 0), ([9, 700, 3], None, 3, 6, 2, 128, 64, 64),
    ([777], None, 8, 32, 8, 128, 64, 64), ([300, 0, 24, 131, 1], [24, 0, 24, 7, 1], 24, 6, 2, 64, 16, 64),
    ([64, 513], [20, 31], 31, 4, 4, 128, 32, 16), ([1030, 129, 128, 127], [40, 3, 40, 17], 40, 8, 2, 128, 16, 64),
    ([260, 60], [60, 60], 60, 3, 1, 256, 16, 256), ([2100], None, 64, 16, 2, 128, 64, 64), ([500, 257], [129, 130], 130, 2, 1, 64, 64, 0),
    ([4000, 10, 200], [70, 10, 70], 70, 4, 2, 64, 128, 16), ([50, 3], [0, 70000], 9, 20, 4, 128, 16, 64), ([6, 20, 33], [9, 9, 9], 9, 32, 2, 64, 1, 64),
    ([1500], None, 300, 1, 1, 128, 256, 64), ([900, 128, 1], [33, 33, 1], 33, 12, 3, 256, 64, 64),
    # enough rows and tokens for the kernel that takes 128 or 256 rows at a time
    ([1100, 0, 40, 1025], [40, 0, 40, 17], 40, 64, 2, 128, 64, 64), ([1200, 1, 700], [16, 1, 9], 16, 64, 8, 128, 16, 16),
    ([900, 1300], None, 150, 64, 8, 64, 128, 64), ([1200, 1281, 31], [30, 29, 30], 30, 32, 8, 64, 16, 0), ([1290, 640], None, 17, 128, 8, 128, 1, 64),
    ([1153, 1152, 1151], [65, 64, 3], 65, 16, 2, 128, 2, 0), ([1400, 129], [128, 128], 128, 16, 8, 64, 4, 16), ([2000, 1500], [257, 256], 257, 4, 2, 128, 256, 64)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_tree(mx, case, dtype):
    lens, nodes, t, hq, hkv, d, page, group = CASES[case]
    b = len(lens)
    codes, scales, table = make_cache(mx, lens, page, hkv, d, group, case)
    q = (torch.randn(b, t, hq, d, generator=torch.Generator().manual_seed(case)) * 1.5).to(DT[dtype]).cuda()
    mask = mx.tree_mask(trees(b, t, case))[0].cuda()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    m = None if nodes is None else torch.tensor(nodes, dtype=torch.int32, device="cuda")
    out = mx.convrot_mx4_tree_attention(q, codes, scales, table, n, mask, m, convrot_groupsize=group)
    nodes = nodes or [t] * b
    check(out, reference(q, codes, scales, table, lens, nodes, mask, d ** -0.5, group), q)
    for i in range(b):
        assert not out[i, nodes[i]:].any()                                        # padding
    again = mx.convrot_mx4_tree_attention(q, codes, scales, table, n, mask, m, convrot_groupsize=group)
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))


@pytest.mark.parametrize("t,hq,hkv,d", [(4, 8, 2, 128), (48, 8, 2, 128), (150, 3, 3, 64), (40, 64, 2, 128), (16, 64, 8, 128), (150, 64, 8, 64), (30, 32, 8, 64)])
def test_any_mask(mx, t, hq, hkv, d):
    """Masks that are no trees: rows that see nothing of a sequence without context, forward references, one mask for all,
    views with strides."""
    lens, nodes = [t, 500 if hq < 32 else 1200, t - 1], [t, t, t]
    codes, scales, table = make_cache(mx, lens, 16, hkv, d, 64, t)
    q = torch.randn(3, t, hq, d, generator=torch.Generator().manual_seed(t)).bfloat16().cuda()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    mask = (torch.rand(t, t, generator=torch.Generator().manual_seed(1)) < 0.3).cuda()
    mask[1] = False
    out = mx.convrot_mx4_tree_attention(q, codes, scales, table, n, mask)
    # (a sequence shorter than its nodes: the first node does not exist)
    ref = reference(q[:2], codes, scales, table[:2], lens[:2], nodes[:2], mask, d ** -0.5, 64)
    check(out[:2], ref, q[:2])
    assert not out[0, 1].any() and out[1, 1].any()
    for wide in (mask.expand(3, t, t), mask.repeat(3, 1, 1), torch.cat((mask, mask), 1)[:, :t],
                 mask.t().contiguous().t(), mask.repeat_interleave(2, 0)[::2]):
        assert torch.equal(mx.convrot_mx4_tree_attention(q, codes, scales, table, n, wide).view(torch.int16), out.view(torch.int16))
    assert not mx.convrot_mx4_tree_attention(q[:1], codes, scales, table[:1], n[:1], torch.zeros_like(mask)).any()


def test_sequence_shorter_than_its_nodes(mx):
    """Nodes at negative positions do not exist, their columns of the mask are not looked at."""
    t, lens = 40, [25]
    codes, scales, table = make_cache(mx, lens, 16, 2, 128, 64, 3)
    q = torch.randn(1, t, 8, 128, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    mask = torch.ones(t, t, dtype=torch.bool, device="cuda").tril()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = mx.convrot_mx4_tree_attention(q, codes, scales, table, n, mask)
    chain = mx.convrot_mx4_attention(q, codes, scales, table, n)                  # a chain, the same rule
    assert not out[0, :15].any()
    # each is off by half a step of its own, eps / 2 of the value at most: eps together
    near = (out.float() - chain.float()).abs() <= torch.finfo(out.dtype).eps * chain.float().abs() * 1.01 + 2.0 ** -12
    assert near.all()


@pytest.mark.parametrize("t,hq", [(6, 4), (60, 8), (60, 64)])
def test_strides_scale_lengths_and_bad_pages(mx, t, hq):
    lens = [90, 64] if hq < 64 else [1500, 1000]
    codes, scales, table = make_cache(mx, lens, 16, 2, 64, 64, 4)
    qkv = torch.randn(2, t, 3, hq, 64, generator=torch.Generator().manual_seed(1)).half().cuda()
    q = qkv[:, :, 1]
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    mask = torch.ones(t, t, dtype=torch.bool, device="cuda").tril()
    out = mx.convrot_mx4_tree_attention(q, codes, scales, table, n, mask, softmax_scale=0.3)
    check(out, reference(q, codes, scales, table, lens, [t, t], mask, 0.3, 64), q)
    odd = torch.zeros(q.numel() + 1, dtype=torch.float16, device="cuda")[1:].reshape(q.shape)
    odd.copy_(q)
    assert torch.equal(mx.convrot_mx4_tree_attention(odd, codes, scales, table, n, mask, softmax_scale=0.3), out)
    for bad in (-1, codes.shape[0], 2 ** 31 - 1):
        tab = table.clone()
        tab[0, 1], tab[1, 3] = bad, bad
        got = mx.convrot_mx4_tree_attention(q, codes, scales, tab, n, mask)
        check(got, reference(q, codes, scales, tab, lens, [t, t], mask, 64 ** -0.5, 64), q)
        assert not mx.convrot_mx4_tree_attention(q, codes, scales, torch.full_like(table, bad), n, mask).any()
    cut = mx.convrot_mx4_tree_attention(q, codes, scales, table[:, :4].contiguous(), torch.tensor([900, -3], dtype=torch.int32, device="cuda"), mask)
    check(cut, reference(q, codes, scales, table[:, :4], [64, 0], [t, t], mask, 64 ** -0.5, 64), q)


@pytest.mark.parametrize("t,d,hq", [(5, 128, 4), (70, 128, 4), (70, 64, 4), (20, 256, 4), (70, 128, 128), (100, 64, 128)])
def test_nan_in_the_cache(mx, t, d, hq):
    """A NaN block of a key or a value reaches the nodes that see its token, and no others."""
    many = hq // 2
    lens = [200] if hq < 64 else [200 + 1040]
    codes, scales, table = make_cache(mx, lens, 16, 2, d, 0, 7)
    q = torch.randn(1, t, hq, d, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    mask = mx.tree_mask(trees(1, t, 5))[0].cuda()
    clean = mx.convrot_mx4_tree_attention(q, codes, scales, table, n, mask, convrot_groupsize=0)

    def at(j):
        return int(table[0, j // 16]), j % 16
    node, n0 = t // 2, lens[0]
    for kind, j in ((0, n0 - t + node), (1, n0 - t + node), (1, n0 - t)):
        held = scales.clone()
        p, o = at(j)
        held[p, kind, 1, o, 1] = 255
        out = mx.convrot_mx4_tree_attention(q, codes, held, table, n, mask, convrot_groupsize=0)
        sees = mask[0, :, j - (n0 - t)]
        bad = out.isnan()
        want = torch.zeros_like(bad)
        want[0, sees, many:, (slice(None) if kind == 0 else slice(32, 64))] = True
        assert torch.equal(bad, want), (kind, j)
        assert torch.equal(out[~want], clean[~want])
    held = scales.clone()                                                         # in the context: all nodes
    p, o = at(3)
    held[p, 1, 0, o, 0] = 255
    out = mx.convrot_mx4_tree_attention(q, codes, held, table, n, mask, convrot_groupsize=0)
    assert out[0, :, :many, :32].isnan().all() and int(out.isnan().sum()) == t * many * 32
    held = scales.clone()                                                         # behind the sequence: nobody
    held[at(n0)[0], :, :, at(n0)[1]:] = 255
    assert torch.equal(mx.convrot_mx4_tree_attention(q, codes, held, table, n, mask, convrot_groupsize=0), clean)


@pytest.mark.parametrize("t,d,hq", [(5, 128, 4), (70, 128, 4), (70, 64, 4), (50, 128, 64), (60, 64, 64)])
@pytest.mark.parametrize("spread", [30.0, 1e4])
def test_values_and_keys_of_mixed_magnitudes(mx, t, d, hq, spread):
    lens = [333, 150] if hq < 64 else [1333, 150]
    codes, scales, table = make_cache(mx, lens, 16, 2, d, 64, 11, spread)
    q = (torch.randn(2, t, hq, d, generator=torch.Generator().manual_seed(3)) * 4).bfloat16().cuda()
    mask = mx.tree_mask(trees(2, t, 6))[0].cuda()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = mx.convrot_mx4_tree_attention(q, codes, scales, table, n, mask)
    check(out, reference(q, codes, scales, table, lens, [t, t], mask, d ** -0.5, 64), q)


@pytest.mark.parametrize("t,hq", [(8, 8), (64, 8), (64, 32)])
def test_streams_and_graphs(mx, t, hq):
    """A captured call replayed with other tables, lengths and masks, and two graphs at once on two streams."""
    lens = [3000, 700]
    codes, scales, table = make_cache(mx, lens, 64, 2, 128, 64, 8)
    g = torch.Generator().manual_seed(4)
    qs = [torch.randn(2, t, hq, 128, generator=g).bfloat16().cuda() for _ in range(2)]
    mask = mx.tree_mask(trees(2, t, 6))[0].cuda()
    n, m = torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.tensor([t, t - 1], dtype=torch.int32, device="cuda")
    call = lambda q: mx.convrot_mx4_tree_attention(q, codes, scales, table, n, mask, m)      # noqa: E731
    call(qs[0])
    graphs, outs = [], []
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(q))
        graphs.append(graph)
    n.copy_(torch.tensor([1000, 650]))
    m.copy_(torch.tensor([t // 2, t]))
    mask.copy_(mask.flip(0))
    want = [call(q) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(4):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(outs, want))


@pytest.mark.parametrize("t,d,hq", [(6, 128, 4), (50, 128, 64), (60, 64, 64)])
def test_keys_far_apart_and_scores_that_grow(mx, t, d, hq):
    """Keys of one tile whose scales lie more than 2^23 apart, and scores that rise from tile to tile, so that the
    reference moves and what was summed gets a new scale."""
    lens = [1300]
    codes, scales, table = make_cache(mx, lens, 16, 2, d, 64, 21)
    j = torch.arange(lens[0])
    slots = (table[0].cpu().long()[j // 16] * 16 + j % 16).cuda()
    k, v = mx.convrot_mx4_cache_read(codes, scales, slots, torch.float32, 64)
    k = k * (0.02 * 1.003 ** j.cuda())[:, None, None]                             # 0.02 .. 1: a row's largest score moves up and up
    k[::7] *= 2.0 ** -40
    mx.convrot_mx4_cache_append(codes, scales, k, v, slots, 64)
    q = (torch.randn(1, t, hq, d, generator=torch.Generator().manual_seed(3)) * 20).bfloat16().cuda()
    mask = mx.tree_mask(trees(1, t, 6))[0].cuda()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = mx.convrot_mx4_tree_attention(q, codes, scales, table, n, mask)
    check(out, reference(q, codes, scales, table, lens, [t], mask, d ** -0.5, 64), q)
    back = mx.convrot_mx4_tree_attention(q, codes, scales, table, n, mask, softmax_scale=-0.05)
    check(back, reference(q, codes, scales, table, lens, [t], mask, -0.05, 64), q)
    flat = mx.convrot_mx4_tree_attention(q, codes, scales, table, n, mask, softmax_scale=0.0)
    check(flat, reference(q, codes, scales, table, lens, [t], mask, 0.0, 64), q)


@pytest.mark.parametrize("b,t,hq,hkv,d,longest", [(41, 20, 24, 8, 64, 1000), (23, 24, 64, 8, 128, 1000), (481, 33, 8, 1, 64, 200), (64, 64, 8, 1, 64, 16384)])
def test_the_order_of_a_ragged_batch_does_not_matter(mx, b, t, hq, hkv, d, longest):
    """More blocks than multiprocessors (sequences go by their lengths, up to 480 of them; the last batch's long ones are split,
    the others stay whole): lengths that are the same, zero,
    negative and beyond the table; each sequence's result is the same wherever it stands, in a replayed graph of other lengths too."""
    g = torch.Generator().manual_seed(b)
    lens = torch.randint(0, longest + 1, (b,), generator=g, dtype=torch.int32)
    lens[0], lens[1], lens[2], lens[3:6], lens[6] = longest, 0, -5, 77, 2 ** 31 - 1
    nodes = torch.randint(0, t + 1, (b,), generator=g, dtype=torch.int32)
    codes, scales, table = make_cache(mx, [longest] * b, 16, hkv, d, 64, b)
    q = torch.randn(b, t, hq, d, generator=g).bfloat16().cuda()
    mask = mx.tree_mask(trees(b, t, b))[0].cuda()
    n, m = lens.cuda(), nodes.cuda()
    out = mx.convrot_mx4_tree_attention(q, codes, scales, table, n, mask, m)
    some = [0, 1, 2, 3, 4, 6, b // 2, b - 1] if longest < 2000 else [0, 1, 3, b // 2]
    held = [min(max(int(lens[i]), 0), table.shape[1] * 16) for i in some]
    check(out[some], reference(q[some], codes, scales, table[some], held, nodes[some], mask[some], d ** -0.5, 64), q[some])
    order = torch.randperm(b, generator=g).cuda()
    turned = mx.convrot_mx4_tree_attention(q[order].contiguous(), codes, scales, table[order].contiguous(), n[order].contiguous(), mask[order].contiguous(), m[order].contiguous())
    assert torch.equal(turned.view(torch.int16), out[order].view(torch.int16))
    live = n.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held_out = mx.convrot_mx4_tree_attention(q, codes, scales, table, live, mask, m)
    for now in (n, n.flip(0).contiguous(), torch.full_like(n, longest), torch.zeros_like(n)):
        live.copy_(now)
        graph.replay()
        assert torch.equal(held_out.view(torch.int16), mx.convrot_mx4_tree_attention(q, codes, scales, table, now, mask, m).view(torch.int16))
