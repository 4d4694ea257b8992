"""GPU test of the block operators together: a block that verifies drafted trees, in the order of its use.

The nodes on an accepted path see what the same tokens see as a chain, so their attention differs by the
order of sums and the roundings of weights alone (bf16 outputs: a step, 2^-8 relative to the mean); the output
projection quantizes it to 4 bits, where a value near a midpoint may then take the other code.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import _int4
    assert _int4.is_available()
    return _int4


def make_block(layers, hidden, heads, kv_heads, d, **how):
    torch.manual_seed(3)
    block = layers.Mx4SelfAttention(hidden, heads, kv_heads, d, device="cuda", **how)
    for lin in (block.qkv, block.out):
        made = layers.Mx4ConvRotLinear.from_linear(torch.nn.Linear(lin.in_features, lin.out_features, bias=False, device="cuda"))
        lin.weight, lin.weight_scale = made.weight, made.weight_scale
    return block


@pytest.mark.parametrize("d,sections,interleaved", [(64, None, False), (128, (8, 28, 28), True), (128, (32,), False)])
def test_tree_verification(lib, d, sections, interleaved):
    from _int4 import mx4_layers as layers
    from _int4.int8_eager import quantize_convrot_w8a8_weight
    from _int4.linear import Int4ConvRotLinear
    hidden, heads, kv = 512, 8, 2
    freqs = lib.rope_freqs(sections or d // 2)
    block = make_block(layers, hidden, heads, kv, d, freqs=freqs, sections=sections, interleaved=interleaved)
    up = Int4ConvRotLinear(hidden, 256, bias=False, device="cuda", mode="int8")
    q, s = quantize_convrot_w8a8_weight(torch.randn(256, hidden, device="cuda") * 0.02, up._qgs)
    up._q.copy_(q), up._qs.copy_(s)
    gain = torch.rand(hidden, device="cuda").bfloat16()

    def place(p):                                                 # positions on the block's axes: (t, 2t, 3t)
        p = torch.as_tensor(p, device="cuda")
        return torch.stack([p * (i + 1) for i in range(3)], -1) if sections and len(sections) == 3 else p

    prompts = [37, 5, 64]
    x = [torch.randn(n + 12, hidden, device="cuda").bfloat16() for n in prompts]
    parents = torch.tensor([[-1, 0, 0, 2, 1, 3, 5], [-1, -1, 1, 2, 3, 4, 0], [-1, 0, 1, 2, 3, 4, 5]])
    nodes = torch.tensor([7, 6, 3], dtype=torch.int32)
    paths = [[0, 2, 3, 5, 6], [1, 2, 3], [0, 1, 2]]
    mask, depth = lib.tree_mask(parents)
    drafted = torch.randn(3, 7, hidden, device="cuda").bfloat16()
    cache = layers.Mx4KVCache(64, kv, d, page=16)
    seqs = [cache.add() for _ in prompts]
    chain = [cache.add() for _ in prompts]
    for group in (seqs, chain):
        for seq, n, xs in zip(group, prompts, x):
            for at in range(0, n, 30):
                block.prefill(xs[at:min(n, at + 30)], cache, seq, place(torch.arange(at, min(n, at + 30))))
    # the trees of all sequences in one call, padded to seven nodes
    slots = torch.full((3, 7), -1, dtype=torch.int64)
    for i, seq in enumerate(seqs):
        slots[i, :nodes[i]] = torch.tensor(cache.extend(seq, int(nodes[i])))
    table, lens = cache.tables(seqs)
    pos = place((torch.tensor(prompts)[:, None] + depth).flatten()).reshape(3, 7, *([3] if sections and len(sections) == 3 else []))
    y = block(drafted, cache, slots.flatten().cuda(), table, lens, pos, mask.cuda(), nodes.cuda())
    out, hid = up.forward_rmsnorm(y, gain, drafted)
    assert torch.equal(hid, (y.float() + drafted.float()).bfloat16()) and out.shape == (3, 7, 256)
    for i, (seq, one) in enumerate(zip(seqs, chain)):
        path = paths[i]
        new = torch.tensor(cache.extend(one, len(path)), device="cuda")
        t1, l1 = cache.tables([one])
        want = block(drafted[None, i, path], cache, new, t1, l1, place(prompts[i] + torch.arange(len(path)))[None])[0]
        got = y[i, path]
        rel = float((got.double() - want.double()).norm() / want.double().norm())
        assert rel < 0.03, rel
        # accepted: the cache holds what the chain's holds, byte for byte
        cache.accept(seq, int(nodes[i]), path)
        a, b = (torch.tensor(cache.slots(z), device="cuda") for z in (seq, one))
        for t in (cache.codes, cache.scales):
            assert torch.equal(t[a // 16, :, :, a % 16], t[b // 16, :, :, b % 16])
    # and decodes on as the chain does
    nxt = torch.randn(3, 1, hidden, device="cuda").bfloat16()
    outs = []
    for group in (seqs, chain):
        sl = torch.tensor([cache.extend(z, 1)[0] for z in group], device="cuda")
        table, lens = cache.tables(group)
        p = place(lens.long() - 1)
        outs.append(block(nxt, cache, sl, table, lens, p[:, None]))
    assert torch.equal(outs[0], outs[1])


def test_a_captured_verification_step(lib):
    """Projection, append with positions, tree attention and output projection as one graph, replayed for other trees."""
    from _int4 import mx4_layers as layers
    block = make_block(layers, 256, 8, 2, 64, freqs=lib.rope_freqs(32))
    cache = layers.Mx4KVCache(64, 2, 64, page=16)
    seqs = [cache.add(), cache.add()]
    for seq, n in zip(seqs, (90, 33)):
        block.prefill(torch.randn(n, 256, device="cuda").bfloat16(), cache, seq)
    x = torch.randn(2, 5, 256, device="cuda").bfloat16()
    slots = torch.tensor([cache.extend(s, 5) for s in seqs], device="cuda").flatten()
    table, lens = cache.tables(seqs)
    mask, depth = (t.cuda() for t in lib.tree_mask([[-1, 0, 0, 1, 2], [-1, 0, 1, 2, 3]]))
    pos, nodes = (lens[:, None] - 5 + depth), torch.tensor([5, 5], dtype=torch.int32, device="cuda")
    call = lambda: block(x, cache, slots, table, lens, pos, mask, nodes)         # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    x.copy_(torch.randn_like(x))
    mask.copy_(mask.flip(0)), pos.copy_(pos.flip(0)), nodes.copy_(torch.tensor([5, 2]))
    graph.replay()
    got = out.clone()
    held = cache.codes.clone()
    assert torch.equal(got, call()) and torch.equal(held, cache.codes)
