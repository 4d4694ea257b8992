"""What needs no GPU of the block operators: refusals before any launch, tree masks, the cache's bookkeeping."""
import ctypes

import pytest
import torch

import _int4
from _int4 import cuda_loader
from _int4.mx4_layers import Mx4KVCache, Mx4SelfAttention


@pytest.fixture(scope="module")
def lib():
    return cuda_loader.library()


def refuse(lib, rc, text):
    assert rc == -1
    assert text in lib.ck_convrot_last_error(), lib.ck_convrot_last_error()


def sections(*n):
    return (ctypes.c_int * len(n))(*n)


def rope(lib, x=16, dtype=1, out=16, b=1, t=4, h=2, d=64, pos=16, kind=1, freqs=16, sec=(32,), axes=None):
    axes = len(sec) if axes is None else axes
    return lib.ck_rope(x, dtype, 0, 128, 64, out, b, t, h, d, pos, kind, 0, 1, 0, freqs, sections(*sec), axes, 0, 0, None)


def test_rope_refusals(lib):
    for how, text in ((dict(dtype=3), b"dtype"), (dict(d=63), b"even"), (dict(d=0), b"even"), (dict(t=-1), b"negative"), (dict(sec=(20, 13)), b"more pairs"),
                      (dict(sec=(33,)), b"more pairs"), (dict(sec=(-1, 5)), b"negative"), (dict(sec=(1,) * 9), b"1 to 8 axes"), (dict(axes=0), b"1 to 8 axes"),
                      (dict(kind=3), b"positions must be"), (dict(x=0), b"null"), (dict(out=0), b"null"), (dict(pos=0), b"null positions"),
                      (dict(freqs=0), b"null positions"), (dict(x=17), b"aligned"), (dict(out=15), b"aligned"), (dict(pos=20), b"aligned"),
                      (dict(freqs=20), b"aligned"), (dict(b=2 ** 31 - 1, t=2 ** 31 - 1, h=2 ** 31 - 1), b"too large")):
        refuse(lib, rope(lib, **how), text)
    assert rope(lib, t=0, x=0) == 0 and rope(lib, h=0, x=0) == 0 and rope(lib, b=0) == 0


def append(lib, codes=16, pages=4, heads=2, d=64, page=16, group=64, q=16, k=16, v=16, dtype=1, hq=4, q_out=16, slots=16, t=3, sec=(32,)):
    return lib.ck_mx4_cache_append_rope(codes, 16, pages, heads, d, page, group, q, k, v, dtype, hq, 256, 64, 128, 64, 128, 64, q_out, slots, t,
                                        16, 1, 1, 0, 16, sections(*sec), len(sec), 0, None)


def test_append_rope_refusals(lib):
    for how, text in ((dict(d=96), b"head dimension"), (dict(group=256), b"multiple of G"), (dict(page=48), b"power of two"), (dict(heads=0), b"heads"),
                      (dict(codes=24), b"aligned"), (dict(dtype=5), b"dtype"), (dict(t=-1), b"negative"), (dict(hq=-1), b"negative"), (dict(k=0), b"null"),
                      (dict(slots=0), b"null"), (dict(q=0), b"null"), (dict(q_out=0), b"null"), (dict(v=17), b"aligned"), (dict(slots=20), b"aligned"),
                      (dict(q_out=17), b"aligned"), (dict(sec=(33,)), b"more pairs"), (dict(t=2 ** 31 - 1, heads=64), b"too many tokens"),
                      (dict(t=2 ** 31 - 1, heads=1, hq=2), b"too many tokens")):
        refuse(lib, append(lib, **how), text)
    assert append(lib, t=0, k=0) == 0


def tree(lib, q=16, dtype=1, pages=8, page=16, table=16, ld=4, per=4, lens=16, nodes=16, mask=16, seq=16, row=4, out=16, b=1, t=4, hq=4, hkv=2, d=64,
         group=64, work=0, size=0):
    return lib.ck_mx4_tree_attention(q, dtype, 1, 1, 1, 16, 16, pages, page, table, ld, per, lens, nodes, mask, seq, row, out, b, t, hq, hkv, d, group,
                                     ctypes.c_float(1.0), work, size, None)


def test_tree_attention_refusals(lib):
    for how, text in ((dict(dtype=0), b"queries must be"), (dict(hq=3), b"multiple"), (dict(t=0), b"multiple"), (dict(b=-1), b"multiple"), (dict(ld=3), b"table"),
                      (dict(per=2 ** 26, ld=2 ** 26, page=64), b"block table longer"), (dict(seq=-1), b"mask strides"), (dict(row=-4), b"mask strides"),
                      (dict(mask=0), b"null"), (dict(lens=0), b"null"), (dict(out=0), b"null"), (dict(q=17), b"aligned"), (dict(nodes=18), b"aligned"),
                      (dict(out=24), b"aligned"), (dict(b=2 ** 20, t=2 ** 10, hq=4), b"too many query rows"), (dict(d=100), b"head dimension"),
                      (dict(pages=2 ** 28, page=16, hkv=2), b"2^32")):
        refuse(lib, tree(lib, **how), text)
    assert tree(lib, b=0) == 0
    need = lib.ck_mx4_tree_attention_workspace_size(1, 64, 16, 2, 128, 65536)
    assert need > 0
    refuse(lib, tree(lib, t=64, hq=16, d=128, per=1024, ld=1024, page=64, pages=2000, work=256, size=need - 1), b"workspace smaller")
    refuse(lib, tree(lib, t=64, hq=16, d=128, per=1024, ld=1024, page=64, pages=2000, work=128, size=need), b"256-byte")


def norm(lib, x=16, r=16, dtype=1, ldx=256, ldr=256, gain=16, gtype=1, w=16, ws=16, bias=16, btype=1, hidden=16, out=16, otype=1, m=3, n=8, k=256, group=256,
         work=256, size=1 << 20):
    return lib.ck_convrot_w8a8_linear_rmsnorm(x, r, dtype, ldx, ldr, gain, gtype, ctypes.c_float(1e-6), w, ws, bias, btype, hidden, out, otype, m, n, k, group,
                                              work, size, None)


def test_rmsnorm_linear_refusals(lib):
    for how, text in ((dict(m=-1), b">= 0"), (dict(k=0), b"K > 0"), (dict(dtype=3), b"dtype"), (dict(group=0), b"G must"), (dict(group=32), b"G must"),
                      (dict(k=320), b"multiple of G"), (dict(k=16384 + 256, ldx=20000, ldr=20000), b"16384"), (dict(otype=2), b"out_dtype"), (dict(gtype=4), b"norm_dtype"),
                      (dict(btype=-1), b"bias_dtype"), (dict(ldx=255), b"strides"), (dict(ldr=100), b"strides"), (dict(x=0), b"null"), (dict(hidden=0), b"null"),
                      (dict(w=0), b"null"), (dict(ws=0), b"null"), (dict(out=0), b"null"), (dict(x=17), b"aligned"), (dict(r=17), b"aligned"),
                      (dict(hidden=24), b"16-byte"), (dict(w=24), b"16-byte"), (dict(out=24), b"16-byte"), (dict(gain=17), b"aligned"), (dict(bias=17), b"aligned"),
                      (dict(ws=18), b"aligned"), (dict(work=0), b"workspace"), (dict(work=128), b"256-byte"), (dict(size=100), b"smaller")):
        refuse(lib, norm(lib, **how), text)
    assert norm(lib, m=0, x=0) == 0


def test_cpu_tensors_and_shapes_are_value_errors():
    freqs, x = torch.ones(32, dtype=torch.float64), torch.zeros(3, 2, 64)
    pos = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        _int4.apply_rope(x, pos, freqs)
    for bad, text in ((dict(freqs=freqs.float()), "float64"), (dict(freqs=torch.ones(33, dtype=torch.float64)), "do not fit"), (dict(positions=pos.double()), "int32"),
                      (dict(positions=pos[:2]), "positions"), (dict(sections=(16, 15)), "add up"), (dict(sections=(16, 16)), "positions"),
                      (dict(sections=()), "1 to 8"), (dict(x=x[..., :63]), "even"), (dict(x=x[0, 0]), "heads"), (dict(x=x.double()), "dtype"),
                      (dict(positions=pos[:, None].expand(3, 2)), "positions")):
        with pytest.raises(ValueError, match=text):
            _int4.apply_rope(**{**dict(x=x, positions=pos, freqs=freqs), **bad})
    with pytest.raises(TypeError):
        _int4.apply_rope(x, pos, freqs, sections=3)
    codes, scales = _int4.mx4_cache_empty(2, 16, 2, 64, device="cpu")
    q, k, slots = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int64)
    for bad, text in ((dict(k=k[:, :1]), "keys"), (dict(v=k.half()), "keys"), (dict(q=q.half()), "queries"), (dict(q=q[:2]), "queries"), (dict(slots=slots.int()), "slots"),
                      (dict(slots=slots[:2]), "slots"), (dict(positions=pos[:2]), "positions"), (dict(convrot_groupsize=32), "convrot_groupsize"), (dict(), "CUDA")):
        with pytest.raises(ValueError, match=text):
            _int4.convrot_mx4_cache_append_rope(**{**dict(codes=codes, scales=scales, q=q, k=k, v=k, slots=slots, positions=pos, freqs=freqs), **bad})
    q, table, lens, mask = torch.zeros(1, 3, 4, 64).half(), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.ones(3, 3, dtype=torch.bool)
    for bad, text in ((dict(tree_mask=mask.int()), "bool"), (dict(tree_mask=mask[:2]), "tree_mask"), (dict(tree_mask=mask.expand(2, 3, 3)), "tree_mask"),
                      (dict(tree_lens=lens.long()), "tree_lens"), (dict(tree_lens=torch.ones(2, dtype=torch.int32)), "tree_lens"), (dict(q=q.float()), "queries"),
                      (dict(q=q[:, :, :3]), "multiple"), (dict(block_table=table.long()), "block_table"), (dict(seq_lens=lens.long()), "seq_lens"), (dict(), "CUDA")):
        with pytest.raises(ValueError, match=text):
            _int4.convrot_mx4_tree_attention(**{**dict(q=q, codes=codes, scales=scales, block_table=table, seq_lens=lens, tree_mask=mask), **bad})
    x, w, ws = torch.zeros(3, 256), torch.zeros(8, 256, dtype=torch.int8), torch.ones(8)
    for bad, text in ((dict(qweight=w.int()), "int8"), (dict(x=x[:, :128]), "match"), (dict(wscales=ws[:4]), "wscales"), (dict(convrot_groupsize=0), "groupsize"),
                      (dict(bias=ws.double()), "bias"), (dict(norm_weight=ws), "norm_weight"), (dict(residual=x[:2]), "residual"), (dict(residual=x.half()), "residual"),
                      (dict(), "CUDA")):
        with pytest.raises(ValueError, match=text):
            _int4.convrot_w8a8_linear_rmsnorm(**{**dict(x=x, qweight=w, wscales=ws), **bad})


def test_tree_mask():
    mask, depth = _int4.tree_mask([-1, 0, 0, 2, -1, 3])
    names = [[0], [0, 1], [0, 2], [0, 2, 3], [4], [0, 2, 3, 5]]
    assert depth.tolist() == [0, 1, 1, 2, 0, 3]
    assert [torch.nonzero(row).flatten().tolist() for row in mask] == names
    both, depths = _int4.tree_mask(torch.tensor([[-1, 0, 1], [-1, -1, -1]], dtype=torch.int32))
    assert both.shape == (2, 3, 3) and depths.tolist() == [[0, 1, 2], [0, 0, 0]]
    assert torch.equal(both[0], torch.ones(3, 3, dtype=torch.bool).tril()) and torch.equal(both[1], torch.eye(3, dtype=torch.bool))
    for bad in ([0], [-1, 1], [-2], [[-1, 2, 0]]):
        with pytest.raises(ValueError, match="parent"):
            _int4.tree_mask(bad)
    for bad in (torch.zeros(3), torch.zeros(1, 1, 1, dtype=torch.int64)):
        with pytest.raises(ValueError, match="whole numbers"):
            _int4.tree_mask(bad)


def test_rope_freqs():
    f = _int4.rope_freqs((2, 3), theta=100.0, device="cpu")
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 0.1, 1.0, 100 ** (-1 / 3), 100 ** (-2 / 3)], dtype=torch.float64))
    assert _int4.rope_freqs(0, device="cpu").numel() == 0
    for bad in ((), (-1,)):
        with pytest.raises(ValueError):
            _int4.rope_freqs(bad, device="cpu")


def test_accept_moves_the_kept_nodes_and_gives_pages_back():
    cache = Mx4KVCache(6, 1, 64, page=4, device="cpu")
    other, seq = cache.add(), cache.add()
    cache.extend(other, 3)
    cache.extend(seq, 6)
    new = cache.extend(seq, 9)                                    # nodes 0 .. 8
    codes = torch.randint(0, 255, cache.codes.shape, dtype=torch.uint8)
    scales = torch.randint(0, 255, cache.scales.shape, dtype=torch.uint8)
    cache.codes.copy_(codes), cache.scales.copy_(scales)
    at = lambda t, s: t[s // 4, :, :, s % 4]                      # noqa: E731
    kept, held = [1, 2, 5, 7], cache.slots(seq)[:6]
    cache.accept(seq, 9, kept)
    assert cache.length(seq) == 10 and cache.slots(seq)[:6] == held and len(cache._pages[seq]) == 3 and len(cache._free) == 2
    for i, node in enumerate(kept):
        assert torch.equal(at(cache.codes, cache.slots(seq)[6 + i]), at(codes, new[node]))
        assert torch.equal(at(cache.scales, cache.slots(seq)[6 + i]), at(scales, new[node]))
    for s in held + cache.slots(other):
        assert torch.equal(at(cache.codes, s), at(codes, s))
    cache.accept(seq, 4, [])
    assert cache.length(seq) == 6 and len(cache._pages[seq]) == 2
    for nodes, bad in ((7, [0]), (3, [3]), (3, [1, 1]), (3, [2, 0]), (3, [-1]), (-1, [])):
        with pytest.raises(ValueError, match="kept nodes"):
            cache.accept(seq, nodes, bad)
    cache.free(seq), cache.free(other)
    assert sorted(cache._free) == list(range(6))


def test_block_positions_that_do_not_fit():
    freqs = _int4.rope_freqs(32, device="cpu")
    plain = Mx4SelfAttention(64, 2, 1, 64, device="cpu")
    turned = Mx4SelfAttention(64, 2, 1, 64, device="cpu", freqs=freqs)
    axes = Mx4SelfAttention(64, 2, 1, 64, device="cpu", freqs=freqs, sections=(8, 24))
    pos = torch.arange(5)
    for block, given, text in ((plain, pos, "without frequencies"), (turned, pos[:4], "expected"), (turned, pos.double(), "expected"), (axes, pos, "expected"), (axes, None, "needs")):
        cache = Mx4KVCache(4, 1, 64, page=16, device="cpu")
        seq = cache.add()
        with pytest.raises(ValueError, match=text):
            block.prefill(torch.zeros(5, 64), cache, seq, given)
        assert cache.length(seq) == 0
    assert "freqs" not in turned.state_dict()


def test_block_positions_of_other_orders_and_a_cast_block():
    freqs = _int4.rope_freqs(32, device="cpu")
    turned = Mx4SelfAttention(64, 2, 1, 64, device="cpu", freqs=freqs)
    axes = Mx4SelfAttention(64, 2, 1, 64, device="cpu", freqs=freqs, sections=(8, 24))
    assert torch.equal(turned._positions(torch.arange(6).view(2, 3), 2, 3), torch.arange(6))
    assert axes._positions(torch.zeros(2, 3, 2), 2, 3).shape == (6, 2) and axes._positions(torch.zeros(6, 2), 2, 3).shape == (6, 2)
    # as many numbers, but not in the tokens' order
    for block, bad in ((turned, torch.zeros(3, 2)), (axes, torch.zeros(2, 6)), (axes, torch.zeros(2, 2, 3)), (axes, torch.zeros(12))):
        with pytest.raises(ValueError, match="expected"):
            block._positions(bad, 2, 3)
    with pytest.raises(ValueError, match="frequencies on"):
        turned._positions(torch.zeros(6, device="meta"), 2, 3)
    for cast in (turned.half(), turned.to(torch.bfloat16), turned.float()):
        assert cast.freqs.dtype == torch.float64 and torch.equal(cast.freqs, freqs)
    with pytest.raises(ValueError, match="tree_mask"):            # (before anything is written)
        turned(torch.zeros(1, 2, 64), None, None, None, None, torch.arange(2), tree_lens=torch.ones(1, dtype=torch.int32))
