"""GPU tests of the MX4 operators against plain implementations in 64 bits.

Tolerances. Quantization and the cache are determined bit for bit by the fp32
rotation's order, so codes, scales and read-back values are compared exactly
with a restatement in that order; against the 64-bit rotation a code may differ
only where the value lies within the rotation's rounding error of a midpoint
(12 roundings of 2^-24, each of at most the group's sum of magnitudes over
sqrt(G)). The linear's products are exact; its fp32 sums lose at most one unit
2^-23 of the sum of magnitudes for each of the K / 32 partial sums, plus the
output's rounding. Attention rounds the rotated queries and the probabilities
to 11 bits: scores move by at most 2^-11 of scale * sum |q||k|, which moves a
probability by twice that relatively.
"""
import math

import numpy as np
import pytest
import torch

from oracle import mx4_oracle as orc

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
UNIT = {"bf16": 2.0 ** -9, "f16": 2.0 ** -12, "f32": 2.0 ** -25}      # half the largest relative rounding error: above its root mean square


@pytest.fixture(scope="module")
def mx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import _int4
    assert _int4.is_available()
    return _int4


def rows(m, k, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g)
    x[:, torch.randperm(k, generator=g)[:max(1, k // 100)]] *= 20
    return x.to(DT[dtype]).cuda()


def f64(t):
    return t.detach().double().cpu().numpy()


def check_quantized(mx, x, group):
    m, k = x.reshape(-1, x.shape[-1]).shape
    codes, scales = mx.quantize_convrot_mx4(x, group)
    torch.cuda.synchronize()
    assert codes.shape == (*x.shape[:-1], k // 2)
    got_c = orc.unpack(codes.reshape(m, k // 2).cpu().numpy())
    tiles = scales.cpu().numpy()
    got_e = orc.untile(tiles, m, k)
    x32 = x.reshape(m, k).float().cpu().numpy()
    want_c, want_e = orc.quantize(x32, group)
    assert np.array_equal(got_e, want_e)
    assert np.array_equal(orc.decode(got_c, got_e), orc.decode(want_c, want_e), equal_nan=True)
    full = tiles.reshape(tiles.shape[0], tiles.shape[1], 32, 4, 4).transpose(0, 3, 2, 1, 4)
    full = full.reshape(tiles.shape[0] * 128, -1)
    assert not full[m:].any() and not full[:, k // 32:].any()              # padding is written
    return got_c, got_e, x32


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m,k,group", [
    (1, 32, 0), (1, 32, 16), (3, 96, 16), (5, 160, 0), (129, 64, 64), (2, 256, 256), (127, 768, 256), (33, 1088, 64),
    (128, 1024, 256), (300, 3840, 256), (7, 15360, 64), (1, 4096, 16), (65, 1280, 256), (17, 2080, 16)])
def test_quantize_bit_exact(mx, m, k, group, dtype):
    x = rows(m, k, dtype, seed=m * 7 + k + group)
    c, e, x32 = check_quantized(mx, x, group)
    y = orc.rotate64(x32, group)
    c64, e64 = orc.encode(y)
    if not group:
        assert np.array_equal(e, e64) and np.array_equal(orc.decode(c, e), orc.decode(c64, e64))
        return
    slack = 12 * 2.0 ** -24 * np.repeat(np.abs(x32.astype(np.float64)).reshape(m, -1, group).sum(-1), group, -1) / math.sqrt(group)
    err = np.abs(orc.decode(c, e) - y)
    best = np.abs(orc.decode(c64, e64) - y)
    same_scale = np.repeat(e == e64, 32, -1)
    assert (np.abs(err - best)[same_scale] <= 2 * slack[same_scale]).all()
    assert (~same_scale).mean() < 1e-3


def test_quantize_special_blocks(mx):
    x = torch.randn(9, 512, generator=torch.Generator().manual_seed(1))
    x[0] = 0.0
    x[1] = 1e-40
    x[2, 5] = float("inf")
    x[3, 70] = float("nan")
    x[4] = 3e38
    x[5] *= 1e-38
    x[6] = -0.0
    x[7, ::3] = 6.0
    x[8] = torch.arange(512) / 64.0 - 4
    for dt in ("f32", "bf16"):
        check_quantized(mx, x.to(DT[dt]).cuda(), 0)
        check_quantized(mx, x[[0, 2, 3, 5, 6, 7, 8]].to(DT[dt]).cuda(), 256)


def test_quantize_strided_and_unaligned_rows(mx):
    base = torch.randn(40, 1000, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    for x in (base[:, 3:3 + 512], base[::2, 8:8 + 256], base[:, 100:356].t().contiguous().t()):
        c, s = mx.quantize_convrot_mx4(x, 64)
        c2, s2 = mx.quantize_convrot_mx4(x.clone(memory_format=torch.contiguous_format), 64)
        assert torch.equal(c, c2) and torch.equal(s, s2)
    x3 = base[:, :768].reshape(5, 8, 768)
    c, s = mx.quantize_convrot_mx4(x3, 256)
    assert c.shape == (5, 8, 384)


@pytest.mark.parametrize("out", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m,k,group", [(1, 32, 0), (3, 96, 16), (130, 1088, 64), (33, 3840, 256), (5, 15360, 0)])
def test_dequantize(mx, m, k, group, out):
    x = rows(m, k, "bf16", seed=m + k)
    codes, scales = mx.quantize_convrot_mx4(x, group)
    v = orc.decode(orc.unpack(codes.cpu().numpy()), orc.untile(scales.cpu().numpy(), m, k))
    for g in {0, group}:
        got = mx.dequantize_convrot_mx4(codes, scales, g, DT[out])
        want = torch.from_numpy(orc.rotate(v.astype(np.float32), g)).to(DT[out])
        assert torch.equal(got.cpu(), want)


def test_empty_inputs(mx):
    x = torch.empty(0, 256, dtype=torch.bfloat16, device="cuda")
    c, s = mx.quantize_convrot_mx4(x, 256)
    assert c.shape == (0, 128) and s.shape == (0, 2, 512)
    assert mx.dequantize_convrot_mx4(c, s).shape == (0, 256)
    w, ws = mx.quantize_convrot_mx4(torch.randn(64, 256, device="cuda"), 256)
    assert mx.convrot_mx4_linear(x, w, ws).shape == (0, 64)


def check_linear(mx, m, n, k, group, dtype, bias, seed, x=None):
    x = rows(m, k, dtype, seed) if x is None else x
    g = torch.Generator().manual_seed(seed + 1)
    w = (torch.randn(n, k, generator=g) * 0.02).cuda()
    b = (torch.randn(n, generator=g) * 0.01).to(DT[bias]).cuda() if bias else None
    qw, ws = mx.quantize_convrot_mx4(w, group)
    out = mx.convrot_mx4_linear(x, qw, ws, b, convrot_groupsize=group)
    assert out.shape == (m, n) and out.dtype == DT[dtype]
    sel = torch.arange(m) if m <= 300 else torch.unique(torch.cat([torch.randint(0, m, (200,), generator=g), torch.tensor([0, m - 1])]))
    qx, xs = mx.quantize_convrot_mx4(x, group)
    xv = mx.dequantize_convrot_mx4(qx, xs, 0, torch.float32)[sel.cuda()].double()
    wv = mx.dequantize_convrot_mx4(qw, ws, 0, torch.float32).double()
    ref = xv @ wv.t()
    mag = xv.abs() @ wv.abs().t()
    if b is not None:
        ref = ref + b.double()
        mag = mag + b.double().abs()
    tol = (k // 32 + 2) * 2.0 ** -23 * mag + 1.01 * UNIT[dtype] * 2 * ref.abs() + 2.0 ** -25
    err = (out[sel.cuda()].double() - ref).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    # a random walk of the same roundings: the whole matrix is far nearer than the bound
    rel = float(err.norm() / ref.norm())
    assert rel <= UNIT[dtype] * 1.2 + math.sqrt(k / 32) * 2.0 ** -22, rel


@pytest.mark.parametrize("m,n,k,group,dtype,bias", [
    (1, 1, 32, 0, "bf16", None), (1, 64, 64, 64, "bf16", "bf16"), (2, 130, 96, 16, "f16", "f32"), (3, 257, 160, 0, "f32", "f16"),
    (16, 1000, 512, 256, "bf16", "bf16"), (17, 72, 4096, 64, "bf16", None), (64, 384, 1088, 64, "f16", "f16"),
    (65, 129, 288, 16, "bf16", "f32"), (127, 513, 768, 256, "bf16", None), (128, 256, 256, 256, "f32", "f32"),
    (129, 255, 1280, 256, "bf16", "bf16"), (255, 120, 2304, 256, "f16", None), (256, 512, 3840, 256, "bf16", "bf16"),
    (300, 1111, 544, 16, "bf16", "bf16"), (513, 640, 4096, 256, "f16", "f16"), (1, 15360, 3840, 256, "bf16", "bf16"),
    (4, 3840, 15360, 256, "bf16", None), (33, 2048, 7680, 256, "bf16", "bf16"), (777, 3001, 992, 0, "bf16", "f16"),
    (1024, 2304, 1536, 256, "f32", "f32"), (2500, 1792, 1024, 64, "bf16", "bf16"), (4097, 4104, 640, 64, "bf16", "f16")])
def test_linear(mx, m, n, k, group, dtype, bias):
    check_linear(mx, m, n, k, group, dtype, bias, seed=m + n + k)


def test_linear_strided_input_and_other_stream(mx):
    base = rows(50, 1200, "bf16", 3)
    check_linear(mx, 50, 320, 512, 64, "bf16", "bf16", 4, x=base[:, 7:7 + 512])
    w, ws = mx.quantize_convrot_mx4(torch.randn(256, 1024, device="cuda") * 0.02, 256)
    x = rows(70, 1024, "bf16", 5)
    want = mx.convrot_mx4_linear(x, w, ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mx.convrot_mx4_linear(x.reshape(2, 35, 1024), w, ws)
    side.synchronize()
    assert torch.equal(got.reshape(70, 256), want)


def test_linear_repeats_and_rows_are_independent(mx):
    """The same bits every time, and a row's result does not change with non-finite neighbours."""
    w, ws = mx.quantize_convrot_mx4(torch.randn(520, 2048, device="cuda") * 0.02, 256)
    for m in (5, 40, 300):
        x = rows(m, 2048, "bf16", m)
        want = mx.convrot_mx4_linear(x, w, ws)
        for _ in range(3):
            assert torch.equal(mx.convrot_mx4_linear(x, w, ws), want)
        y = x.clone()
        y[m // 2, 9] = float("nan")
        got = mx.convrot_mx4_linear(y, w, ws)
        keep = torch.arange(m, device="cuda") != m // 2
        assert torch.equal(got[keep], want[keep])
        assert bool(got[m // 2].isnan().all())


def test_linear_in_a_graph(mx):
    w, ws = mx.quantize_convrot_mx4(torch.randn(512, 1024, device="cuda") * 0.02, 256)
    x = rows(200, 1024, "bf16", 8)
    want = mx.convrot_mx4_linear(x, w, ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mx.convrot_mx4_linear(x, w, ws)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


# --------------------------------------------------------------------- cache


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("t,heads,d,page,group", [
    (1, 1, 64, 16, 64), (1, 8, 128, 16, 64), (5, 3, 64, 1, 16), (33, 8, 128, 64, 64), (100, 2, 256, 32, 256), (17, 5, 256, 128, 0),
    (257, 4, 64, 16, 0), (1000, 8, 128, 64, 16)])
def test_cache_append_and_read(mx, t, heads, d, page, group, dtype):
    g = torch.Generator().manual_seed(t + d)
    pages = -(-t // page) + 3
    codes, scales = mx.mx4_cache_empty(pages, page, heads, d)
    qkv = rows(t, 3 * heads * d, dtype, t).reshape(t, 3, heads, d)
    k, v = qkv[:, 1], qkv[:, 2]                                           # strided views
    slots = torch.randperm(pages * page, generator=g)[:t].cuda()
    mx.convrot_mx4_cache_append(codes, scales, k, v, slots, group)
    kr, vr = mx.convrot_mx4_cache_read(codes, scales, slots, DT[dtype], group)
    for src, got, i in ((k, kr, 0), (v, vr, 1)):
        c, e = orc.quantize(src.float().cpu().numpy(), group)
        at, off = (slots // page).cpu().numpy(), (slots % page).cpu().numpy()
        held_c = orc.unpack(codes.cpu().numpy()[at, i, :, off])
        held_e = scales.cpu().numpy()[at, i, :, off]
        assert np.array_equal(held_e, e)
        assert np.array_equal(orc.decode(held_c, held_e), orc.decode(c, e))
        want = torch.from_numpy(orc.rotate(orc.decode(c, e).astype(np.float32), group)).to(DT[dtype])
        assert torch.equal(got.cpu(), want)
    written = torch.zeros(pages * page, dtype=torch.bool)
    written[slots.cpu()] = True
    rest = (~written).reshape(pages, page)
    assert not codes.cpu().transpose(2, 3).transpose(1, 2)[rest].any()    # no other slot was touched


def test_cache_skips_slots_outside_and_keeps_what_is_there(mx):
    codes, scales = mx.mx4_cache_empty(4, 16, 2, 64)
    k = rows(6, 128, "bf16", 0).reshape(6, 2, 64)
    slots = torch.tensor([0, -1, 63, 64, 1 << 40, 17], device="cuda")
    mx.convrot_mx4_cache_append(codes, scales, k, k * 2, slots, 64)
    kr, vr = mx.convrot_mx4_cache_read(codes, scales, slots, torch.float32, 64)
    for i in (1, 3, 4):
        assert not kr[i].any() and not vr[i].any()
    for i in (0, 2, 5):
        assert torch.equal(vr[i], 2 * kr[i]) and kr[i].any()
    before = codes.clone()
    mx.convrot_mx4_cache_append(codes, scales, k[:0], k[:0], slots[:0], 64)
    assert torch.equal(codes, before)
    kr, _ = mx.convrot_mx4_cache_read(codes, scales, slots[:0], torch.bfloat16, 64)
    assert kr.shape == (0, 2, 64)


def test_cache_non_finite_blocks(mx):
    codes, scales = mx.mx4_cache_empty(1, 16, 1, 128)
    k = torch.randn(3, 1, 128, generator=torch.Generator().manual_seed(0)).cuda()
    k[1, 0, 40] = float("inf")
    k[2, 0, 100] = float("nan")
    slots = torch.arange(3, device="cuda")
    mx.convrot_mx4_cache_append(codes, scales, k, k, slots, 0)
    kr, _ = mx.convrot_mx4_cache_read(codes, scales, slots, torch.float32, 0)
    assert bool(kr[0].isfinite().all())
    assert kr[1, 0].isnan().nonzero().flatten().tolist() == list(range(32, 64))
    assert kr[2, 0].isnan().nonzero().flatten().tolist() == list(range(96, 128))


# --------------------------------------------------------------------- attention


def make_cache(mx, lens, page, hkv, d, group, seed, per=None, vscale=1.0, poison=True):
    """A cache whose pages lie anywhere; every slot no sequence owns holds NaN blocks."""
    b = len(lens)
    g = torch.Generator().manual_seed(seed)
    per = max(1, max(-(-n // page) for n in lens)) if per is None else per
    pages = b * per + 2
    codes, scales = mx.mx4_cache_empty(pages, page, hkv, d)
    if poison:
        codes.fill_(0x73)
        scales.fill_(255)
    table = torch.randperm(pages, generator=g)[:b * per].reshape(b, per).int()
    ks, vs = [], []
    for i, n in enumerate(lens):
        k = torch.randn(n, hkv, d, generator=g)
        k[..., 3] *= 6
        v = torch.randn(n, hkv, d, generator=g) * vscale
        j = torch.arange(n)
        slots = table[i].long()[j // page] * page + j % page
        mx.convrot_mx4_cache_append(codes, scales, k.cuda(), v.cuda(), slots.cuda(), group)
        kv = []
        for which in (0, 1):
            held = codes.cpu().numpy()[(slots // page).numpy(), which, :, (slots % page).numpy()]
            he = scales.cpu().numpy()[(slots // page).numpy(), which, :, (slots % page).numpy()]
            kv.append(orc.decode(orc.unpack(held), he).reshape(n, hkv, d))
        ks.append(kv[0])
        vs.append(kv[1])
    return codes, scales, table.cuda(), ks, vs


def check_attention(q, out, ks, vs, lens, group, scale, dtype):
    ref, spread, reach = orc.attention64(orc.rotate64(f64(q), group), ks, vs, lens, scale)
    ref, got = orc.rotate64(ref, group), f64(out)
    assert np.isfinite(got).all()
    d = q.shape[-1]
    g = max(group, 1)
    # rotation back mixes a group's errors: at most their sum over sqrt(G)
    spread = np.repeat(spread.reshape(*spread.shape[:-1], d // g, g).sum(-1), g, -1) / math.sqrt(g)
    tol = (2 * 2.0 ** -11 * reach[..., None] + 2.0 ** -10) * spread + 2.02 * UNIT[dtype] * np.abs(ref) + 1e-7 * spread + 2.0 ** -25
    err = np.abs(got - ref)
    assert (err <= tol).all(), (err / tol).max()
    norm = np.linalg.norm(ref)
    if norm:
        assert np.linalg.norm(got - ref) / norm <= 1.2 * UNIT[dtype] + 2.0 ** -10
    return ref


CASES = [
    # lens, tq, hq, hkv, d, page, group
    ([1], 1, 1, 1, 64, 16, 64), ([7], 1, 8, 8, 128, 16, 64), ([16], 1, 8, 1, 128, 16, 64), ([17, 0, 1, 33], 1, 8, 2, 64, 16, 16),
    ([100, 3, 0, 257], 4, 8, 2, 128, 32, 64), ([5, 64, 65], 8, 12, 4, 128, 64, 0), ([300], 3, 6, 2, 256, 32, 256), ([31, 129], 1, 16, 1, 256, 128, 64),
    ([2, 1, 0], 4, 4, 4, 64, 1, 64), ([700, 12], 1, 64, 4, 128, 64, 64), ([515], 2, 32, 1, 64, 16, 16), ([1500, 1, 900], 1, 5, 5, 128, 16, 64),
    ([40, 90], 16, 8, 2, 128, 16, 64), ([3000], 1, 8, 2, 128, 64, 64), ([130], 33, 3, 1, 64, 32, 64)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(mx, case, dtype):
    lens, tq, hq, hkv, d, page, group = CASES[case]
    codes, scales, table, ks, vs = make_cache(mx, lens, page, hkv, d, group, case)
    q = (torch.randn(len(lens), tq, hq, d, generator=torch.Generator().manual_seed(case)) * 1.5).to(DT[dtype]).cuda()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = mx.convrot_mx4_attention(q, codes, scales, table, n, convrot_groupsize=group)
    check_attention(q, out, ks, vs, lens, group, d ** -0.5, dtype)
    for i, length in enumerate(lens):
        empty = max(0, tq - length)
        assert not out[i, :empty].any()
    again = mx.convrot_mx4_attention(q, codes, scales, table, n, convrot_groupsize=group)
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))


def test_attention_long_table_many_splits(mx):
    """A table far longer than the sequences (as a serving engine keeps it)."""
    lens = [2000, 5, 0, 64]
    codes, scales, table, ks, vs = make_cache(mx, lens, 16, 2, 128, 64, 3, per=125)
    wide = torch.full((4, 4096), -1, dtype=torch.int32, device="cuda")
    wide[:, :125] = table
    q = torch.randn(4, 1, 8, 128, generator=torch.Generator().manual_seed(9)).bfloat16().cuda()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = mx.convrot_mx4_attention(q, codes, scales, wide, n)
    check_attention(q, out, ks, vs, lens, 64, 128 ** -0.5, "bf16")


def test_attention_strides_scale_and_length_cut(mx):
    lens = [50, 20]
    codes, scales, table, ks, vs = make_cache(mx, lens, 16, 2, 64, 64, 4)
    qkv = torch.randn(2, 3, 3, 4, 64, generator=torch.Generator().manual_seed(1)).half().cuda()
    q = qkv[:, :, 1]                                                       # [2, 3, 4, 64], strided
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = mx.convrot_mx4_attention(q, codes, scales, table, n, softmax_scale=0.3)
    check_attention(q, out, ks, vs, lens, 64, 0.3, "f16")
    odd = torch.zeros(2 * 3 * 4 * 64 + 1, dtype=torch.float16, device="cuda")[1:].reshape(2, 3, 4, 64)
    odd.copy_(q)                                                           # rows not 16-byte aligned
    assert torch.equal(mx.convrot_mx4_attention(odd, codes, scales, table, n, softmax_scale=0.3), out)
    # a length beyond the table is cut to it; negative lengths see nothing
    cut = mx.convrot_mx4_attention(q[:1], codes, scales, table[:1, :2].contiguous(), torch.tensor([900], dtype=torch.int32, device="cuda"))
    check_attention(q[:1], cut, [ks[0][:32]], [vs[0][:32]], [32], 64, 64 ** -0.5, "f16")
    none = mx.convrot_mx4_attention(q, codes, scales, table, torch.tensor([-3, 0], dtype=torch.int32, device="cuda"))
    assert not none.any()


def test_attention_pages_outside_the_cache_are_hidden(mx):
    lens = [48]
    codes, scales, table, ks, vs = make_cache(mx, lens, 16, 1, 64, 64, 5)
    q = torch.randn(1, 1, 2, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for bad in (-1, codes.shape[0], 2 ** 31 - 1):
        t = table.clone()
        t[0, 1] = bad
        out = mx.convrot_mx4_attention(q, codes, scales, t, n)
        keep = np.r_[0:16, 32:48]
        check_attention(q, out, [ks[0][keep]], [vs[0][keep]], [32], 64, 64 ** -0.5, "bf16")
        all_bad = torch.full_like(table, bad)
        assert not mx.convrot_mx4_attention(q, codes, scales, all_bad, n).any()


@pytest.mark.parametrize("vscale", [1e-12, 1e-3, 1e5, 1e14])
def test_attention_value_magnitudes(mx, vscale):
    """Values far from 1 (the result keeps its relative precision; bf16 holds the range)."""
    lens = [200, 33]
    codes, scales, table, ks, vs = make_cache(mx, lens, 16, 2, 128, 64, 6, vscale=vscale)
    q = torch.randn(2, 1, 4, 128, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = mx.convrot_mx4_attention(q, codes, scales, table, n)
    check_attention(q, out.double() / vscale, ks, [v / vscale for v in vs], lens, 64, 128 ** -0.5, "bf16")


def test_attention_values_of_mixed_magnitudes(mx):
    """Tokens whose values differ by a factor of 10^6: the result is as near as its own sum of p |v|."""
    lens = [64]
    codes, scales, table, ks, vs = make_cache(mx, lens, 16, 1, 64, 64, 7)
    j = torch.arange(0, 64, 2)
    slots = (table[0].cpu().long()[j // 16] * 16 + j % 16).cuda()
    big = torch.randn(32, 1, 64, generator=torch.Generator().manual_seed(3)).cuda()
    kr, _ = mx.convrot_mx4_cache_read(codes, scales, slots, torch.float32, 64)
    mx.convrot_mx4_cache_append(codes, scales, kr, big * 1e6, slots, 64)
    for which, held in ((0, ks), (1, vs)):
        s = (table[0].cpu().long()[torch.arange(64) // 16] * 16 + torch.arange(64) % 16)
        c = codes.cpu().numpy()[(s // 16).numpy(), which, :, (s % 16).numpy()]
        e = scales.cpu().numpy()[(s // 16).numpy(), which, :, (s % 16).numpy()]
        held[0] = orc.decode(orc.unpack(c), e).reshape(64, 1, 64)
    q = torch.randn(1, 1, 4, 64, generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = mx.convrot_mx4_attention(q, codes, scales, table, n)
    check_attention(q, out, ks, vs, lens, 64, 0.125, "bf16")


@pytest.mark.parametrize("qscale", [1e-6, 1.0, 3e4])
def test_attention_query_magnitudes(mx, qscale):
    """Queries outside half precision's comfortable range (bf16 holds them)."""
    lens = [77]
    codes, scales, table, ks, vs = make_cache(mx, lens, 16, 1, 64, 16, 8)
    q = (torch.randn(1, 1, 4, 64, generator=torch.Generator().manual_seed(4)) * qscale).bfloat16().cuda()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = mx.convrot_mx4_attention(q, codes, scales, table, n, softmax_scale=0.1 / qscale, convrot_groupsize=16)
    check_attention(q, out, ks, vs, lens, 16, 0.1 / qscale, "bf16")


def test_attention_visible_nan_reaches_only_its_row(mx):
    lens = [30, 30]
    codes, scales, table, ks, vs = make_cache(mx, lens, 16, 1, 64, 0, 9)
    q = torch.randn(2, 1, 2, 64, generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = mx.convrot_mx4_attention(q, codes, scales, table, n, convrot_groupsize=0)
    scales[table[1, 1].long(), 1, 0, 2, 0] = 255                           # a value block of a token that is seen
    out = mx.convrot_mx4_attention(q, codes, scales, table, n, convrot_groupsize=0)
    assert torch.equal(out[0], want[0])
    assert bool(out[1, :, :, :32].isnan().all()) and torch.equal(out[1, :, :, 32:], want[1, :, :, 32:])


def test_refusals(mx):
    x = torch.randn(4, 64, device="cuda")
    c, s = mx.quantize_convrot_mx4(x, 64)
    cases = [
        lambda: mx.quantize_convrot_mx4(x.double(), 64), lambda: mx.quantize_convrot_mx4(x, 48), lambda: mx.quantize_convrot_mx4(x[:, :48], 16),
        lambda: mx.dequantize_convrot_mx4(c, s[:, :, :256]), lambda: mx.dequantize_convrot_mx4(c.int(), s),
        lambda: mx.dequantize_convrot_mx4(c, s, 256), lambda: mx.dequantize_convrot_mx4(c, s, 0, torch.int8),
        lambda: mx.convrot_mx4_linear(x[:, :32], c, s), lambda: mx.convrot_mx4_linear(x, c, s, torch.zeros(3, device="cuda"), 64),
        lambda: mx.convrot_mx4_linear(x, c, s, torch.zeros(4), 64), lambda: mx.convrot_mx4_linear(x, c, s.cpu(), None, 64)]
    codes, scales = mx.mx4_cache_empty(2, 16, 2, 64)
    kv = torch.zeros(3, 2, 64, device="cuda")
    slots = torch.zeros(3, dtype=torch.int64, device="cuda")
    q = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16, device="cuda")
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    lens = torch.ones(1, dtype=torch.int32, device="cuda")
    cases += [
        lambda: mx.convrot_mx4_cache_append(codes, scales, kv, kv[:2], slots), lambda: mx.convrot_mx4_cache_append(codes, scales, kv, kv, slots.int()),
        lambda: mx.convrot_mx4_cache_append(codes, scales, kv[..., :32], kv[..., :32], slots), lambda: mx.convrot_mx4_cache_append(codes, scales, kv, kv, slots, 256),
        lambda: mx.convrot_mx4_cache_read(codes, scales[:1], slots), lambda: mx.convrot_mx4_cache_read(codes, scales, slots, torch.int32),
        lambda: mx.convrot_mx4_attention(q.float(), codes, scales, table, lens), lambda: mx.convrot_mx4_attention(q[:, :, :3], codes, scales, table, lens),
        lambda: mx.convrot_mx4_attention(q, codes, scales, table.long(), lens), lambda: mx.convrot_mx4_attention(q, codes, scales, table, lens.long()),
        lambda: mx.convrot_mx4_attention(q[..., :32], codes, scales, table, lens), lambda: mx.convrot_mx4_attention(q, codes, scales, table, lens.cpu())]
    for i, call in enumerate(cases):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"refusal {i} was accepted")


@pytest.mark.parametrize("m,n,k,group,dtype,bias", [
    (333, 3840, 4096, 256, "bf16", "bf16"), (130, 520, 2080, 16, "f16", None), (257, 255, 4128, 0, "f32", "f32"), (500, 2049, 7680, 64, "bf16", "f16")])
def test_linear_few_tiles_long_k(mx, m, n, k, group, dtype, bias):
    """Sizes with few output tiles and a long K (the product may be split along K)."""
    check_linear(mx, m, n, k, group, dtype, bias, seed=m + n)
    w, ws = mx.quantize_convrot_mx4(torch.randn(n, k, device="cuda") * 0.02, group)
    x = rows(m, k, dtype, 1)
    want = mx.convrot_mx4_linear(x, w, ws, None, group)
    assert all(torch.equal(mx.convrot_mx4_linear(x, w, ws, None, group), want) for _ in range(3))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,nan_at", [([1, 1], 0), ([129, 129], 128), ([40, 40], 39), ([3000, 3000], 2999), ([1500, 1500], 7)])
def test_attention_visible_nan_key_spoils_its_sequence(mx, lens, nan_at, dtype):
    """Also where the key is the only one that a warp or a block meets."""
    codes, scales, table, _, _ = make_cache(mx, lens, 16, 1, 128, 64, 11)
    q = torch.randn(2, 1, 2, 128, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = mx.convrot_mx4_attention(q, codes, scales, table, n, convrot_groupsize=64)
    scales[table[1, nan_at // 16].long(), 0, 0, nan_at % 16, 2] = 255
    out = mx.convrot_mx4_attention(q, codes, scales, table, n, convrot_groupsize=64)
    assert torch.equal(out[0], want[0]) and bool(want.isfinite().all())
    assert bool(out[1].isnan().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 40, 1500])
def test_attention_nan_query_spoils_its_row(mx, n, dtype):
    codes, scales, table, _, _ = make_cache(mx, [n], 16, 2, 128, 64, 12)
    q = torch.randn(1, 1, 4, 128, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    want = mx.convrot_mx4_attention(q, codes, scales, table, lens, convrot_groupsize=0)
    q[0, 0, 2, 70] = math.nan
    out = mx.convrot_mx4_attention(q, codes, scales, table, lens, convrot_groupsize=0)
    assert bool(out[0, 0, 2].isnan().all())
    assert all(torch.equal(out[0, 0, h], want[0, 0, h]) for h in (0, 1, 3))


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,tq,d", [(3, 3, 64), (40, 3, 128), (33, 4, 128), (300, 2, 256), (1500, 5, 64)])
def test_attention_nan_of_the_newest_token_stays_hidden(mx, n, tq, d, dtype, which):
    """The newest token's key or value block is NaN: only the last row sees it."""
    codes, scales, table, ks, vs = make_cache(mx, [n], 16, 1, d, 64, 13)
    q = torch.randn(1, tq, 2, d, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    scales[table[0, (n - 1) // 16].long(), which, 0, (n - 1) % 16, 1] = 255
    out = mx.convrot_mx4_attention(q, codes, scales, table, lens, convrot_groupsize=64)
    assert bool(out[0, -1, :, 0:64].isnan().all())
    check_attention(q[:, :-1], out[:, :-1], [ks[0][:-1]], [vs[0][:-1]], [n - 1], 64, 1 / math.sqrt(d), "bf16" if dtype == torch.bfloat16 else "f16")
