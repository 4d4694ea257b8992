"""GPU tests of the W8A8 linear behind a root-mean-square norm, against the definition in 64 bits.

Tolerance. The rotated row is off by at most 12 roundings of 2^-24 of each group's magnitudes over
sqrt(G), plus some five for the sum, the gain and the scale. A code may differ by one where the 64-bit
value lies that near to a midpoint; each such code may move the output by |w| s s_w. The product is
exact; scales, bias and the sum lose 2^-21 of the output's terms, then half a step of the type is lost.
"""
import numpy as np
import pytest
import torch

from oracle import mx4_oracle as orc

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.fixture(scope="module")
def lib():
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


def weight(n, k, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8).cuda(), (torch.rand(n, generator=g) * 1e-3 + 1e-4).cuda()


def f64(t):
    return t.detach().double().cpu().numpy()


def check(got, x, r, gain, w, ws, bias, group, eps=1e-6):
    out, hidden = got
    h32 = x.float() if r is None else x.float() + r.float()
    assert hidden.dtype == x.dtype and torch.equal(hidden, h32.to(x.dtype))
    assert out.dtype == x.dtype and out.shape == (*x.shape[:-1], w.shape[0])
    k = x.shape[-1]
    h = f64(x) if r is None else f64(x) + f64(r)
    h = h.reshape(-1, k)
    rstd = 1 / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    hg = h * (f64(gain) if gain is not None else 1.0) * rstd
    y = orc.rotate64(hg, group)
    s = np.maximum(np.abs(y).max(-1, keepdims=True), 1e-10) / 127
    c = np.rint(y / s)
    near = np.repeat(np.abs(hg).reshape(h.shape[0], -1, group).sum(-1), group, -1) / group ** 0.5 * 17 * 2.0 ** -24 / s + 127 * 2.0 ** -21
    edge = np.abs(np.abs(y / s) % 1 - 0.5) <= near
    w64, ws64 = f64(w), f64(ws)
    terms = (c @ w64.T) * s * ws64
    want = terms + (f64(bias) if bias is not None else 0.0)
    moved = (edge.astype(np.float64) @ np.abs(w64).T) * s * ws64
    step = torch.finfo(x.dtype)
    slack = moved + 2.0 ** -20 * (np.abs(terms) + np.abs(want)) + np.abs(want) * step.eps / 2 * 1.001 + 2.0 ** -24 * (x.dtype == torch.float16)
    err = np.abs(f64(out).reshape(want.shape) - want)
    assert (err <= slack).all(), float((err - slack).max())


CASES = [  # m, n, k, group, residual, gain dtype, bias dtype
    (1, 16, 16, 16, False, None, None), (1, 40, 64, 64, True, "f32", "f32"), (3, 129, 256, 256, True, "bf16", None), (5, 64, 112, 16, True, "f16", "bf16"),
    (127, 72, 768, 256, False, "bf16", "bf16"), (130, 300, 1088, 64, True, "bf16", "f16"), (33, 257, 4096, 256, True, "bf16", None),
    (2, 96, 4112, 16, True, "f32", None), (9, 128, 5120, 256, True, None, "bf16"), (4, 64, 8448, 256, True, "bf16", None),
    (3, 33, 15360, 64, True, "bf16", "bf16"), (2, 24, 16384, 256, False, "bf16", None), (700, 512, 512, 64, True, "bf16", None),
    (1, 1000, 3840, 256, True, "bf16", "bf16"), (8, 520, 2048, 256, True, "bf16", None), (17, 136, 1280, 16, True, "bf16", None), (64, 1024, 640, 64, False, "f16", None)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_linear(lib, case, dtype):
    m, n, k, group, residual, gain, bias = CASES[case]
    x = rows(m, k, dtype, case)
    r = rows(m, k, dtype, case + 100) if residual else None
    g = torch.Generator().manual_seed(case)
    gain = (1 + 0.2 * torch.randn(k, generator=g)).to(DT[gain]).cuda() if gain else None
    bias = torch.randn(n, generator=g).to(DT[bias]).cuda() if bias else None
    w, ws = weight(n, k, case)
    got = lib.convrot_w8a8_linear_rmsnorm(x, w, ws, bias, norm_weight=gain, residual=r, convrot_groupsize=group)
    check(got, x, r, gain, w, ws, bias, group)
    again = lib.convrot_w8a8_linear_rmsnorm(x, w, ws, bias, norm_weight=gain, residual=r, convrot_groupsize=group)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    if r is None:
        assert got[1] is x


def test_rows_do_not_depend_on_their_number(lib):
    """A token gives the same codes alone and in a batch: outputs are equal bit for bit."""
    w, ws = weight(200, 1024, 1)
    x, r = rows(150, 1024, "bf16", 2), rows(150, 1024, "bf16", 3)
    whole, _ = lib.convrot_w8a8_linear_rmsnorm(x, w, ws, residual=r)
    for m in (1, 2, 4, 5, 8, 16, 31, 65, 130):
        part, _ = lib.convrot_w8a8_linear_rmsnorm(x[:m], w, ws, residual=r[:m])
        assert torch.equal(part, whole[:m]), m


def test_strides_shapes_and_alignment(lib):
    w, ws = weight(48, 256, 4)
    base = rows(40, 1000, "bf16", 5)
    for x in (base[:, 3:259], base[::2, 8:264], base[:, 100:356].t().contiguous().t(), base[:, :512].reshape(5, 8, 512)[..., 256:], base[0, :256]):
        r = x.flip(0)
        check(lib.convrot_w8a8_linear_rmsnorm(x, w, ws[:, None], residual=r), x, r, None, w, ws, None, 256)
    wide = torch.randint(-9, 9, (48, 300), dtype=torch.int8).cuda()[:, 20:276]
    check(lib.convrot_w8a8_linear_rmsnorm(base[:, :256], wide, ws.double()), base[:, :256], None, None, wide, ws, None, 256)
    x = torch.empty(0, 256, dtype=torch.bfloat16, device="cuda")
    out, hidden = lib.convrot_w8a8_linear_rmsnorm(x, w, ws, residual=x)
    assert out.shape == (0, 48) and hidden.shape == (0, 256)
    out, hidden = lib.convrot_w8a8_linear_rmsnorm(base[:, :256], w[:0], ws[:0], residual=base[:, :256])
    assert out.shape == (40, 0) and torch.equal(hidden, base[:, :256] * 2)


def test_special_rows(lib):
    """Zeros give the bias, NaN and infinities their own row's NaN only, large and tiny rows keep their precision."""
    w, ws = weight(32, 512, 6)
    x = rows(8, 512, "f32", 7)
    x[0] = 0
    x[1, 5], x[2, 300], x[3, 0] = float("nan"), float("inf"), float("-inf")
    x[4] *= 1e15
    x[5] *= 1e-30
    x[6] *= 1e-15
    bias = torch.randn(32).cuda()
    out, _ = lib.convrot_w8a8_linear_rmsnorm(x, w, ws, bias)
    assert torch.equal(out[0], bias) and out[1:4].isnan().all() and out[4:].isfinite().all()
    keep = torch.tensor([4, 6, 7], device="cuda")
    check((out[keep], x[keep]), x[keep], None, None, w, ws, bias, 256)
    tiny = rows(2, 512, "f32", 8) * 1e-15
    check(lib.convrot_w8a8_linear_rmsnorm(tiny, w, ws, eps=0.0), tiny, None, None, w, ws, None, 256, eps=0.0)


def test_streams_and_graphs_with_workspaces_of_their_own(lib):
    """Two captured graphs replayed on two streams at once do not share scratch."""
    w, ws = weight(256, 1024, 9)
    xs, outs, graphs, streams = [], [], [], []
    for i in range(2):
        x = rows(300, 1024, "bf16", 10 + i)
        lib.convrot_w8a8_linear_rmsnorm(x, w, ws)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(lib.convrot_w8a8_linear_rmsnorm(x, w, ws, residual=x)[0])
        xs.append(x)
        graphs.append(graph)
        streams.append(torch.cuda.Stream())
    want = [lib.convrot_w8a8_linear_rmsnorm(x, w, ws, residual=x)[0] for x in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_layer(lib):
    from _int4.int8_eager import quantize_convrot_w8a8_weight
    from _int4.linear import Int4ConvRotLinear
    layer = Int4ConvRotLinear(512, 96, device="cuda", mode="int8")
    q, s = quantize_convrot_w8a8_weight(torch.randn(96, 512, device="cuda") * 0.02, layer._qgs)
    layer._q.copy_(q)
    layer._qs.copy_(s)
    layer.bias.copy_(torch.randn(96))
    x, r, g = rows(5, 512, "bf16", 1), rows(5, 512, "bf16", 2), torch.rand(512, device="cuda").bfloat16()
    got = layer.forward_rmsnorm(x, g, r)
    check(got, x, r, g, q, s, layer.bias, layer._qgs)
    # int4 layers and adapters: the same through torch's norm, up to their own quantization
    layer.set_dynamic_lora([(torch.zeros(8, 512), torch.zeros(96, 8), 8.0, 1.0)])
    near, hidden = layer.forward_rmsnorm(x, g, r)
    assert torch.equal(hidden, got[1]) and (near - got[0]).float().norm() <= 0.02 * got[0].float().norm()
