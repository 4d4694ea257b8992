"""GPU tests of the rotary positions against the definition in 64 bits.

Tolerance. Sine and cosine are rounded to fp32 (2^-25), the two products and their sum by 2^-24 each: an
output is off by (|a| + |b|) 2^-22 at most for a pair (a, b), then by half a step of its type. In 64 bits
an angle A itself carries the product's rounding here and in the reference, 2^-53 each, which counts
from positions of some 2^30 on: (|a| + |b|) |A| 2^-51.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import _int4
    assert _int4.is_available()
    return _int4


def turned64(x, positions, freqs, sections, interleaved, inverse):
    """(the turned heads, the error of each channel's pair) in 64 bits, pair by pair."""
    x, f = x.double().cpu(), freqs.cpu()
    lead = x.shape[:-2]
    n = f.numel()
    sections = sections or (n,)
    p = positions.double().cpu()
    p = p.expand(*lead, len(sections)) if len(sections) > 1 else p.expand(lead)[..., None]
    out, size = x.clone(), torch.zeros_like(x)
    i = 0
    for axis, many in enumerate(sections):
        for _ in range(many):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
            angle = (p[..., axis] * f[i] * (-1 if inverse else 1))[..., None]
            out[..., a] = x[..., a] * angle.cos() - x[..., b] * angle.sin()
            out[..., b] = x[..., a] * angle.sin() + x[..., b] * angle.cos()
            size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs()) * (2.0 ** -22 + angle.abs() * 2.0 ** -51)
            i += 1
    return out, size


def check(got, x, positions, freqs, sections=None, interleaved=True, inverse=False):
    want, size = turned64(x, positions, freqs, sections, interleaved, inverse)
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    step = torch.finfo(x.dtype)
    slack = size + want.abs() * (step.eps / 2 * 1.001) + step.smallest_normal * step.eps
    assert ((got.double().cpu() - want).abs() <= slack).all()
    rest = 2 * freqs.numel()
    assert torch.equal(got[..., rest:], x[..., rest:])


CASES = [  # lead, heads, D, sections, interleaved
    ((1,), 1, 2, (1,), True), ((1,), 1, 64, (32,), False), ((3, 5), 7, 128, (64,), False), ((2, 33), 24, 64, (16,), False),
    ((17,), 5, 128, (8, 28, 28), True), ((4, 9), 3, 256, (16, 56, 56), False), ((33,), 40, 96, (5, 7, 9, 3), True),
    ((6,), 2, 80, (13, 17), False), ((), 8, 128, (64,), True), ((2, 3, 4), 6, 32, (16,), True), ((257,), 16, 128, (0, 64), False),
    ((5,), 3, 10, (2,), False), ((1000,), 11, 72, (36,), False)]


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_rope(lib, case, dtype, inverse):
    lead, heads, d, sections, interleaved = CASES[case]
    g = torch.Generator().manual_seed(case)
    x = (torch.randn(*lead, heads, d, generator=g) * 3).to(DT[dtype]).cuda()
    axes = len(sections)
    p = torch.randint(0, 5000, (*lead, axes) if axes > 1 else lead, generator=g)
    freqs = lib.rope_freqs(sections)
    for kind in (torch.int64, torch.int32, torch.float32):
        got = lib.apply_rope(x, p.to(kind).cuda(), freqs, sections=sections, interleaved=interleaved, inverse=inverse)
        check(got, x, p.cuda(), freqs, sections, interleaved, inverse)
    if axes == 1:
        assert torch.equal(lib.apply_rope(x, p.cuda(), freqs, interleaved=interleaved, inverse=inverse),
                           lib.apply_rope(x, p.cuda(), freqs, sections=sections, interleaved=interleaved, inverse=inverse))


def test_far_negative_and_fractional_positions(lib):
    x = torch.randn(6, 4, 128, generator=torch.Generator().manual_seed(0)).cuda()
    freqs = lib.rope_freqs(64)
    p = torch.tensor([0, 1, -7, 1000003, 2 ** 31 + 5, 2 ** 40], device="cuda")
    check(lib.apply_rope(x, p, freqs), x, p, freqs)
    p = torch.tensor([0.5, -2.25, 1e6 + 0.5, 1e-3, 0.0, 3.0], device="cuda")
    check(lib.apply_rope(x, p, freqs), x, p, freqs)


def test_strides_broadcast_positions_and_unaligned_rows(lib):
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(2, 31, 12, 64, generator=g).bfloat16().cuda()
    freqs = lib.rope_freqs(32)
    p = torch.arange(31, device="cuda")
    for x in (qkv[:, :, :5], qkv[:, :, 3:4], qkv[:, ::3, 2:9:2], qkv.transpose(1, 2)[:, :, :12].transpose(1, 2),
              qkv.permute(2, 1, 0, 3).transpose(0, 1), qkv[..., 2:50], qkv[1:2].expand(3, -1, -1, -1)):
        pos = p[:x.shape[-3]] if x.shape[0] != 31 else p[:x.shape[-3]].reshape(-1)
        f = freqs[:x.shape[-1] // 2]
        check(lib.apply_rope(x, pos, f, interleaved=False), x, pos, f, None, False)
    odd = torch.randn(31 * 4 * 64 + 1, generator=g).half().cuda()[1:].reshape(31, 4, 64)
    check(lib.apply_rope(odd, p, freqs), odd, p, freqs)
    per = torch.randint(0, 99, (2, 1, 3), generator=g).cuda()                      # one place for all tokens of a batch entry
    check(lib.apply_rope(qkv, per, lib.rope_freqs((8, 12, 12)), sections=(8, 12, 12)), qkv, per, lib.rope_freqs((8, 12, 12)), (8, 12, 12))
    t = qkv.transpose(-1, -2).contiguous().transpose(-1, -2)                       # D not contiguous
    check(lib.apply_rope(t, p, freqs), t, p, freqs)


def test_gradient_is_the_rotation_back(lib):
    """The derivative by x in direction g: <rope(x), g> = <x, rope back(g)>, and differences of a linear map."""
    gen = torch.Generator().manual_seed(2)
    x, g = (torch.randn(9, 3, 128, generator=gen).cuda() for _ in range(2))
    p, freqs = torch.arange(9, device="cuda") * 17, lib.rope_freqs((16, 24, 24))
    pos = torch.stack((p, p + 1, 2 * p), -1)
    for interleaved in (True, False):
        how = dict(sections=(16, 24, 24), interleaved=interleaved)
        back = lib.apply_rope(g, pos, freqs, inverse=True, **how)
        dx = torch.zeros_like(x)
        dx[4, 1] = torch.randn(128, generator=gen).cuda()
        diff = (lib.apply_rope(x + dx, pos, freqs, **how).double() - lib.apply_rope(x, pos, freqs, **how).double())
        bound = float((x.abs().sum() + dx.abs().sum()) * g.abs().max()) * 2.0 ** -20
        assert abs(float((diff * g.double()).sum() - (dx.double() * back.double()).sum())) <= bound
        assert (lib.apply_rope(lib.apply_rope(x, pos, freqs, **how), pos, freqs, inverse=True, **how) - x).abs().max() <= float(x.abs().max()) * 2.0 ** -18


def test_special_values_streams_and_graphs(lib):
    x = torch.randn(4, 2, 64, generator=torch.Generator().manual_seed(3)).cuda()
    x[1, 0, 3] = float("nan")
    x[2, 1, 7] = float("inf")
    freqs, p = lib.rope_freqs(32), torch.arange(4, device="cuda")
    out = lib.apply_rope(x, p, freqs, interleaved=False)
    bad = ~torch.isfinite(out)
    assert bad[1, 0, 3] and bad[1, 0, 35] and int(bad[1].sum()) == 2 and bad[2, 1, 7] and bad[2, 1, 39] and int(bad[2].sum()) == 2
    assert int(bad.sum()) == 4
    stream = torch.cuda.Stream()
    y = torch.randn(300, 8, 128, device="cuda").bfloat16()
    p, freqs = torch.arange(300, device="cuda"), lib.rope_freqs(64)
    want = lib.apply_rope(y, p, freqs)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = lib.apply_rope(y, p, freqs)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = lib.apply_rope(y, p, freqs)
    y.copy_(y.flip(0))
    p.add_(5)
    graph.replay()
    assert torch.equal(held, lib.apply_rope(y, p, freqs))


def test_empty(lib):
    freqs = lib.rope_freqs(32)
    for shape in ((0, 4, 64), (2, 0, 4, 64), (3, 0, 64), (2, 3, 0, 4, 64), (0, 2, 3, 4, 64), (2, 3, 5, 0, 64)):
        assert lib.apply_rope(torch.empty(shape, device="cuda"), torch.zeros(shape[:-2], dtype=torch.int64, device="cuda"), freqs).shape == shape
    x = torch.randn(3, 2, 64, device="cuda")
    assert torch.equal(lib.apply_rope(x, torch.arange(3, device="cuda"), freqs[:0]), x)        # no pair is turned
