"""GPU tests of the cache append with positions.

Keys go through the fp32 steps of ``apply_rope`` and then those of ``convrot_mx4_cache_append``, so their
codes are those of the two calls on float32 tensors, bit for bit, and values those of the plain append.
Against 64 bits a code may differ only where the value lies within the steps' rounding error of a
midpoint: (|a| + |b|) 2^-22 from the positions and 12 roundings of 2^-24 of the group's magnitudes.
"""
import numpy as np
import pytest
import torch

from oracle import mx4_oracle as orc
from test_gpu_rope import check, turned64

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.fixture(scope="module")
def mx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import _int4
    assert _int4.is_available()
    return _int4


def inputs(tokens, hq, hkv, d, dtype, seed):
    x = torch.randn(tokens, hq + 2 * hkv, d, generator=torch.Generator().manual_seed(seed))
    x[..., 3] *= 8
    return x.to(DT[dtype]).cuda().split((hq, hkv, hkv), 1)


CASES = [  # tokens, hq, hkv, D, page, group, sections, interleaved
    (1, 4, 1, 64, 16, 64, (32,), False), (1, 0, 1, 128, 16, 0, (64,), True), (7, 32, 8, 128, 16, 64, (64,), False),
    (33, 6, 3, 64, 32, 16, (8, 12, 12), False), (5, 2, 2, 256, 64, 256, (128,), False), (65, 3, 1, 256, 16, 64, (64,), True),
    (130, 5, 5, 64, 1, 0, (13,), False), (19, 8, 4, 128, 128, 64, (8, 28, 28), True), (300, 1, 1, 128, 64, 16, (32,), False),
    (12, 14, 7, 128, 16, 64, (3, 5), True), (257, 24, 8, 64, 16, 64, (16,), True), (40, 9, 3, 256, 32, 0, (20, 44, 64), False),
    (4001, 32, 8, 128, 64, 64, (64,), False), (5003, 15, 5, 64, 16, 16, (13,), False), (2049, 0, 8, 256, 128, 256, (16, 56, 56), True)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_append(mx, case, dtype):
    tokens, hq, hkv, d, page, group, sections, interleaved = CASES[case]
    q, k, v = inputs(tokens, hq, hkv, d, dtype, case)
    pages = -(-tokens // page) + 2
    g = torch.Generator().manual_seed(case)
    slots = torch.randperm(pages * page, generator=g)[:tokens].cuda()
    pos = torch.randint(0, 3000, (tokens, len(sections)) if len(sections) > 1 else (tokens,), generator=g).cuda()
    freqs = mx.rope_freqs(sections)
    how = dict(sections=sections, interleaved=interleaved)
    codes, scales = mx.mx4_cache_empty(pages, page, hkv, d)
    codes.fill_(0x5A)
    scales.fill_(0x7B)
    c2, s2 = codes.clone(), scales.clone()
    out = mx.convrot_mx4_cache_append_rope(codes, scales, q if hq else None, k, v, slots, pos, freqs, convrot_groupsize=group, **how)
    if hq:
        check(out, q, pos, freqs, **how)
        assert torch.equal(out, mx.apply_rope(q, pos, freqs, **how))
    else:
        assert out is None
    k32 = mx.apply_rope(k.float(), pos, freqs, **how)
    mx.convrot_mx4_cache_append(c2, s2, k32, v.float(), slots, group)
    assert torch.equal(codes, c2) and torch.equal(scales, s2)                     # (slots without a token are left alone)
    # against 64 bits
    y, size = turned64(k, pos, freqs, sections, interleaved, False)
    at = slots.cpu().numpy()
    c = orc.unpack(codes.cpu().numpy()[at // page, 0, :, at % page])
    e = scales.cpu().numpy()[at // page, 0, :, at % page]
    y64 = orc.rotate64(y.numpy(), group)
    c64, e64 = orc.encode(y64)
    width = group or 1
    spread = np.repeat((size.numpy() + np.abs(y.numpy()) * 12 * 2.0 ** -24).reshape(-1, width).sum(-1), width).reshape(y64.shape) / width ** 0.5
    same = np.repeat(e == e64, 32, -1)
    err, best = np.abs(orc.decode(c, e) - y64), np.abs(orc.decode(c64, e64) - y64)
    assert (np.abs(err - best)[same] <= 2 * spread[same] + 1e-30).all()
    assert (~same).mean() < 1e-2


def test_slots_outside_strides_and_graph(mx):
    """Skipped slots write nothing (their queries are turned), views of a projection, unaligned rows; a graph of the call."""
    tokens, hq, hkv, d = 21, 4, 2, 128
    y = torch.randn(tokens, (hq + 2 * hkv) * d + 8, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    freqs, pos = mx.rope_freqs(64), torch.arange(tokens, device="cuda", dtype=torch.int32) * 3
    slots = torch.arange(tokens).cuda()
    slots[3], slots[7], slots[20] = -1, 2 ** 40, 32
    for off in (0, 8, 3):
        q, k, v = y[:, off:off + (hq + 2 * hkv) * d].unflatten(1, (-1, d)).split((hq, hkv, hkv), 1)
        codes, scales = mx.mx4_cache_empty(2, 16, hkv, d)
        out = mx.convrot_mx4_cache_append_rope(codes, scales, q, k, v, slots, pos, freqs)
        assert torch.equal(out, mx.apply_rope(q, pos, freqs, interleaved=False))
        c2, s2 = mx.mx4_cache_empty(2, 16, hkv, d)
        mx.convrot_mx4_cache_append(c2, s2, mx.apply_rope(k.float(), pos, freqs, interleaved=False), v.float(), slots)
        assert torch.equal(codes, c2) and torch.equal(scales, s2)
        assert not codes[1, :, :, 5:].any()
    version = codes._version
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = mx.convrot_mx4_cache_append_rope(codes, scales, q, k, v, slots, pos, freqs)
    assert codes._version == version + 1
    codes.zero_(), scales.zero_()
    pos.add_(11)
    graph.replay()
    mx.convrot_mx4_cache_append(c2, s2, mx.apply_rope(k.float(), pos, freqs, interleaved=False), v.float(), slots)
    assert torch.equal(codes, c2) and torch.equal(scales, s2) and torch.equal(held, mx.apply_rope(q, pos, freqs, interleaved=False))


def test_special_values(mx):
    """A NaN or an infinity makes its block NaN (the group's blocks, rotated), as in the plain append."""
    q, k, v = inputs(4, 0, 2, 128, "f32", 9)
    k, v = k.clone(), v.clone()
    k[1, 0, 5], k[2, 1, 70], v[3, 0, 100] = float("nan"), float("inf"), float("-inf")
    freqs, slots = mx.rope_freqs(64), torch.arange(4, device="cuda")
    for group in (0, 64):
        codes, scales = mx.mx4_cache_empty(1, 16, 2, 128)
        mx.convrot_mx4_cache_append_rope(codes, scales, None, k, v, slots, slots, freqs, convrot_groupsize=group)
        c2, s2 = mx.mx4_cache_empty(1, 16, 2, 128)
        mx.convrot_mx4_cache_append(c2, s2, mx.apply_rope(k, slots, freqs, interleaved=False), v, slots, group)
        assert torch.equal(scales, s2) and (scales == 255).any()
        fine = (scales != 255).repeat_interleave(16, -1)
        assert torch.equal(codes[fine], c2[fine])


def test_empty(mx):
    codes, scales = mx.mx4_cache_empty(1, 16, 2, 64)
    q, k, v = (torch.empty(0, h, 64, device="cuda") for h in (4, 2, 2))
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert mx.convrot_mx4_cache_append_rope(codes, scales, q, k, v, none, none, mx.rope_freqs(32)).shape == (0, 4, 64)
