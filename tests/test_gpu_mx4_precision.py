"""GPU tests of the precision and range of attention over the MX4 cache.

``oracle/mx4_oracle.py`` derives the bounds: MOST_APART is the share of outputs that
may differ from the nearest value of their type when every operand keeps 22 bits.
"""
import math

import numpy as np
import pytest
import torch

from oracle import mx4_oracle as orc
from test_gpu_mx4 import DT, f64, make_cache, mx  # noqa: F401

pytestmark = pytest.mark.gpu


def expected(q, ks, vs, lens, group, scale):
    out, _, _ = orc.attention64(orc.rotate64(f64(q), group), ks, vs, lens, scale)
    return orc.rotate64(out, group)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lens,tq,hq,hkv,d,group", [
    ([300], 1, 64, 8, 128, 64), ([200, 57], 4, 24, 8, 64, 64), ([3000], 2, 32, 4, 128, 64), ([700], 3, 16, 2, 128, 16), ([700], 8, 8, 1, 64, 64),
    ([150, 9], 2, 16, 2, 256, 256), ([2500], 1, 32, 4, 256, 0)])
def test_attention_outputs_are_the_nearest_values(mx, lens, tq, hq, hkv, d, group, dtype):  # noqa: F811
    codes, scales, table, ks, vs = make_cache(mx, lens, 16, hkv, d, group, 20)
    q = (torch.randn(len(lens), tq, hq, d, generator=torch.Generator().manual_seed(5)) * 1.5).to(DT[dtype]).cuda()
    out = mx.convrot_mx4_attention(q, codes, scales, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), convrot_groupsize=group)
    apart = orc.rounded_apart(f64(out), expected(q, ks, vs, lens, group, 1 / math.sqrt(d)), dtype)
    assert apart <= orc.MOST_APART[dtype], apart


def set_values(codes, scales, table, at, v):
    """Writes values v [N, heads, D] (64 bits), unrotated, as the cache's tokens 0 .. of its only sequence."""
    c, e = orc.encode(v)
    page = codes.shape[3]
    j = torch.arange(v.shape[0])
    pages, off = table[0].cpu().long()[j // page], j % page
    codes[pages.cuda(), at, :, off.cuda()] = torch.from_numpy(orc.pack(c)).cuda()
    scales[pages.cuda(), at, :, off.cuda()] = torch.from_numpy(e).cuda()
    return orc.decode(c, e)


@pytest.mark.parametrize("dtype,ratio", [("bf16", 2.0 ** 6), ("bf16", 2.0 ** 9), ("bf16", 2.0 ** 14), ("bf16", 2.0 ** 20), ("bf16", 2.0 ** 40), ("bf16", 2.0 ** 100),
                                         ("f16", 2.0 ** 6), ("f16", 2.0 ** 9), ("f16", 2.0 ** 12)])
@pytest.mark.parametrize("each", [True, False])
@pytest.mark.parametrize("n,tq,hq,d", [(70, 1, 16, 64), (300, 2, 8, 128), (1500, 1, 32, 128), (300, 16, 2, 128), (200, 8, 2, 256), (500, 32, 1, 64)])
def test_attention_channels_of_different_magnitudes(mx, n, tq, hq, d, each, ratio, dtype):  # noqa: F811
    """Channel blocks whose values differ by a ratio, in every token or (not ``each``) with the
    large block in the even tokens and the others in the odd ones only: every channel keeps
    the precision of its own values."""
    codes, scales, table, ks, vs = make_cache(mx, [n], 16, 1, d, 0, 21)
    v = np.random.default_rng(3).standard_normal((n, 1, d))
    v[..., 32:64] *= ratio
    if not each:
        v[::2, :, :32] = v[::2, :, 64:] = 0
        v[1::2, :, 32:64] = 0
    vs = [set_values(codes, scales, table, 1, v)]
    q = torch.randn(1, tq, hq, d, generator=torch.Generator().manual_seed(6)).to(DT[dtype]).cuda()
    out = f64(mx.convrot_mx4_attention(q, codes, scales, table, torch.tensor([n], dtype=torch.int32, device="cuda"), convrot_groupsize=0))
    ref = expected(q, ks, vs, [n], 0, 1 / math.sqrt(d))
    for part in (slice(0, 32), slice(32, 64), slice(64, d)):
        apart = orc.rounded_apart(out[..., part], ref[..., part], dtype) if part.stop > part.start else 0.0
        assert apart <= 2 * orc.MOST_APART[dtype], (part, apart)               # (twice: down to 512 outputs a part)


@pytest.mark.parametrize("d,bits", [(64, 16), (128, 24), (128, 27), (256, 20)])
def test_attention_of_many_small_weights(mx, d, bits):  # noqa: F811
    """One token outweighs thousands by 2^bits and has no values in a block that they have. A
    weight is off by 2^-25 where the largest product of weight and values is 2^8 at
    least, so an output by 2^-33 of that product for each token, beside the 2^-17 of every operand."""
    n = 4000
    codes, scales, table, _, _ = make_cache(mx, [n], 64, 1, d, 0, 22)
    k = np.zeros((n, 1, d))
    k[0, 0, 0] = 4.0
    v = np.full((n, 1, d), 1.5)
    v[0, :, :32] = 0
    ks, vs = [set_values(codes, scales, table, 0, k)], [set_values(codes, scales, table, 1, v)]
    q = torch.zeros(1, 1, 8, d, dtype=torch.bfloat16, device="cuda")
    q[0, 0, :, 0] = torch.linspace(0.9, 1.1, 8)
    scale = bits * math.log(2) / 4
    out = f64(mx.convrot_mx4_attention(q, codes, scales, table, torch.tensor([n], dtype=torch.int32, device="cuda"), scale, 0))
    ref = expected(q, ks, vs, [n], 0, scale)
    tol = 2.0 ** -8 * np.abs(ref) + 2.0 ** -17 * np.abs(ref) + n * 2.0 ** -33 * 1.5
    err = np.abs(out - ref)
    assert (err <= tol).all(), (err / tol).max()


def test_attention_of_far_blocks_and_a_hidden_nan(mx):  # noqa: F811
    """Values far apart and a NaN block in the newest token: rows that do not see it keep their result."""
    n, tq, d = 75, 3, 128
    codes, scales, table, ks, _ = make_cache(mx, [n], 16, 1, d, 0, 26)
    v = np.random.default_rng(4).standard_normal((n, 1, d))
    v[:, :, 64:96] *= 2.0 ** 30
    vs = [set_values(codes, scales, table, 1, v)]
    scales[table[0, (n - 1) // 16].long(), 1, 0, (n - 1) % 16, 1] = 255
    q = torch.randn(1, tq, 4, d, generator=torch.Generator().manual_seed(9)).bfloat16().cuda()
    out = f64(mx.convrot_mx4_attention(q, codes, scales, table, torch.tensor([n], dtype=torch.int32, device="cuda"), convrot_groupsize=0))
    ref = expected(q, ks, vs, [n], 0, d ** -0.5)
    seen = np.zeros((tq, 1, d), bool)
    seen[-1, :, 32:64] = True
    assert np.array_equal(np.isnan(out[0]), np.broadcast_to(seen, out[0].shape))
    apart = orc.rounded_apart(np.where(seen, 0, out[0]), np.where(seen, 0, ref[0]), "bf16")
    assert apart <= 2 * orc.MOST_APART["bf16"], apart


def test_attention_keys_of_the_smallest_scale(mx):  # noqa: F811
    """Keys whose scale byte is 0 (2^-127) are not zeros: queries of 2^120 bring the scores near 1."""
    n, d = 60, 128
    codes, scales, table, _, vs = make_cache(mx, [n], 16, 1, d, 0, 23)
    rng = np.random.default_rng(1)
    ks = [set_values(codes, scales, table, 0, rng.standard_normal((n, 1, d)) * 2.0 ** -126)]
    assert ks[0].any() and not scales[table[0].long(), 0, 0].reshape(-1, d // 32)[:n].any()
    q = (torch.randn(1, 1, 64, d, generator=torch.Generator().manual_seed(7)) * 2.0 ** 120).bfloat16().cuda()
    out = mx.convrot_mx4_attention(q, codes, scales, table, torch.tensor([n], dtype=torch.int32, device="cuda"), 8.0, 0)
    apart = orc.rounded_apart(f64(out), expected(q, ks, vs, [n], 0, 8.0), "bf16")
    assert apart <= orc.MOST_APART["bf16"], apart


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("size", [3e2, 1e4, 1e6, -1e4, -1e6, -1e9, 1e12])
@pytest.mark.parametrize("n,d", [(1, 64), (40, 128), (3000, 64)])
def test_attention_of_large_scores(mx, n, d, size, dtype):  # noqa: F811
    """Two tokens share the highest score, all others are far below it: the result is the
    mean of their values, however large the scores are."""
    codes, scales, table, _, vs = make_cache(mx, [n], 16, 1, d, 0, 27)
    k = np.full((n, 1, d), 0.5 if size > 0 else 1.0)
    best = sorted({n // 3, n - 1})
    k[best] = 1.0 if size > 0 else 0.5
    set_values(codes, scales, table, 0, k)
    q = torch.ones(1, 1, 2, d, dtype=DT[dtype], device="cuda") * math.copysign(1.0, size)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    out = mx.convrot_mx4_attention(q, codes, scales, table, lens, abs(size) / d, 0)
    want = torch.from_numpy(vs[0][best].mean(0)).to(DT[dtype])
    assert torch.equal(out[0, 0].cpu().float(), want.repeat(2, 1).float())


@pytest.mark.parametrize("n", [1, 40, 3000])
def test_attention_of_very_low_scores(mx, n):  # noqa: F811
    """All of a row's scores lie below -1e30: the highest one's values are the result."""
    d = 64
    codes, scales, table, _, vs = make_cache(mx, [n], 16, 1, d, 0, 24)
    k = np.full((n, 1, d), 1.5e17)
    k[n // 2] = 1e17
    set_values(codes, scales, table, 0, k)
    q = torch.full((1, 1, 2, d), -2e18, dtype=torch.bfloat16, device="cuda")
    out = mx.convrot_mx4_attention(q, codes, scales, table, torch.tensor([n], dtype=torch.int32, device="cuda"), 0.25, 0)
    assert np.array_equal(f64(out)[0, 0], np.repeat(vs[0][n // 2], 2, 0))
    none = mx.convrot_mx4_attention(q, codes, scales, table, torch.zeros(1, dtype=torch.int32, device="cuda"), 0.25, 0)
    assert not none.any()


@pytest.mark.parametrize("vscale", [2.0 ** 124, 2.0 ** 110, 2.0 ** -124])
@pytest.mark.parametrize("b,n", [(1, 30), (1, 500), (3, 4000), (40, 6000)])
def test_attention_values_at_the_ends_of_the_range(mx, b, n, vscale):  # noqa: F811
    """Sums of many values stay in fp32's range, and tiny ones are not flushed (one block,
    a cluster, and the separate join, whose sequences share their pages)."""
    d = 64
    codes, scales, table, ks, _ = make_cache(mx, [n], 64, 1, d, 0, 25)
    v = np.clip(np.random.default_rng(2).standard_normal((n, 1, d)), -3, 3) + 1
    v = [set_values(codes, scales, table, 1, v * vscale)]
    q = torch.randn(1, 1, 8, d, generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    lens = torch.full((b,), n, dtype=torch.int32, device="cuda")
    out = f64(mx.convrot_mx4_attention(q.repeat(b, 1, 1, 1), codes, scales, table.repeat(b, 1), lens, convrot_groupsize=0))
    ref = np.repeat(expected(q, ks, v, [n], 0, d ** -0.5), b, 0)
    err = np.abs(out - ref)
    # half a spacing, 2^-17 of the operands; fp32 sums below its normal range: 2^-149 each
    assert (err <= (2.0 ** -8 + 2.0 ** -16) * np.abs(ref) + 2.0 ** -134).all(), (err / np.abs(ref)).max()
