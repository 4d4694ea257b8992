"""GPU tests of the cache append with positions for many tokens: queries, values and keys by launches of their own.

That begins where a call has more than 64 tasks of 32 units (128 values each) a multiprocessor; the number of tokens
is made from the device's and checked against that, so that every case is known to lie beyond it (or, the
last token taken away, below). The same codes, bit for bit, as by ``apply_rope`` and the plain append.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

BITS = {torch.bfloat16: torch.int16, torch.float16: torch.int16, torch.float32: torch.int32}


@pytest.fixture(scope="module")
def mx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import _int4
    assert _int4.is_available()
    return _int4


def first_apart(hq, hkv, d):
    """The least number of tokens that takes launches of their own."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    units = (hkv + 1) // 2 if d == 64 else hkv * d // 128
    apart = lambda t: (2 * t * units + t * hq * d // 128) // 32 > 64 * sms      # noqa: E731
    t = (64 * sms * 32) * 128 // (2 * units * 128 + hq * d)
    while not apart(t):
        t += 1
    assert apart(t) and not apart(t - 1)
    return t


CASES = [  # hq, hkv, D, page, group, sections, interleaved, dtype, layout
    (32, 8, 128, 64, 64, (64,), False, torch.bfloat16, "projection"), (3, 5, 64, 16, 64, (8, 12, 12), False, torch.float16, "projection"),
    (8, 2, 256, 64, 256, (128,), True, torch.bfloat16, "contiguous"), (0, 3, 256, 32, 256, (20, 44), False, torch.float32, "contiguous"),
    (7, 7, 128, 16, 16, (16,), True, torch.bfloat16, "unaligned"), (16, 4, 128, 128, 0, (5, 27), False, torch.bfloat16, "turned"),
    (1, 1, 64, 8, 16, (13,), True, torch.bfloat16, "contiguous"), (24, 8, 64, 64, 64, (32,), True, torch.float16, "turned")]


@pytest.mark.parametrize("more", [-1, 0, 77])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_many_tokens(mx, case, more):
    hq, hkv, d, page, group, sections, interleaved, dtype, layout = CASES[case]
    tokens = first_apart(hq, hkv, d) + more
    g = torch.Generator(device="cuda").manual_seed(case)
    heads = hq + 2 * hkv
    if layout == "projection":
        x = torch.randn(tokens, heads, d, generator=g, device="cuda").to(dtype)
        q, k, v = x.split((hq, hkv, hkv), 1)
    else:
        q, k, v = (torch.randn(tokens, h, d, generator=g, device="cuda").to(dtype) for h in (hq, hkv, hkv))
        if layout == "unaligned":
            q, k, v = (torch.cat((t.flatten()[:1], t.flatten()))[1:].reshape(t.shape) for t in (q, k, v))
        if layout == "turned":                                    # heads outside, tokens inside
            q, k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    pages = -(-tokens // page) + 3
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    slots[::13], slots[5], slots[tokens - 1] = -1, pages * page, 2 ** 40
    axes = len(sections)
    pos = torch.randint(0, 40000, (tokens, axes) if axes > 1 else (tokens,), generator=g, device="cuda")
    freqs = mx.rope_freqs(sections)
    how = dict(sections=sections, interleaved=interleaved)
    codes, scales = mx.mx4_cache_empty(pages, page, hkv, d)
    codes.fill_(0x5A)
    scales.fill_(0x7B)
    c2, s2 = codes.clone(), scales.clone()
    out = mx.convrot_mx4_cache_append_rope(codes, scales, q if hq else None, k, v, slots, pos, freqs, convrot_groupsize=group, **how)
    if hq:
        assert torch.equal(out.view(BITS[dtype]), mx.apply_rope(q, pos, freqs, **how).view(BITS[dtype]))
    else:
        assert out is None
    mx.convrot_mx4_cache_append(c2, s2, mx.apply_rope(k.float(), pos, freqs, **how), v.float(), slots, group)
    assert torch.equal(codes, c2) and torch.equal(scales, s2)
    # the same tokens in small calls
    c3, s3 = torch.full_like(codes, 0x5A), torch.full_like(scales, 0x7B)
    step = -(-tokens // 9)
    for at in range(0, tokens, step):
        cut = slice(at, at + step)
        part = mx.convrot_mx4_cache_append_rope(c3, s3, q[cut] if hq else None, k[cut], v[cut], slots[cut].contiguous(), pos[cut], freqs, convrot_groupsize=group, **how)
        if hq:
            assert torch.equal(part, out[cut])
    assert torch.equal(codes, c3) and torch.equal(scales, s3)
