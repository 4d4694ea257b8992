"""GPU tests of rotary positions on a part of the head: the channels behind the pairs are copied, bit for bit.

Whatever these channels hold (infinities, NaN, zeros of either sign) neither changes nor reaches a
neighbour, interleaved or in halves, in chunks of 16 bytes or single values; the turned channels are
those of the same heads with zeros behind them.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BITS = {torch.bfloat16: torch.int16, torch.float16: torch.int16, torch.float32: torch.int32}


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import _int4
    assert _int4.is_available()
    return _int4


def heads(tokens, h, d, rest, dtype, seed):
    """Heads whose channels from `rest` on hold special values between ordinary ones."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, h, d, generator=g)
    special = torch.tensor([float("inf"), float("-inf"), float("nan"), -0.0, 0.0, 1.0])
    pick = torch.randint(0, 12, (tokens, h, d - rest), generator=g)
    x[..., rest:] = torch.where(pick < 6, special[pick.clamp(max=5)], x[..., rest:])
    return x.to(DT[dtype]).cuda()


def unaligned(x):
    y = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].reshape(x.shape)
    return y.copy_(x)


def bits(t):
    return t.contiguous().view(BITS[t.dtype])


PARTS = [(64, 16), (128, 32), (128, 16), (128, 48), (256, 64), (80, 8), (128, 13), (64, 4), (96, 1)]     # D, pairs


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("part", range(len(PARTS)))
def test_channels_behind_the_pairs_are_copied(lib, part, dtype, interleaved):
    d, pairs = PARTS[part]
    x = heads(37, 3, d, 2 * pairs, dtype, part)
    freqs, pos = lib.rope_freqs(pairs), torch.arange(37, device="cuda") * 5
    bare = x.clone()
    bare[..., 2 * pairs:] = 0
    want = lib.apply_rope(bare, pos, freqs, interleaved=interleaved)[..., :2 * pairs]
    for given in (x, unaligned(x)):
        for inverse in (False, True):
            out = lib.apply_rope(given, pos, freqs, interleaved=interleaved, inverse=inverse)
            assert torch.equal(bits(out[..., 2 * pairs:]), bits(x[..., 2 * pairs:]))
            assert out[..., :2 * pairs].isfinite().all()
            if not inverse:
                assert torch.equal(bits(out[..., :2 * pairs]), bits(want))


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("tokens,hq,hkv,d,pairs", [(9, 6, 2, 128, 32), (9, 6, 2, 64, 16), (9, 3, 1, 256, 48), (2100, 32, 8, 256, 32)])
def test_queries_and_keys_on_their_way_into_the_cache(lib, tokens, hq, hkv, d, pairs, interleaved):
    """The same of a call's queries (by the same launch, and in one of their own where there are many tokens); keys as
    those of the two calls, blocks of NaN where the copied channels hold one."""
    x = heads(tokens, hq + 2 * hkv, d, 2 * pairs, "bf16", tokens)
    freqs, pos = lib.rope_freqs(pairs), torch.arange(tokens, device="cuda") * 3
    slots = torch.arange(tokens, device="cuda")
    pages = -(-tokens // 64)
    for given in (x, unaligned(x)):
        q, k, v = given.split((hq, hkv, hkv), 1)
        codes, scales = lib.mx4_cache_empty(pages, 64, hkv, d)
        out = lib.convrot_mx4_cache_append_rope(codes, scales, q, k, v, slots, pos, freqs, interleaved=interleaved, convrot_groupsize=0)
        assert torch.equal(bits(out[..., 2 * pairs:]), bits(q[..., 2 * pairs:]))
        assert torch.equal(bits(out), bits(lib.apply_rope(q, pos, freqs, interleaved=interleaved)))
        c2, s2 = lib.mx4_cache_empty(pages, 64, hkv, d)
        turned = k.float()
        turned[..., 2 * pairs:] = 0
        turned = lib.apply_rope(turned, pos, freqs, interleaved=interleaved)
        turned[..., 2 * pairs:] = k[..., 2 * pairs:].float()
        lib.convrot_mx4_cache_append(c2, s2, turned, v.float(), slots, 0)
        assert torch.equal(scales, s2)
        fine = (scales != 255).repeat_interleave(16, -1)
        assert torch.equal(codes[fine], c2[fine])
