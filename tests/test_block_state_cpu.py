"""Bookkeeping of the cache and the trees where a call fails or has nothing to do (no GPU needed)."""
import pytest
import torch

import _int4
from _int4.mx4_layers import Mx4KVCache, Mx4SelfAttention


def test_a_prefill_that_fails_on_its_way_to_the_cache_reserves_no_tokens():
    """Frequencies of the wrong type, of more pairs than a head, sections that do not add up, tensors that the kernels
    do not take: the sequence keeps its length and its pages."""
    f = _int4.rope_freqs(32, device="cpu")
    for how in (dict(freqs=f.float()), dict(freqs=_int4.rope_freqs(64, device="cpu")), dict(freqs=f, sections=(8, 25)), dict(freqs=f), dict()):
        block = Mx4SelfAttention(64, 2, 1, 64, device="cpu", **how)
        block.project = lambda x: (torch.zeros(len(x), 2, 64), torch.zeros(len(x), 1, 64), torch.zeros(len(x), 1, 64))
        cache = Mx4KVCache(4, 1, 64, page=16, device="cpu")
        seq = cache.add()
        cache.extend(seq, 7)
        free, held = list(cache._free), list(cache._pages[seq])
        axes = (2,) if "sections" in how else ()
        with pytest.raises(ValueError):
            block.prefill(torch.zeros(20, 64), cache, seq, torch.zeros(20, *axes) if "freqs" in how else None)
        assert cache.length(seq) == 7 and cache._pages[seq] == held and sorted(cache._free) == sorted(free)


def test_accept_takes_caches_made_in_inference_mode():
    with torch.inference_mode():
        cache = Mx4KVCache(2, 1, 64, page=4, device="cpu")
        codes = torch.randint(0, 255, cache.codes.shape, dtype=torch.uint8)
        cache.codes.copy_(codes)
    seq = cache.add()
    new = cache.extend(seq, 6)
    cache.accept(seq, 5, [1, 3])
    assert cache.length(seq) == 3
    for to, node in enumerate((1, 3)):
        s, t = cache.slots(seq)[1 + to], new[1 + node]
        assert torch.equal(cache.codes[s // 4, :, :, s % 4], codes[t // 4, :, :, t % 4])
    plain = Mx4KVCache(2, 1, 64, page=4, device="cpu")
    seq = plain.add()
    plain.extend(seq, 6)
    before = plain.codes._version
    plain.accept(seq, 5, [1, 3])
    assert plain.codes._version > before                          # (written in place)


def test_trees_without_nodes():
    for shape in ((0,), (3, 0), (0, 0), (0, 5)):
        mask, depth = _int4.tree_mask(torch.zeros(shape, dtype=torch.int64))
        assert mask.shape == (*shape, shape[-1]) and mask.dtype == torch.bool and depth.shape == shape and depth.dtype == torch.int64
    with pytest.raises(ValueError, match="whole numbers"):
        _int4.tree_mask(torch.zeros(3, dtype=torch.complex64))
