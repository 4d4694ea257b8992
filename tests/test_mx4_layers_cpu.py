"""State dicts of the MX4 layers (no GPU needed)."""
import pytest
import torch

from _int4.mx4_layers import Mx4ConvRotLinear


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_linear_loads_a_bias_in_its_own_type(dtype):
    m = Mx4ConvRotLinear(64, 3, device="cpu")
    m.bias = torch.tensor([1 / 3, -1e-3, 7.123]).to(dtype)
    clone = Mx4ConvRotLinear(64, 3, device="cpu")
    clone.load_state_dict(m.state_dict())
    assert clone.bias.dtype == dtype and torch.equal(clone.bias, m.bias)
    assert clone.bias.data_ptr() != m.bias.data_ptr()


def test_linear_state_dict_carries_the_rotation_group():
    """Codes mean nothing without the group that their rows were rotated in."""
    m = Mx4ConvRotLinear(256, 3, device="cpu", convrot_groupsize=16)
    clone = Mx4ConvRotLinear(256, 3, device="cpu")
    assert clone.groupsize == 256
    clone.load_state_dict(m.state_dict())
    assert clone.groupsize == 16
    block = torch.nn.Sequential(Mx4ConvRotLinear(64, 2, device="cpu", convrot_groupsize=0))
    other = torch.nn.Sequential(Mx4ConvRotLinear(64, 2, device="cpu"))
    other.load_state_dict(block.state_dict())
    assert other[0].groupsize == 0
    old = {k: v for k, v in m.state_dict().items() if k != "convrot_groupsize"}       # written without it
    keep = Mx4ConvRotLinear(256, 3, device="cpu", convrot_groupsize=64)
    keep.load_state_dict(old)
    assert keep.groupsize == 64
    for bad in (32, 256):
        with pytest.raises(RuntimeError, match="convrot_groupsize"):
            Mx4ConvRotLinear(64, 2, device="cpu").load_state_dict({**block[0].state_dict(), "convrot_groupsize": torch.tensor(bad)})


def test_prefill_that_fails_reserves_no_tokens():
    from _int4.mx4_layers import Mx4KVCache, Mx4SelfAttention
    block = Mx4SelfAttention(64, 2, 1, 64, device="cpu")
    cache = Mx4KVCache(4, 1, 64, page=16, device="cpu")
    seq = cache.add()
    with pytest.raises(ValueError):
        block.prefill(torch.zeros(5, 64), cache, seq)             # (not on a CUDA device)
    assert cache.length(seq) == 0 and cache.slots(seq) == []
