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
