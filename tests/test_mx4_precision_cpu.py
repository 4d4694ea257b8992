"""The bound that the GPU tests of attention's precision use tells one f16 value an operand from two."""
import numpy as np
import pytest
import torch

from oracle import mx4_oracle as orc


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_bound_tells_one_f16_term_from_two(dtype):
    rng = np.random.default_rng(0)
    q = orc.rotate64(rng.standard_normal((128, 128)) * 1.5, 64)
    k, v = (orc.decode(*orc.quantize64(rng.standard_normal((300, 128)), 64)) for _ in range(2))
    scale = 128 ** -0.5
    s = q @ k.T * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    ref = p @ v / p.sum(-1, keepdims=True)
    to = {"bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    shares = [orc.rounded_apart(torch.from_numpy(orc.attention_f16_terms(q, k, v, scale, n)).to(to).double().numpy(), ref, dtype)
              for n in (1, 2)]
    assert shares[1] <= orc.MOST_APART[dtype] < shares[0] / 4, shares
