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
