"""GPU tests of the MX4 cache at unit numbers beyond 2^30."""
import pytest
import torch

from test_gpu_mx4 import mx  # noqa: F401

pytestmark = pytest.mark.gpu


def test_append_of_more_than_2_30_units(mx):  # noqa: F811
    """Keys and values broadcast over their tokens: 2 * T * 128 units, above 2^30. All slots
    but a few lie outside the cache."""
    t, heads, d, page = (1 << 22) + 37, 128, 128, 16
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(1, heads, d, generator=g).bfloat16().cuda() for _ in range(2))
    slots = torch.full((t,), -1, dtype=torch.int64, device="cuda")
    kept = torch.tensor([0, 1, t // 2, t - 2, t - 1], device="cuda")
    slots[kept] = torch.arange(5, device="cuda") * 7
    codes, scales = mx.mx4_cache_empty(3, page, heads, d)
    mx.convrot_mx4_cache_append(codes, scales, k.expand(t, -1, -1), v.expand(t, -1, -1), slots, 64)
    one_c, one_s = mx.mx4_cache_empty(3, page, heads, d)
    mx.convrot_mx4_cache_append(one_c, one_s, k.repeat(5, 1, 1), v.repeat(5, 1, 1), slots[kept], 64)
    assert torch.equal(codes, one_c) and torch.equal(scales, one_s)
