"""GPU test: the cache's tensors know that append writes them."""
import pytest
import torch

from test_gpu_mx4 import mx  # noqa: F401

pytestmark = pytest.mark.gpu


def test_append_raises_the_version_counters(mx):  # noqa: F811
    k = torch.randn(3, 2, 64, device="cuda")
    slots = torch.arange(3, device="cuda")
    codes, scales = mx.mx4_cache_empty(2, 16, 2, 64)
    was = codes._version, scales._version
    mx.convrot_mx4_cache_append(codes, scales, k, k, slots)
    assert codes._version > was[0] and scales._version > was[1]
    now = codes._version
    mx.convrot_mx4_cache_read(codes, scales, slots)
    assert codes._version == now
    with torch.inference_mode():                                                     # tensors without a version
        codes, scales = mx.mx4_cache_empty(2, 16, 2, 64)
        mx.convrot_mx4_cache_append(codes, scales, k, k, slots)
    mx.convrot_mx4_cache_append(codes, scales, k, k, slots)
    read, _ = mx.convrot_mx4_cache_read(codes, scales, slots, torch.float32)
    assert bool(read.isfinite().all()) and bool(read.any())
