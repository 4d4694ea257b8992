"""GPU tests of the few-row MX4 linear where K does not fill a cluster's slices: with 33 to
35, 41, 42 or 49 stages of 256 the last of eight ranks has none and sends zeros at once."""
import pytest

from test_gpu_mx4 import check_linear, mx  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 8, 20, 32, 64, 100])
@pytest.mark.parametrize("n,k", [(512, 8448), (1536, 8960), (512, 10496), (130, 12544)])
def test_linear_with_an_empty_slice(mx, m, n, k):  # noqa: F811
    for dtype in ("bf16", "f16") if m in (8, 20) else ("bf16",):
        check_linear(mx, m, n, k, 256, dtype, "bf16", seed=m + n)
