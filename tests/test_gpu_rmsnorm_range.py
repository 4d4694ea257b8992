"""GPU tests of the W8A8 linear behind a norm at the ends of fp32's range: finite rows whose squares, or whose
products with the gain, leave it. Definition and tolerance of test_gpu_w8a8_rmsnorm.py, relative to each row.
"""
import pytest
import torch

from test_gpu_w8a8_rmsnorm import DT, check, rows, weight

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import _int4
    assert _int4.is_available()
    return _int4


@pytest.mark.parametrize("m", [1, 5, 40])
@pytest.mark.parametrize("k,group", [(64, 16), (512, 256), (1088, 64), (3840, 256), (8192, 256)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_whose_squares_leave_the_range(lib, dtype, k, group, m):
    """Rows of 10^16 to some 10^38 beside ordinary ones, with and without a residual and a gain."""
    x = rows(m, k, "f32", m)
    peak = x.abs().amax(-1, keepdim=True)
    factor = torch.tensor([3.0e38, 1.0, 1e25, 3e19, 1e18, 1e16], device="cuda").repeat(m)[:m, None]
    x = torch.where(factor > 1, x / peak * factor, x).to(DT[dtype])
    w, ws = weight(72, k, 1)
    gain = (1 + 0.2 * torch.randn(k, generator=torch.Generator().manual_seed(2))).cuda()
    bias = torch.randn(72, generator=torch.Generator().manual_seed(3)).cuda()
    check(lib.convrot_w8a8_linear_rmsnorm(x, w, ws, bias, convrot_groupsize=group), x, None, None, w, ws, bias, group)
    check(lib.convrot_w8a8_linear_rmsnorm(x, w, ws, bias, gain, convrot_groupsize=group), x, None, gain, w, ws, bias, group)
    half = (x.float() / 2).to(x.dtype)
    check(lib.convrot_w8a8_linear_rmsnorm(half, w, ws, None, gain, half, convrot_groupsize=group), half, half, gain, w, ws, None, group)


@pytest.mark.parametrize("k,group", [(512, 256), (1088, 64), (8192, 256)])
def test_products_with_the_gain_that_leave_the_range(lib, k, group):
    """h g beyond fp32's range, where h g / rms(h) is within it; h's squares within it or not."""
    w, ws = weight(40, k, 1)
    for size, by in ((1e17, 1e24), (1e10, 1e30), (1e30, 1e10)):
        x = rows(3, k, "f32", 4)
        x = x / x.abs().amax(-1, keepdim=True) * size
        gain = (1 + 0.2 * torch.randn(k, generator=torch.Generator().manual_seed(2))).cuda() * by
        check(lib.convrot_w8a8_linear_rmsnorm(x, w, ws, None, gain, convrot_groupsize=group), x, None, gain, w, ws, None, group)


@pytest.mark.parametrize("k,group", [(512, 256), (1088, 64), (8192, 256)])
def test_rows_whose_squares_vanish(lib, k, group):
    """Without eps, rows of 10^-37 to 10^-19 are normalised like others, and a row of zeros is 0 / 0."""
    w, ws = weight(40, k, 1)
    x = rows(4, k, "f32", 4)
    x = x / x.abs().amax(-1, keepdim=True) * torch.tensor([1e-19, 1e-25, 1e-30, 1e-34], device="cuda")[:, None]
    check(lib.convrot_w8a8_linear_rmsnorm(x, w, ws, eps=0.0, convrot_groupsize=group), x, None, None, w, ws, None, group, eps=0.0)
    out, _ = lib.convrot_w8a8_linear_rmsnorm(torch.zeros_like(x), w, ws, eps=0.0, convrot_groupsize=group)
    assert out.isnan().all()


@pytest.mark.parametrize("k", [512, 1024, 8192])
def test_rows_that_are_not_finite_spoil_themselves_alone(lib, k):
    """Beside huge and ordinary rows, in blocks that take several rows at a time."""
    x = rows(23, k, "bf16", 5)
    plain, _ = lib.convrot_w8a8_linear_rmsnorm(x, *weight(40, k, 1), None)
    y = x.clone()
    y[3] *= 1e30
    y[7, 9], y[8, k - 1], y[20, 0] = float("inf"), float("nan"), float("-inf")
    out, _ = lib.convrot_w8a8_linear_rmsnorm(y, *weight(40, k, 1), None)
    bad = torch.zeros(23, dtype=torch.bool, device="cuda")
    bad[[7, 8, 20]] = True
    assert out[bad].isnan().all() and out[~bad].isfinite().all()
    bad[3] = True
    assert torch.equal(out[~bad], plain[~bad])
    check((out[3:4], y[3:4]), y[3:4], None, None, *weight(40, k, 1), None, 256)
