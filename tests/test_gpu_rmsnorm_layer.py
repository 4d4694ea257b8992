"""GPU tests of ``Int4ConvRotLinear.forward_rmsnorm`` for layers and rows that the one-pass kernel does not take."""
import pytest
import torch

from test_gpu_w8a8_rmsnorm import rows, weight

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def Layer():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import _int4
    assert _int4.is_available()
    from _int4.linear import Int4ConvRotLinear
    return Int4ConvRotLinear


def plain(layer, x, gain, residual, eps):
    h = x.double() if residual is None else x.double() + residual.double()
    y = h / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    return layer(((y * gain.double()) if gain is not None else y).to(x.dtype)), h.to(x.dtype)


@pytest.mark.parametrize("k,group,kind,other", [
    (16640, 256, torch.bfloat16, torch.bfloat16),                 # more inputs than the kernel's rows
    (1024, 1024, torch.bfloat16, torch.bfloat16),                 # a rotation group that it does not have
    (512, 256, torch.bfloat16, torch.float32)])                   # a residual stream of another type
def test_layers_that_forward_takes(Layer, k, group, kind, other):
    layer = Layer(k, 72, device="cuda", convrot_groupsize=group, mode="int8")
    q, s = weight(72, k, 1)
    layer._q.copy_(q)
    layer._qs.copy_(s)
    layer.bias.copy_(torch.randn(72, generator=torch.Generator().manual_seed(1)))
    x, r = rows(9, k, "f32", 1).to(kind), rows(9, k, "f32", 2).to(other)
    gain = (1 + 0.2 * torch.randn(k, generator=torch.Generator().manual_seed(2))).bfloat16().cuda()
    assert layer(x).isfinite().all()
    for residual in (None, r):
        out, hidden = layer.forward_rmsnorm(x, gain, residual)
        want, h = plain(layer, x, gain, residual, 1e-6)
        assert out.dtype == x.dtype and hidden.dtype == x.dtype
        # the layer rounds what the norm gives it to x's type and to int8, 2^-9 of a value and 1/254 of the row's
        # largest: rows rounded from 32 and from 64 bits differ by a step of either now and then
        assert (out.double() - want.double()).norm() <= 0.01 * want.double().norm()
        assert (hidden.double() - h.double()).abs().max() <= float(h.double().abs().max()) * torch.finfo(kind).eps
