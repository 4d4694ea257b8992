"""GPU tests of the layers on the MX4 operators, alone and together.

The block's distance from float32 is the format's: a value keeps 1 + 1 significant
bits, a relative error of about 0.12 (root mean square) per quantized operand, so
a product of two quantized operands is about 0.16 off and the block, two such
products and an attention over a quantized cache, less than 0.4. Against the
block computed in 64 bits from the same quantized values the error is the
roundings' alone: bf16 outputs of the projection, of the attention and of the
block, 2^-9 each (root mean square under half the largest rounding).
"""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def layers():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from _int4 import mx4_layers
    return mx4_layers


def test_linear_from_linear(layers):
    import _int4
    lin = torch.nn.Linear(320, 100, device="cuda", dtype=torch.bfloat16)
    m = layers.Mx4ConvRotLinear.from_linear(lin)
    x = torch.randn(2, 7, 320, device="cuda").bfloat16()
    y = m(x)
    assert y.shape == (2, 7, 100)
    q, s = _int4.quantize_convrot_mx4(lin.weight.detach(), 64)
    assert torch.equal(y, _int4.convrot_mx4_linear(x, q, s, lin.bias.detach(), 64))
    clone = layers.Mx4ConvRotLinear(320, 100, device="cuda")
    clone.bias = clone.bias.to(torch.bfloat16)
    clone.load_state_dict(m.state_dict())
    assert torch.equal(clone(x), y)


def test_block_decodes_like_prefill(layers):
    """Tokens decoded one by one give what the same tokens give as one chunk."""
    torch.manual_seed(0)
    block = layers.Mx4SelfAttention(512, 8, 2, 64, device="cuda")
    for lin in (block.qkv, block.out):
        src = torch.nn.Linear(lin.in_features, lin.out_features, bias=False, device="cuda")
        made = layers.Mx4ConvRotLinear.from_linear(src)
        lin.weight, lin.weight_scale = made.weight, made.weight_scale
    x = torch.randn(40, 512, device="cuda").bfloat16()
    cache = layers.Mx4KVCache(8, 2, 64, page=16)
    whole = cache.add()
    want = block.prefill(x, cache, whole)
    step = cache.add()
    block.prefill(x[:23], cache, step)
    got = []
    at = 23
    for t in (1, 1, 4, 1, 10):
        slots = torch.tensor(cache.extend(step, t), device="cuda")
        table, lens = cache.tables([step])
        got.append(block(x[None, at:at + t], cache, slots, table, lens)[0])
        at += t
    got = torch.cat(got)
    rel = float((got.double() - want[23:].double()).norm() / want[23:].double().norm())
    # the attention's bf16 output differs by roundings; requantized to 4 bits for the
    # output projection a value near a midpoint may then take the other code
    assert rel < 0.03, rel


def test_example_runs(layers):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import mx4_decode
    r = mx4_decode.run(hidden=512, heads=8, kv_heads=2, head_dim=64, batch=3, prompt=90, chunk=32, tokens=5, page=16)
    assert r["rel"] < 0.4 and r["us_per_step"] > 0
