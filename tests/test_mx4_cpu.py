"""MX4 host logic without a GPU: the format's restatement, scale tiles, refusals."""
import ctypes

import numpy as np
import pytest
import torch

import _int4
from _int4 import cuda_loader, mx4
from oracle import mx4_oracle as orc


@pytest.fixture(scope="module")
def lib():
    return cuda_loader.library()


def test_encode_is_nearest_with_ties_to_even():
    x = np.zeros((1, 32))
    x[0, 0] = 6.0                                             # amplitude in [4, 8): unit scale
    probe = np.concatenate([orc.MIDPOINTS, orc.GRID, [5.1, 7.9, 0.2, 2.6]])
    x[0, 1:1 + len(probe)] = probe
    c, e = orc.encode(x)
    assert e[0, 0] == 127
    want = [0, 2, 2, 4, 4, 6, 6] + list(range(8)) + [7, 7, 0, 5]
    assert c[0, 1:1 + len(probe)].tolist() == want


def test_scale_of_tiny_huge_zero_and_bad_blocks():
    x = np.zeros((1, 6 * 32), np.float32)
    x[0, 32] = 1e-45
    x[0, 64] = 3e38
    x[0, 96] = np.inf
    x[0, 128] = np.nan
    x[0, 160] = 2.0 ** -126
    _, e = orc.encode(x)
    assert e[0].tolist() == [0, 0, 252, 255, 255, 0]


def test_rotation_is_an_involution_and_matches_the_matrix():
    x = np.random.default_rng(0).standard_normal((3, 512)).astype(np.float32)
    for g in (16, 64, 256):
        np.testing.assert_allclose(orc.rotate(x, g), orc.rotate64(x, g), atol=2e-6)
        np.testing.assert_allclose(orc.rotate64(orc.rotate64(x, g), g), x, atol=1e-12)


@pytest.mark.parametrize("rows,k", [(1, 32), (5, 96), (128, 128), (129, 160), (300, 4096)])
def test_scale_tiles_round_trip(rows, k):
    s = torch.randint(0, 256, (rows, k // 32), dtype=torch.uint8)
    t = _int4.mx4_scales_from_rows(s)
    assert t.shape == mx4._scale_tiles(rows, k)
    assert torch.equal(_int4.mx4_scales_to_rows(t, rows, k), s)
    assert np.array_equal(orc.untile(t.numpy(), rows, k), s.numpy())
    r, b = rows - 1, k // 32 - 1
    assert t[r // 128, b // 4, (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4] == s[r, b]


def test_python_entries_refuse_cpu_tensors_and_bad_arguments():
    x = torch.zeros(2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        _int4.quantize_convrot_mx4(x, 64)
    for bad, group, text in ((torch.zeros(2, 48), 16, "multiple of 32"), (x, 32, "convrot_groupsize"), (torch.zeros(2, 96), 64, "not divisible"),
                             (x.double(), 64, "unsupported dtype")):
        with pytest.raises(ValueError, match=text):
            _int4.quantize_convrot_mx4(bad, group)
    with pytest.raises(TypeError):
        _int4.quantize_convrot_mx4(None, 64)
    with pytest.raises(TypeError):
        _int4.quantize_convrot_mx4(x, "64")
    codes = torch.zeros(3, 64, dtype=torch.uint8)
    scales = torch.zeros(1, 1, 512, dtype=torch.uint8)
    for call, text in ((lambda: _int4.dequantize_convrot_mx4(codes, scales), "CUDA"),
                       (lambda: _int4.dequantize_convrot_mx4(codes, scales[:, :, :8].contiguous()), "do not match"),
                       (lambda: _int4.convrot_mx4_linear(torch.zeros(2, 128), codes, scales, torch.zeros(3), 64), "CUDA"),
                       (lambda: _int4.convrot_mx4_linear(torch.zeros(2, 128), codes, scales, torch.zeros(4), 64), "bias"),
                       (lambda: _int4.convrot_mx4_linear(torch.zeros(2, 64), codes, scales), "does not match")):
        with pytest.raises(ValueError, match=text):
            call()
    with pytest.raises(ValueError, match="power of two"):
        _int4.mx4_cache_empty(1, 48, 1, 64, device="cpu")
    with pytest.raises(ValueError, match="head_dim"):
        _int4.mx4_cache_empty(1, 16, 1, 96, device="cpu")
    with pytest.raises(ValueError, match="tiles"):
        _int4.mx4_scales_to_rows(torch.zeros(1, 1, 512, dtype=torch.uint8), 129, 128)


def refuse(lib, rc, text):
    assert rc == -1
    assert text in lib.ck_convrot_last_error()


def test_c_entries_refuse_before_any_launch(lib):
    q = lib.ck_mx4_quant
    refuse(lib, q(16, 1, 64, 16, 16, 2, 48, 16, None), b"K must be")
    refuse(lib, q(16, 1, 64, 16, 16, 2, 64, 32, None), b"G must be")
    refuse(lib, q(16, 1, 96, 16, 16, 2, 96, 64, None), b"multiple of G")
    refuse(lib, q(16, 3, 64, 16, 16, 2, 64, 64, None), b"dtype")
    refuse(lib, q(16, 1, 32, 16, 16, 2, 64, 64, None), b"ldx")
    refuse(lib, q(17, 1, 64, 16, 16, 2, 64, 64, None), b"aligned")
    refuse(lib, q(16, 1, 64, 8, 16, 2, 64, 64, None), b"aligned")
    refuse(lib, q(0, 1, 64, 16, 16, 2, 64, 64, None), b"null")
    refuse(lib, q(16, 1, 64, 16, 16, -1, 64, 64, None), b"negative")
    assert q(0, 1, 64, 0, 0, 0, 64, 64, None) == 0                                   # nothing to do
    lin = lib.ck_mx4_linear
    assert lib.ck_mx4_linear_workspace_size(8, 64) == 0
    need = lib.ck_mx4_linear_workspace_size(20, 64)
    assert need == 768 + 512
    refuse(lib, lin(16, 1, 64, 16, 16, 0, 0, 16, 20, 8, 64, 64, 256, need - 1, None), b"workspace")
    refuse(lib, lin(16, 1, 64, 16, 16, 0, 0, 16, 20, 8, 64, 64, 128, need, None), b"256-byte")
    refuse(lib, lin(16, 1, 64, 16, 16, 16, 7, 16, 4, 8, 64, 64, 0, 0, None), b"bias_dtype")
    refuse(lib, lin(16, 1, 64, 16, 16, 0, 0, 8, 4, 8, 64, 64, 0, 0, None), b"out must")
    refuse(lib, lin(16, 1, 63, 16, 16, 0, 0, 16, 4, 8, 64, 64, 0, 0, None), b"ldx")
    assert lin(16, 1, 64, 16, 16, 0, 0, 16, 4, 0, 64, 64, 0, 0, None) == 0
    app = lib.ck_mx4_cache_append
    refuse(lib, app(16, 16, 4, 2, 96, 16, 0, 16, 16, 1, 1, 1, 1, 1, 16, 3, None), b"head dimension")
    refuse(lib, app(16, 16, 4, 2, 64, 24, 0, 16, 16, 1, 1, 1, 1, 1, 16, 3, None), b"power of two")
    refuse(lib, app(16, 16, 4, 2, 64, 16, 256, 16, 16, 1, 1, 1, 1, 1, 16, 3, None), b"multiple of G")
    refuse(lib, app(16, 16, 4, 2, 64, 16, 64, 16, 16, 1, 1, 1, 1, 1, 0, 3, None), b"null")
    refuse(lib, app(8, 16, 4, 2, 64, 16, 64, 16, 16, 1, 1, 1, 1, 1, 16, 3, None), b"aligned")
    assert app(16, 16, 4, 2, 64, 16, 64, 0, 0, 1, 1, 1, 1, 1, 0, 0, None) == 0
    rd = lib.ck_mx4_cache_read
    refuse(lib, rd(16, 16, 4, 2, 64, 16, 64, 16, 3, 16, 8, 1, None), b"aligned")
    refuse(lib, rd(16, 16, 4, 2, 64, 16, 64, 16, 3, 16, 16, 9, None), b"dtype")
    att = lib.ck_mx4_attention

    def attention(dtype=1, hq=4, tq=1, b=2, out=16, table=16, ld=4, per=4, page=16):
        return att(16, dtype, 1, 1, 1, 16, 16, 8, page, table, ld, per, 16, out, b, tq, hq, 2, 64, 64,
                   ctypes.c_float(1.0), 0, 0, None)
    refuse(lib, attention(dtype=0), b"bf16")
    refuse(lib, attention(hq=3), b"multiple")
    refuse(lib, attention(tq=0), b"multiple")
    refuse(lib, attention(out=8), b"16 bytes")
    refuse(lib, attention(table=0), b"null")
    refuse(lib, attention(ld=3), b"block table")
    assert attention(b=0) == 0


def test_cache_pages_of_sequences():
    from _int4.mx4_layers import Mx4KVCache
    c = Mx4KVCache(5, 1, 64, page=16, device="cpu")
    a, b = c.add(), c.add()
    assert c.extend(a, 17) == list(range(16)) + [16]
    assert c.extend(b, 1) == [32]
    assert c.extend(a, 1) == [17] and c.length(a) == 18
    assert c.slots(a) == list(range(18))
    table, lens = c.tables([b, a])
    assert table.tolist() == [[2, -1], [0, 1]] and lens.tolist() == [1, 18]
    with pytest.raises(RuntimeError, match="free pages"):
        c.extend(b, 48)
    assert c.length(b) == 1
    c.free(a)
    assert c.extend(b, 63) == list(range(33, 48)) + list(range(0, 32)) + list(range(48, 64))
    assert c.tables([b])[0].tolist() == [[2, 0, 1, 3]]


def test_linear_module_refuses_and_shapes():
    from _int4.mx4_layers import Mx4ConvRotLinear, Mx4SelfAttention
    with pytest.raises(ValueError):
        Mx4ConvRotLinear(48, 8)
    m = Mx4ConvRotLinear(320, 24, convrot_groupsize=0)
    assert m.weight.shape == (24, 160) and m.weight_scale.shape == (1, 3, 512) and m.groupsize == 0
    assert Mx4ConvRotLinear(320, 24).groupsize == 64
    with pytest.raises(ValueError):
        Mx4SelfAttention(64, 5, 2, 64)
