"""What the MX4 C entries refuse before any launch (no GPU needed)."""
import pytest

from _int4 import cuda_loader


@pytest.fixture(scope="module")
def lib():
    return cuda_loader.library()


def refuse(lib, rc, text):
    assert rc == -1
    assert text in lib.ck_convrot_last_error()


@pytest.mark.parametrize("group", [0, 64])
@pytest.mark.parametrize("dtype,size", [(0, 4), (1, 2), (2, 2)])
def test_dequant_refuses_an_unaligned_output(lib, group, dtype, size):
    """Values are stored 16 bytes at a time."""
    for at in (size, 8, 24):
        refuse(lib, lib.ck_mx4_dequant(16, 16, at, dtype, 3, 64, group, None), b"out must be 16-byte aligned")
    assert lib.ck_mx4_dequant(16, 16, 2, dtype, 0, 64, group, None) == 0             # nothing to do


@pytest.mark.parametrize("m", [4, 20])
def test_linear_refuses_a_bias_that_is_not_aligned_to_its_type(lib, m):
    for kind, at in ((0, 18), (1, 17), (2, 33)):
        refuse(lib, lib.ck_mx4_linear(16, 1, 64, 16, 16, at, kind, 16, m, 8, 64, 64, 256, 1 << 20, None), b"bias is not aligned")


def test_attention_refuses_tables_at_the_end_of_32_bit_positions(lib):
    """Token positions, and those of the chunks and groups that end behind the last token, are 32-bit numbers."""
    import ctypes

    def attention(per, page):
        return lib.ck_mx4_attention(16, 1, 1, 1, 1, 16, 16, 8, page, 16, per, per, 16, 16, 1, 1, 4, 2, 64, 64,
                                    ctypes.c_float(1.0), 0, 0, None)
    for per, page in ((2 ** 31 - 1, 1), (2 ** 27 - 1, 16), (2 ** 31 - 1000, 1), (2 ** 25, 64)):
        refuse(lib, attention(per, page), b"block table longer")
    refuse(lib, attention(2 ** 26 - 64, 32), b"workspace")                          # accepted as a length


def test_cache_shapes_that_the_kernels_do_not_take_are_value_errors():
    import torch

    import _int4
    slots = torch.zeros(1, dtype=torch.int64)
    for page, heads, text in ((48, 1, "power of two"), (1 << 17, 1, "power of two"), (16, 0, "heads")):
        codes = torch.empty(0, 2, heads, page, 32, dtype=torch.uint8)
        scales = torch.empty(0, 2, heads, page, 2, dtype=torch.uint8)
        kv = torch.zeros(1, heads, 64)
        with pytest.raises(ValueError, match=text):
            _int4.convrot_mx4_cache_read(codes, scales, slots)
        with pytest.raises(ValueError, match=text):
            _int4.convrot_mx4_cache_append(codes, scales, kv, kv, slots)
        with pytest.raises(ValueError, match=text):
            _int4.mx4_cache_empty(0, page, heads, 64, device="cpu")
