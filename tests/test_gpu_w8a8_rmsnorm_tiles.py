"""GPU tests of the W8A8 linear behind a norm at the sizes that take the GEMM's wide tiles.

256 x 256 tiles are the choice from half as many of them as pairs of multiprocessors on, in bf16 with N a multiple
of 8 256 x 192 ones where their waves are shorter by more than a tenth. Sizes are made from the device's number of
multiprocessors and the rule is repeated here, so that each case is known to reach its tiles. Definition and tolerance
of test_gpu_w8a8_rmsnorm.py for some of the rows; all rows bit for bit those of the same call in pieces of 16 rows,
another kernel.
"""
import pytest
import torch

from test_gpu_w8a8_rmsnorm import check, rows, weight

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import _int4
    assert _int4.is_available()
    return _int4


def tile_columns(m, n, dtype):
    pairs = torch.cuda.get_device_properties(0).multi_processor_count // 2
    wide, narrow = -(-m // 256) * -(-n // 256), -(-m // 256) * -(-n // 192)
    if 2 * wide < pairs:
        return 128
    return 192 if dtype == "bf16" and n % 8 == 0 and -(-narrow // pairs) * 5 < -(-wide // pairs) * 6 else 256


# columns of a tile, rows, N by the number of pairs of multiprocessors, K, group, type
CASES = [(192, 509, lambda p: 192 * (p // 2 - 5), 512, 64, "bf16"), (192, 511, lambda p: 192 * (p // 2 - 5) + 8, 512, 64, "bf16"),
         (192, 513, lambda p: 192 * (p // 3) - 120, 256, 256, "bf16"), (192, 255, lambda p: 192 * (p - 2) + 136, 512, 256, "bf16"),
         (192, 400, lambda p: 192 * (p // 2 - 3), 3840, 256, "bf16"), (192, 301, lambda p: 192 * (p // 2 - 3) - 64, 5120, 256, "bf16"),
         (256, 512, lambda p: 256 * (p // 2) - 8, 512, 64, "bf16"), (256, 511, lambda p: 256 * (p // 2), 3840, 256, "bf16"),
         (256, 257, lambda p: 256 * (p // 2) - 88, 4096, 64, "bf16"), (256, 509, lambda p: 256 * (p // 2) - 101, 256, 64, "bf16"),
         (256, 510, lambda p: 256 * (p // 2) - 24, 512, 256, "f32"), (256, 333, lambda p: 256 * (p // 2) - 3, 512, 64, "f16"),
         (128, 509, lambda p: 200 * (p // 8), 512, 64, "bf16"), (128, 300, lambda p: 96 * (p // 8) + 5, 512, 64, "f16")]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_wide_tiles(lib, case):
    columns, m, width, k, group, dtype = CASES[case]
    n = width(torch.cuda.get_device_properties(0).multi_processor_count // 2)
    assert tile_columns(m, n, dtype) == columns
    x, r = rows(m, k, dtype, case), rows(m, k, dtype, case + 100)
    g = torch.Generator().manual_seed(case)
    gain, bias = (1 + 0.2 * torch.randn(k, generator=g)).bfloat16().cuda(), torch.randn(n, generator=g).cuda()
    w, ws = weight(n, k, case)
    out, hidden = lib.convrot_w8a8_linear_rmsnorm(x, w, ws, bias, gain, r, convrot_groupsize=group)
    for at in range(0, m, 16):
        part, h = lib.convrot_w8a8_linear_rmsnorm(x[at:at + 16], w, ws, bias, gain, r[at:at + 16], convrot_groupsize=group)
        assert torch.equal(part, out[at:at + 16]) and torch.equal(h, hidden[at:at + 16]), at
    some = torch.tensor([0, 1, 127, 128, 254, m // 2, m - 2, m - 1], device="cuda")
    check((out[some], hidden[some]), x[some], r[some], gain, w, ws, bias, group)
    plain, same = lib.convrot_w8a8_linear_rmsnorm(x, w, ws, convrot_groupsize=group)
    assert same is x
    check((plain[some], x[some]), x[some], None, None, w, ws, None, group)
