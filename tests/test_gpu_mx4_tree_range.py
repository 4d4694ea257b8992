"""GPU tests of the tree attention where scores or keys leave the ordinary range. Reference and tolerance of
test_gpu_mx4_tree.py; the larger sizes reach the kernel that takes 128 or 256 rows at a time.
"""
import pytest
import torch

from test_gpu_mx4_tree import check, make_cache, reference, trees

pytestmark = pytest.mark.gpu

SIZES = [(6, 128, 4), (50, 128, 64), (60, 64, 64), (16, 128, 64), (16, 64, 64)]        # nodes, D, query heads (on 2)

LONG = [(6, 128, 4, 1250), (50, 128, 64, 1250), (60, 64, 64, 1250), (16, 128, 16, 9000), (16, 64, 16, 20000)]     # and tokens


@pytest.fixture(scope="module")
def mx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import _int4
    assert _int4.is_available()
    return _int4


def slots_of(table, n):
    j = torch.arange(n)
    return (table[0].cpu().long()[j // 16] * 16 + j % 16).cuda()


@pytest.mark.parametrize("t,d,hq", SIZES)
def test_scores_that_jump_within_a_tile(mx, t, d, hq):
    """The largest score comes behind tokens of the same 128 whose weights are laid down already: they get a new scale."""
    lens = [1300]
    codes, scales, table = make_cache(mx, lens, 16, 2, d, 64, 31)
    slots = slots_of(table, lens[0])
    k, v = mx.convrot_mx4_cache_read(codes, scales, slots, torch.float32, 64)
    q = torch.randn(1, 1, 1, d, generator=torch.Generator().manual_seed(3)).cuda()
    # one direction for all rows and some tokens: scores of 0 to 60 that rise at places 20, 50, 70, 101 and 127 of a tile
    for tile in range(0, lens[0] - 128, 128):
        for step, at in enumerate((20, 50, 70, 101, 127)):
            k[tile + at] = q[0, 0] * d ** 0.5 / float((q * q).sum()) * (12.0 * (step + 1) + tile / 128)
    mx.convrot_mx4_cache_append(codes, scales, k, v, slots, 64)
    q = (q + 0.02 * torch.randn(1, t, hq, d, generator=torch.Generator().manual_seed(4)).cuda()).bfloat16()
    mask = mx.tree_mask(trees(1, t, 6))[0].cuda()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = mx.convrot_mx4_tree_attention(q, codes, scales, table, n, mask)
    check(out, reference(q, codes, scales, table, lens, [t], mask, d ** -0.5, 64), q)


@pytest.mark.parametrize("t,d,hq,tokens", LONG)
def test_tiny_queries_meet_huge_keys(mx, t, d, hq, tokens):
    """Queries of 2^-113 and keys of 2^104: scores that count, of rows whose factor is about the least normal number."""
    lens = [tokens]
    codes, scales, table = make_cache(mx, lens, 16, 2, d, 64, 33)
    scales[:, 0] = (scales[:, 0].int() + 104).clamp(max=254).to(torch.uint8)
    q = (torch.randn(1, t, hq, d, generator=torch.Generator().manual_seed(3)) * 2.0 ** -113).bfloat16().cuda()
    mask = mx.tree_mask(trees(1, t, 6))[0].cuda()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for scale in (2.0 ** -4, -2.0 ** -3, 2.0 ** 5):
        out = mx.convrot_mx4_tree_attention(q, codes, scales, table, n, mask, softmax_scale=scale)
        check(out, reference(q, codes, scales, table, lens, [t], mask, scale, 64), q)
