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


@pytest.mark.parametrize("every", [1, 9])
@pytest.mark.parametrize("t,d,hq,tokens", LONG)
def test_blocks_of_a_key_far_apart(mx, t, d, hq, tokens, every):
    """Blocks of 32 channels of one key whose scales lie up to 2^90 apart, and heads whose queries look at one block each:
    every block keeps its own precision, that of scale byte 0 included."""
    lens = [tokens]
    codes, scales, table = make_cache(mx, lens, 16, 2, d, 0, 35)
    blocks = d // 32
    step = 24 if blocks == 4 else 40
    low = [step * (blocks - 1 - c) - step * (blocks - 1) // 2 for c in range(blocks)]          # exponents added to the blocks'
    far = torch.zeros(codes.shape[0] * 16, dtype=torch.bool)
    far[::every] = True
    far = far.reshape(-1, 1, 16, 1).cuda()
    shift = torch.tensor(low, dtype=torch.int32, device="cuda")
    scales[:, 0] = torch.where(far, scales[:, 0].int() + shift, scales[:, 0].int()).clamp(1, 254).to(torch.uint8)
    g = torch.Generator().manual_seed(3)
    q = torch.zeros(1, t, hq, d)
    for h in range(hq):
        c = h % blocks
        q[:, :, h, 32 * c:32 * c + 32] = torch.randn(1, t, 32, generator=g) * 2.0 ** -low[c]
    q = q.bfloat16().cuda()
    mask = mx.tree_mask(trees(1, t, 6))[0].cuda()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def run(q, scales):
        out = mx.convrot_mx4_tree_attention(q, codes, scales, table, n, mask, convrot_groupsize=0)
        check(out, reference(q, codes, scales, table, lens, [t], mask, d ** -0.5, 0), q)
        again = mx.convrot_mx4_tree_attention(q, codes, scales, table, n, mask, convrot_groupsize=0)
        assert torch.equal(out.view(torch.int16), again.view(torch.int16))
    if every == 1:
        run(q, scales)
    else:
        # (ordinary keys beside them: queries that are moderate for both)
        run(q * torch.tensor([2.0 ** min(0, x) for x in low], device="cuda").repeat_interleave(32).bfloat16(), scales)
    # a block of scale byte 0, 2^-127, beside ordinary ones, and one that is NaN
    least = scales.clone()
    least[:, 0] = torch.where(far, scales[:, 0] * 0 + 127, scales[:, 0])
    least[:, 0, :, :, 1] = torch.where(far[..., 0], 0, least[:, 0, :, :, 1])
    q = torch.zeros(1, t, hq, d)
    q[..., 32:64] = torch.randn(1, t, hq, 32, generator=g) * 2.0 ** 124
    q = q.bfloat16().cuda()
    if every == 1:
        run(q, least)
        j = lens[0] - t - 3
        held = least.clone()
        held[int(table[0, j // 16]), 0, :, j % 16, 0] = 255
        assert mx.convrot_mx4_tree_attention(q, codes, held, table, n, mask, convrot_groupsize=0).isnan().all()


@pytest.mark.parametrize("up", [20, 34, 60, 90])
@pytest.mark.parametrize("t,d,hq,tokens", LONG)
def test_scores_of_any_finite_size(mx, t, d, hq, tokens, up):
    """Scores of 2^20 to 2^90 pick the largest; steps of their own fp32 values, 2^66 there, are far above 1."""
    lens = [tokens]
    codes, scales, table = make_cache(mx, lens, 16, 2, d, 64, 37)
    scales[:, 0] = (scales[:, 0].int() + up).clamp(max=254).to(torch.uint8)
    q = torch.randn(1, t, hq, d, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    mask = mx.tree_mask(trees(1, t, 6))[0].cuda()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for scale in (0.1, -0.3):
        out = mx.convrot_mx4_tree_attention(q, codes, scales, table, n, mask, softmax_scale=scale)
        ref, err = reference(q, codes, scales, table, lens, [t], mask, scale, 64)
        check(out, (ref, err), q)
        # (that tolerance grows with the scores, beyond the values: the means are finite and of the values' size)
        assert out.isfinite().all() and float(out.abs().max()) <= 16 * float(abs(ref).max())
