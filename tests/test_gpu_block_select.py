"""Summaries of blocks and their selection against the definitions in 64 bits."""

import pytest
import torch

import flagsparse_amd as fs

from ._blocks_helpers import BLOCK_DTYPES, BLOCK_IDS, Case, randn, select_oracle
from ._rows_helpers import TINY, UNIT

pytestmark = pytest.mark.gpu


def _means_oracle(case, most):
    """(means, bound of the error): n values added in 32 bits, a division, a rounding."""
    u = UNIT[case.dtype]
    want = torch.zeros((len(case.lengths), most, case.heads, case.width), dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(want)
    row = 0
    for b, n in enumerate(case.lengths):
        for i in range(min(most, -(-n // case.block))):
            keys = case.packed_k[row + i * case.block : row + min((i + 1) * case.block, n)].double()
            want[b, i] = keys.mean(0)
            size = (keys.shape[0] + 2) * 2.0**-24 * keys.abs().mean(0)
            bound[b, i] = size + u * (want[b, i].abs() + size) + TINY[case.dtype]
        row += n
    return want, bound


MEANS = [
    ([1, 64, 777], 2, 64, 64, 0),
    ([0, 33, 2000], 3, 128, 32, 0),
    ([500, 0, 129], 1, 80, 64, 16),
    ([1025, 5], 2, 256, 128, 64),
    ([3000], 2, 8, 1024, 32),
]


@pytest.mark.parametrize("dtype", BLOCK_DTYPES, ids=BLOCK_IDS)
@pytest.mark.parametrize("sizes", MEANS, ids=["x".join(map(str, c[1:])) for c in MEANS])
def test_means(sizes, dtype):
    lengths, heads, width, block, page = sizes
    if dtype == torch.float32:
        width = min(width, 128)
    case = Case([0] * len(lengths), lengths, heads, 1, width, block, dtype, 1, page)
    most = -(-max(lengths) // block) + 1
    got = fs.flagsparse_block_means(case.k, case.seqs, max_blocks=most)
    want, bound = _means_oracle(case, most)
    assert bool(((got.double() - want).abs() <= bound).all())
    # fewer blocks than there are: the first ones
    some = fs.flagsparse_block_means(case.k, case.seqs, max_blocks=1)
    assert torch.equal(some, got[:, :1])


@pytest.mark.parametrize("page", [0, 64])
@pytest.mark.parametrize("single", [False, True])
def test_means_update(page, single):
    lengths, start = [200, 64, 130, 5], [199, 63, 64, 5]
    case = Case([1] * 4, lengths, 2, 1, 64, 64, torch.bfloat16, 2, page, single=single)
    whole = fs.flagsparse_block_means(case.k, case.seqs, max_blocks=4)
    kept = torch.full_like(whole, 7.0)
    got = fs.flagsparse_block_means(case.k, case.seqs, start=torch.tensor(start, dtype=torch.int32).cuda(), out=kept)
    assert got is kept
    want = torch.full_like(whole, 7.0)
    want[0, 3], want[1, 0], want[2, 1:3] = whole[0, 3], whole[1, 0], whole[2, 1:3]  # the last has no new key
    assert torch.equal(got, want)


SELECT = [
    # new, lengths, heads, group, width, block, top, first, recent
    ([1, 1, 1], [1, 640, 3000], 2, 4, 64, 64, 8, 1, 1),
    ([300, 0, 17], [300, 50, 2017], 3, 1, 128, 32, 16, 1, 1),
    ([65], [4000], 2, 16, 80, 32, 12, 2, 3),
    ([40], [33000], 1, 3, 64, 64, 24, 0, 1),  # more blocks than are scored at a time
    ([20, 3], [18, 9], 2, 2, 64, 64, 4, 1, 1),  # queries before the first key
    ([2], [30000], 1, 8, 128, 32, 128, 5, 9),
    ([33], [700], 2, 2, 8, 64, 2, 1, 1),  # nothing chosen by score
    ([16], [5000], 1, 2, 40, 32, 6, 0, 6),
]


@pytest.mark.parametrize("dtype", BLOCK_DTYPES, ids=BLOCK_IDS)
@pytest.mark.parametrize("sizes", SELECT, ids=["x".join(map(str, c[2:])) for c in SELECT])
def test_select(sizes, dtype):
    new, lengths, heads, group, width, block, top, first, recent = sizes
    most = -(-max(lengths) // block)
    q = randn((sum(new) + 2, heads * group, width), dtype, 3)
    means = randn((len(new), most, heads, width), dtype, 4)
    case = Case(new, lengths, 1, 1, 8, block, torch.float16, 5, tail=2)
    got = fs.flagsparse_block_select(q, means, case.seqs, top, first, recent)
    seq, pos, _ = case.positions()
    want = select_oracle(q, means, seq, pos, block, top, first, recent)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", BLOCK_DTYPES, ids=BLOCK_IDS)
@pytest.mark.parametrize("sizes", [(4, 64, 64, 8, 1, 1), (16, 128, 32, 100, 3, 4), (1, 80, 64, 4, 1, 3)],
                         ids=lambda c: "x".join(map(str, c)))
def test_select_of_single_tokens(sizes, dtype):
    """One query a sequence, without offsets: each wave takes a part of the blocks."""
    group, width, block, top, first, recent = sizes
    lengths = [0, 1, block * 3, 20011, 70000 if block == 64 else 9000, 640]
    most = -(-max(lengths) // block)
    q = randn((6, 2 * group, width), dtype, 3)
    means = randn((6, most, 2, width), dtype, 4)
    case = Case([1] * 6, lengths, 1, 1, 8, block, torch.float16, 5, page=64, single=True)
    got = fs.flagsparse_block_select(q, means, case.seqs, top, first, recent)
    seq, pos = list(range(6)), [n - 1 for n in lengths]
    assert torch.equal(got, select_oracle(q, means, seq, pos, block, top, first, recent))


def test_select_wide():
    case = Case([70], [4000], 1, 1, 8, 32, torch.float16, 5)
    for dtype in BLOCK_DTYPES[:2]:
        q, means = randn((70, 6, 256), dtype, 3), randn((1, 125, 2, 256), dtype, 4)
        seq, pos, _ = case.positions()
        assert torch.equal(fs.flagsparse_block_select(q, means, case.seqs, 9),
                           select_oracle(q, means, seq, pos, 32, 9, 1, 1))


@pytest.mark.parametrize("tokens", [1, 20])
def test_select_ties_and_what_is_not_a_number(tokens):
    """Equal scores go to the lower block, both zeros are equal, NaN comes last."""
    case = Case([tokens], [64 * 40], 1, 1, 8, 64, torch.float16, 6, single=tokens == 1)
    q = torch.ones((tokens, 1, 8), device="cuda")
    means = torch.zeros((1, 40, 1, 8), device="cuda")
    means[0, 5:20] = 1.0
    means[0, 20:25] = -0.0
    means[0, 25] = float("nan")
    means[0, 26] = float("inf")
    means[0, 27] = -float("inf")
    seq, pos, _ = case.positions()
    for top in (4, 9, 17, 25, 38, 40):
        got = fs.flagsparse_block_select(q, means, case.seqs, top)
        assert torch.equal(got, select_oracle(q, means, seq, pos, 64, top, 1, 1)), top


def test_select_near_ties_go_by_64_bits():
    """Scores that 32-bit sums cannot tell apart."""
    case = Case([17], [64 * 30], 1, 1, 8, 64, torch.float16, 6)
    q = torch.zeros((17, 1, 8), device="cuda")
    q[:] = torch.tensor([1.0, 2.0**-40, 0, 0, 0, 0, 0, 0], device="cuda")
    means = torch.zeros((1, 30, 1, 8), device="cuda")
    means[0, :, 0, 0] = 1000.0
    order = torch.randperm(30, generator=torch.Generator().manual_seed(1))
    means[0, :, 0, 1] = order.float().cuda()
    seq, pos, _ = case.positions()
    got = fs.flagsparse_block_select(q, means, case.seqs, 9)
    assert torch.equal(got, select_oracle(q, means, seq, pos, 64, 9, 1, 1))
