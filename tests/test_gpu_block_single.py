"""The selection's kernel of single tokens: many blocks, which its waves share."""

import pytest
import torch

import flagsparse_amd as fs
from flagsparse_amd import _lib

from ._blocks_helpers import BLOCK_DTYPES, BLOCK_IDS, Case, randn, select_oracle

pytestmark = pytest.mark.gpu
SINGLE = "block_select_single_kernel"

SIZES = [
    # new, lengths, heads, group, width, block, top, first, recent
    ([1, 1, 1], [20480, 22000, 3], 2, 4, 64, 32, 8, 1, 1),
    ([3, 2, 0, 1], [30000, 33, 9, 21000], 3, 2, 128, 32, 100, 3, 4),
    ([1], [32 * 700], 1, 16, 80, 32, 4, 0, 1),
    ([5], [64 * 3001 - 7], 2, 1, 40, 64, 128, 5, 9),
    ([1, 2], [64 * 641, 64 * 640 + 1], 4, 3, 8, 64, 2, 1, 1),  # nothing chosen by score
    ([1], [1024 * 650], 1, 2, 96, 1024, 33, 2, 2),
]


@pytest.mark.parametrize("dtype", BLOCK_DTYPES, ids=BLOCK_IDS)
@pytest.mark.parametrize("sizes", SIZES, ids=["x".join(map(str, c[2:])) for c in SIZES])
def test_select_of_few_tokens_among_many_blocks(sizes, dtype):
    new, lengths, heads, group, width, block, top, first, recent = sizes
    most = -(-max(lengths) // block)
    assert most >= 640
    q = randn((sum(new) + 1, heads * group, width), dtype, 3)
    means = randn((len(new), most, heads, width), dtype, 4)
    seqs = _seqs(new, lengths, block)
    got = fs.flagsparse_block_select(q, means, seqs, top, first, recent)
    assert _lib.last_kernel() == SINGLE
    seq = [b for b, n in enumerate(new) for _ in range(n)] + [-1]
    pos = [p for n, m in zip(lengths, new) for p in range(n - m, n)] + [-1]
    assert torch.equal(got, select_oracle(q, means, seq, pos, block, top, first, recent))


def _seqs(new, lengths, block):
    """Sequences by their lengths alone: the selection reads no keys."""
    offsets = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32).cuda()
    pages = torch.zeros((len(new), 1), dtype=torch.int32, device="cuda")
    return fs.prepare_block_sequences(block, offsets, pages=pages,
                                      k_lengths=torch.tensor(lengths, dtype=torch.int32).cuda())


def test_ties_and_what_is_not_a_number_among_many_blocks():
    """Equal scores go to the lower block, both zeros are equal, NaN comes last, wherever the
    waves' parts of the blocks end."""
    case = Case([1], [64 * 800], 1, 1, 8, 64, torch.float16, 6, single=True)
    q = torch.ones((1, 1, 8), device="cuda")
    means = torch.zeros((1, 800, 1, 8), device="cuda")
    means[0, 90:130] = 1.0
    means[0, 300:330] = -0.0
    means[0, 400:420] = float("nan")
    means[0, 420] = float("inf")
    means[0, 421:780] = -float("inf")
    seq, pos, _ = case.positions()
    for top in (4, 9, 41, 42, 43, 100, 128):
        got = fs.flagsparse_block_select(q, means, case.seqs, top)
        assert _lib.last_kernel() == SINGLE
        assert torch.equal(got, select_oracle(q, means, seq, pos, 64, top, 1, 1)), top
    means[0] = float("nan")
    for top in (4, 128):
        got = fs.flagsparse_block_select(q, means, case.seqs, top)
        assert torch.equal(got, select_oracle(q, means, seq, pos, 64, top, 1, 1)), top


@pytest.mark.parametrize("blocks, tokens, width, single", [
    (639, 1, 64, False), (640, 1, 64, True), (640, 64, 64, True), (640, 65, 64, False), (640, 1, 136, False),
])
def test_either_side_of_the_rule(blocks, tokens, width, single):
    q = randn((tokens, 8, width), torch.bfloat16, 7)
    means = randn((1, blocks, 8, width), torch.bfloat16, 8)
    length = blocks * 32 - 5
    got = fs.flagsparse_block_select(q, means, _seqs([tokens], [length], 32), 12)
    assert (_lib.last_kernel() == SINGLE) == single
    pos = list(range(length - tokens, length))
    assert torch.equal(got, select_oracle(q, means, [0] * tokens, pos, 32, 12, 1, 1))
