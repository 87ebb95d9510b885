"""Attention over selected blocks against its definition in 64 bits over all pairs
of queries and keys."""

import pytest
import torch

import flagsparse_amd as fs

from ._blocks_helpers import BLOCK_DTYPES, BLOCK_IDS, Case, assert_within, oracle, random_blocks, randn

pytestmark = pytest.mark.gpu

# few rows: one token a workgroup; many: a workgroup's tokens share what they select
FEW = [
    # new, lengths, heads, group, width, block, top, page
    ([1, 1, 1], [1, 64, 777], 2, 4, 64, 64, 5, 0),
    ([3, 0, 7, 1], [3, 40, 129, 500], 3, 1, 128, 32, 8, 0),
    ([5, 2], [700, 65], 2, 16, 128, 64, 16, 16),
    ([4], [300], 1, 17, 80, 128, 3, 64),
    ([2, 9], [95, 33], 2, 5, 40, 32, 7, 32),
    ([1, 2], [2100, 90], 2, 40, 96, 1024, 2, 256),
    ([6], [4], 2, 2, 64, 64, 2, 0),  # more queries than keys: the first ones see none
    ([2, 3], [0, 3], 2, 2, 64, 64, 2, 16),
]
MANY = [
    ([1100, 0, 250, 1], [1100, 30, 260, 70], 4, 2, 64, 64, 6, 0),
    ([700, 333], [900, 1333], 4, 4, 128, 64, 9, 0),
    ([2049], [2049], 2, 3, 80, 32, 12, 0),
    ([500, 600], [1000, 640], 4, 1, 128, 32, 5, 16),
    ([1300], [1500], 4, 16, 64, 128, 4, 64),
    ([600, 500], [600, 500], 4, 12, 32, 256, 2, 0),
    ([430, 600], [425, 640], 4, 5, 96, 64, 40, 128),
]


def _ids(cases):
    return ["x".join(map(str, c[2:])) for c in cases]


@pytest.mark.parametrize("dtype", BLOCK_DTYPES, ids=BLOCK_IDS)
@pytest.mark.parametrize("sizes", FEW, ids=_ids(FEW))
def test_few(sizes, dtype):
    new, lengths, heads, group, width, block, top, page = sizes
    case = Case(new, lengths, heads, group, width, block, dtype, 1, page)
    blocks = random_blocks(new, lengths, heads, top, block, 5)
    out, lse = fs.flagsparse_block_attention(case.q, case.k, case.v, blocks, case.seqs, return_lse=True)
    found = oracle(case, blocks, width**-0.5)
    assert_within(lse, found, "lse")
    assert_within(out, found, "out")


@pytest.mark.parametrize("dtype", BLOCK_DTYPES, ids=BLOCK_IDS)
@pytest.mark.parametrize("sizes", MANY, ids=_ids(MANY))
def test_many(sizes, dtype):
    new, lengths, heads, group, width, block, top, page = sizes
    assert sum(new) * heads > 4096
    case = Case(new, lengths, heads, group, width, block, dtype, 2, page, tail=3)
    blocks = random_blocks(new, lengths, heads, top, block, 6, extra=3)
    out, lse = fs.flagsparse_block_attention(case.q, case.k, case.v, blocks, case.seqs, return_lse=True)
    found = oracle(case, blocks, width**-0.5)
    assert_within(lse, found, "lse")
    assert_within(out, found, "out")
    assert not out[-3:].any() and bool((lse[-3:] == -float("inf")).all())  # tokens of no sequence


@pytest.mark.parametrize("tokens", [5, 2100], ids=["few", "many"])
@pytest.mark.parametrize("width", [136, 256])
@pytest.mark.parametrize("dtype", BLOCK_DTYPES[:2], ids=BLOCK_IDS[:2])
def test_wide(tokens, width, dtype):
    case = Case([tokens], [tokens + 70], 2, 4, width, 64, dtype, 3)
    blocks = random_blocks([tokens], [tokens + 70], 2, 6, 64, 7)
    out, lse = fs.flagsparse_block_attention(case.q, case.k, case.v, blocks, case.seqs, 0.11, return_lse=True)
    found = oracle(case, blocks, 0.11)
    assert_within(lse, found, "lse")
    assert_within(out, found, "out")


GRAD = [
    ([1], [1], 1, 1, 64, 64, 1),
    ([70, 0, 3], [70, 0, 5], 2, 2, 64, 64, 2),
    ([300, 129], [300, 129], 2, 4, 128, 64, 4),
    ([257], [300], 3, 1, 80, 32, 5),
    ([200, 31, 1], [200, 40, 77], 2, 5, 64, 32, 3),
    ([150], [150], 2, 16, 128, 128, 2),
    ([2500], [2500], 1, 2, 64, 64, 6),  # the first block's list in several pieces
    ([190], [512], 1, 33, 40, 256, 2),
]


@pytest.mark.parametrize("dtype", BLOCK_DTYPES, ids=BLOCK_IDS)
@pytest.mark.parametrize("sizes", GRAD, ids=_ids(GRAD))
def test_grad(sizes, dtype):
    new, lengths, heads, group, width, block, top = sizes
    case = Case(new, lengths, heads, group, width, block, dtype, 4, tail=2, key_tail=5)
    blocks = random_blocks(new, lengths, heads, top, block, 8, extra=2)
    grad = randn(case.q.shape, dtype, 9)
    scale = width**-0.5
    out, lse = fs.flagsparse_block_attention(case.q, case.k, case.v, blocks, case.seqs, return_lse=True)
    dq, dk, dv = fs.flagsparse_block_attention_grad(grad, case.q, case.k, case.v, blocks, case.seqs, out, lse)
    found = oracle(case, blocks, scale, grad)
    assert_within(dq, found, "dq")
    assert_within(dv, found, "dv")
    assert_within(dk, found, "dk")
    assert not dq[-2:].any() and not dk[-5:].any() and not dv[-5:].any()  # of no sequence


@pytest.mark.parametrize("width", [192, 256])
@pytest.mark.parametrize("block", [32, 64])
@pytest.mark.parametrize("dtype", BLOCK_DTYPES[:2], ids=BLOCK_IDS[:2])
def test_grad_wide(width, block, dtype):
    case = Case([333], [350], 2, 2, width, block, dtype, 5)
    blocks = random_blocks([333], [350], 2, 4, block, 9)
    grad = randn(case.q.shape, dtype, 10)
    out, lse = fs.flagsparse_block_attention(case.q, case.k, case.v, blocks, case.seqs, 0.07, return_lse=True)
    got = fs.flagsparse_block_attention_grad(grad, case.q, case.k, case.v, blocks, case.seqs, out, lse, 0.07)
    found = oracle(case, blocks, 0.07, grad)
    for t, name in zip(got, ("dq", "dk", "dv")):
        assert_within(t, found, name)


@pytest.mark.parametrize("tokens", [3, 70])
@pytest.mark.parametrize("group", [96, 97, 128])
@pytest.mark.parametrize("width", [128, 256])
def test_large_groups(tokens, group, width):
    """One key-value head of many query heads: a token's rows take several waves, or more than a workgroup has."""
    case = Case([tokens], [tokens + 130], 64 if tokens > 3 else 1, group, width, 64, torch.bfloat16, 11)
    if tokens > 3:
        assert tokens * case.heads > 4096
    blocks = random_blocks([tokens], [tokens + 130], case.heads, 3, 64, 12)
    out, lse = fs.flagsparse_block_attention(case.q, case.k, case.v, blocks, case.seqs, return_lse=True)
    found = oracle(case, blocks, width**-0.5)
    assert_within(lse, found, "lse")
    assert_within(out, found, "out")
    if tokens > 3 or (group > 96 and width > 128):  # (the gradient of such groups is refused)
        return
    grad = randn(case.q.shape, torch.bfloat16, 13)
    got = fs.flagsparse_block_attention_grad(grad, case.q, case.k, case.v, blocks, case.seqs, out, lse)
    found = oracle(case, blocks, width**-0.5, grad)
    for t, name in zip(got, ("dq", "dk", "dv")):
        assert_within(t, found, name)


@pytest.mark.parametrize("group", [1, 3])
def test_many_blocks_in_several_windows(group):
    """More blocks than a workgroup's table holds at a time."""
    tokens, length = 2100, 60000
    case = Case([tokens], [length], 2, group, 32, 32, torch.bfloat16, 14)
    blocks = random_blocks([tokens], [length], 2, 5, 32, 15)
    out, lse = fs.flagsparse_block_attention(case.q, case.k, case.v, blocks, case.seqs, return_lse=True)
    rows = torch.arange(0, tokens, 97)
    for t in rows.tolist():
        p = length - tokens + t
        one = Case([1], [p + 1], 2, group, 32, 32, torch.bfloat16, 14)
        one.q, one.packed_k, one.packed_v = case.q[t : t + 1], case.packed_k[: p + 1], case.packed_v[: p + 1]
        found = oracle(one, blocks[t : t + 1], 32**-0.5)
        assert_within(lse[t : t + 1], found, "lse")
        assert_within(out[t : t + 1], found, "out")
