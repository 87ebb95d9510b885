"""Operators over blocks at their edges: scores that are all minus infinity, lists in
several pieces, windows of the gradients' walks, memory around the arrays."""

import pytest
import torch

import flagsparse_amd as fs

from ._blocks_helpers import BLOCK_DTYPES, BLOCK_IDS, Case, assert_within, oracle, random_blocks, randn

pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.mark.parametrize("page", [0, 16], ids=["rows", "pages"])
@pytest.mark.parametrize("tokens", [1, 9, 1100])
@pytest.mark.parametrize("dtype", BLOCK_DTYPES, ids=BLOCK_IDS)
def test_scores_that_are_all_minus_infinity(dtype, tokens, page):
    """Their softmax is 0 / 0; a row with other keys too leaves them out, one without keys is zero."""
    heads, group, width, block = 4, 2, 64, 64
    length = tokens + 200
    case = Case([tokens], [length], heads, group, width, block, dtype, 60, page)
    case.q[:, :, 0] = case.q[:, :, 0].abs() + 0.5
    blocks = random_blocks([tokens], [length], heads, 4, block, 61)
    blocks[0::5, :, :] = 1  # nothing but the block of the bad keys
    blocks[1::5, 0, :] = -1
    blocks[2::5, 1, :2] = 1
    seen = case.seen(blocks)
    bad = seen[:, :, 64:128].any(2) & ~seen[:, :, :64].any(2) & ~seen[:, :, 128:].any(2)  # (heads, tokens)
    empty = ~seen.any(2)
    seen[:, :, 64:128] = False
    found = oracle(case, blocks, width**-0.5, seen=seen)
    for j in range(64, 128):
        row = case.k[int(case.pages[0, j // page]), j % page] if page else case.packed_k[j]
        row.zero_()
        row[:, 0] = -INF
    out, lse = fs.flagsparse_block_attention(case.q, case.k, case.v, blocks, case.seqs, return_lse=True)
    by_head = out.view(tokens, heads, group, width).transpose(0, 1)
    assert bad.any() and (tokens == 1 or empty.any())
    assert bool(torch.isnan(by_head[bad]).all())
    assert not by_head[empty].any()
    none = (bad | empty).t()[:, :, None].expand(tokens, heads, group).reshape(tokens, heads * group)
    assert bool((lse[none] == -INF).all())
    rows = bad.t()[:, :, None].expand(tokens, heads, group).reshape(tokens, heads * group)
    want, bound = found["out"]
    off = (out.double() - want).abs() <= bound
    assert bool(off[~rows].all())
    if page:
        return
    grad = randn(case.q.shape, dtype, 62)
    dq, _, dv = fs.flagsparse_block_attention_grad(grad, case.q, case.k, case.v, blocks, case.seqs, out, lse)
    assert bool(torch.isnan(dq[rows]).all())
    assert bool(torch.isnan(dv[64:128][case.seen(blocks)[:, bad.any(0), 64:128].any(1).t()]).all())
