"""Operators over blocks at their edges: scores that are all minus infinity, lists in
several pieces, windows of the gradients' walks, memory around the arrays."""

import pytest
import torch

import flagsparse_amd as fs
from flagsparse_amd import blocks as block_module

from ._blocks_bounds import gradient_bounds, worst
from ._blocks_helpers import BLOCK_DTYPES, BLOCK_IDS, Case, oracle, random_blocks, randn

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


@pytest.mark.parametrize("bad", [None, float("nan")], ids=["finite", "nan"])
@pytest.mark.parametrize("dtype", BLOCK_DTYPES, ids=BLOCK_IDS)
def test_lists_of_more_entries_than_a_window_holds(dtype, bad):
    """One selection for eight heads, blocks of 1024 keys: the first block's list has 9000
    tokens, in pieces of more than 1024."""
    tokens, heads, width, block = 9000, 8, 16, 1024
    case = Case([tokens], [tokens], heads, 1, width, block, dtype, 63)
    blocks = torch.zeros((tokens, 1, 2), dtype=torch.int32)
    blocks[:, 0, 1] = torch.arange(tokens) // block
    blocks = blocks.cuda()
    assert tokens * 2 * heads * (block // 64) > 2048 * 1024  # entries a piece
    grad = randn(case.q.shape, dtype, 64)
    out, lse = fs.flagsparse_block_attention(case.q, case.k, case.v, blocks, case.seqs, return_lse=True)
    given = grad.clone()
    row = 5000  # sees the keys below 1024 and from 4096 on
    if bad is not None:
        grad[row], given[row] = 0.0, bad
    got = fs.flagsparse_block_attention_grad(given, case.q, case.k, case.v, blocks, case.seqs, out, lse)
    for h in (0, 5):
        one = Case([tokens], [tokens], 1, 1, width, block, dtype, 63)
        one.q, one.packed_k, one.packed_v = (t[:, h : h + 1] for t in (case.q, case.packed_k, case.packed_v))
        part = slice(h, h + 1)
        found = gradient_bounds(one, blocks, width**-0.5, grad[:, part], out[:, part], lse[:, part])
        keys = torch.zeros(tokens, dtype=torch.bool, device="cuda")
        rows = keys.clone()
        if bad is not None:
            keys[:1024] = keys[4096 : row + 1] = True
            rows[row] = True
        for t, name, apart in zip(got, ("dq", "dk", "dv"), (rows, keys, keys)):
            want, bound = found[name]
            assert bool(torch.isnan(t[:, part][apart]).all())
            off = worst(t[:, part][~apart], want[~apart], bound[~apart])
            assert off <= 1.0, (name, h, off)
        del found


@pytest.mark.parametrize("wanted", ["q", "k", "v", "kv", "qv"])
@pytest.mark.parametrize("tokens", [70, 1500])
def test_gradients_that_are_not_wanted_are_not_computed(tokens, wanted, monkeypatch):
    case = Case([tokens, 30], [tokens + 40, 30], 4, 2, 64, 64, torch.bfloat16, 65, tail=3, key_tail=4)
    blocks = random_blocks([tokens, 30], [tokens + 40, 30], 4, 3, 64, 66, extra=3)
    grad = randn(case.q.shape, torch.bfloat16, 67)
    out, lse = fs.flagsparse_block_attention(case.q, case.k, case.v, blocks, case.seqs, return_lse=True)
    want = dict(zip("qkv", fs.flagsparse_block_attention_grad(grad, case.q, case.k, case.v, blocks, case.seqs, out, lse)))
    computed = []
    inner = block_module._attention_grad
    monkeypatch.setattr(block_module, "_attention_grad", lambda *a, **b: computed.append(inner(*a, **b)) or computed[-1])
    leaves = {n: t.clone().requires_grad_(n in wanted) for n, t in zip("qkv", (case.q, case.k, case.v))}
    result = fs.flagsparse_block_attention(*leaves.values(), blocks, case.seqs)
    got = torch.autograd.grad(result, [leaves[n] for n in wanted], grad)
    assert all(torch.equal(g, want[n]) for g, n in zip(got, wanted))
    dq, dk, dv = computed.pop()
    assert (dq is None) == ("q" not in wanted) and (dk is None) == (dv is None) == (wanted == "q")
