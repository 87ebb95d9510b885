"""Operators over blocks at their edges: scores that are all minus infinity, lists in
several pieces, windows of the gradients' walks, memory around the arrays."""

import pytest
import torch

import flagsparse_amd as fs
from flagsparse_amd import _lib, blocks as block_module

from ._blocks_bounds import attention_bounds, gradient_bounds, worst
from ._blocks_helpers import BLOCK_DTYPES, BLOCK_IDS, Case, offsets, oracle, random_blocks, randn

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


WINDOWS = [
    # dtype, group, width, context: more blocks of 32 keys than a workgroup's table holds at a time
    (torch.float16, 1, 64, 30000),
    (torch.bfloat16, 3, 64, 30000),
    (torch.bfloat16, 1, 128, 40000),
    (torch.float32, 1, 64, 40000),
    (torch.float32, 1, 128, 50000),
]


@pytest.mark.parametrize("sizes", WINDOWS, ids=["x".join(map(str, c)).replace("torch.", "") for c in WINDOWS])
def test_gradients_in_several_windows(sizes):
    dtype, group, width, context = sizes
    tokens = 250
    case = Case([tokens], [context], 2, group, width, 32, dtype, 68)
    blocks = random_blocks([tokens], [context], 2, 6, 32, 69)
    grad = randn(case.q.shape, dtype, 70)
    out, lse = fs.flagsparse_block_attention(case.q, case.k, case.v, blocks, case.seqs, return_lse=True)
    got = fs.flagsparse_block_attention_grad(grad, case.q, case.k, case.v, blocks, case.seqs, out, lse)
    found = gradient_bounds(case, blocks, width**-0.5, grad, out, lse)
    off = {name: worst(t, *found[name]) for t, name in zip(got, ("dq", "dk", "dv"))}
    assert max(off.values()) <= 1.0, off


LARGE_BLOCKS = [
    ([700, 3], [1500, 600], 2, 3, 64, 512, 2),
    ([1100, 90], [1100, 2100], 4, 2, 128, 1024, 2),
    ([5], [2600], 2, 4, 80, 512, 3),
]


@pytest.mark.parametrize("dtype", BLOCK_DTYPES, ids=BLOCK_IDS)
@pytest.mark.parametrize("sizes", LARGE_BLOCKS, ids=["x".join(map(str, c[2:])) for c in LARGE_BLOCKS])
def test_large_blocks(sizes, dtype):
    new, lengths, heads, group, width, block, top = sizes
    case = Case(new, lengths, heads, group, width, block, dtype, 71, tail=2, key_tail=3)
    blocks = random_blocks(new, lengths, heads, top, block, 72, extra=2)
    grad = randn(case.q.shape, dtype, 73)
    out, lse = fs.flagsparse_block_attention(case.q, case.k, case.v, blocks, case.seqs, return_lse=True)
    got = fs.flagsparse_block_attention_grad(grad, case.q, case.k, case.v, blocks, case.seqs, out, lse)
    found = gradient_bounds(case, blocks, width**-0.5, grad, out, lse)
    off = {name: worst(t, *found[name]) for t, name in zip(got, ("dq", "dk", "dv"))}
    off["out"] = worst(out, *attention_bounds(case, blocks, width**-0.5))
    assert max(off.values()) <= 1.0, off
    means = fs.flagsparse_block_means(case.k, case.seqs, max_blocks=6)
    at = 0
    for b, n in enumerate(lengths):
        for i in range(6):
            rows = case.packed_k[at + min(i * block, n) : at + min((i + 1) * block, n)].double()
            want = rows.mean(0) if rows.shape[0] else torch.zeros_like(means[b, i]).double()
            size = rows.abs().sum(0) / max(1, rows.shape[0])
            # sums of `block` terms in 32 bits, one division, one rounding
            bound = (block + 2) * 2.0**-24 * size + torch.finfo(dtype).eps / 2 * (want.abs() + size * 2.0**-13) + 2.0**-25
            assert bool(((means[b, i].double() - want).abs() <= bound).all())
        at += n


@pytest.mark.parametrize("tokens", [405, 407], ids=["few", "many"])
@pytest.mark.parametrize("page", [0, 32])
def test_either_side_of_the_rule(tokens, page):
    """Groups of 16 and four heads of 128: 1625 tokens and heads go to the one kernel, more to the other."""
    case = Case([tokens - 5, 5], [tokens + 30, 100], 4, 16, 128, 64, torch.float16, 77, page)
    blocks = random_blocks([tokens - 5, 5], [tokens + 30, 100], 4, 3, 64, 78)
    out, lse = fs.flagsparse_block_attention(case.q, case.k, case.v, blocks, case.seqs, return_lse=True)
    assert _lib.last_kernel() == ("block_attention_few_kernel" if tokens * 4 <= 1625 else "block_attention_kernel")
    assert worst(out, *attention_bounds(case, blocks, 128**-0.5)) <= 1.0


@pytest.mark.parametrize("page", [0, 16], ids=["rows", "pages"])
@pytest.mark.parametrize("group, kernel", [(2, "few_"), (17, "")])
def test_single_tokens_of_many_sequences(page, group, kernel):
    """A decode step of 1200 sequences: no two tokens share a block."""
    n, heads = 1200, 4
    lengths = [(7 * i) % 23 for i in range(n)]
    case = Case([1] * n, lengths, heads, group, 32, 32, torch.bfloat16, 79, page, single=True)
    blocks = torch.zeros((n, 1, 1), dtype=torch.int32, device="cuda")
    out, lse = fs.flagsparse_block_attention(case.q, case.k, case.v, blocks, case.seqs, return_lse=True)
    assert _lib.last_kernel() == f"block_attention_{kernel}kernel"
    for b in range(0, n, 61):
        one = Case([1], [lengths[b]], heads, group, 32, 32, torch.bfloat16, 79)
        rows = slice(sum(lengths[:b]), sum(lengths[: b + 1]))
        one.q, one.packed_k, one.packed_v = case.q[b : b + 1], case.packed_k[rows], case.packed_v[rows]
        if lengths[b] == 0:
            assert not out[b].any() and bool((lse[b] == -INF).all())
        else:
            assert worst(out[b : b + 1], *attention_bounds(one, blocks[b : b + 1], 32**-0.5)) <= 1.0


class _Guarded:
    """A tensor's copy in the middle of a larger one, whose other values are kept in mind."""

    def __init__(self, t, around):
        self.whole = torch.full((t.numel() + 8192,), around, dtype=t.dtype, device="cuda")
        self.middle = self.whole[4096 : 4096 + t.numel()].view(t.shape)
        self.middle.copy_(t)
        self.around = around

    def untouched(self):
        sides = torch.cat([self.whole[:4096], self.whole[-4096:]])
        return bool((torch.isnan(sides) if self.around != self.around else sides == self.around).all())


@pytest.mark.parametrize("tokens", [(40, 30), (1500, 30)], ids=["few", "many"])
@pytest.mark.parametrize("which", ["queries", "keys", "below", "falling"])
def test_lengths_beyond_the_arrays_touch_nothing_around_them(which, tokens):
    """Offsets far past the arrays and below zero: what they say there is not there, and the
    results are those of the offsets brought into range, unless they fall: sequences then
    lie over each other."""
    heads, group, width, block, top = 4, 2, 64, 64, 4
    total, rows = sum(tokens), tokens[0] + 660
    lengths = [tokens[0] + 360, 300]
    wild = torch.tensor([0, 2**31 - 1, 5] if which == "falling" else [0, 2**31 - 9, 2**31 - 1], dtype=torch.int32).cuda()
    if which == "queries":  # all tokens are the first sequence's
        q_offsets, k_offsets, new, lengths = wild, offsets(lengths), [total, 0], lengths
    elif which == "keys":  # all rows are
        q_offsets, k_offsets, new, lengths = offsets(tokens), wild, list(tokens), [rows, 0]
    elif which == "falling":
        q_offsets, k_offsets, new = wild, wild, [total, 0]
    else:  # no sequence has any
        q_offsets, k_offsets, new, lengths = -wild, -wild, [0, 0], [0, 0]
    case = Case(new, lengths, heads, group, width, block, torch.bfloat16, 74, tail=total - sum(new),
                key_tail=rows - sum(lengths))
    blocks = random_blocks([total], [rows], heads, top, block, 75)
    nan = float("nan")
    q, k, v, grad = (_Guarded(t, nan) for t in (case.q, case.packed_k, case.packed_v, randn(case.q.shape, torch.bfloat16, 76)))
    ids = _Guarded(blocks, 1)
    out, dq = (_Guarded(torch.zeros_like(case.q), 7.0) for _ in range(2))
    dk, dv = (_Guarded(torch.zeros_like(case.packed_k), 7.0) for _ in range(2))
    seqs = fs.prepare_block_sequences(block, q_offsets, k_offsets=k_offsets)
    _, lse = fs.flagsparse_block_attention(q.middle, k.middle, v.middle, ids.middle, seqs, out=out.middle, return_lse=True)
    # (by the C entry, whose results lie where they are put)
    lib, described = _lib.lib(), block_module._described(seqs, total, k.middle)
    need = lib.fs_block_attention_grad_workspace_bytes(_lib.FS_BF16, described, heads, group, width, heads, top)
    ws = _Guarded(torch.zeros(need, dtype=torch.uint8, device="cuda"), 7)
    token, row = heads * group * width, heads * width
    rc = lib.fs_block_attention_grad(
        _lib.FS_BF16, described, heads, group, width, heads, top, grad.middle.data_ptr(), q.middle.data_ptr(), token, width,
        k.middle.data_ptr(), row, width, v.middle.data_ptr(), row, width, ids.middle.data_ptr(), heads * top, top,
        width**-0.5, out.middle.data_ptr(), lse.data_ptr(), dq.middle.data_ptr(), dk.middle.data_ptr(),
        dv.middle.data_ptr(), ws.middle.data_ptr(), need, _lib.stream_handle(q.middle.device))
    assert rc == _lib.FS_OK, lib.fs_last_error()
    means = _Guarded(torch.zeros((2, 9, heads, width), dtype=torch.bfloat16, device="cuda"), 7.0)
    fs.flagsparse_block_means(k.middle, seqs, out=means.middle)
    chosen = _Guarded(torch.zeros((total, heads, 5), dtype=torch.int32, device="cuda"), 7)
    fs.flagsparse_block_select(q.middle, means.middle, seqs, 5, out=chosen.middle)
    torch.cuda.synchronize()
    for t in (q, k, v, grad, ids, out, dq, dk, dv, ws, means, chosen):
        assert t.untouched()
    if which == "falling":
        return
    if which != "keys":  # (the selection has no keys: it takes the lengths as they are)
        assert torch.equal(chosen.middle, fs.flagsparse_block_select(case.q, means.middle, case.seqs, 5))
    assert torch.equal(means.middle, fs.flagsparse_block_means(case.packed_k, case.seqs, max_blocks=9))
    assert worst(out.middle, *attention_bounds(case, blocks, width**-0.5)) <= 1.0
    found = gradient_bounds(case, blocks, width**-0.5, grad.middle, out.middle, lse)
    for t, name in ((dq, "dq"), (dk, "dk"), (dv, "dv")):
        assert worst(t.middle, *found[name]) <= 1.0, name


@pytest.mark.parametrize("wanted", ["q", "kv"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["f16", "f32"])
def test_a_captured_backward_of_some_leaves(dtype, wanted):
    """Captured alone, replayed with other values, eager passes in between; on a stream of its own."""
    case = Case([300, 70], [300, 90], 2, 3, 64, 64, dtype, 80)
    blocks = random_blocks([300, 70], [300, 90], 2, 3, 64, 81)
    leaves = {n: t.clone().requires_grad_(n in wanted) for n, t in zip("qkv", (case.q, case.k, case.v))}
    grad = randn(case.q.shape, dtype, 82)

    def step():
        out = fs.flagsparse_block_attention(*leaves.values(), blocks, case.seqs)
        return torch.autograd.grad(out, [leaves[n] for n in wanted], grad)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for turn in range(4):
        size = 2.0 ** (6 * turn - 12)
        grad.copy_(randn(case.q.shape, dtype, 83 + turn) * size)
        with torch.no_grad():
            leaves["v"].copy_(randn(case.v.shape, dtype, 90 + turn))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        with torch.cuda.stream(side):
            want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), turn
