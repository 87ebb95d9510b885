"""Operators over blocks where they can go wrong: what is left out holds infinities or
NaN, pages outside the cache, strides, empty calls, graphs, streams, autograd."""

import pytest
import torch

import flagsparse_amd as fs

from ._blocks_helpers import BLOCK_DTYPES, BLOCK_IDS, Case, assert_within, offsets, oracle, random_blocks, randn, select_oracle

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def _attend(case, blocks, **more):
    return fs.flagsparse_block_attention(case.q, case.k, case.v, blocks, case.seqs, **more)


@pytest.mark.parametrize("bad", [NAN, INF, -INF], ids=["nan", "inf", "-inf"])
@pytest.mark.parametrize("tokens", [9, 1100], ids=["few", "many"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_what_a_query_does_not_see_may_hold_anything(tokens, bad, dtype):
    """Keys and values of a block that some select, and of positions behind a query."""
    case = Case([tokens], [tokens + 200], 4, 2, 64, 64, dtype, 1)
    blocks = random_blocks([tokens], [tokens + 200], 4, 4, 64, 2)
    # block 1: selected by some queries alone, the last keys: behind most queries' positions
    blocks[(torch.arange(tokens) % 5 != 0).nonzero().flatten().cuda()] = torch.where(
        blocks[(torch.arange(tokens) % 5 != 0).nonzero().flatten().cuda()] == 1, 0,
        blocks[(torch.arange(tokens) % 5 != 0).nonzero().flatten().cuda()])
    want, bound = oracle(case, blocks, 64**-0.5)["out"]
    seen = case.seen(blocks)
    rows = [70, 100, tokens + 190, tokens + 199]
    touched = seen[:, :, rows].any(2).t()[:, :, None].expand(tokens, 4, 2).reshape(tokens, 8)
    case.packed_k[70] = bad
    case.packed_v[100] = bad
    case.packed_k[tokens + 190] = bad
    case.packed_v[tokens + 199] = bad
    got = _attend(case, blocks).double()
    # (a row beside one that is not finite is computed anew in 32 bits: as near, not to the bit)
    assert bool(((got - want).abs() <= bound)[~touched].all())
    assert touched.any() and not touched.all()
    if bad != bad:
        assert bool(torch.isnan(got[touched]).all())


@pytest.mark.parametrize("dtype", BLOCK_DTYPES, ids=BLOCK_IDS)
def test_gradients_of_what_is_not_seen_may_hold_anything(dtype):
    """A key's row that is not finite reaches the queries that see it alone; a gradient's
    row that is not, the keys that its query sees."""
    n = 300
    case = Case([n], [n], 2, 2, 64, 64, dtype, 1)
    blocks = random_blocks([n], [n], 2, 3, 64, 2)
    grad = randn(case.q.shape, dtype, 3)
    out, lse = _attend(case, blocks, return_lse=True)

    def run():
        return fs.flagsparse_block_attention_grad(grad, case.q, case.k, case.v, blocks, case.seqs, out, lse)

    def near(got, found, name, where):
        want, bound = found[name]
        assert bool(((got.double() - want).abs() <= bound)[where].all()), name

    grad[200] = 0.5
    found = oracle(case, blocks, 64**-0.5, grad)
    seen = case.seen(blocks)
    grad[200] = NAN
    got = run()
    reached = seen[:, 200].t()[:, :, None].expand(n, 2, 64)  # (rows, heads, width)
    others = (torch.arange(n) != 200).cuda()
    near(got[0], found, "dq", others)
    for t, name in zip(got[1:], ("dk", "dv")):
        near(t, found, name, ~reached)
        assert bool(torch.isnan(t[reached]).all())
    grad[200] = 0.5
    case.packed_k[150] = INF  # not in all selections, and behind 0 .. 149
    reached = seen[:, :, 150].t()[:, :, None, None].expand(n, 2, 2, 64).reshape(n, 4, 64)
    near(run()[0], found, "dq", ~reached)


def test_pages_outside_the_cache_hold_no_keys():
    for tokens in (3, 1500):
        case = Case([tokens, 2], [tokens + 300, 100], 4, 2, 64, 64, torch.bfloat16, 4, page=16)
        blocks = random_blocks([tokens, 2], [tokens + 300, 100], 4, 5, 64, 5)
        seen = case.seen(blocks)
        for page, bad in ((3, -1), (5, case.k.shape[0]), (7, 2**31 - 1), (9, -(2**31))):
            case.pages[0, page] = bad
            seen[:, :, page * 16 : (page + 1) * 16] = False
        out, lse = _attend(case, blocks, return_lse=True)
        found = oracle(case, blocks, 64**-0.5, seen=seen)
        assert_within(lse, found, "lse")
        assert_within(out, found, "out")
        # no page of a sequence is: nothing is seen
        case.pages[:] = -7
        out, lse = _attend(case, blocks, return_lse=True)
        assert not out.any() and bool((lse == -INF).all())
        means = fs.flagsparse_block_means(case.k, case.seqs, max_blocks=30)
        assert not means.any()


def test_lengths_beyond_the_arrays_read_nothing_outside():
    """Offsets and lengths are not checked on the host; what they say past the arrays is not there."""
    case = Case([40, 30], [400, 300], 2, 2, 64, 64, torch.float16, 6)
    blocks = random_blocks([40, 30], [400, 300], 2, 4, 64, 7)
    wild = torch.tensor([0, 2**31 - 1, 5], dtype=torch.int32).cuda()
    for q_offsets, k_offsets in ((wild, offsets([400, 300])), (offsets([40, 30]), wild), (-wild, -wild)):
        seqs = fs.prepare_block_sequences(64, q_offsets, k_offsets=k_offsets)
        out, lse = fs.flagsparse_block_attention(case.q, case.k, case.v, blocks, seqs, return_lse=True)
        fs.flagsparse_block_attention_grad(case.q, case.q, case.k, case.v, blocks, seqs, out, lse)
        fs.flagsparse_block_select(case.q, torch.zeros((2, 7, 2, 64), dtype=torch.float16, device="cuda"), seqs, 4)
        fs.flagsparse_block_means(case.k, seqs, max_blocks=7)
    torch.cuda.synchronize()


@pytest.mark.parametrize("tokens", [40, 1100], ids=["few", "many"])
def test_a_block_named_twice_counts_once(tokens):
    case = Case([tokens], [tokens], 4, 2, 64, 32, torch.bfloat16, 8)
    one = random_blocks([tokens], [tokens], 4, 3, 32, 9)
    twice = torch.cat([one, one.flip(2), one], 2)
    for blocks in (one, twice):
        out, lse = _attend(case, blocks, return_lse=True)
        grads = fs.flagsparse_block_attention_grad(case.q, case.q, case.k, case.v, blocks, case.seqs, out, lse)
        if blocks is one:
            found = oracle(case, one, 64**-0.5, case.q) if tokens < 100 else None
        if found is not None:
            for t, name in zip((out, lse, *grads), ("out", "lse", "dq", "dk", "dv")):
                assert_within(t, found, name)
        elif blocks is one:
            first = (out, *grads)
        else:
            assert all(torch.equal(a, b) for a, b in zip(first, (out, *grads)))


def test_one_selection_for_all_heads():
    case = Case([260], [300], 4, 2, 64, 64, torch.bfloat16, 10)
    shared = random_blocks([260], [300], 1, 3, 64, 11)
    every = shared.expand(-1, 4, -1)
    grad = randn(case.q.shape, torch.bfloat16, 12)
    got = []
    for blocks in (shared, every, every.contiguous()):
        out, lse = _attend(case, blocks, return_lse=True)
        got.append((out, lse, *fs.flagsparse_block_attention_grad(grad, case.q, case.k, case.v, blocks, case.seqs, out, lse)))
    found = oracle(case, every.contiguous(), 64**-0.5, grad)
    for results in got:
        for t, name in zip(results, ("out", "lse", "dq", "dk", "dv")):
            assert_within(t, found, name)


def test_strides_and_alignment():
    """Heads before tokens, rows of a wider tensor, rows that begin off 16 bytes."""
    case = Case([50], [200], 3, 2, 64, 64, torch.float16, 13)
    blocks = random_blocks([50], [200], 3, 4, 64, 14)
    want = _attend(case, blocks, return_lse=True)
    grad = randn(case.q.shape, torch.float16, 15)
    wants = fs.flagsparse_block_attention_grad(grad, case.q, case.k, case.v, blocks, case.seqs, *want)

    def turned(t):
        return t.transpose(0, 1).contiguous().transpose(0, 1)

    def wider(t):
        big = torch.full((*t.shape[:-1], t.shape[-1] + 16), NAN, dtype=t.dtype, device="cuda")
        big[..., 8:-8] = t
        return big[..., 8:-8]

    def off(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape)
        return flat.copy_(t)

    def sparse(t):
        big = torch.full((*t.shape, 2), NAN if t.is_floating_point() else 9, dtype=t.dtype, device="cuda")
        big[..., 0] = t
        return big[..., 0]

    for lay in (turned, wider, off, sparse):
        q, k, v = (lay(t) for t in (case.q, case.k, case.v))
        got = fs.flagsparse_block_attention(q, k, v, sparse(blocks), case.seqs, return_lse=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        grads = fs.flagsparse_block_attention_grad(lay(grad), q, k, v, blocks, case.seqs, *got)
        assert all(torch.equal(a, b) for a, b in zip(grads, wants))
        means = fs.flagsparse_block_means(k, case.seqs, max_blocks=4)
        assert torch.equal(means, fs.flagsparse_block_means(case.k, case.seqs, max_blocks=4))
        assert torch.equal(fs.flagsparse_block_select(q, lay(means), case.seqs, 3),
                           fs.flagsparse_block_select(case.q, means, case.seqs, 3))


def test_heads_before_pages():
    """A cache laid out page by head by row."""
    case = Case([3, 1], [200, 90], 2, 4, 128, 64, torch.bfloat16, 16, page=32)
    blocks = random_blocks([3, 1], [200, 90], 2, 3, 64, 17)
    want = _attend(case, blocks)
    k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (case.k, case.v))
    assert torch.equal(fs.flagsparse_block_attention(case.q, k, v, blocks, case.seqs), want)


def test_out():
    case = Case([30], [200], 2, 2, 64, 64, torch.bfloat16, 18)
    blocks = random_blocks([30], [200], 2, 3, 64, 19)
    want = _attend(case, blocks)
    out = torch.empty_like(case.q)
    assert _attend(case, blocks, out=out) is out and torch.equal(out, want)
    q = case.q.clone()
    assert torch.equal(fs.flagsparse_block_attention(q, case.k, case.v, blocks, case.seqs, out=q), want)
    means = fs.flagsparse_block_means(case.k, case.seqs, max_blocks=4)
    ids = fs.flagsparse_block_select(case.q, means, case.seqs, 3)
    place = torch.empty_like(ids)
    assert fs.flagsparse_block_select(case.q, means, case.seqs, 3, out=place) is place and torch.equal(place, ids)
    kept = torch.full_like(means, 5.0)
    assert torch.equal(fs.flagsparse_block_means(case.k, case.seqs, out=kept), means)


def test_empty_calls():
    empty = torch.zeros((0, 4, 64), dtype=torch.float16, device="cuda")
    keys = randn((40, 2, 64), torch.float16, 20)
    none = torch.zeros((0, 2, 3), dtype=torch.int32, device="cuda")
    seqs = fs.prepare_block_sequences(64, offsets([0, 0]), k_offsets=offsets([30, 5]))
    out, lse = fs.flagsparse_block_attention(empty, keys, keys, none, seqs, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    dq, dk, dv = fs.flagsparse_block_attention_grad(empty, empty, keys, keys, none, seqs, out, lse)
    assert dq.shape == (0, 4, 64) and not dk.any() and not dv.any()
    assert fs.flagsparse_block_select(empty, torch.zeros((2, 1, 2, 64), dtype=torch.float16, device="cuda"), seqs, 3).shape == (0, 2, 3)
    # no sequences, tokens and keys of none
    seqs = fs.prepare_block_sequences(64, offsets([]), k_offsets=offsets([]))
    q, ids = randn((7, 4, 64), torch.float16, 21), torch.zeros((7, 2, 3), dtype=torch.int32, device="cuda")
    out, lse = fs.flagsparse_block_attention(q, keys, keys, ids, seqs, return_lse=True)
    assert not out.any() and bool((lse == -INF).all())
    grads = fs.flagsparse_block_attention_grad(q, q, keys, keys, ids, seqs, out, lse)
    assert not any(t.any() for t in grads)
    assert fs.flagsparse_block_means(keys, seqs, max_blocks=2).shape == (0, 2, 2, 64)
    # no keys at all
    seqs = fs.prepare_block_sequences(64, offsets([7]), k_offsets=offsets([0]))
    out = fs.flagsparse_block_attention(q, keys[:0], keys[:0], ids, seqs)
    assert not out.any()
    # an empty table of pages
    seqs = fs.prepare_block_sequences(64, pages=torch.zeros((7, 0), dtype=torch.int32, device="cuda"),
                                      k_lengths=torch.full((7,), 9, dtype=torch.int32, device="cuda"))
    cache = randn((3, 16, 2, 64), torch.float16, 22)
    assert not fs.flagsparse_block_attention(q, cache, cache, ids, seqs).any()


@pytest.mark.parametrize("tokens", [33, 1100], ids=["few", "many"])
def test_a_step_in_a_graph(tokens):
    """Summaries, selection and attention captured; lengths, pages and values change between replays,
    with eager calls in between."""
    case = Case([tokens, 5], [tokens + 300, 200], 4, 2, 64, 64, torch.bfloat16, 23, page=64)
    for t in (case.k, case.v):  # (another order of pages puts what lies behind the keys among them)
        t.nan_to_num_(0.25)
    start = torch.tensor([tokens + 200, 100], dtype=torch.int32).cuda()
    kept = fs.flagsparse_block_means(case.k, case.seqs, max_blocks=30).clone()
    out = torch.empty_like(case.q)

    def step():
        fs.flagsparse_block_means(case.k, case.seqs, start=start, out=kept)
        blocks = fs.flagsparse_block_select(case.q, kept, case.seqs, 4)
        fs.flagsparse_block_attention(case.q, case.k, case.v, blocks, case.seqs, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    table = case.pages.clone()
    for turn in range(4):
        case.q.copy_(randn(case.q.shape, torch.bfloat16, 30 + turn))
        case.k_lengths.copy_(torch.tensor([tokens + 300 - turn, 200 - 7 * turn], dtype=torch.int32))
        case.pages.copy_(table.flip(1) if turn == 2 else table)
        graph.replay()
        torch.cuda.synchronize()
        got, summaries = out.clone(), kept.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(out, got) and torch.equal(kept, summaries), turn


def test_a_training_step_in_a_graph():
    case = Case([200, 90], [200, 90], 2, 4, 128, 64, torch.bfloat16, 24)
    blocks = random_blocks([200, 90], [200, 90], 2, 4, 64, 25)
    grad = randn(case.q.shape, torch.bfloat16, 26)
    leaves = [t.clone().requires_grad_() for t in (case.q, case.k, case.v)]

    def step():
        out = fs.flagsparse_block_attention(*leaves, blocks, case.seqs)
        return (out.detach(), *torch.autograd.grad(out, leaves, grad))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for turn in range(3):
        with torch.no_grad():
            leaves[0].copy_(randn(case.q.shape, torch.bfloat16, 40 + turn))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), turn


def test_calls_on_two_streams_at_once():
    cases = [Case([700], [900], 8, 2, 64, 64, torch.bfloat16, 50 + i) for i in range(2)]
    blocks = [random_blocks([700], [900], 8, 4, 64, 60 + i) for i in range(2)]
    grads = [randn(c.q.shape, torch.bfloat16, 70 + i) for i, c in enumerate(cases)]

    def run(i):
        out, lse = _attend(cases[i], blocks[i], return_lse=True)
        return (out, lse, *fs.flagsparse_block_attention_grad(grads[i], cases[i].q, cases[i].k, cases[i].v, blocks[i],
                                                              cases[i].seqs, out, lse))

    want = [run(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = [None, None]
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = run(i)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_autograd_and_differences():
    """The Function's gradients are the named call's, and those of differences in 32 bits."""
    case = Case([90, 20], [90, 20], 2, 2, 32, 32, torch.float32, 27)
    blocks = random_blocks([90, 20], [90, 20], 2, 3, 32, 28)
    grad = randn(case.q.shape, torch.float32, 29)
    leaves = [t.clone().requires_grad_() for t in (case.q, case.k, case.v)]
    out, lse = fs.flagsparse_block_attention(*leaves, blocks, case.seqs, scale=0.2, return_lse=True)
    assert out.requires_grad and not lse.requires_grad
    got = torch.autograd.grad(out, leaves, grad)
    named = fs.flagsparse_block_attention_grad(grad, *(t.detach() for t in leaves), blocks, case.seqs, out.detach(), lse, 0.2)
    assert all(torch.equal(a, b) for a, b in zip(got, named))
    found = oracle(case, blocks, 0.2, grad)
    for t, name in zip(got, ("dq", "dk", "dv")):
        assert_within(t, found, name)

    def value(*x):
        with torch.no_grad():
            return float((fs.flagsparse_block_attention(*x, blocks, case.seqs, scale=0.2).double() * grad.double()).sum())

    h = 2.0**-7
    for i in range(3):
        d = randn(leaves[i].shape, torch.float32, 80 + i)
        up = [t.detach() + h * d if j == i else t.detach() for j, t in enumerate(leaves)]
        down = [t.detach() - h * d if j == i else t.detach() for j, t in enumerate(leaves)]
        slope = (value(*up) - value(*down)) / (2 * h)
        want = float((got[i].double() * d.double()).sum())
        size = float((got[i].double() * d.double()).norm()) + abs(want)
        # second differences of order h^2 and results off by some 2^-20 over 2 h
        assert abs(slope - want) <= 40 * h * h * size + 2.0**-18 / h * float(grad.double().norm())
    # only one operand wants a gradient
    q = case.q.clone().requires_grad_()
    fs.flagsparse_block_attention(q, case.k, case.v, blocks, case.seqs, scale=0.2).backward(grad)
    assert torch.equal(q.grad, got[0])
    # lengths overwritten between the passes are noticed
    out = fs.flagsparse_block_attention(*leaves, blocks, case.seqs)
    case.seqs.k_offsets.add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_float16_gradients_of_small_and_large_values():
    """dS goes through 16 bits: a power of two keeps its small values, whatever the gradient's size."""
    case = Case([300], [300], 2, 2, 64, 64, torch.float16, 31)
    blocks = random_blocks([300], [300], 2, 3, 64, 32)
    base = randn(case.q.shape, torch.float16, 33)
    out, lse = _attend(case, blocks, return_lse=True)
    for size in (2.0**-11, 1.0, 2.0**11):
        grad = base * size
        got = fs.flagsparse_block_attention_grad(grad, case.q, case.k, case.v, blocks, case.seqs, out, lse)
        found = oracle(case, blocks, 64**-0.5, grad)
        for t, name in zip(got, ("dq", "dk", "dv")):
            assert_within(t, found, name)


def test_the_same_twice_and_after_others():
    case = Case([1200], [1200], 4, 4, 64, 64, torch.bfloat16, 34)
    blocks = random_blocks([1200], [1200], 4, 6, 64, 35)
    grad = randn(case.q.shape, torch.bfloat16, 36)

    def run():
        out, lse = _attend(case, blocks, return_lse=True)
        return (out, lse, *fs.flagsparse_block_attention_grad(grad, case.q, case.k, case.v, blocks, case.seqs, out, lse))

    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(), first))


def test_prompt_then_decode_with_summaries_kept():
    """A prompt in two chunks, then single tokens, over one cache: every step is the whole sequence's last
    rows, whose selection and attention follow the definitions."""
    heads, group, width, block, total = 2, 4, 64, 64, 700
    dtype = torch.bfloat16
    q = randn((total, heads * group, width), dtype, 37)
    k, v = randn((total, heads, width), dtype, 38), randn((total, heads, width), dtype, 39)
    pages = torch.tensor([[5, 2, 9, 0, 7, 1, 8, 3, 4, 6, 11]], dtype=torch.int32).cuda()
    cache_k = torch.full((12, 64, heads, width), NAN, dtype=dtype, device="cuda")
    cache_v = torch.full_like(cache_k, NAN)
    kept = torch.zeros((1, 11, heads, width), dtype=dtype, device="cuda")
    at = 0
    for new in (300, 390, 1, 1, 1, 1, 6):
        for p in range(at, at + new):
            cache_k[pages[0, p // 64], p % 64], cache_v[pages[0, p // 64], p % 64] = k[p], v[p]
        lengths = torch.tensor([at + new], dtype=torch.int32).cuda()
        seqs = fs.prepare_block_sequences(block, None if new == 1 else offsets([new]), pages=pages, k_lengths=lengths)
        fs.flagsparse_block_means(cache_k, seqs, start=torch.tensor([at], dtype=torch.int32).cuda(), out=kept)
        rows = slice(at, at + new)
        blocks = fs.flagsparse_block_select(q[rows], kept, seqs, 5)
        want = select_oracle(q[rows], kept, [0] * new, list(range(at, at + new)), block, 5, 1, 1)
        assert torch.equal(blocks, want)
        out = fs.flagsparse_block_attention(q[rows], cache_k, cache_v, blocks, seqs)
        case = Case([new], [at + new], heads, group, width, block, dtype, 1)
        case.q, case.packed_k, case.packed_v = q[rows], k[: at + new], v[: at + new]
        assert_within(out, oracle(case, blocks, width**-0.5), "out")
        at += new


@pytest.mark.parametrize("tokens", [2, 1100], ids=["few", "many"])
@pytest.mark.parametrize("page", [0, 64], ids=["rows", "pages"])
def test_keys_behind_32_bits(page, tokens):
    """Keys 4.3 billion elements into their array: bit for bit those of a short one."""
    heads, width, block, length = 4, 128, 64, 1500
    case = Case([tokens], [length], heads, 1, width, block, torch.bfloat16, 21)
    blocks = random_blocks([tokens], [length], heads, 5, block, 22)
    want, want_lse = _attend(case, blocks, return_lse=True)
    want_means = fs.flagsparse_block_means(case.k, case.seqs, 24)
    rows = 2**32 // (heads * width) + 20000 // block * block
    k = torch.zeros((rows, heads, width), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    k[-length:], v[-length:] = case.k, case.v
    if page:
        at = rows // page * page - 1536
        k[at : at + length], v[at : at + length] = case.k, case.v
        table = (torch.arange(24, dtype=torch.int32) + at // page)[None].cuda()
        seqs = fs.prepare_block_sequences(block, offsets([tokens]), pages=table,
                                          k_lengths=torch.tensor([length], dtype=torch.int32).cuda())
        k, v = (x[: rows // page * page].view(-1, page, heads, width) for x in (k, v))
    else:
        seqs = fs.prepare_block_sequences(block, offsets([0, tokens]), k_offsets=offsets([rows - length, length]))
    out, lse = fs.flagsparse_block_attention(case.q, k, v, blocks, seqs, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    if page:
        assert torch.equal(fs.flagsparse_block_means(k, seqs, 24), want_means)
        return
    grad = randn(case.q.shape, torch.bfloat16, 23)
    want_grads = fs.flagsparse_block_attention_grad(grad, case.q, case.k, case.v, blocks, case.seqs, want, want_lse)
    grads = fs.flagsparse_block_attention_grad(grad, case.q, k, v, blocks, seqs, out, lse)
    assert torch.equal(grads[0], want_grads[0])
    for got, of in zip(grads[1:], want_grads[1:]):
        assert torch.equal(got[-length:], of)
        assert not got[:-length].any()


def test_one_sequence_of_millions_of_keys():
    """Blocks at both ends of a sequence of 8.4 million keys; its blocks are selected by means."""
    heads, width, block, n = 4, 128, 64, 131072 + 7
    length = n * block - 9
    k = torch.zeros((n * block, heads, width), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    near = Case([3], [9 * block - 9], heads, 2, width, block, torch.bfloat16, 24)
    k[:block], v[:block] = near.k[:block], near.v[:block]
    k[length - near.rows + block : length], v[length - near.rows + block : length] = near.k[block:], near.v[block:]
    k, v = k[:length], v[:length]
    seqs = fs.prepare_block_sequences(block, offsets([3]), k_offsets=offsets([length]))
    ids = torch.tensor([[0, 3, 5, 8], [0, 1, 7, 8], [0, 2, 4, 6]], dtype=torch.int32)[:, None].expand(3, heads, 4).contiguous().cuda()
    far = torch.where(ids > 0, ids + (n - 9), ids)
    want = fs.flagsparse_block_attention(near.q, near.k, near.v, ids, near.seqs)
    assert torch.equal(fs.flagsparse_block_attention(near.q, k, v, far, seqs), want)
    means = fs.flagsparse_block_means(k, seqs, n)
    assert torch.equal(means[:, [0, *range(n - 8, n)]], fs.flagsparse_block_means(near.k, near.seqs, 9))
    assert not means[:, 1 : n - 8].any()
    got = fs.flagsparse_block_select(near.q, means, seqs, 6)
    assert torch.equal(got, select_oracle(near.q, means, [0] * 3, [length - 3, length - 2, length - 1], block, 6, 1, 1))
