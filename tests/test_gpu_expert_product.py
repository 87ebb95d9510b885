"""The experts' products and their gradients (expert_product.hip) against 64-bit
products on the CPU: types, both matrix layouts, sizes that end inside tiles,
steps and 16-byte pieces, experts without rows, rows of no expert, strides."""

import pytest
import torch

import flagsparse_amd as fs
from flagsparse_amd import _lib
from tests._rows_helpers import assert_sum, randn, random_experts

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float16, torch.bfloat16, torch.float32]
IDS = ["f16", "bf16", "f32"]


def _route(counts, dropped=0):
    """A route of one slot a token with the given rows an expert, in order."""
    ids = torch.cat([torch.full((n,), e) for e, n in enumerate(counts)] + [torch.full((dropped,), -1)])
    return fs.prepare_expert_route(ids.int()[:, None].to(DEV), len(counts))


def _oracle(rows, matrices, route, op):
    x, w, off = rows.cpu().double(), matrices.cpu().double(), route.offsets.tolist()
    w = w.transpose(1, 2) if op == "trans" else w
    out, mag = torch.zeros(len(x), w.shape[2], dtype=torch.float64), torch.zeros(len(x), w.shape[2], dtype=torch.float64)
    for e in range(len(w)):
        a, b = off[e], off[e + 1]
        out[a:b], mag[a:b] = x[a:b] @ w[e], x[a:b].abs() @ w[e].abs()
    return out, mag


def _oracle_matrices(grad, rows, matrices, route, op):
    g, x, off = grad.cpu().double(), rows.cpu().double(), route.offsets.tolist()
    out, mag = torch.zeros(matrices.shape, dtype=torch.float64), torch.zeros(matrices.shape, dtype=torch.float64)
    for e in range(len(matrices)):
        a, b = (g, x) if op == "trans" else (x, g)
        a, b = a[off[e] : off[e + 1]], b[off[e] : off[e + 1]]
        out[e], mag[e] = a.T @ b, a.abs().T @ b.abs()
    return out, mag


def _check(dtype, op, counts, inner, outer, dropped=0, seed=0):
    route = _route(counts, dropped)
    n, most = route.n_rows, max(counts)
    rows, grad = randn((n, inner), dtype, seed + 1), randn((n, outer), dtype, seed + 2)
    shape = (len(counts), outer, inner) if op == "trans" else (len(counts), inner, outer)
    matrices = randn(shape, dtype, seed + 3)
    if dropped:
        rows[n - dropped :], grad[n - dropped :] = float("nan"), float("inf")
    got = fs.flagsparse_expert_product(rows, matrices, route, op=op)
    assert got.dtype == dtype and _lib.last_kernel().startswith("expert_product")
    want, mag = _oracle(rows, matrices, route, op)
    assert_sum(got, want, mag, inner)
    assert not bool(got[n - dropped :].any())
    grad_rows, grad_matrices = fs.flagsparse_expert_product_grad(grad, rows, matrices, route, op=op)
    want, mag = _oracle(grad, matrices, route, "non" if op == "trans" else "trans")
    assert grad_rows.dtype == dtype and grad_rows.shape == rows.shape
    assert_sum(grad_rows, want, mag, outer)
    want, mag = _oracle_matrices(grad, rows, matrices, route, op)
    assert grad_matrices.dtype == dtype and grad_matrices.shape == matrices.shape
    assert_sum(grad_matrices, want, mag, most)
    for e, count in enumerate(counts):
        if count == 0:
            assert not bool(grad_matrices[e].any())


# rows an expert around the tiles' sizes, none, one; a route of nothing but lost slots
COUNTS = [(1,), (0, 1, 0), (16, 17, 15), (0, 0, 5, 0), (31, 0, 33, 64), (127, 128, 129, 1), (255, 300, 0, 257), (0, 0)]


@pytest.mark.parametrize("counts", COUNTS, ids=str)
@pytest.mark.parametrize("op", ["non", "trans"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_rows_an_expert(dtype, op, counts):
    _check(dtype, op, counts, 136, 200, dropped=13)


# inner and outer sizes at and off steps (64 and 32 elements), tiles, 16-byte pieces and odd
SIZES = [(1, 1), (8, 8), (7, 9), (64, 128), (63, 129), (65, 127), (72, 264), (200, 31), (33, 300), (256, 256), (264, 520),
         (130, 134), (1000, 24)]


@pytest.mark.parametrize("inner,outer", SIZES, ids=[f"{a}x{b}" for a, b in SIZES])
@pytest.mark.parametrize("op", ["non", "trans"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_sizes(dtype, op, inner, outer):
    _check(dtype, op, (3, 0, 150, 40), inner, outer, dropped=2, seed=inner)


# few rows an expert, as at decoding, and many, as in training
@pytest.mark.parametrize("n_tokens,slots,n_experts", [(1, 1, 8), (1, 8, 64), (2, 6, 60), (16, 4, 32), (700, 2, 4), (1500, 3, 3)])
@pytest.mark.parametrize("op", ["non", "trans"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_routed(dtype, op, n_tokens, slots, n_experts):
    counts = torch.bincount(random_experts(n_tokens, slots, n_experts, n_tokens).reshape(-1).long(), minlength=n_experts)
    for inner, outer in ((512, 384), (520, 1032)):
        _check(dtype, op, counts.tolist(), inner, outer, seed=outer)


# enough and large enough tiles for the largest ones, of rows and of the matrices' gradient; two leave a last
# round that is split, two have rows of whole words but not of whole 16 bytes
@pytest.mark.parametrize("counts,inner,outer", [((700, 1, 513, 900), 264, 5512), ((256, 0, 1024), 40, 12808),
                                                ((300, 0, 5, 260), 2056, 2080),
                                                ((1024, 1000, 300, 700), 1032, 5512),
                                                ((900, 1400, 0, 1900), 2056, 2080),
                                                ((700, 1, 513, 900), 266, 5510), ((300, 0, 5, 260), 2054, 2090)],
                         ids=["rows", "short", "matrices", "rows_split", "matrices_split", "rows_words",
                              "matrices_words"])
@pytest.mark.parametrize("op", ["non", "trans"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_many_tiles(dtype, op, counts, inner, outer):
    _check(dtype, op, counts, inner, outer, dropped=70)


# many rows and small matrices: tiles of every size split along the rows
@pytest.mark.parametrize("counts,inner,outer", [((5000, 0, 3300), 40, 24), ((2100, 2500, 1800), 136, 300),
                                                ((4099, 3999), 65, 127), ((7000, 9000), 258, 202)], ids=str)
@pytest.mark.parametrize("op", ["non", "trans"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_many_rows_small_matrices(dtype, op, counts, inner, outer):
    _check(dtype, op, counts, inner, outer, dropped=9)


@pytest.mark.parametrize("op", ["non", "trans"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_neighbours_do_not_leak(dtype, op):
    """NaN and infinities in one expert's rows and matrix stay in its results,
    also where tiles and steps reach past the expert's last row."""
    counts = (5, 70, 3, 130)
    route = _route(counts)
    rows, grad = randn((208, 96), dtype, 1), randn((208, 80), dtype, 2)
    matrices = randn((4, 80, 96) if op == "trans" else (4, 96, 80), dtype, 3)
    clean = (fs.flagsparse_expert_product(rows, matrices, route, op=op),
             *fs.flagsparse_expert_product_grad(grad, rows, matrices, route, op=op))
    rows[75:78], grad[75:78], matrices[2] = float("nan"), float("inf"), float("nan")
    out, grad_rows, grad_matrices = (fs.flagsparse_expert_product(rows, matrices, route, op=op),
                                     *fs.flagsparse_expert_product_grad(grad, rows, matrices, route, op=op))
    for got, want in ((out, clean[0]), (grad_rows, clean[1])):
        assert torch.equal(got[:75], want[:75]) and torch.equal(got[78:], want[78:])
        assert bool(torch.isnan(got[75:78]).all())
    others = [0, 1, 3]
    assert torch.equal(grad_matrices[others], clean[2][others]) and bool(torch.isnan(grad_matrices[2]).all())


def test_strides_views_and_out():
    route = _route((40, 3, 90), 7)
    big, g = randn((140, 3 * 96), torch.bfloat16, 1), randn((140, 2 * 64), torch.bfloat16, 2)
    matrices = randn((3, 96, 64), torch.bfloat16, 3)
    for cut in (slice(0, 96), slice(1, 97), slice(None, None, 3)):
        rows, grad = big[:, cut], g[:, :64]
        want = fs.flagsparse_expert_product(rows.contiguous(), matrices, route)
        assert torch.equal(fs.flagsparse_expert_product(rows, matrices, route), want)
        grads = fs.flagsparse_expert_product_grad(grad.contiguous(), rows.contiguous(), matrices, route)
        assert all(torch.equal(a, b) for a, b in zip(fs.flagsparse_expert_product_grad(grad, rows, matrices, route), grads))
        out = torch.full_like(want, 5.0)
        assert fs.flagsparse_expert_product(rows, matrices, route, out=out) is out and torch.equal(out, want)
    rows = big[:, :96]
    want, mag = _oracle(rows, matrices, route, "non")
    flipped = matrices.transpose(1, 2).contiguous()
    sliced = randn((6, 96, 64), torch.bfloat16, 3)
    sliced[::2] = matrices
    for m, op in ((matrices, 0), (flipped, "trans"), (flipped, "conj"), (flipped.transpose(1, 2), "non"),
                  (matrices.transpose(1, 2), "trans"), (sliced[::2], None)):
        assert_sum(fs.flagsparse_expert_product(rows, m, route, op=op), want, mag, 96)
    # matrices that start off 16 bytes
    store = torch.empty(3 * 96 * 64 + 1, dtype=torch.bfloat16, device=DEV)
    off = store[1:].view(3, 96, 64).copy_(matrices)
    assert_sum(fs.flagsparse_expert_product(rows, off, route), want, mag, 96)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_rows_far_apart(dtype):
    # a tile's rows further apart than the offsets of the loads that go straight to LDS
    route = _route((200, 100))
    store = torch.zeros((300, (1 << 22) // torch.empty(0, dtype=dtype).element_size() + 8), dtype=dtype, device=DEV)
    rows, matrices = store[:, :40], randn((2, 40, 24), dtype, 2)
    rows.copy_(randn((300, 40), dtype, 1))
    want, mag = _oracle(rows, matrices, route, "non")
    assert_sum(fs.flagsparse_expert_product(rows, matrices, route), want, mag, 40)
    grad = randn((300, 24), dtype, 3)
    _, got = fs.flagsparse_expert_product_grad(grad, rows, matrices, route)
    want, mag = _oracle_matrices(grad, rows, matrices, route, "non")
    assert_sum(got, want, mag, 200)


def test_empty_sizes():
    route, none = _route((2, 0, 1)), _route((0, 0, 0))
    for a, b in ((0, 8), (8, 0)):
        rows, grad = torch.ones((3, a), device=DEV), torch.ones((3, b), device=DEV)
        matrices = torch.ones((3, a, b), device=DEV)
        out = fs.flagsparse_expert_product(rows, matrices, route)
        assert out.shape == (3, b) and not bool(out.any())
        gr, gm = fs.flagsparse_expert_product_grad(grad, rows, matrices, route)
        assert gr.shape == (3, a) and gm.shape == matrices.shape and not bool(gr.any())
    rows = torch.ones((0, 8), device=DEV)
    matrices = torch.ones((3, 8, 8), device=DEV)
    assert fs.flagsparse_expert_product(rows, matrices, none).shape == (0, 8)
    gr, gm = fs.flagsparse_expert_product_grad(rows, rows, matrices, none)
    assert gr.shape == (0, 8) and not bool(gm.any())


def test_runs_repeat():
    route = _route((300, 1, 0, 411), 9)
    rows, grad = randn((721, 776), torch.bfloat16, 1), randn((721, 392), torch.bfloat16, 2)
    matrices = randn((4, 776, 392), torch.bfloat16, 3)

    def f():
        return (fs.flagsparse_expert_product(rows, matrices, route),
                *fs.flagsparse_expert_product_grad(grad, rows, matrices, route))

    first = f()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(f(), first))


def test_offsets_past_32_bits():
    # 600,000 rows of 4096 elements: 2.4 G; one matrix for the last rows
    n = 600_000
    route = _route((n - 300, 300))
    rows = torch.zeros((n, 4096), dtype=torch.bfloat16, device=DEV)
    rows[-300:] = randn((300, 4096), torch.bfloat16, 1)
    matrices = randn((2, 4096, 16), torch.bfloat16, 2)
    got = fs.flagsparse_expert_product(rows, matrices, route)
    x, w = rows[-300:].cpu().double(), matrices[1].cpu().double()
    assert_sum(got[-300:], x @ w, x.abs() @ w.abs(), 4096)
    assert not bool(got[:-300].any())
    grad = randn((n, 16), torch.bfloat16, 3)
    gr, gm = fs.flagsparse_expert_product_grad(grad, rows, matrices, route)
    g = grad[-300:].cpu().double()
    assert_sum(gm[1], x.T @ g, x.abs().T @ g.abs(), 300)
    assert_sum(gr[-300:], g @ w.T, g.abs() @ w.abs().T, 16)
    assert not bool(gm[0].any())


@pytest.mark.parametrize("op", ["non", "trans"])
def test_autograd_matches_formula_and_differences(op):
    route = _route((3, 0, 5), 2)
    rows = randn((10, 12), torch.float32, 1).requires_grad_()
    matrices = randn((3, 7, 12) if op == "trans" else (3, 12, 7), torch.float32, 2).requires_grad_()
    seed = randn((10, 7), torch.float32, 3)
    out = fs.flagsparse_expert_product(rows, matrices, route, op=op)
    gr, gm = torch.autograd.grad(out, (rows, matrices), seed)
    want, mag = _oracle(seed, matrices.detach(), route, "non" if op == "trans" else "trans")
    assert_sum(gr, want, mag, 7)
    want, mag = _oracle_matrices(seed, rows.detach(), matrices.detach(), route, op)
    assert_sum(gm, want, mag, 5)
    with torch.no_grad():  # differences of a function linear in each argument, in 64 bits outside the product
        def f(a, b):
            return (fs.flagsparse_expert_product(a, b, route, op=op).double() * seed.double()).sum()

        size = float((out.detach().double().abs() * seed.double().abs()).sum()) + 1000.0
        for r, h in ((0, 0), (7, 11), (9, 3)):
            step = torch.zeros_like(rows)
            step[r, h] = 8.0
            diff = float(f(rows + step, matrices) - f(rows - step, matrices)) / 16
            assert abs(diff - float(gr[r, h])) <= 32 * 2.0**-24 * size
        for at in ((0, 0, 0), (2, 3, 5), (1, 1, 1)):
            step = torch.zeros_like(matrices)
            step[at] = 8.0
            diff = float(f(rows, matrices + step) - f(rows, matrices - step)) / 16
            assert abs(diff - float(gm[at])) <= 32 * 2.0**-24 * size
    # a frozen operand gets none
    frozen = matrices.detach()
    fs.flagsparse_expert_product(rows, frozen, route, op=op).sum().backward()
    assert rows.grad is not None and frozen.grad is None


def test_other_stream_and_graph():
    experts = random_experts(300, 2, 6, 1, 0.1)
    x, w = randn((300, 128), torch.float16, 2), randn((6, 128, 96), torch.float16, 3)
    grad = randn((600, 96), torch.float16, 4)

    def step():
        route = fs.prepare_expert_route(experts, 6)
        rows = fs.flagsparse_expert_dispatch(x, route)
        return (fs.flagsparse_expert_product(rows, w, route), *fs.flagsparse_expert_product_grad(grad, rows, w, route))

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (5, 6, 7):
        experts.copy_(random_experts(300, 2, 6, seed, 0.1))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    route = _route((2, 1))
    rows, matrices, grad = torch.ones((3, 8), device=DEV), torch.ones((2, 8, 4), device=DEV), torch.ones((3, 4), device=DEV)
    with pytest.raises(TypeError, match="route must be a PreparedExpertRoute"):
        fs.flagsparse_expert_product(rows, matrices, None)
    with pytest.raises(TypeError, match="rows dtype must be one of: float16, bfloat16, float32"):
        fs.flagsparse_expert_product(rows.double(), matrices.double(), route)
    with pytest.raises(TypeError, match="matrices dtype must match rows dtype"):
        fs.flagsparse_expert_product(rows, matrices.half(), route)
    with pytest.raises(ValueError, match="matrices must be on the same CUDA device"):
        fs.flagsparse_expert_product(rows, matrices.cpu(), route)
    with pytest.raises(ValueError, match="matrices must be a 3D tensor with 2 matrices"):
        fs.flagsparse_expert_product(rows, matrices[:1], route)
    with pytest.raises(ValueError, match="rows must have width 4"):
        fs.flagsparse_expert_product(rows, matrices, route, op="trans")
    with pytest.raises(ValueError, match="op must be one of"):
        fs.flagsparse_expert_product(rows, matrices, route, op="bad")
    with pytest.raises(ValueError, match="rows must be a 2D tensor with 3 rows"):
        fs.flagsparse_expert_product(rows[:2], matrices, route)
    with pytest.raises(ValueError, match="out shape/dtype must match result"):
        fs.flagsparse_expert_product(rows, matrices, route, out=rows)
    with pytest.raises(ValueError, match="out cannot be given"):
        fs.flagsparse_expert_product(rows, matrices.clone().requires_grad_(), route, out=grad)
    with pytest.raises(ValueError, match="grad must have width 4"):
        fs.flagsparse_expert_product_grad(rows, rows, matrices, route)
    with pytest.raises(TypeError, match="grad dtype must match rows dtype"):
        fs.flagsparse_expert_product_grad(grad.half(), rows, matrices, route)
