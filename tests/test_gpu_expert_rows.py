"""Routing of tokens to experts (select_sort.hip) and rows into expert order and
back (expert_rows.hip) against the definitions in 64 bits on the CPU."""

import pytest
import torch

import flagsparse_amd as fs
from flagsparse_amd import _lib
from tests._rows_helpers import ROW_DTYPES, ROW_IDS, assert_sum, randn, random_experts, route_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _same_route(route, experts, num_experts):
    order, inverse, offsets = route_oracle(experts, num_experts)
    assert route.order.dtype == route.inverse.dtype == route.offsets.dtype == torch.int32
    assert torch.equal(route.offsets.cpu(), offsets)
    assert torch.equal(route.order.cpu(), order)
    assert torch.equal(route.inverse.cpu(), inverse)


@pytest.mark.parametrize("num_experts", [1, 2, 7, 8, 63, 64, 255, 256, 511, 512, 1023])
@pytest.mark.parametrize("n_tokens,slots", [(1, 1), (1, 8), (3, 2), (64, 1), (65, 1), (511, 8), (512, 8), (4097, 1),
                                            (3001, 6)])
def test_route(n_tokens, slots, num_experts):
    for dtype, dropped in ((torch.int32, 0.0), (torch.int64, 0.3)):
        experts = random_experts(n_tokens, slots, num_experts, n_tokens + num_experts, dropped, dtype)
        _same_route(fs.prepare_expert_route(experts, num_experts), experts, num_experts)


def test_route_special_ids():
    for fill in (0, 6, 7, -1, 2**31 - 1, -(2**31), 2**32 + 1, -(2**63), 2**63 - 1):
        experts = torch.full((300, 3), fill, dtype=torch.int64, device=DEV)
        experts[17, 1] = 2
        route = fs.prepare_expert_route(experts, 7)
        _same_route(route, experts, 7)
    assert int(fs.prepare_expert_route(experts, 7).offsets[-1]) == 1
    empty = fs.prepare_expert_route(experts[:0], 7)
    assert empty.offsets.tolist() == [0] * 8 and empty.order.numel() == 0 and empty.n_rows == 0
    _same_route(fs.prepare_expert_route(experts.t().contiguous().t(), 7), experts, 7)


def test_route_many_tiles():
    # within and beyond the tiles that a scatter adds up itself
    for n_tokens in (40000, 4096 * 520 // 4 + 5):
        experts = random_experts(n_tokens, 4, 60, n_tokens, 0.05)
        route = fs.prepare_expert_route(experts, 60)
        flat = experts.reshape(-1).long()
        key = torch.where((flat >= 0) & (flat < 60), flat, 60)
        order = torch.sort(key.cpu(), stable=True)[1]
        assert torch.equal(route.order.cpu().long(), order)
        assert torch.equal(route.inverse.reshape(-1).cpu().long()[order], torch.arange(len(order)))
        assert torch.equal(route.offsets[1:].cpu().long(), torch.cumsum(torch.bincount(key.cpu(), minlength=61), 0)[:60])


CASES = [(1, 1, 1, 0.0), (1, 8, 16, 0.0), (5, 2, 3, 0.5), (130, 6, 20, 0.1), (64, 9, 33, 1.0), (333, 3, 8, 0.02)]
CASE_IDS = [f"{t}x{k}of{e}" for t, k, e, _ in CASES]


def _case(case, seed=0):
    n_tokens, slots, num_experts, dropped = case
    experts = random_experts(n_tokens, slots, num_experts, seed + n_tokens, dropped)
    route = fs.prepare_expert_route(experts, num_experts)
    inverse = route_oracle(experts, num_experts)[1].long()
    inside = ((experts >= 0) & (experts < num_experts)).cpu()
    return route, inverse, inside


@pytest.mark.parametrize("width", [1, 5, 8, 100, 127, 512, 2056])
@pytest.mark.parametrize("case", CASES, ids=CASE_IDS)
@pytest.mark.parametrize("dtype", ROW_DTYPES, ids=ROW_IDS)
def test_dispatch_combine_and_gradients(dtype, case, width):
    route, inverse, inside = _case(case)
    n_tokens, slots = inverse.shape
    x = randn((n_tokens, width), dtype, 1)
    rows = fs.flagsparse_expert_dispatch(x, route)
    want = torch.zeros((n_tokens * slots, width), dtype=dtype)
    for j in range(slots):
        want[inverse[inside[:, j], j]] = x.cpu()[inside[:, j]]
    assert rows.dtype == dtype and torch.equal(rows.cpu(), want)

    y = randn((n_tokens * slots, width), dtype, 2)
    y[inverse[~inside].to(DEV)] = float("nan")  # rows of no expert are not read
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    weights = randn((n_tokens, slots), wide, 3)
    weights[~inside.to(DEV)] = float("inf")
    term = torch.where(inside[:, :, None], y.cpu().double()[inverse], 0.0)
    term_w = term * torch.where(inside, weights.cpu().double(), 0.0)[:, :, None]
    assert_sum(fs.flagsparse_expert_combine(y, route, weights), term_w.sum(1), term_w.abs().sum(1), slots)
    assert_sum(fs.flagsparse_expert_combine(y, route), term.sum(1), term.abs().sum(1), slots)
    assert_sum(fs.flagsparse_expert_dispatch_grad(y, route), term.sum(1), term.abs().sum(1), slots)

    grad = randn((n_tokens, width), dtype, 4)
    grad_rows, grad_weights = fs.flagsparse_expert_combine_grad(grad, y, route, weights)
    product = grad.cpu().double()[:, None, :] * torch.where(inside, weights.cpu().double(), 0.0)[:, :, None]
    want = torch.zeros((n_tokens * slots, width), dtype=torch.float64)
    want[inverse.reshape(-1)] = product.reshape(-1, width)
    assert grad_rows.dtype == dtype and grad_weights.dtype == wide
    assert_sum(grad_rows, want, want.abs(), 1)
    dots = term * grad.cpu().double()[:, None, :]
    assert_sum(grad_weights, dots.sum(2), dots.abs().sum(2), width, arithmetic=wide)


def test_strides_and_out():
    route, inverse, inside = _case((70, 3, 5, 0.1))
    x, y = randn((70, 3 * 48), torch.bfloat16, 1), randn((210, 3 * 48), torch.bfloat16, 2)
    w = randn((3, 70), torch.float32, 3).t()
    for cut in (slice(0, 48), slice(1, 48), slice(None, None, 3)):
        xc, yc = x[:, cut].contiguous(), y[:, cut].contiguous()
        rows, back = fs.flagsparse_expert_dispatch(xc, route), fs.flagsparse_expert_combine(yc, route, w.contiguous())
        assert torch.equal(fs.flagsparse_expert_dispatch(x[:, cut], route), rows)
        assert torch.equal(fs.flagsparse_expert_combine(y[:, cut], route, w), back)
        grads = fs.flagsparse_expert_combine_grad(xc, yc, route, w.contiguous())
        assert all(torch.equal(a, b) for a, b in zip(fs.flagsparse_expert_combine_grad(x[:, cut], y[:, cut], route, w), grads))
        out = torch.full_like(rows, 7.0)
        assert fs.flagsparse_expert_dispatch(xc, route, out=out) is out and torch.equal(out, rows)
        room = torch.zeros((70, 2 * back.shape[1]), dtype=back.dtype, device=DEV)
        assert torch.equal(fs.flagsparse_expert_combine(yc, route, w, out=room[:, ::2]), back)
        assert torch.equal(room[:, ::2], back) and not bool(room[:, 1::2].any())
        out = torch.full_like(back, 7.0)
        assert fs.flagsparse_expert_dispatch_grad(yc, route, out=out) is out
        assert torch.equal(out, fs.flagsparse_expert_combine(yc, route))


def test_offsets_past_32_bits():
    n_tokens, slots, width = 70_000, 4, 8192  # 2.3 G elements of rows
    experts = random_experts(n_tokens, slots, 8, 1)
    route = fs.prepare_expert_route(experts, 8)
    x = (torch.arange(n_tokens, device=DEV) % 251).to(torch.bfloat16)[:, None].expand(n_tokens, width).contiguous()
    rows = fs.flagsparse_expert_dispatch(x, route)
    last = route.order[-5:].long()
    assert torch.equal(rows[-5:], x[last // slots])
    w = torch.ones((n_tokens, slots), device=DEV)
    out = fs.flagsparse_expert_combine(rows, route, w)
    assert torch.equal(out[-3:], (x[-3:].float() * slots).bfloat16())
    del out
    grad_rows, grad_w = fs.flagsparse_expert_combine_grad(x, rows, route, w)
    assert torch.equal(grad_rows[-5:], rows[-5:])
    assert torch.equal(grad_w[-1], (x[-1, 0].float() ** 2 * width).expand(slots))


def test_more_slots_than_one_grid_dimension_has_threads_for():
    n_tokens = 34_000_000  # 68 M slots, a wave each: over 2^32 threads
    experts = torch.zeros((n_tokens, 2), dtype=torch.int32, device=DEV)
    experts[:, 1] = 1
    experts[-3, 0] = -1
    route = fs.prepare_expert_route(experts, 2)
    assert route.offsets.tolist() == [0, n_tokens - 1, 2 * n_tokens - 1]
    grad = torch.ones((n_tokens, 8), dtype=torch.float16, device=DEV)
    rows = torch.full((2 * n_tokens, 8), 2.0, dtype=torch.float16, device=DEV)
    grad_rows, grad_weights = fs.flagsparse_expert_combine_grad(grad, rows, route, torch.full((n_tokens, 2), 0.5, device=DEV))
    assert bool((grad_rows[:-1] == 0.5).all()) and not bool(grad_rows[-1].any())
    assert float(grad_weights[-3, 0]) == 0.0 and int((grad_weights == 16.0).sum()) == 2 * n_tokens - 1


def test_autograd_matches_formula_and_differences():
    route, inverse, inside = _case((9, 3, 4, 0.2))
    x = randn((9, 5), torch.float64, 1).requires_grad_()
    w = randn((9, 3), torch.float64, 2).requires_grad_()
    scale = randn((27, 5), torch.float64, 3)
    seed = randn((9, 5), torch.float64, 4)

    def f(x, w):
        rows = fs.flagsparse_expert_dispatch(x, route)
        return (fs.flagsparse_expert_combine(rows * scale, route, w) * seed).sum()

    gx, gw = torch.autograd.grad(f(x, w), (x, w))
    s = scale.cpu()[inverse] * inside[:, :, None]
    xd, wd, sd = x.detach().cpu(), w.detach().cpu(), seed.cpu()
    want_x = (s * wd[:, :, None]).sum(1) * sd
    want_w = (s * (xd * sd)[:, None, :]).sum(2)
    assert torch.allclose(gx.cpu(), want_x, rtol=1e-13, atol=1e-13)
    assert torch.allclose(gw.cpu(), want_w, rtol=1e-13, atol=1e-13)
    with torch.no_grad():  # differences of a function linear in each argument
        for t, h in ((0, 0), (4, 3), (8, 4)):
            step = torch.zeros_like(x)
            step[t, h] = 0.5
            assert abs(float(f(x + step, w) - f(x - step, w) - gx[t, h])) < 1e-12
        for t, j in ((0, 0), (4, 2), (8, 1)):
            step = torch.zeros_like(w)
            step[t, j] = 0.5
            assert abs(float(f(x, w + step) - f(x, w - step) - gw[t, j])) < 1e-12
    # without weights
    x2 = x.detach().requires_grad_()
    (fs.flagsparse_expert_combine(fs.flagsparse_expert_dispatch(x2, route), route) * seed).sum().backward()
    assert torch.allclose(x2.grad.cpu(), sd * inside.sum(1, keepdim=True), rtol=1e-14, atol=0)


def test_other_stream_and_graph():
    experts = random_experts(600, 4, 12, 1, 0.1)
    x, w = randn((600, 72), torch.float16, 2), randn((600, 4), torch.float32, 3)

    def step():
        route = fs.prepare_expert_route(experts, 12)
        rows = fs.flagsparse_expert_dispatch(x, route)
        return (route.order, route.offsets, rows, fs.flagsparse_expert_combine(rows, route, w),
                *fs.flagsparse_expert_combine_grad(x, rows, route, w))

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
        experts.copy_(random_experts(600, 4, 12, seed, 0.1))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_kernel_names():
    fs.prepare_expert_route(random_experts(5000, 1, 3, 1), 3)
    assert _lib.last_kernel() == "select_scatter_kernel"
    route, _, _ = _case((4, 2, 3, 0.0))
    assert _lib.last_kernel() == "select_small_kernel"
    x = randn((4, 8), torch.float32, 1)
    rows = fs.flagsparse_expert_dispatch(x, route)
    assert _lib.last_kernel() == "expert_dispatch_kernel"
    fs.flagsparse_expert_combine(rows, route)
    assert _lib.last_kernel() == "expert_combine_kernel"
    fs.flagsparse_expert_combine_grad(x, rows, route, torch.ones((4, 2), device=DEV))
    assert _lib.last_kernel() == "expert_combine_grad_kernel"


def test_refusals():
    experts = random_experts(4, 2, 3, 1)
    with pytest.raises(TypeError, match="experts must be a torch.Tensor"):
        fs.prepare_expert_route([[0]], 3)
    with pytest.raises(ValueError, match="experts must be a 2D tensor"):
        fs.prepare_expert_route(experts[0], 3)
    with pytest.raises(TypeError, match="experts dtype must be"):
        fs.prepare_expert_route(experts.float(), 3)
    with pytest.raises(ValueError, match="experts must be a CUDA tensor"):
        fs.prepare_expert_route(experts.cpu(), 3)
    for bad in (0, -1, 1024):
        with pytest.raises(ValueError, match="num_experts must be in 1..1023"):
            fs.prepare_expert_route(experts, bad)
    with pytest.raises(ValueError, match="at least one slot"):
        fs.prepare_expert_route(experts[:, :0], 3)
    route = fs.prepare_expert_route(experts, 3)
    x, rows, w = (torch.ones(s, device=DEV) for s in ((4, 8), (8, 8), (4, 2)))
    with pytest.raises(TypeError, match="route must be a PreparedExpertRoute"):
        fs.flagsparse_expert_dispatch(x, experts)
    with pytest.raises(TypeError, match="x dtype must be one of"):
        fs.flagsparse_expert_dispatch(x.int(), route)
    with pytest.raises(ValueError, match="x must be a CUDA tensor"):
        fs.flagsparse_expert_dispatch(x.cpu(), route)
    with pytest.raises(ValueError, match="x must be a 2D tensor with 4 rows"):
        fs.flagsparse_expert_dispatch(rows, route)
    with pytest.raises(ValueError, match="rows must be a 2D tensor with 8 rows"):
        fs.flagsparse_expert_combine(x, route, w)
    with pytest.raises(TypeError, match="weights dtype must be torch.float32"):
        fs.flagsparse_expert_combine(rows, route, w.half())
    with pytest.raises(ValueError, match="weights must have shape"):
        fs.flagsparse_expert_combine(rows, route, w.t())
    with pytest.raises(ValueError, match="weights must be on the same CUDA device"):
        fs.flagsparse_expert_combine(rows, route, w.cpu())
    with pytest.raises(ValueError, match="out shape/dtype must match result"):
        fs.flagsparse_expert_combine(rows, route, w, out=rows)
    with pytest.raises(ValueError, match="out cannot be given"):
        fs.flagsparse_expert_combine(rows, route, w.requires_grad_(), out=x)
    with pytest.raises(ValueError, match="grad must have width 8"):
        fs.flagsparse_expert_combine_grad(x[:, :4], rows, route, w.detach())
    with pytest.raises(TypeError, match="grad dtype must match rows dtype"):
        fs.flagsparse_expert_combine_grad(x.half(), rows, route, w.detach())
