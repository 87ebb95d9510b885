"""A route prepared on one stream and used on another, dropped right after the call,
and inside a graph captured on a stream of its own."""

import pytest
import torch

import flagsparse_amd as fs
from tests._rows_helpers import randn, random_experts

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _step(route, x, matrices, weights):
    rows = fs.flagsparse_expert_product(fs.flagsparse_expert_dispatch(x, route), matrices, route)
    return (rows, fs.flagsparse_expert_combine(rows, route, weights),
            *fs.flagsparse_expert_combine_grad(x, rows, route, weights))


def _operands(n):
    return randn((n, 64), torch.bfloat16, 1), randn((6, 64, 64), torch.bfloat16, 2), randn((n, 2), torch.float32, 3)


def test_dropped_after_a_call_on_another_stream():
    operands = _operands(3000)
    experts = [random_experts(3000, 2, 6, seed, 0.1) for seed in range(8)]
    want = [_step(fs.prepare_expert_route(e, 6), *operands) for e in experts]
    side = torch.cuda.Stream()
    for e, w in zip(experts, want):
        route = fs.prepare_expert_route(e, 6)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = _step(route, *operands)
        places = route.order.untyped_storage().nbytes()
        del route
        # the next owner of memory of that size, on the stream that prepared the route
        torch.full((places,), 0, dtype=torch.uint8, device=DEV)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, w))


def test_prepared_before_a_graph_that_uses_it():
    x, matrices, weights = _operands(500)
    route = fs.prepare_expert_route(random_experts(500, 2, 6, 1, 0.1), 6)
    _step(route, x, matrices, weights)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _step(route, x, matrices, weights)
    for _ in range(3):
        x.mul_(1.5)
        want = _step(route, x, matrices, weights)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
