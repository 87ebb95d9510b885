"""What the routed operators keep for their backward passes: only operands that a
wanted gradient reads.  Others may change before the backward pass, and their
memory is not held."""

import pytest
import torch

import flagsparse_amd as fs
from tests._rows_helpers import ROW_DTYPES, ROW_IDS, randn, random_experts

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _saved_by(call):
    """(result, the tensors saved for its backward pass)."""
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t.data_ptr()) or t, lambda t: t):
        return call(), saved


@pytest.mark.parametrize("op", ["non", "trans"])
def test_product_keeps_the_other_operand(op):
    route = fs.prepare_expert_route(random_experts(60, 2, 4, 1, 0.1), 4)
    rows, matrices = randn((120, 24), torch.float32, 2), randn((4, 24, 24), torch.float32, 3)
    seed = randn((120, 24), torch.float32, 4)
    want = fs.flagsparse_expert_product_grad(seed, rows, matrices, route, op=op)
    for k, frozen in ((0, 1), (1, 0)):
        operands = [rows.clone(), matrices.clone()]
        leaf = operands[k].requires_grad_()
        operands[k] = leaf * 1.0
        out, saved = _saved_by(lambda: fs.flagsparse_expert_product(*operands, route, op=op))
        assert saved == [operands[frozen].data_ptr()]
        operands[k].mul_(3.0)  # its own gradient does not read it
        (got,) = torch.autograd.grad(out, leaf, seed)
        assert torch.equal(got, want[k])
    both = [t.clone().requires_grad_() for t in (rows, matrices)]
    out, saved = _saved_by(lambda: fs.flagsparse_expert_product(*both, route, op=op))
    assert sorted(saved) == sorted(t.data_ptr() for t in both)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, both, seed), want))


@pytest.mark.parametrize("width", [0, 1, 7, 136, 515])
@pytest.mark.parametrize("dtype", ROW_DTYPES, ids=ROW_IDS)
def test_combine_keeps_the_other_operand(dtype, width):
    experts = random_experts(90, 3, 5, 1, 0.1)
    route = fs.prepare_expert_route(experts, 5)
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    rows, weights, seed = randn((270, width), dtype, 2), randn((90, 3), wide, 3), randn((90, width), dtype, 4)
    lost = ((experts < 0) | (experts >= 5)).reshape(-1)[route.order.long()]
    rows[lost] = float("nan")
    want = fs.flagsparse_expert_combine_grad(seed, rows, route, weights)
    for k, frozen in ((0, 1), (1, 0)):
        operands = [rows.clone(), weights.clone()]
        leaf = operands[k].requires_grad_()
        operands[k] = leaf * 1.0
        out, saved = _saved_by(lambda: fs.flagsparse_expert_combine(operands[0], route, operands[1]))
        assert saved == [operands[frozen].data_ptr()]
        operands[k].mul_(3.0)
        (got,) = torch.autograd.grad(out, leaf, seed)
        assert got.dtype == want[k].dtype and torch.equal(got, want[k])
    both = [t.clone().requires_grad_() for t in (rows, weights)]
    out = fs.flagsparse_expert_combine(both[0], route, both[1])
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, both, seed), want))
    # without weights nothing is kept
    leaf = rows.clone().requires_grad_()
    out, saved = _saved_by(lambda: fs.flagsparse_expert_combine(leaf, route))
    assert saved == []
    (got,) = torch.autograd.grad(out, leaf, seed)
    assert torch.equal(got, fs.flagsparse_expert_dispatch(seed, route))


def test_combine_gradients_alone_past_the_caches():
    # over 256 MB each way, rows of whole words that end off 16 bytes
    route = fs.prepare_expert_route(random_experts(20000, 4, 8, 1, 0.02), 8)
    rows, weights = randn((80000, 8), torch.float16, 2).repeat(1, 254)[:, :2026], randn((20000, 4), torch.float32, 3)
    rows, seed = rows.contiguous(), randn((20000, 8), torch.float16, 4).repeat(1, 254)[:, :2026].contiguous()
    want = fs.flagsparse_expert_combine_grad(seed, rows, route, weights)
    for k in (0, 1):
        operands = [rows, weights]
        operands[k] = operands[k].clone().requires_grad_()
        out = fs.flagsparse_expert_combine(operands[0], route, operands[1])
        (got,) = torch.autograd.grad(out, operands[k], seed)
        assert torch.equal(got, want[k])


def test_combine_grad_rows_are_products_in_32_bits():
    # the same rounding in every element: that of the 32-bit product
    route = fs.prepare_expert_route(random_experts(3000, 4, 8, 1), 8)
    rows, seed = randn((12000, 515), torch.float16, 2), randn((3000, 515), torch.float16, 4)
    weights = randn((3000, 4), torch.float32, 3)
    grad_rows, _ = fs.flagsparse_expert_combine_grad(seed, rows, route, weights)
    order = route.order.long()
    want = (weights.reshape(-1)[order][:, None] * seed[order // 4].float()).half()
    assert torch.equal(grad_rows, want)
