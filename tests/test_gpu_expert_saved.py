"""What the routed operators keep for their backward passes: only operands that a
wanted gradient reads.  Others may change before the backward pass, and their
memory is not held."""

import pytest
import torch

import flagsparse_amd as fs
from tests._rows_helpers import randn, random_experts

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
