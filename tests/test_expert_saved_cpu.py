"""The routed operators' saved tensors with the library replaced by a recorder (no
GPU): an operand that no wanted gradient reads may be written between the forward
and the backward pass."""

import pytest
import torch

import flagsparse_amd as fs
from flagsparse_amd import _lib
from flagsparse_amd.expert import PreparedExpertRoute


@pytest.fixture
def launched(monkeypatch):
    calls = []

    class Library:
        def __getattr__(self, name):
            return lambda *args: calls.append((name, args)) or 0

    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    monkeypatch.setattr(_lib, "lib", lambda: Library())
    monkeypatch.setattr(_lib, "stream_handle", lambda device: 11)
    return calls


def _route(n_tokens, slots=1, experts=2):
    n = n_tokens * slots
    return PreparedExpertRoute(n_tokens, slots, experts, torch.zeros(2 * n + experts + 1, dtype=torch.int32))


@pytest.mark.parametrize("changed", ["rows", "matrices"])
def test_product_operand_with_a_gradient_may_change(launched, changed):
    rows, matrices = torch.ones(4, 8), torch.ones(2, 8, 8)
    t = (rows if changed == "rows" else matrices).requires_grad_() * 1.0
    out = fs.flagsparse_expert_product(t if changed == "rows" else rows, t if changed == "matrices" else matrices, _route(4))
    t.mul_(2.0)
    out.sum().backward()  # reads the other one
    names = [name for name, _ in launched if not name.endswith("bytes")]
    assert names == ["fs_expert_product", "fs_expert_product" if changed == "rows" else "fs_expert_product_grad_matrices"]
