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
    return PreparedExpertRoute(n_tokens, slots, experts, torch.zeros(2 * n + experts + 1, dtype=torch.int32), 11)


@pytest.mark.parametrize("changed", ["rows", "matrices"])
def test_product_operand_with_a_gradient_may_change(launched, changed):
    rows, matrices = torch.ones(4, 8), torch.ones(2, 8, 8)
    t = (rows if changed == "rows" else matrices).requires_grad_() * 1.0
    operands = (t, matrices) if changed == "rows" else (rows, t)
    out = fs.flagsparse_expert_product(*operands, _route(4))
    t.mul_(2.0)
    out.sum().backward()  # reads the other one
    names = [name for name, _ in launched if not name.endswith("bytes")]
    assert names == ["fs_expert_product",
                     "fs_expert_product" if changed == "rows" else "fs_expert_product_grad_matrices"]


def test_combine_operand_with_a_gradient_may_change(launched):
    route = _route(4, 2)
    # each gradient alone: the call names no operand that it does not need
    for changed in ("rows", "weights"):
        rows, weights = torch.ones(8, 8), torch.ones(4, 2)
        t = (rows if changed == "rows" else weights).requires_grad_() * 1.0
        operands = (t, route, weights) if changed == "rows" else (rows, route, t)
        out = fs.flagsparse_expert_combine(*operands)
        t.mul_(2.0)
        out.sum().backward()
        (_, _), (name, args) = launched
        launched.clear()
        assert name == "fs_expert_combine_grad"
        given = [args[k] is not None for k in (7, 11, 12, 13)]  # rows, weights, and their gradients
        assert given == ([False, True, True, False] if changed == "rows" else [True, False, False, True])
    # without weights nothing is kept
    rows = torch.ones(8, 8, requires_grad=True) * 1.0
    out = fs.flagsparse_expert_combine(rows, route)
    rows.mul_(2.0)
    out.sum().backward()
    assert [name for name, _ in launched] == ["fs_expert_combine", "fs_expert_dispatch"]


def test_c_combine_grad_refusals():
    lib = _lib.load_library()
    fake, f32 = 4096, _lib.FS_F32

    def call(width, rows, weights, grad_rows, grad_weights):
        return lib.fs_expert_combine_grad(f32, 4, 2, width, 4, fake, 8, rows, 8, fake, fake, weights, grad_rows,
                                          grad_weights, None)

    for args in ((8, fake, None, fake, fake), (8, None, fake, fake, fake), (8, fake, fake, None, None),
                 (8, None, fake, None, fake), (8, fake, None, fake, None)):
        assert call(*args) == _lib.FS_E_INVALID
        assert "bad pointer or stride" in lib.fs_last_error().decode()
    assert call(0, None, fake, None, None) == 0  # of no columns there is nothing to write
