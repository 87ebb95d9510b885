"""Forward-mode tangents, which the row operators do not propagate: an error, not a
result without them (no GPU: the checks before any launch)."""

import pytest
import torch
from torch.autograd import forward_ad

import flagsparse_amd as fs
from flagsparse_amd import _lib
from flagsparse_amd.expert import PreparedExpertRoute


@pytest.fixture
def launched(monkeypatch):
    """The library calls made, with tensors taken for GPU tensors."""
    calls = []

    class Library:
        def __getattr__(self, name):
            return lambda *args: calls.append(name) or 0

    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    monkeypatch.setattr(_lib, "lib", lambda: Library())
    monkeypatch.setattr(_lib, "stream_handle", lambda device: 11)
    return calls


def test_tangents_are_refused(launched):
    tokens, route = torch.arange(4), PreparedExpertRoute(4, 1, 2, torch.zeros(11, dtype=torch.int32), 11)
    x, w, m = torch.ones(4, 8), torch.ones(4, 1), torch.ones(2, 8, 8)
    calls = {
        "table": lambda t: fs.flagsparse_embedding(t(x), tokens),
        "grad of tokens": lambda t: fs.flagsparse_embedding_grad(t(x), tokens, 4),
        "x": lambda t: fs.flagsparse_expert_dispatch(t(x), route),
        "grad of dispatch": lambda t: fs.flagsparse_expert_dispatch_grad(t(x), route),
        "rows": lambda t: fs.flagsparse_expert_combine(t(x), route, w),
        "weights": lambda t: fs.flagsparse_expert_combine(x, route, t(w)),
        "grad of combine": lambda t: fs.flagsparse_expert_combine_grad(t(x), x, route, w),
        "rows of combine": lambda t: fs.flagsparse_expert_combine_grad(x, t(x), route, w),
        "weights of combine": lambda t: fs.flagsparse_expert_combine_grad(x, x, route, t(w)),
        "rows of product": lambda t: fs.flagsparse_expert_product(t(x), m, route),
        "matrices": lambda t: fs.flagsparse_expert_product(x, t(m), route),
        "grad of product": lambda t: fs.flagsparse_expert_product_grad(t(x), x, m, route),
        "matrices of product": lambda t: fs.flagsparse_expert_product_grad(x, x, t(m), route),
    }
    for name, call in calls.items():
        with forward_ad.dual_level():
            call(lambda v: v)  # none of its own inside the level
            assert launched, name
            launched.clear()
            for grad in (torch.no_grad(), torch.enable_grad()):
                with grad, pytest.raises(NotImplementedError, match=f"{name.split(' ')[0]} has a forward-mode tangent"):
                    call(lambda v: forward_ad.make_dual(v, torch.ones_like(v)))
            assert not launched, name
        call(lambda v: v)
        launched.clear()
