"""Where the row operators write, with the library and the stream replaced by
recorders (no GPU): a result given with out= that shares memory with an operand
is written elsewhere and copied, since the kernels' workgroups read operands
while others write."""

import ctypes
from types import SimpleNamespace

import pytest
import torch

import flagsparse_amd.embedding as embedding
import flagsparse_amd.expert as expert
from flagsparse_amd import _lib
from flagsparse_amd._rows import check_out

VALUE = 7.0


@pytest.fixture
def written(monkeypatch):
    """The addresses that the calls' kernels would write, in order."""
    calls = []

    def call(at):
        def function(*args):
            calls.append(args[at])
            return 0
        return function

    lib = SimpleNamespace(
        fs_embedding=call(9), fs_embedding_grad=call(11), fs_embedding_grad_workspace_bytes=lambda *a: 64,
        fs_expert_dispatch=call(9), fs_expert_combine=call(10), fs_expert_product=call(10),
        fs_expert_product_workspace_bytes=lambda *a: 0)
    monkeypatch.setattr(_lib, "lib", lambda: lib)
    monkeypatch.setattr(_lib, "stream_handle", lambda device: 11)
    monkeypatch.setattr(embedding, "_check_tokens", lambda *a: None)
    monkeypatch.setattr(embedding, "check_out", lambda *a: None)
    return calls


def _route(n_tokens, slots=1, experts=2):
    n = n_tokens * slots
    return expert.PreparedExpertRoute(n_tokens, slots, experts, torch.zeros(2 * n + experts + 1, dtype=torch.int32), 11)


def _calls(x, out, tokens):
    """Every call that takes out=, with x (8 x 8, or a view of as many values) among its operands."""
    route = _route(8)
    matrices = torch.ones(2, 8, 8)
    return {
        "embedding": lambda: embedding._lookup(x, tokens, 1.0, out),
        "embedding_grad": lambda: embedding.flagsparse_embedding_grad(x, tokens, 8, out=out),
        "dispatch": lambda: expert._dispatch(x, route, out),
        "combine": lambda: expert._combine(x, route, None, out),
        "combine_weights": lambda: expert._combine(torch.ones(8, 8), route, x.reshape(-1)[:8].reshape(8, 1), out),
        "product_rows": lambda: expert._product(x, matrices, route, False, 8, 8, out),
    }


NAMES = ["embedding", "embedding_grad", "dispatch", "combine", "combine_weights", "product_rows"]


@pytest.mark.parametrize("name", NAMES)
def test_out_sharing_memory_is_written_last(written, name):
    store, tokens = torch.zeros(200), torch.arange(8)
    x = store[64:128].view(8, 8)
    # the operand itself, its first and its last element
    for start in (64, 1, 71 if name == "combine_weights" else 127):
        out = store[start : start + 64].view(8, 8)
        assert _calls(x, out, tokens)[name]() is out
        at = written.pop()
        assert not (store.data_ptr() < at + 4 * 64 and at < store.data_ptr() + 4 * 200), start
    # next to it: no copy
    for start in (0, 128):
        out = store[start : start + 64].view(8, 8)
        assert _calls(x, out, tokens)[name]() is out
        assert written.pop() == out.data_ptr()


def test_out_sharing_memory_with_tokens_and_matrices(written):
    tokens = torch.arange(32, dtype=torch.int64)
    out = tokens.view(torch.float32).view(8, 8)
    for call in (lambda: embedding._lookup(torch.ones(8, 8), tokens[:8], 1.0, out),
                 lambda: embedding.flagsparse_embedding_grad(torch.ones(8, 8), tokens[:8], 8, out=out)):
        assert call() is out and written.pop() != out.data_ptr()
    matrices = torch.ones(2, 8, 8)
    for m in (matrices, matrices.transpose(1, 2)):
        out = matrices[1]
        assert expert._product(torch.ones(8, 8), m, _route(8), False, 8, 8, out) is out
        assert written.pop() != out.data_ptr()


def test_the_result_reaches_out(monkeypatch, written):
    """What the kernel writes elsewhere is copied; a strided out is, as before."""
    x = torch.zeros(8, 8)

    def write(*args):
        for i in range(64):
            ctypes.c_float.from_address(args[9] + 4 * i).value = VALUE + i
        return 0

    monkeypatch.setattr(_lib.lib(), "fs_expert_dispatch", write)
    want = VALUE + torch.arange(64.0).view(8, 8)
    assert torch.equal(expert._dispatch(x, _route(8), x), want) and torch.equal(x, want)
    wide = torch.zeros(8, 16)
    expert._dispatch(torch.zeros(8, 8), _route(8), wide[:, ::2])
    assert torch.equal(wide[:, ::2], want) and not bool(wide[:, 1::2].any())


@pytest.mark.parametrize("name", NAMES)
def test_autograd_learns_of_the_write(written, name):
    """A backward pass that needs the values which out= replaced raises, where the
    kernel writes out itself and where the result is copied."""
    x, tokens = torch.ones(8, 8), torch.arange(8)
    for out in (torch.ones(8, 8), torch.ones(8, 16)[:, ::2], x):
        factor = torch.ones(8, 8, requires_grad=True)
        product = factor * out
        with torch.no_grad():
            _calls(x, out, tokens)[name]()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            product.sum().backward()


def test_out_with_a_graph_is_refused(monkeypatch):
    """out's graph would go on to give the gradient of the values it held before."""
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    held = torch.ones(8, 8, requires_grad=True) * 2.0
    with pytest.raises(ValueError, match="out cannot be given where a gradient is recorded"):
        check_out(held, held.device, (8, 8), torch.float32)
    with torch.no_grad():
        check_out(held, held.device, (8, 8), torch.float32)
    check_out(held.detach(), held.device, (8, 8), torch.float32)
