"""The example model: gradients of the operators together against the same model
in plain 64-bit torch, training that learns, decoding of single tokens."""

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "routed_layer.py")


def _example():
    spec = importlib.util.spec_from_file_location("routed_layer", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _plain(params, tokens, experts, slots, scale):
    """The model in 64 bits on the CPU, each slot by itself, with the given choice of experts."""
    table, router, into, back = params
    x = table[tokens] * scale
    scores = torch.softmax(x @ router, dim=1)
    weights = torch.gather(scores, 1, experts)
    weights = weights / weights.sum(dim=1, keepdim=True)
    out = x
    for j in range(slots):
        h = torch.nn.functional.silu(torch.einsum("th,tfh->tf", x, into[experts[:, j]]))
        out = out + weights[:, j : j + 1] * torch.einsum("tf,thf->th", h, back[experts[:, j]])
    return out @ table.t()


def test_gradients_match_plain_torch():
    ex = _example()
    model = ex.RoutedLayer(vocab=97, width=48, hidden=40, experts=5, slots=2, dtype=torch.float32, seed=1)
    tokens = torch.randint(0, 97, (150,), generator=torch.Generator().manual_seed(2)).cuda()
    targets = torch.randint(0, 97, (150,), generator=torch.Generator().manual_seed(3)).cuda()
    loss = torch.nn.functional.cross_entropy(model(tokens), targets)
    grads = torch.autograd.grad(loss, model.parameters())
    with torch.no_grad():
        x = model.table[tokens] * model.scale
        experts = torch.topk(torch.softmax(x @ model.router, dim=1), 2, dim=1)[1].cpu()
    params = [p.detach().cpu().double().requires_grad_() for p in model.parameters()]
    want = torch.nn.functional.cross_entropy(_plain(params, tokens.cpu(), experts, 2, model.scale), targets.cpu())
    wants = torch.autograd.grad(want, params)
    # sums of at most 150 x 97 products in 32 bits, normwise: 1e4 half units in the last place
    loss, want = float(loss.detach()), float(want.detach())
    assert abs(loss - want) < 1e4 * 2.0**-24 * want
    for got, ref in zip(grads, wants):
        assert float((got.cpu().double() - ref).norm()) < 1e4 * 2.0**-24 * float(ref.norm())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_learns_and_decodes(dtype):
    ex = _example()
    model = ex.RoutedLayer(vocab=128, width=64, hidden=96, experts=4, slots=2, dtype=dtype, seed=4)
    successor = torch.randperm(128, generator=torch.Generator().manual_seed(5)).cuda()
    losses = ex.train(model, successor, 80, tokens_a_step=1024, rate=1e-2)
    assert losses[-1] < 0.5 * losses[0]
    token, want = torch.tensor(9), []
    for _ in range(6):
        token = successor.cpu()[token]
        want.append(int(token))
    assert ex.decode(model, torch.tensor(9, device="cuda"), 6).tolist() == want
