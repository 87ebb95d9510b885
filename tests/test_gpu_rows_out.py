"""The row operators with a result given by out= that shares memory with an
operand: the same result as without."""

import pytest
import torch

import flagsparse_amd as fs
from tests._rows_helpers import randn, random_experts

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float16, torch.bfloat16, torch.float32]
IDS = ["f16", "bf16", "f32"]


def _calls(n, width, dtype):
    """name -> (a call of x (n, width) and out) for each operator that takes out=."""
    tokens = torch.randint(0, n, (n,), generator=torch.Generator().manual_seed(1)).to(DEV)
    route = fs.prepare_expert_route(random_experts(n, 1, 3, 2, 0.1), 3)
    weights, matrices = randn((n, 1), torch.float32, 3), randn((3, width, width), dtype, 4)
    return {
        "embedding": lambda x, out=None: fs.flagsparse_embedding(x, tokens, scale=3.0, out=out),
        "embedding_grad": lambda x, out=None: fs.flagsparse_embedding_grad(x, tokens, n, out=out),
        "dispatch": lambda x, out=None: fs.flagsparse_expert_dispatch(x, route, out=out),
        "dispatch_grad": lambda x, out=None: fs.flagsparse_expert_dispatch_grad(x, route, out=out),
        "combine": lambda x, out=None: fs.flagsparse_expert_combine(x, route, weights, out=out),
        "product": lambda x, out=None: fs.flagsparse_expert_product(x, matrices, route, out=out),
        "product_trans": lambda x, out=None: fs.flagsparse_expert_product(x, matrices, route, op="trans", out=out),
    }


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,width", [(9, 8), (700, 72), (5000, 264)])
def test_out_shares_memory_with_the_rows(n, width, dtype):
    values = randn((n, width), dtype, 5)
    for name, call in _calls(n, width, dtype).items():
        want = call(values)
        for shift in (0, 3, width, n * width - 1):  # where out begins behind the rows
            store = torch.zeros(2 * n * width, dtype=dtype, device=DEV)
            x, out = store[: n * width].view(n, width), store[shift : shift + n * width].view(n, width)
            x.copy_(values)
            assert call(x, out) is out
            assert torch.equal(out, want), (name, shift)
        # every second row and column of a tensor that is its own operand
        store = torch.zeros((2 * n, 2 * width), dtype=dtype, device=DEV)
        x = store[::2, ::2]
        x.copy_(values)
        assert torch.equal(call(x, x), want) and torch.equal(x, want), name


def test_out_shares_memory_with_weights_and_matrices():
    route = fs.prepare_expert_route(random_experts(300, 64, 5, 2, 0.1), 5)
    rows, weights = randn((300 * 64, 64), torch.float32, 1), randn((300, 64), torch.float32, 2)
    want = fs.flagsparse_expert_combine(rows, route, weights)
    assert torch.equal(fs.flagsparse_expert_combine(rows, route, weights, out=weights), want)
    assert torch.equal(weights, want)
    route = fs.prepare_expert_route(random_experts(96, 1, 5, 2, 0.1), 5)
    rows, matrices = randn((96, 96), torch.float32, 3), randn((5, 96, 96), torch.float32, 4)
    want = fs.flagsparse_expert_product(rows, matrices, route)
    assert torch.equal(fs.flagsparse_expert_product(rows, matrices, route, out=matrices[2]), want)
