"""Row operators at sizes where code of its own begins: results stored past the
caches (256 MB in all), and sorts of every number of tiles.  Values are whole
numbers whose sums are exact in 32 bits, so results are compared for equality."""

import pytest
import torch

import flagsparse_amd as fs
from tests._rows_helpers import ROW_DTYPES, ROW_IDS, random_experts

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _whole(shape, dtype, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.randint(-3, 4, shape, device=DEV, generator=g).to(dtype)


def _tokens(n, n_rows, seed):
    """A few words of many tokens (64 and 65 among them), the rest anywhere."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, n_rows, (n,), generator=g)
    at = torch.randperm(n, generator=g)
    first = 0
    for word, count in ((7, n // 4), (n_rows - 1, 64), (0, 65), (n_rows // 2, 200)):
        ids[at[first : first + count]] = word
        first += count
    return ids.to(DEV)


# gradient type, result type, width (rows of whole words that end off 16 bytes, and one that does not), tokens: after
# a longer sort, and beside zeros that end inside the table
@pytest.mark.parametrize("dtype,out,width", [
    (torch.float32, torch.float32, 1003), (torch.float16, torch.float32, 1003), (torch.bfloat16, torch.float32, 520),
    (torch.bfloat16, torch.bfloat16, 1002), (torch.float16, torch.float16, 2040), (torch.float64, torch.float64, 501),
    (torch.float16, torch.float16, 1001)], ids=str)
@pytest.mark.parametrize("n", [3000, 20000])
def test_gradient_past_the_caches(dtype, out, width, n):
    size = torch.empty(0, dtype=out).element_size()
    n_rows = (300 << 20) // (width * size)
    tokens, grad = _tokens(n, n_rows, n + width), _whole((n, width), dtype, width)
    for padding in (None, 7):
        got = fs.flagsparse_embedding_grad(grad, tokens, n_rows, padding_idx=padding, dtype=out)
        want = torch.zeros((n_rows, width), dtype=torch.float64, device=DEV).index_add_(0, tokens, grad.double())
        if padding is not None:
            want[padding] = 0
        assert got.dtype == out and torch.equal(got, want.to(out))
        del want
    assert torch.equal(fs.flagsparse_embedding_grad(grad, tokens, n_rows, padding_idx=7, dtype=out), got)


@pytest.mark.parametrize("width", [1002, 1004])
@pytest.mark.parametrize("dtype", ROW_DTYPES, ids=ROW_IDS)
def test_moves_past_the_caches(dtype, width):
    size = torch.empty(0, dtype=dtype).element_size()
    n_tokens, slots = (75 << 20) // (width * size), 4
    experts = random_experts(n_tokens, slots, 9, 1, 0.05)
    route = fs.prepare_expert_route(experts, 9)
    routed, order = int(route.offsets[-1]), route.order.long()
    x = _whole((n_tokens, width), dtype, 2)
    rows = fs.flagsparse_expert_dispatch(x, route)
    want = x[order // slots]
    want[routed:] = 0
    assert torch.equal(rows, want)
    rows[routed:] = float("nan")
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    weights = _whole((n_tokens, slots), wide, 3)
    inside = ((experts >= 0) & (experts < 9)).to(wide)
    for w in (weights, None):
        got = fs.flagsparse_expert_combine(rows, route, w)
        factor = (inside if w is None else inside * w).sum(1, keepdim=True)
        assert torch.equal(got, (x.to(wide) * factor).to(dtype))
    grad = _whole((n_tokens, width), dtype, 4)
    grad_rows, grad_weights = fs.flagsparse_expert_combine_grad(grad, rows, route, weights)
    want = (grad[order // slots].to(wide) * weights.reshape(-1)[order][:, None]).to(dtype)
    want[routed:] = 0
    assert torch.equal(grad_rows, want)
    assert torch.equal(grad_weights, inside * (grad.to(wide) * x.to(wide)).sum(1, keepdim=True))


# around the sizes at which tiles grow: 512 positions to 32768, 1024 to 65536, 2048 to 524288, then 4096
SIZES = [4097, 32767, 32768, 32769, 65535, 65536, 65537, 131072, 131073, 524288, 524289]


@pytest.mark.parametrize("n", SIZES)
@pytest.mark.parametrize("num_experts", [1, 8, 64, 256, 1023])
def test_routes_of_every_number_of_tiles(n, num_experts):
    for dtype, dropped in ((torch.int32, 0.0), (torch.int64, 0.2)):
        experts = random_experts(n, 1, num_experts, n + num_experts, dropped, dtype)
        route = fs.prepare_expert_route(experts, num_experts)
        flat = experts.reshape(-1).cpu().long()
        key = torch.where((flat >= 0) & (flat < num_experts), flat, num_experts)
        order = torch.sort(key, stable=True)[1]
        assert torch.equal(route.order.cpu().long(), order)
        assert torch.equal(route.inverse.reshape(-1).cpu().long()[order], torch.arange(n))
        counts = torch.bincount(key, minlength=num_experts + 1)[:num_experts]
        assert route.offsets.tolist() == [0, *torch.cumsum(counts, 0).tolist()]


@pytest.mark.parametrize("n", SIZES)
@pytest.mark.parametrize("n_rows", [900, 5000, 131072, 1048577, (1 << 20) + (1 << 18)])
def test_gradients_of_every_number_of_tiles(n, n_rows):
    """One to three passes of the sort; a token's value tells it from its neighbours."""
    tokens = _tokens(n, n_rows, n)
    tokens[::11] = -1
    grad = (torch.arange(n, device=DEV, dtype=torch.float64) % 1000 + 1)[:, None]
    got = fs.flagsparse_embedding_grad(grad, tokens.int() if n % 2 else tokens, n_rows)
    inside = (tokens >= 0).cpu()
    want = torch.bincount(tokens.cpu()[inside], grad.cpu()[inside, 0], minlength=n_rows)
    assert torch.equal(got[:, 0].cpu(), want)
