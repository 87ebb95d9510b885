"""Embedding lookup and its gradient (embedding.hip, select_sort.hip) against the
definitions in 64 bits on the CPU: types, odd widths and strides, segments at the
lengths where their sums are cut, tokens outside the table, padding, empties."""

import pytest
import torch

import flagsparse_amd as fs
from flagsparse_amd import _lib
from tests._rows_helpers import ROW_DTYPES, ROW_IDS, assert_sum, randn

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _lookup_oracle(table, tokens, scale):
    wide = torch.float64 if table.dtype == torch.float64 else torch.float32
    t, ids = table.cpu().to(wide), tokens.cpu().long()
    inside = (ids >= 0) & (ids < t.shape[0])
    rows = torch.zeros((*ids.shape, t.shape[1]), dtype=wide)
    rows[inside] = t[ids[inside]] * torch.tensor(scale, dtype=wide)
    return rows.to(table.dtype)


def _grad_oracle(grad, tokens, n_rows, scale, padding=None):
    """(gradient, sum of magnitudes, longest segment) in 64 bits."""
    ids = tokens.cpu().reshape(-1).long()
    g = grad.cpu().double().reshape(ids.numel(), -1) * scale
    keep = (ids >= 0) & (ids < n_rows)
    if padding is not None:
        keep &= ids != padding
    out, mag = torch.zeros(n_rows, g.shape[1], dtype=torch.float64), torch.zeros(n_rows, g.shape[1], dtype=torch.float64)
    out.index_add_(0, ids[keep], g[keep])
    mag.index_add_(0, ids[keep], g[keep].abs())
    longest = int(torch.bincount(ids[keep], minlength=1).max()) if bool(keep.any()) else 0
    return out, mag, longest


@pytest.mark.parametrize("width", [1, 3, 7, 8, 9, 64, 100, 513, 2048, 4104])
@pytest.mark.parametrize("dtype", ROW_DTYPES, ids=ROW_IDS)
def test_lookup(dtype, width):
    table = randn((37, width), dtype, width)
    for index in (torch.int32, torch.int64):
        tokens = torch.tensor([[0, 36, 5], [5, 1, 0]], dtype=index, device=DEV)
        for scale in (1.0, 0.3):
            got = fs.flagsparse_embedding(table, tokens, scale=scale)
            assert got.shape == (2, 3, width) and got.dtype == dtype
            assert torch.equal(got.cpu(), _lookup_oracle(table, tokens, scale))


@pytest.mark.parametrize("dtype", ROW_DTYPES, ids=ROW_IDS)
def test_lookup_outside_and_special_values(dtype):
    table = randn((5, 40), dtype, 1)
    table[2, 3], table[2, 4], table[0, 0] = float("nan"), float("inf"), float("nan")
    tokens = torch.tensor([-1, 5, 2, 4, 2**31 + 1, -(2**40)], device=DEV)
    got = fs.flagsparse_embedding(table, tokens, scale=2.0).cpu()
    want = _lookup_oracle(table, tokens, 2.0)
    assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0)) and bool((got[[0, 1, 4, 5]] == 0).all())
    assert bool(torch.isnan(got[2, 3])) and bool(torch.isinf(got[2, 4]))
    # no row at all
    assert not bool(fs.flagsparse_embedding(table[:0], tokens).any())
    assert fs.flagsparse_embedding(table, tokens[:0]).shape == (0, 40)


def test_lookup_strides_and_out():
    big = randn((50, 3 * 72), torch.bfloat16, 2)
    tokens = torch.arange(0, 50, 3, device=DEV)
    for table in (big[:, :72], big[:, 1:72], big[:, ::3], big[::2], big.t().contiguous().t()):
        ids = tokens.clamp(max=table.shape[0] - 1)
        want = _lookup_oracle(table, ids, 0.5)
        assert torch.equal(fs.flagsparse_embedding(table, ids, scale=0.5).cpu(), want)
        out = torch.empty_like(want, device=DEV)
        assert fs.flagsparse_embedding(table, ids, scale=0.5, out=out) is out
        assert torch.equal(out.cpu(), want)
        wide = torch.zeros((len(ids), 2 * table.shape[1]), dtype=torch.bfloat16, device=DEV)
        out = wide[:, ::2]
        assert fs.flagsparse_embedding(table, ids[:, None].flip(0).flip(0)[:, 0], scale=0.5, out=out) is out
        assert torch.equal(out.cpu(), want) and not bool(wide[:, 1::2].any())


def test_lookup_offsets_past_32_bits():
    table = torch.zeros((300_000, 8192), dtype=torch.bfloat16, device=DEV)
    rows = torch.tensor([299_999, 262_144, 131_072, 0], device=DEV)
    table[rows] = torch.arange(1, 5, device=DEV).bfloat16()[:, None]
    got = fs.flagsparse_embedding(table, rows.int())
    assert bool((got == torch.arange(1, 5, device=DEV).bfloat16()[:, None]).all())


@pytest.mark.parametrize("width", [1, 7, 8, 65, 512, 1030, 2048])
@pytest.mark.parametrize("dtype", ROW_DTYPES, ids=ROW_IDS)
def test_gradient(dtype, width):
    tokens = torch.randint(0, 90, (777,), generator=torch.Generator().manual_seed(width)).to(DEV)
    tokens[100:300] = 41  # a long segment among short ones
    grad = randn((777, width), dtype, width + 1)
    for scale in (1.0, 0.7):
        got = fs.flagsparse_embedding_grad(grad, tokens.int(), 113, scale=scale)
        want, mag, n = _grad_oracle(grad, tokens, 113, scale)
        assert got.dtype == dtype and got.shape == (113, width)
        assert_sum(got, want, mag, n + 1)
    if grad.element_size() == 2:
        got = fs.flagsparse_embedding_grad(grad, tokens, 113, scale=0.7, dtype=torch.float32)
        assert got.dtype == torch.float32
        assert_sum(got, want, mag, n + 1)


# around the 64 positions at which segments are cut, from every phase
@pytest.mark.parametrize("lengths", [
    (64,), (65,), (63, 64, 65), (1, 64, 1, 65, 2, 66), (128,), (129,), (127, 1, 128), (64, 64, 64), (3, 61, 64, 65),
    (200, 300, 5), (65, 65, 65, 65), (1000,), (5,) * 40, (1,) * 200, (130, 62, 2, 64, 190),
], ids=str)
def test_gradient_segment_lengths(lengths):
    ids = torch.cat([torch.full((n,), 2 * k, dtype=torch.int64) for k, n in enumerate(lengths)])
    ids = ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(len(ids)))].to(DEV)
    n_rows = 2 * len(lengths) + 1
    for width in (5, 300):
        grad = randn((len(ids), width), torch.float32, len(ids))
        got = fs.flagsparse_embedding_grad(grad, ids, n_rows)
        want, mag, longest = _grad_oracle(grad, ids, n_rows, 1.0)
        assert_sum(got, want, mag, longest)
        assert not bool(got[1::2].any())
        again = fs.flagsparse_embedding_grad(grad, ids, n_rows)
        assert torch.equal(got, again)


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 4095, 4096, 4097, 9000])
@pytest.mark.parametrize("n_rows", [1, 2, 16, 1023, 1024, 5000, 70001, 1048577])
def test_gradient_sorts_of_every_size(n, n_rows):
    """One and more passes of the sort, one and more tiles, one value per token
    that tells it from the others."""
    g = torch.Generator().manual_seed(n + n_rows)
    ids = (torch.rand(n, generator=g) ** 3 * n_rows).long().clamp(max=n_rows - 1)
    ids[::7] = ids[0]
    if n > 3:
        ids[1], ids[2] = -5, n_rows
    grad = torch.arange(1, n + 1, dtype=torch.float64)[:, None]
    want, _, _ = _grad_oracle(grad, ids, n_rows, 1.0)
    got = fs.flagsparse_embedding_grad(grad.to(DEV), ids.to(DEV), n_rows)
    assert torch.equal(got.cpu(), want)  # sums of small whole numbers


def test_gradient_many_tiles_scanned_by_launches():
    n, n_rows = 4096 * 513 + 17, 3000  # more tiles than a scatter adds up itself
    ids = torch.randint(0, n_rows, (n,), generator=torch.Generator().manual_seed(3))
    grad = (torch.arange(n, dtype=torch.float64) % 1000)[:, None]
    want, _, _ = _grad_oracle(grad, ids, n_rows, 1.0)
    got = fs.flagsparse_embedding_grad(grad.to(DEV), ids.int().to(DEV), n_rows)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("n", [5, 300, 1025, 4096])
@pytest.mark.parametrize("dtype", ROW_DTYPES, ids=ROW_IDS)
def test_gradient_of_tables_larger_than_what_the_sort_zeroes(dtype, n):
    """Beside a short sort the first 64 or 96 MB of the table are zeroed; the rows
    after them are not, and rows have odd sizes and begin at one element."""
    width = 1003
    n_rows = (104 << 20) // (width * torch.empty(0, dtype=dtype).element_size())
    g = torch.Generator().manual_seed(n)
    tokens = torch.randint(0, n_rows, (n,), generator=g)
    tokens[0], tokens[1], tokens[2], tokens[3] = 0, n_rows - 1, 7, n_rows - 2  # (7 and n_rows - 2: padding)
    grad = torch.randint(-3, 4, (n, width), generator=g).to(dtype)  # sums of whole values: exact
    for padding in (7, n_rows - 2):
        room = torch.full((1 + n_rows * width,), float("nan"), dtype=dtype, device=DEV)
        out = room[1:].view(n_rows, width)
        fs.flagsparse_embedding_grad(grad.to(DEV), tokens.to(DEV), n_rows, padding_idx=padding, out=out)
        rows, at = torch.unique(tokens, return_inverse=True)
        want = torch.zeros(len(rows), width, dtype=torch.float64).index_add_(0, at, grad.double())
        want[rows == padding] = 0
        assert torch.equal(out[rows.to(DEV)].cpu().double(), want)
        out[rows.to(DEV)] = 0
        assert bool((out == 0).all()) and bool(torch.isnan(room[0]))


@pytest.mark.parametrize("length", [1, 64, 65, 500])
def test_gradient_padding_and_outside(length):
    ids = torch.cat([torch.full((length,), 3), torch.arange(8), torch.full((length,), -1), torch.full((length,), 8)])
    ids = ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(length))].to(DEV)
    grad = randn((len(ids), 24), torch.bfloat16, length)
    nowhere = (ids == 3) | (ids < 0) | (ids >= 8)
    grad[nowhere] = float("nan")
    for padding in (3, -5):
        got = fs.flagsparse_embedding_grad(grad, ids, 8, padding_idx=padding)
        want, mag, n = _grad_oracle(torch.where(nowhere[:, None], 0, grad), ids, 8, 1.0, padding=3)
        assert_sum(got, want, mag, n)
        assert not bool(got[3].any())


def test_gradient_empty_and_strided():
    g = randn((6, 40), torch.float16, 5)
    ids = torch.tensor([[1, 1, 0], [2, 1, 0]], device=DEV)
    assert not bool(fs.flagsparse_embedding_grad(g[:0], ids[:0, 0], 7).any())
    assert fs.flagsparse_embedding_grad(g, ids.reshape(-1), 0).shape == (0, 40)
    assert fs.flagsparse_embedding_grad(g[:, :0], ids.reshape(-1), 5).shape == (5, 0)
    for grad in (g[:, :24], g[:, 1:24], g[:, ::2], g.t().contiguous().t(), g[:1].expand(6, 40)):
        want, mag, n = _grad_oracle(grad, ids, 4, 1.0)
        got = fs.flagsparse_embedding_grad(grad.reshape(2, 3, -1) if grad.is_contiguous() else
                                           grad.unflatten(0, (2, 3)), ids, 4)
        assert_sum(got, want, mag, n)
    out = torch.full((4, 40), 9.0, dtype=torch.float16, device=DEV)
    assert fs.flagsparse_embedding_grad(g, ids.reshape(-1), 4, out=out) is out
    want, mag, n = _grad_oracle(g, ids, 4, 1.0)
    assert_sum(out, want, mag, n)


def test_autograd_matches_formula_and_differences():
    table = randn((11, 6), torch.float64, 1).requires_grad_()
    ids = torch.tensor([3, 3, 0, 10, 7, 3, -1, 11], device=DEV)

    def f(t):
        return fs.flagsparse_embedding(t, ids, scale=1.7, padding_idx=7)

    out = f(table)
    seed = randn(out.shape, torch.float64, 2)
    (got,) = torch.autograd.grad(out, table, seed)
    want, mag, n = _grad_oracle(seed, ids, 11, 1.7, padding=7)
    assert_sum(got, want, mag, n + 1)
    # central differences of a linear function: exact but for rounding
    base = table.detach()
    for v, h in ((3, 2), (0, 5), (10, 0), (9, 1)):
        step = torch.zeros_like(base)
        step[v, h] = 0.5
        diff = ((f(base + step) - f(base - step)) * seed).sum()
        assert abs(float(diff - got[v, h])) <= 1e-13 * float((f(base).abs() * seed.abs()).sum())
    half = randn((11, 6), torch.bfloat16, 1).requires_grad_()
    fs.flagsparse_embedding(half, ids).float().sum().backward()
    assert half.grad.dtype == torch.bfloat16 and float(half.grad[3, 0]) == 3.0


def test_other_stream_and_graph():
    table = randn((300, 264), torch.bfloat16, 1)
    ids = torch.randint(0, 300, (1000,), generator=torch.Generator().manual_seed(2)).to(DEV)
    grad = randn((1000, 264), torch.bfloat16, 3)
    want = fs.flagsparse_embedding(table, ids, scale=3.0), fs.flagsparse_embedding_grad(grad, ids, 300)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = fs.flagsparse_embedding(table, ids, scale=3.0), fs.flagsparse_embedding_grad(grad, ids, 300)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = fs.flagsparse_embedding(table, ids, scale=3.0), fs.flagsparse_embedding_grad(grad, ids, 300)
    for seed in (5, 6, 7):
        ids.copy_(torch.randint(0, 300, (1000,), generator=torch.Generator().manual_seed(seed)))
        want = fs.flagsparse_embedding(table, ids, scale=3.0), fs.flagsparse_embedding_grad(grad, ids, 300)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_kernel_names():
    table, ids = randn((4, 8), torch.float32, 1), torch.tensor([1], device=DEV)
    fs.flagsparse_embedding(table, ids)
    assert _lib.last_kernel() == "embedding_kernel"
    fs.flagsparse_embedding_grad(table[:1], ids, 4)
    assert _lib.last_kernel() == "embedding_grad_kernel"


def test_refusals():
    table, ids = randn((4, 8), torch.float32, 1), torch.tensor([1, 2], device=DEV)
    with pytest.raises(TypeError, match="must be torch.Tensor"):
        fs.flagsparse_embedding([1.0], ids)
    with pytest.raises(TypeError, match="table dtype must be one of"):
        fs.flagsparse_embedding(table.to(torch.complex64), ids)
    with pytest.raises(TypeError, match="tokens dtype must be"):
        fs.flagsparse_embedding(table, ids.to(torch.int16))
    with pytest.raises(ValueError, match="must be CUDA tensors"):
        fs.flagsparse_embedding(table.cpu(), ids)
    with pytest.raises(ValueError, match="table must be a 2D tensor"):
        fs.flagsparse_embedding(table[0], ids)
    with pytest.raises(ValueError, match="padding_idx must be within"):
        fs.flagsparse_embedding(table, ids, padding_idx=4)
    with pytest.raises(ValueError, match="out shape/dtype must match result"):
        fs.flagsparse_embedding(table, ids, out=torch.empty((2, 7), device=DEV))
    with pytest.raises(ValueError, match="out cannot be given"):
        fs.flagsparse_embedding(table.requires_grad_(), ids, out=torch.empty((2, 8), device=DEV))
    grad = torch.ones((2, 8), device=DEV)
    with pytest.raises(ValueError, match="grad must have the shape of tokens plus a width"):
        fs.flagsparse_embedding_grad(grad[:1], ids, 4)
    with pytest.raises(ValueError, match="num_rows must be non-negative"):
        fs.flagsparse_embedding_grad(grad, ids, -1)
    with pytest.raises(TypeError, match="dtype must be grad's"):
        fs.flagsparse_embedding_grad(grad, ids, 4, dtype=torch.float16)
    with pytest.raises(ValueError, match="out must be a CUDA tensor"):
        fs.flagsparse_embedding_grad(grad, ids, 4, out=torch.empty((4, 8)))
