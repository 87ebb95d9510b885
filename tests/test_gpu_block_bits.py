"""Bits of the operators over blocks: 16-bit results are off by their own rounding and
little else, whatever the sizes of weights and gradients beside each other."""

import math

import pytest
import torch

import flagsparse_amd as fs

from ._blocks_bounds import attention_bounds, gradient_bounds, worst
from ._blocks_helpers import BLOCK_DTYPES, BLOCK_IDS, Case, random_blocks, randn

pytestmark = pytest.mark.gpu
INF = float("inf")

SIZES = [
    # new, lengths, heads, group, width, block, top, page
    ([5, 3], [700, 65], 2, 4, 64, 32, 4, 0),
    ([1, 1], [90, 300], 2, 16, 128, 64, 2, 16),
    ([4], [90], 1, 3, 32, 32, 2, 0),
    ([1100], [1150], 4, 3, 32, 32, 2, 0),
    ([600, 450], [600, 700], 4, 8, 128, 64, 2, 16),
    ([1030], [1030], 4, 2, 64, 32, 5, 32),
]


@pytest.mark.parametrize("dtype", BLOCK_DTYPES, ids=BLOCK_IDS)
@pytest.mark.parametrize("sizes", SIZES, ids=["x".join(map(str, c[2:])) for c in SIZES])
def test_weights_keep_their_bits(sizes, dtype):
    new, lengths, heads, group, width, block, top, page = sizes
    case = Case(new, lengths, heads, group, width, block, dtype, 90, page)
    blocks = random_blocks(new, lengths, heads, top, block, 91)
    got = fs.flagsparse_block_attention(case.q, case.k, case.v, blocks, case.seqs)
    off = worst(got, *attention_bounds(case, blocks, width**-0.5))
    assert off <= 1.0, f"{off} times the bound"


@pytest.mark.parametrize("dtype", BLOCK_DTYPES, ids=BLOCK_IDS)
@pytest.mark.parametrize("tokens", [2, 1100], ids=["few", "many"])
def test_many_small_weights_add_up(tokens, dtype):
    """One key with nearly all the weight, 8000 with 2^-26 of it each: their part of the
    result is 8000 times that."""
    length, block, heads, width = 8192 + tokens, 1024, 4, 64
    case = Case([tokens], [length], heads, 1, width, block, dtype, 92)
    case.q.zero_()
    case.packed_k.zero_()
    case.packed_v.fill_(1.0)
    # scores of 0 and 26 in powers of two; the exponent is rounded to the type once, here
    case.q[:, :, 0] = 1.0
    case.packed_k[5, :, 0] = 26.0
    case.packed_v[5] = 0.0
    scale = math.log(2.0)
    blocks = torch.arange(8, dtype=torch.int32).expand(tokens, heads, 8).contiguous().cuda()
    got = fs.flagsparse_block_attention(case.q, case.k, case.v, blocks, case.seqs, scale)
    n = 8191.0
    want = n * 2.0**-26 / (1 + n * 2.0**-26)
    # scores off by some 2^-24 of 26, sums of 8192 terms, one rounding, float16's last step
    bound = want * (2.0**-16 + 2 * 8192 * 2.0**-24) + torch.finfo(dtype).eps / 2 * want + 2.0**-25
    assert float((got.double() - want).abs().max()) <= bound


def _gradients(case, blocks, grad):
    out, lse = fs.flagsparse_block_attention(case.q, case.k, case.v, blocks, case.seqs, return_lse=True)
    return out, lse, fs.flagsparse_block_attention_grad(grad, case.q, case.k, case.v, blocks, case.seqs, out, lse)


GRAD = [
    # new, lengths, heads, group, width, block, top
    ([90], [90], 2, 2, 32, 32, 2),
    ([70, 0, 30], [70, 0, 45], 2, 3, 64, 64, 1),
    ([100], [180], 1, 4, 128, 64, 2),
    ([129, 40], [129, 40], 2, 1, 80, 32, 3),
]


@pytest.mark.parametrize("dtype", BLOCK_DTYPES, ids=BLOCK_IDS)
@pytest.mark.parametrize("sizes", GRAD, ids=["x".join(map(str, c[2:])) for c in GRAD])
def test_gradients_keep_their_bits(sizes, dtype):
    new, lengths, heads, group, width, block, top = sizes
    case = Case(new, lengths, heads, group, width, block, dtype, 93)
    blocks = random_blocks(new, lengths, heads, top, block, 94)
    grad = randn(case.q.shape, dtype, 95)
    out, lse, got = _gradients(case, blocks, grad)
    found = gradient_bounds(case, blocks, width**-0.5, grad, out, lse)
    off = {name: worst(t, *found[name]) for t, name in zip(got, ("dq", "dk", "dv"))}
    assert max(off.values()) <= 1.0, off


@pytest.mark.parametrize("tokens", [90, 700])
@pytest.mark.parametrize("large", [2.0**13, INF, float("nan")], ids=["2^13", "inf", "nan"])
@pytest.mark.parametrize("dtype", BLOCK_DTYPES, ids=BLOCK_IDS)
def test_small_gradients_beside_large_ones(dtype, large, tokens):
    """Gradients of 2^-13 beside a row 2^26 times as large, or one that is not finite: what
    that row has no part in keeps its bits."""
    case = Case([tokens], [tokens], 2, 2, 64, 32, dtype, 96)
    blocks = random_blocks([tokens], [tokens], 2, 2, 32, 97)
    grad = randn(case.q.shape, dtype, 98) * 2.0**-13
    row = tokens - 20
    grad[row] = randn(case.q.shape[1:], dtype, 99) * (large if large < INF else 1.0)
    shown = grad.clone()
    if not large < INF:
        grad[row] = large
    out, lse, got = _gradients(case, blocks, grad)
    found = gradient_bounds(case, blocks, 64**-0.5, shown, out, lse)
    reached = case.seen(blocks)[:, row].t()[:, :, None].expand(case.packed_k.shape)
    rows = torch.arange(tokens, device="cuda") == row
    off = {}
    for t, name, apart in zip(got, ("dq", "dk", "dv"), (rows, reached, reached)):
        want, bound = found[name]
        if not large < INF:
            assert not torch.isfinite(t[apart]).any()
            t, want, bound = t[~apart], want[~apart], bound[~apart]
        off[name] = worst(t, want, bound)
    assert max(off.values()) <= 1.0, off


@pytest.mark.parametrize("size", [2.0**-14, 1.0, 2.0**13])
@pytest.mark.parametrize("width", [64, 128])
def test_float16_gradients_of_small_weights(width, size):
    """Scores that differ by 60 and more: weights down to 2^-90, and gradients of scores
    that grow from step to step."""
    case = Case([200], [200], 2, 2, width, 32, torch.float16, 100)
    case.q *= 4.0
    case.packed_k *= torch.linspace(0.0, 3.0, 200, device="cuda")[:, None, None].half()
    blocks = random_blocks([200], [200], 2, 4, 32, 101)
    grad = randn(case.q.shape, torch.float16, 102) * size
    out, lse, got = _gradients(case, blocks, grad)
    found = gradient_bounds(case, blocks, width**-0.5, grad, out, lse)
    off = {name: worst(t, *found[name]) for t, name in zip(got, ("dq", "dk", "dv"))}
    assert max(off.values()) <= 1.0, off
