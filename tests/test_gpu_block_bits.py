"""Bits of the operators over blocks: 16-bit results are off by their own rounding and
little else, whatever the sizes of weights and gradients beside each other."""

import math

import pytest
import torch

import flagsparse_amd as fs

from ._blocks_bounds import attention_bounds, worst
from ._blocks_helpers import BLOCK_DTYPES, BLOCK_IDS, Case, random_blocks

pytestmark = pytest.mark.gpu

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
