"""The experts' products on paths that the other sizes do not reach: few rows with
operands off 16 bytes and off whole words, 128 x 128 tiles through registers and by
words, and more experts than a wave has lanes, in every size of tiles."""

import pytest
import torch

import flagsparse_amd as fs
from flagsparse_amd import _lib
from tests._rows_helpers import randn, random_experts
from tests.test_gpu_expert_product import DTYPES, IDS, _check, _route

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _counts(n_tokens, slots, n_experts):
    experts = random_experts(n_tokens, slots, n_experts, n_tokens)
    return torch.bincount(experts.reshape(-1).long(), minlength=n_experts).tolist()


# decode steps; 16-bit rows of 513 and 385 go through registers, of 514 and 386 by words (in the few-rows kernel,
# whose waves are eight where few tiles leave the chip idle: up to 12 chosen experts here, and four with 32)
@pytest.mark.parametrize("n_tokens,slots,n_experts", [(1, 1, 8), (1, 8, 64), (2, 6, 60), (16, 4, 32), (33, 2, 8)])
@pytest.mark.parametrize("inner,outer", [(513, 385), (514, 386), (31, 65), (2049, 71)], ids=str)
@pytest.mark.parametrize("op", ["non", "trans"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_few_rows_off_16_bytes(dtype, op, inner, outer, n_tokens, slots, n_experts):
    counts = _counts(n_tokens, slots, n_experts)
    _check(dtype, op, counts, inner, outer, dropped=3, seed=outer)
    route = _route(counts)
    rows = randn((route.n_rows, inner), dtype, 1)
    matrices = randn((n_experts, outer, inner) if op == "trans" else (n_experts, inner, outer), dtype, 2)
    fs.flagsparse_expert_product(rows, matrices, route, op=op)
    assert _lib.last_kernel() == "expert_product_few_kernel"


# 48 rows an expert and 66 columns of 128 x 128 tiles an expert: of rows, of the rows' gradient (sizes exchanged)
# and of the matrices'; the last with more than 1024 rows an expert
@pytest.mark.parametrize("counts", [(30, 0, 100, 62), (1, 130, 31, 40), (1100, 1200, 900, 1400)], ids=str)
@pytest.mark.parametrize("inner,outer", [(67, 8321), (8321, 67), (66, 8322), (8322, 66)], ids=str)
@pytest.mark.parametrize("op", ["non", "trans"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_tiles_of_128_off_16_bytes(dtype, op, inner, outer, counts):
    _check(dtype, op, counts, inner, outer, dropped=5)


# experts beyond the first 64, with and without rows, and slots of none; rows an expert: few, a 64-row tile's, a
# 128-row tile's, large tiles'
@pytest.mark.parametrize("n_experts", [64, 65, 128, 200, 1023])
@pytest.mark.parametrize("rows", [1, 20, 60, 140])
@pytest.mark.parametrize("op", ["non", "trans"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_many_experts(dtype, op, rows, n_experts):
    g = torch.Generator().manual_seed(n_experts + rows)
    counts = torch.randint(0, 2 * rows + 1, (n_experts,), generator=g)
    counts[::7] = 0
    counts[63], counts[-1] = rows, rows + 3
    _check(dtype, op, counts.tolist(), 40, 72, dropped=11)
    if n_experts < 200:  # more columns
        _check(dtype, op, counts.tolist(), 24, 776, dropped=0)
