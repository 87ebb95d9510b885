"""Bounds of the operators over blocks as near as 32-bit arithmetic comes: weights
keep the bits of two 16-bit parts, so that what a 16-bit result is
off by is its own rounding, next to which the rest is small."""

import math

import torch

from ._blocks_helpers import U32
from ._rows_helpers import TINY, UNIT


def _parts(dtype):
    """Relative error of a value held in two parts of a 16-bit type (each rounded by half
    a step at most): the product of both; nothing of float32."""
    return 0.0 if dtype == torch.float32 else UNIT[dtype] ** 2


class _Pairs:
    """All pairs of queries and keys of a case in 64 bits, (heads, group, tokens, rows)."""

    def __init__(self, case, blocks, scale):
        self.case, self.scale = case, scale
        self.H, self.G, self.D, self.T = case.heads, case.group, case.width, case.tokens
        self.seen = case.seen(blocks)
        self.mask = self.seen[:, None]
        self.q = self.by_head(case.q)
        self.k, self.v = (x.double().transpose(0, 1)[:, None].contiguous() for x in (case.packed_k, case.packed_v))
        self.s = scale * torch.matmul(self.q, self.k.transpose(2, 3).contiguous())
        self.s_size = scale * torch.matmul(self.q.abs(), self.k.abs().transpose(2, 3).contiguous())

    def by_head(self, x):
        return x.double().reshape(self.T, self.H, self.G, self.D).permute(1, 2, 0, 3).contiguous()

    def by_token(self, x):
        return x.permute(2, 0, 1, 3).reshape(self.T, self.H * self.G, self.D)

    def score_error(self, lse):
        """Of a weight, relative: D products added in 32 bits, scaled and shifted, each a
        rounding of values no larger than the sizes; the exponential two units more."""
        e = (self.D + 4) * U32 * self.s_size + 4 * U32 * (self.s_size + lse.abs()) + 4 * U32
        return torch.where(self.mask, e, 0.0)


def attention_bounds(case, blocks, scale):
    """(result in 64 bits, bound of its error)."""
    x = _Pairs(case, blocks, scale)
    s = x.s.masked_fill(~x.mask, -math.inf)
    lse = torch.logsumexp(s, 3, keepdim=True)
    empty = torch.isinf(lse)
    lse = torch.where(empty, 0.0, lse)
    p = torch.where(empty, 0.0, torch.exp(s - lse))
    e_row = x.score_error(lse).amax(3, keepdim=True)
    n = x.seen.sum(2).max().item()
    out = torch.matmul(p, x.v)
    # float16's second part ends at 2^-24 of a weight that is 2^7 where its score is the
    # largest; weights and their sum off by e, sums of 2 n terms
    floor = 2.0**-32 if case.dtype == torch.float16 else 0.0
    err = torch.matmul(p * (2 * e_row + _parts(case.dtype) + (4 * n + 16) * U32) + floor * x.mask, x.v.abs())
    err = 1.01 * err
    u = UNIT[case.dtype]
    return x.by_token(out), x.by_token(err + u * (out.abs() + err) + TINY[case.dtype])


def worst(got, want, bound):
    """The largest error in units of its bound."""
    off = (got.double() - want).abs() / (bound + 1e-300)
    return torch.where(torch.isnan(off), math.inf, off).max().item()
