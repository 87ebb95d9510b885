"""Bounds of the operators over blocks as near as 32-bit arithmetic comes: weights and
gradients of scores keep the bits of two 16-bit parts, so that what a 16-bit result is
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


def gradient_bounds(case, blocks, scale, grad, out, lse):
    """{name: (gradient in 64 bits, bound)} of the call with these results of the forward
    pass, as they were rounded."""
    x = _Pairs(case, blocks, scale)
    dtype = case.dtype
    u, parts = UNIT[dtype], _parts(dtype)
    g, o = x.by_head(grad), x.by_head(out)
    lse = lse.double().view(x.T, x.H, x.G).permute(1, 2, 0)[..., None]
    shown = torch.where(torch.isinf(lse), 0.0, lse)
    p = torch.where(x.mask, torch.exp(x.s - shown), 0.0)
    e = x.score_error(shown)
    vt = x.v.transpose(2, 3).contiguous()
    dp, dp_size = torch.matmul(g, vt), torch.matmul(g.abs(), vt.abs())
    delta, delta_size = (g * o).sum(3, keepdim=True), (g * o).abs().sum(3, keepdim=True)
    ds = p * (dp - delta)
    ds_err = p * (1.1 * (e + 4 * U32) * (dp.abs() + delta.abs()) + (x.D + 4) * U32 * (dp_size + delta_size)
                  + 2 * U32 * (dp.abs() + delta.abs()))
    ds_err = torch.where(x.mask, ds_err + parts * (ds.abs() + ds_err), 0.0)
    # float16: a power of two of a row (of a key) keeps its largest value at 2^8 or above,
    # and the second part ends at 2^-24; weights times 2^15
    small, floor = (2.0**-33, 2.0**-40) if dtype == torch.float16 else (0.0, 0.0)
    large = ds.abs() + ds_err
    row_err = ds_err + small * large.amax(3, keepdim=True) * x.mask
    key_err = ds_err + small * large.amax((1, 2), keepdim=True) * x.mask
    p_err = torch.where(x.mask, p * (1.1 * e + 4 * U32 + parts) + floor, 0.0)
    n = x.seen.sum(2).max().item()  # keys of a query
    rows = x.G * x.seen.sum(1).max().item()  # queries of a key

    def keys(y):
        return y.sum(1).transpose(0, 1)

    found = {}
    for name, value, size in (
        ("dq", x.by_token(scale * torch.matmul(ds, x.k)),
         x.by_token(scale * torch.matmul(row_err + (2 * n + 16) * U32 * ds.abs(), x.k.abs()))),
        ("dk", keys(scale * torch.matmul(ds.transpose(2, 3).contiguous(), x.q)),
         keys(scale * torch.matmul((key_err + (2 * rows + 64) * U32 * ds.abs()).transpose(2, 3).contiguous(), x.q.abs()))),
        ("dv", keys(torch.matmul(p.transpose(2, 3).contiguous(), g)),
         keys(torch.matmul((p_err + (2 * rows + 64) * U32 * p).transpose(2, 3).contiguous(), g.abs()))),
    ):
        size = 1.01 * size
        found[name] = (value, size + u * (value.abs() + size) + TINY[dtype])
    return found


def worst(got, want, bound):
    """The largest error in units of its bound.  What may lie past half a step behind the
    type's largest value may be infinite."""
    info = torch.finfo(got.dtype)
    past = want.abs() + bound >= info.max * (2.0 - info.eps / 2) / (2.0 - info.eps)
    off = (got.double() - want).abs() / (bound + 1e-300)
    off = torch.where(past & torch.isinf(got) & ((got > 0) == (want > 0)), 0.0, off)
    return torch.where(torch.isnan(off), math.inf, off).max().item()
