"""Helpers of the tests of the operators over blocks: sequences, the definitions in
64 bits over all pairs of queries and keys, and rounding-error bounds."""

import math

import torch

import flagsparse_amd as fs

from ._rows_helpers import TINY, UNIT

BLOCK_DTYPES = [torch.float16, torch.bfloat16, torch.float32]
BLOCK_IDS = ["f16", "bf16", "f32"]
U32 = 2.0**-24


def offsets(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32).cuda()


def randn(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g, dtype=torch.float64).to(dtype).cuda()


def random_blocks(new, lengths, heads, top, block, seed, extra=0):
    """Random blocks of each query's sequence, some behind its own, negative or named
    again; the query's own block and the first one mostly among them."""
    g = torch.Generator().manual_seed(seed)
    rows = []
    for n, m in zip(lengths, new):
        for p in range(n - m, n):
            most = max(p, 0) // block + 2
            ids = torch.randint(-1, most, (heads, top), generator=g)
            if top > 1:
                ids[torch.rand(heads, generator=g) < 0.8, 0] = max(p, 0) // block
                ids[torch.rand(heads, generator=g) < 0.5, -1] = 0
            rows.append(ids)
    for _ in range(extra):
        rows.append(torch.randint(-1, 3, (heads, top), generator=g))
    return torch.stack(rows).int().cuda()


class Case:
    """Ragged sequences with packed rows or pages, and where each query and key is."""

    def __init__(self, new, lengths, heads, group, width, block, dtype, seed, page=0, tail=0, key_tail=0, single=False):
        self.new, self.lengths, self.heads, self.group, self.width = new, lengths, heads, group, width
        self.block, self.dtype, self.page = block, dtype, page
        tokens, rows = sum(new) + tail, sum(lengths) + key_tail
        self.tokens, self.rows = tokens, rows
        self.q = randn((tokens, heads * group, width), dtype, seed)
        self.packed_k = randn((rows, heads, width), dtype, seed + 1)
        self.packed_v = randn((rows, heads, width), dtype, seed + 2)
        q_offsets = None if single else offsets(new)
        if page:
            per = [-(-n // page) for n in lengths]
            g = torch.Generator().manual_seed(seed + 3)
            ids = torch.randperm(sum(per) + 2, generator=g)[: sum(per)].tolist()
            table = torch.full((len(lengths), max(per + [1]) + 1), -1, dtype=torch.int32)
            self.k = torch.full((sum(per) + 2, page, heads, width), float("nan"), dtype=dtype, device="cuda")
            self.v = torch.full_like(self.k, float("nan"))
            at = row = 0
            for i, n in enumerate(lengths):
                for j in range(per[i]):
                    table[i, j] = ids[at]
                    here = min(page, n - j * page)
                    self.k[ids[at], :here] = self.packed_k[row : row + here]
                    self.v[ids[at], :here] = self.packed_v[row : row + here]
                    at, row = at + 1, row + here
            self.pages = table.cuda()
            self.k_lengths = torch.tensor(lengths, dtype=torch.int32).cuda()
            self.seqs = fs.prepare_block_sequences(block, q_offsets, pages=self.pages, k_lengths=self.k_lengths)
        else:
            self.k, self.v = self.packed_k, self.packed_v
            self.seqs = fs.prepare_block_sequences(block, q_offsets, k_offsets=offsets(lengths))

    def positions(self):
        """Sequence and position of each query (-1: none), first row of each sequence."""
        seq, pos, first = [], [], [0]
        for b, (n, m) in enumerate(zip(self.lengths, self.new)):
            seq += [b] * m
            pos += list(range(n - m, n))
            first.append(first[-1] + n)
        extra = self.tokens - len(seq)
        return seq + [-1] * extra, pos + [-1] * extra, first

    def seen(self, blocks):
        """(heads, tokens, rows) truth values, by the definition."""
        seq, pos, first = self.positions()
        out = torch.zeros((self.heads, self.tokens, self.rows), dtype=torch.bool)
        ids = blocks.cpu().tolist()
        for t in range(self.tokens):
            if seq[t] < 0:
                continue
            for h in range(self.heads):
                for b in ids[t][h if len(ids[t]) > 1 else 0]:
                    a, e = b * self.block, min((b + 1) * self.block, pos[t] + 1)
                    if b >= 0 and e > a:
                        out[h, t, first[seq[t]] + a : first[seq[t]] + e] = True
        return out.cuda()


def oracle(case, blocks, scale, grad=None, seen=None):
    """Results in 64 bits and the bounds of their errors: a dict of (value, bound)."""
    H, G, D, T = case.heads, case.group, case.width, case.tokens
    u = UNIT[case.dtype]
    seen = case.seen(blocks) if seen is None else seen
    mask = seen[:, None]

    def by_head(x):
        return x.double().view(T, H, G, D).permute(1, 2, 0, 3)

    def by_token(x):
        return x.permute(2, 0, 1, 3).reshape(T, H * G, D)

    q = by_head(case.q)
    k, v = (x.double().transpose(0, 1)[:, None] for x in (case.packed_k, case.packed_v))
    s = scale * (q @ k.transpose(2, 3))
    s_size = scale * (q.abs() @ k.abs().transpose(2, 3))
    s = s.masked_fill(~mask, -math.inf)
    lse = torch.logsumexp(s, 3, keepdim=True)
    empty = torch.isinf(lse)
    p = torch.where(empty, 0.0, torch.exp(s - torch.where(empty, 0.0, lse)))
    # a score: D products added in 32 bits, scaled and shifted (two roundings of values
    # no larger than the sizes), then the exponential, off by two units at most
    e = torch.where(mask, (D + 4) * U32 * s_size + 4 * U32 * (s_size + lse.abs().nan_to_num(0.0, 0.0, 0.0)) + 4 * U32, 0.0)
    n = seen.sum(2).max().item()
    e_row = e.amax(3, keepdim=True)
    narrow = u if u > U32 else 0.0
    floor = 2.0**-25 if case.dtype == torch.float16 else 0.0  # of a weight of at most 1
    out = p @ v
    # weights off by e and rounded to the type, their sum off by e, sums of n terms
    out_err = (p * (2 * e_row + narrow + (2 * n + 8) * U32)) @ v.abs() + floor * (mask.double() @ v.abs())
    out_err = 1.01 * out_err
    out_err = out_err + u * (out.abs() + out_err) + TINY[case.dtype]
    lse_err = e_row + (n + 8) * U32 + 4 * U32 * lse.abs().nan_to_num(0.0, 0.0, 0.0)
    found = {"out": (by_token(out), by_token(out_err)),
             "lse": (lse[..., 0].permute(2, 0, 1).reshape(T, H * G), lse_err[..., 0].permute(2, 0, 1).reshape(T, H * G))}
    if grad is None:
        return found
    g = by_head(grad)
    dp, dp_size = g @ v.transpose(2, 3), g.abs() @ v.abs().transpose(2, 3)
    delta = (g * out).sum(3, keepdim=True)
    # from the forward result as it was rounded
    delta_err = ((g.abs() * out_err).sum(3, keepdim=True) + (D + 2) * U32 * (g.abs() * (out.abs() + out_err)).sum(3, keepdim=True))
    e_p = e + lse_err
    ds = p * (dp - delta)
    # float16: smallest step of a value times the power of two that brings the largest
    # gradient to [1, 2)
    step = 2.0**-24 * g.abs().max().item() if case.dtype == torch.float16 else 0.0
    ds_err = p * (1.1 * (e_p + 4 * U32) * (dp.abs() + delta.abs()) + (D + 4) * U32 * dp_size + 1.1 * delta_err)
    ds_err = torch.where(mask, ds_err + narrow * (ds.abs() + ds_err) + step, 0.0)
    p_err = torch.where(mask, p * (1.1 * e_p + narrow) + floor, 0.0)
    scores = (2 * T * G + 2 * n + 64) * U32

    def keys(x):  # sums over the group's heads and all queries
        return x.sum(1).transpose(0, 1)

    for name, value, size in (
        ("dq", by_token(scale * (ds @ k)), by_token(scale * ((ds_err + scores * ds.abs()) @ k.abs()))),
        ("dk", keys(scale * (ds.transpose(2, 3) @ q)), keys(scale * ((ds_err + scores * ds.abs()).transpose(2, 3) @ q.abs()))),
        ("dv", keys(p.transpose(2, 3) @ g), keys((p_err + scores * p).transpose(2, 3) @ g.abs())),
    ):
        size = 1.01 * size
        found[name] = (value, size + u * (value.abs() + size) + TINY[case.dtype])
    return found


def assert_within(got, found, name):
    want, bound = found[name]
    got = got.double()
    assert got.shape == want.shape
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    off = torch.where(same, 0.0, (got - want).abs() / (bound + 1e-300))
    worst = off.max().item() if off.numel() else 0.0
    assert bool((off <= 1.0).all()), f"{name}: {worst} times the bound, {int((~(off <= 1.0)).sum())} of {off.numel()}"


def select_oracle(q, means, seqs_of, pos, block, top, first, recent):
    """Blocks of each query by sorting all scores in 64 bits, on the CPU."""
    tokens, n_seqs = q.shape[0], means.shape[0]
    heads = means.shape[2]
    summed = q.double().cpu().view(tokens, heads, -1, q.shape[2]).sum(2)
    m = means.double().cpu()
    out = torch.full((tokens, heads, top), -1, dtype=torch.int32)
    for t in range(tokens):
        if seqs_of[t] < 0 or pos[t] < 0:
            continue
        own = pos[t] // block
        for h in range(heads):
            forced = set(range(min(first, own + 1))) | set(range(max(0, own - recent + 1), own + 1))
            among = [b for b in range(min(own + 1, m.shape[1])) if b not in forced]
            score = (m[seqs_of[t], : own + 1, h] @ summed[t, h]).tolist()
            among.sort(key=lambda b: (-math.inf if math.isnan(score[b]) else score[b], -b), reverse=True)
            ids = sorted(forced | set(among[: top - len(forced)] if top > len(forced) else []))
            out[t, h, : len(ids)] = torch.tensor(ids, dtype=torch.int32)
    return out.cuda()
