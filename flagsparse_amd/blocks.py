"""Attention over selected blocks of keys: blocks' summaries, each query's selection
by a cheap score, and the attention over what was selected, with its gradients.

``prepare_block_sequences`` describes sequences of different lengths, in packed
rows or in the pages of a cache.  A block is ``block_size`` consecutive keys of a
sequence.  Query heads share a key-value head in groups, and a group its
selection.

    means      m[b] = mean of the keys of block b
    select     the first blocks, the most recent ones up to the query's own, and of
               the others the largest sum over the group of <q[t], m[b]>
    attention  out[t] = softmax over the keys j <= position(t) of the selected
               blocks (scale <q[t], k[j]>) v[j]

The selection is a matrix queries x blocks with ``top`` entries a row, and the
attention a product of dense matrices sampled there, a softmax along the rows and
that sparse matrix times the values, in one pass (csrc/block_means.hip,
block_select.hip, block_attention.hip, block_attention_grad.hip).  Values:
float16, bfloat16, float32; sums and softmax statistics run in 32 bits, scores of
blocks in 64, all in a fixed order.  Lengths, offsets and pages stay on the device
and nothing synchronises: a program may overwrite them in place between calls, in
a captured graph too.  They are not checked, but nothing outside the tensors is
read or written whatever they hold.  ``flagsparse_block_attention`` is
differentiable once in queries, keys and values of packed rows; the selection
carries no gradient.

The reference has no counterpart; names, checks and errors follow its other
operators (sparse_operations/spmm_coo.py:335-395, 619-625).
"""

import ctypes
import math

import torch

from . import _lib
from ._rows import check_out, done, into, recording, refuse_tangent, tangents

BLOCK_SIZES = (32, 64, 128, 256, 512, 1024)
MAX_SELECTED_BLOCKS = 128
MAX_GROUP = 128
BLOCK_VALUE_CODES = {
    torch.float16: _lib.FS_F16,
    torch.bfloat16: _lib.FS_BF16,
    torch.float32: _lib.FS_F32,
}
_INT32_MAX = 2**31 - 1
_MAX_KEYS = _INT32_MAX - 2047


class PreparedBlockSequences:
    """Sequences of queries and keys (``prepare_block_sequences``).

    It holds the tensors that describe them, not copies: what they hold when a
    call runs is what counts.
    """

    __slots__ = ("block_size", "q_offsets", "k_offsets", "pages", "k_lengths", "n_seqs", "device")

    def __init__(self, block_size, q_offsets, k_offsets, pages, k_lengths, n_seqs, device):
        self.block_size, self.q_offsets, self.k_offsets = block_size, q_offsets, k_offsets
        self.pages, self.k_lengths, self.n_seqs, self.device = pages, k_lengths, n_seqs, device


def _check_lengths(t, what, n=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a torch.Tensor")
    if t.dtype != torch.int32:
        raise TypeError(f"{what} dtype must be torch.int32")
    if t.ndim != 1 or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous 1D tensor")
    if n is not None and t.shape[0] != n:
        raise ValueError(f"{what} must have {n} elements, got {t.shape[0]}")


def prepare_block_sequences(block_size, q_offsets=None, k_offsets=None, pages=None, k_lengths=None):
    """Describe sequences for the operators over blocks.  No device work.

    block_size  keys a block: 32, 64, 128, 256, 512 or 1024
    q_offsets   (B + 1,) int32: query tokens of sequence b are rows q_offsets[b] to
                q_offsets[b + 1] - 1; None: one a sequence, row b
    k_offsets   (B + 1,) int32: its keys in packed rows; or
    pages       (B, n) int32: the pages of its keys in a cache, in order, and
    k_lengths   (B,) int32: how many keys they hold

    Offsets begin at 0 and do not decrease.  Queries are the last positions of
    their sequence.  Tokens behind the last sequence have no keys, a page outside
    the cache holds none.
    """
    block_size = int(block_size)
    if block_size not in BLOCK_SIZES:
        raise ValueError(f"block_size must be one of {BLOCK_SIZES}, got {block_size}")
    if (k_offsets is None) == (pages is None):
        raise ValueError("either k_offsets or pages must be given")
    if k_offsets is not None:
        if k_lengths is not None:
            raise ValueError("k_lengths goes with pages")
        _check_lengths(k_offsets, "k_offsets")
        n_seqs, device = k_offsets.shape[0] - 1, k_offsets.device
        if n_seqs < 0:
            raise ValueError("k_offsets must have at least one element")
    else:
        if not isinstance(pages, torch.Tensor):
            raise TypeError("pages must be a torch.Tensor")
        if pages.dtype != torch.int32:
            raise TypeError("pages dtype must be torch.int32")
        if pages.ndim != 2 or (pages.shape[1] > 1 and pages.stride(1) != 1) or pages.stride(0) < 0:
            raise ValueError("pages must be a 2D tensor of contiguous rows")
        n_seqs, device = pages.shape[0], pages.device
        if k_lengths is None:
            raise ValueError("k_lengths must be given with pages")
        _check_lengths(k_lengths, "k_lengths", n_seqs)
    if q_offsets is not None:
        _check_lengths(q_offsets, "q_offsets", n_seqs + 1)
    for t, what in ((q_offsets, "q_offsets"), (k_offsets, "k_offsets"), (pages, "pages"), (k_lengths, "k_lengths")):
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError(f"{what} must be a CUDA tensor")
        if t.device != device:
            raise ValueError(f"{what} must be on the same CUDA device as the keys' lengths")
    return PreparedBlockSequences(block_size, q_offsets, k_offsets, pages, k_lengths, n_seqs, device)


def _check_values(t, what, seqs, ndim):
    if not isinstance(seqs, PreparedBlockSequences):
        raise TypeError("seqs must be a PreparedBlockSequences")
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a torch.Tensor")
    if t.dtype not in BLOCK_VALUE_CODES:
        raise TypeError(f"{what} dtype must be one of: float16, bfloat16, float32")
    if not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    if t.device != seqs.device:
        raise ValueError(f"{what} must be on the same CUDA device as the sequences")
    if t.ndim != ndim:
        raise ValueError(f"{what} must be a {ndim}D tensor, got shape {tuple(t.shape)}")
    if tangents():
        refuse_tangent(t, what)


def _check_keys(k, what, seqs):
    """Keys or values: (rows, heads, width), or (pages, page rows, heads, width)."""
    _check_values(k, what, seqs, 3 if seqs.pages is None else 4)
    heads, width = k.shape[-2:]
    most = 128 if k.dtype == torch.float32 else 256
    if not 8 <= width <= most or width % 8:
        raise ValueError(f"{what} width must be a multiple of 8 from 8 to {most}, got {width}")
    if heads < 1:
        raise ValueError(f"{what} must have at least one head")
    if seqs.pages is not None:
        page = k.shape[1]
        if page < 16 or page > 1 << 20 or page & (page - 1):
            raise ValueError(f"pages must have a power of two of rows, at least 16, got {page}")
    elif k.shape[0] > _MAX_KEYS:
        raise ValueError(f"{what} rows exceed the int32 range")


def _check_queries(q, what, seqs, heads, width, dtype):
    _check_values(q, what, seqs, 3)
    if q.dtype != dtype:
        raise TypeError(f"{what} dtype must match the keys'")
    if q.shape[2] != width:
        raise ValueError(f"{what} must have width {width}, got {q.shape[2]}")
    group = q.shape[1] // heads
    if group * heads != q.shape[1] or not 1 <= group <= MAX_GROUP:
        raise ValueError(f"{what} heads must be 1 to {MAX_GROUP} times the {heads} key-value heads, got {q.shape[1]}")
    if seqs.q_offsets is None and q.shape[0] != seqs.n_seqs:
        raise ValueError(f"without q_offsets {what} must have {seqs.n_seqs} tokens, got {q.shape[0]}")
    return group


def _check_blocks(blocks, q, heads):
    if not isinstance(blocks, torch.Tensor):
        raise TypeError("blocks must be a torch.Tensor")
    if blocks.dtype != torch.int32:
        raise TypeError("blocks dtype must be torch.int32")
    if blocks.device != q.device:
        raise ValueError("blocks must be on the same CUDA device as the queries")
    if blocks.ndim != 3 or blocks.shape[0] != q.shape[0] or blocks.shape[1] not in (1, heads):
        raise ValueError(f"blocks must have shape ({q.shape[0]}, {heads} or 1, top), got {tuple(blocks.shape)}")
    if not 1 <= blocks.shape[2] <= MAX_SELECTED_BLOCKS:
        raise ValueError(f"blocks must name 1 to {MAX_SELECTED_BLOCKS} blocks a query, got {blocks.shape[2]}")


def _check_gradient(group, width, dtype):
    """A workgroup of the queries' gradient holds a group's rows: 96 where they are wide."""
    if group > 96 and width * dtype.itemsize > 256:
        raise ValueError(f"gradients of rows of more than 256 bytes need groups of up to 96 heads, got {group}")


def _scale_of(scale, width):
    scale = width**-0.5 if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError("scale must be positive and finite")
    return scale


def _described(seqs, n_tokens, k):
    """The C entry points' description of the sequences; without k, which the selection
    does not read, their lengths alone."""
    q_offsets = seqs.q_offsets
    if seqs.pages is None:
        c = _lib.FsBlockSeqs(seqs.n_seqs, n_tokens, _MAX_KEYS if k is None else k.shape[0],
                             None if q_offsets is None else q_offsets.data_ptr(), seqs.k_offsets.data_ptr(), None, None,
                             0, 0, 0, 0, 0, seqs.block_size)
    else:
        pages, page = seqs.pages, 1 << 20 if k is None else k.shape[1]
        # (an empty table has no address of its own: any other will do, nothing is read)
        c = _lib.FsBlockSeqs(seqs.n_seqs, n_tokens, 0, None if q_offsets is None else q_offsets.data_ptr(), None,
                             seqs.k_lengths.data_ptr(), pages.data_ptr() or seqs.k_lengths.data_ptr() or 16,
                             pages.stride(0), pages.shape[1], 0 if k is None else k.shape[0], page,
                             page.bit_length() - 1, seqs.block_size)
    return ctypes.byref(c)


def _heads_major(t):
    """A tensor whose last dimension is contiguous and whose distances are not negative."""
    return t if t.stride(-1) == 1 else t.contiguous()


def _cache_rows(k):
    """(k, distances of pages, rows and heads): rows at multiples of 16 bytes; a copy
    where they are not."""
    size = k.element_size()

    def fits(t):
        return t.stride(-1) == 1 and not (t.data_ptr() & 15 or any(s * size & 15 for s in t.stride()[:-1]))

    if not fits(k) or k.stride(-3) > 1 << 22:
        k = k.contiguous()
        if not fits(k):
            k = k.clone()
    return k, (0 if k.ndim == 3 else k.stride(0), k.stride(-3), k.stride(-2))


def flagsparse_block_means(k, seqs, max_blocks=None, start=None, out=None):
    """The mean of each block's keys: (B, max_blocks, heads, width).

    k is (rows, heads, width), or (pages, page rows, heads, width) with pages.
    Blocks without keys are zero.  ``start``, (B,) int32, updates summaries that a
    program keeps, which ``out`` then has to give: only blocks that hold a key at
    position start[b] or behind it are written.  Sums run in 32 bits, rounded
    once.  Carries no gradient.
    """
    _check_values(k, "k", seqs, 3 if isinstance(seqs, PreparedBlockSequences) and seqs.pages is None else 4)
    _check_keys(k, "k", seqs)
    heads, width = k.shape[-2:]
    if out is None:
        if start is not None:
            raise ValueError("out must be given with start")
        if max_blocks is None:
            raise ValueError("max_blocks must be given without out")
        max_blocks = int(max_blocks)
        if not 0 <= max_blocks <= _INT32_MAX:
            raise ValueError("max_blocks out of range")
    else:
        most = out.shape[1] if isinstance(out, torch.Tensor) and out.ndim == 4 else 0
        if max_blocks is not None and int(max_blocks) != most:
            raise ValueError(f"out must hold max_blocks blocks, got {most}")
        max_blocks = most
        check_out(out, k.device, (seqs.n_seqs, most, heads, width), k.dtype)
    if start is not None:
        _check_lengths(start, "start", seqs.n_seqs)
        if start.device != seqs.device:
            raise ValueError("start must be on the same CUDA device as the sequences")
    shape = (seqs.n_seqs, max_blocks, heads, width)
    if out is None:
        result = k.new_zeros(shape)
    elif start is not None:
        # (the other blocks stay: written where it lies, or a copy with all of them)
        result = into(out, k, start)
        if result is not out:
            result.copy_(out)
    else:
        result = into(out, k).zero_()
    k = k.detach() if k.stride(-1) == 1 else k.detach().contiguous()
    page, row, head = 0 if k.ndim == 3 else k.stride(0), k.stride(-3), k.stride(-2)
    rc = _lib.lib().fs_block_means(
        BLOCK_VALUE_CODES[k.dtype], _described(seqs, 0 if seqs.q_offsets is not None else seqs.n_seqs, k), heads, width,
        _lib.ptr(k) or 16, page, row, head, None if start is None else start.data_ptr(), max_blocks, _lib.ptr(result),
        result.stride(0), result.stride(1), result.stride(2), _lib.stream_handle(k.device))
    if rc:
        _lib.check(rc, "fs_block_means")
    return result if out is None else done(out, result)


def flagsparse_block_select(q, means, seqs, top, first=1, recent=1, out=None):
    """The blocks that each query attends to: (T, heads, top) int32, ascending, -1 behind.

    q is (T, heads * group, width), means (B, blocks, heads, width)
    (``flagsparse_block_means``).  The ``first`` blocks of the sequence and the
    ``recent`` ones up to the query's own are taken in any case, and of those in
    between the ones with the largest sum over the group of <q[t], means[b]>;
    equal ones by their number, not-a-numbers last.  Scores are computed in 64
    bits.  first + recent <= top <= 128.  Carries no gradient.
    """
    _check_values(means, "means", seqs, 4)
    n_seqs, most, heads, width = means.shape
    limit = 128 if means.dtype == torch.float32 else 256
    if not 8 <= width <= limit or width % 8:
        raise ValueError(f"means width must be a multiple of 8 from 8 to {limit}, got {width}")
    if n_seqs != seqs.n_seqs or heads < 1:
        raise ValueError(f"means must hold {seqs.n_seqs} sequences' blocks, got shape {tuple(means.shape)}")
    group = _check_queries(q, "q", seqs, heads, width, means.dtype)
    top, first, recent = int(top), int(first), int(recent)
    if not 1 <= top <= MAX_SELECTED_BLOCKS:
        raise ValueError(f"top must be in 1..{MAX_SELECTED_BLOCKS}, got {top}")
    if first < 0 or recent < 1 or first + recent > top:
        raise ValueError("first must not be negative, recent at least 1, and both together at most top")
    n_tokens = q.shape[0]
    shape = (n_tokens, heads, top)
    if out is not None:
        check_out(out, q.device, shape, torch.int32)
    q, means = _heads_major(q), _heads_major(means)
    result = torch.empty(shape, dtype=torch.int32, device=q.device) if out is None else into(out, q, means)
    rc = _lib.lib().fs_block_select(
        BLOCK_VALUE_CODES[q.dtype], _described(seqs, n_tokens, None), heads, group, width, _lib.ptr(q), q.stride(0),
        q.stride(1), _lib.ptr(means), most, means.stride(0), means.stride(1), means.stride(2), top, first, recent,
        _lib.ptr(result), _lib.stream_handle(q.device))
    if rc:
        _lib.check(rc, "fs_block_select")
    return result if out is None else done(out, result)


def _check_attention(q, k, v, blocks, seqs):
    """(heads, group, width) of an attention's arguments."""
    if not isinstance(seqs, PreparedBlockSequences):
        raise TypeError("seqs must be a PreparedBlockSequences")
    _check_keys(k, "k", seqs)
    _check_keys(v, "v", seqs)
    if v.dtype != k.dtype:
        raise TypeError("v dtype must match k dtype")
    if v.shape != k.shape:
        raise ValueError(f"v must have k's shape {tuple(k.shape)}, got {tuple(v.shape)}")
    heads, width = k.shape[-2:]
    group = _check_queries(q, "q", seqs, heads, width, k.dtype)
    _check_blocks(blocks, q, heads)
    return heads, group, width


def _attention(q, k, v, blocks, seqs, scale, out=None, want_lse=False):
    heads, width = k.shape[-2:]
    group = q.shape[1] // heads
    q = _heads_major(q)
    k, at_k = _cache_rows(k)
    v, at_v = _cache_rows(v)
    if blocks.stride(2) != 1:
        blocks = blocks.contiguous()
    result = q.new_empty(q.shape) if out is None else into(out, q, k, v, blocks)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if want_lse else None
    top, lib, code = blocks.shape[2], _lib.lib(), BLOCK_VALUE_CODES[q.dtype]
    described = _described(seqs, q.shape[0], k)
    need = lib.fs_block_attention_workspace_bytes(code, described, heads, group, width, top)
    ws = _lib.workspace(need, q.device) if need else None
    rc = lib.fs_block_attention(
        code, described, heads, group, width, top, _lib.ptr(q), q.stride(0), q.stride(1), _lib.ptr(k) or 16, *at_k,
        _lib.ptr(v) or 16, *at_v, _lib.ptr(blocks), blocks.stride(0), blocks.stride(1) if blocks.shape[1] > 1 else 0,
        scale, _lib.ptr(result), _lib.ptr(lse), _lib.ptr(ws), need, _lib.stream_handle(q.device))
    if rc:
        _lib.check(rc, "fs_block_attention")
    return (result if out is None else done(out, result)), lse


def _attention_grad(grad, q, k, v, blocks, seqs, scale, out, lse, queries=True, keys=True):
    """(dq, dk, dv): None for the queries', or for the keys' and values', where not wanted."""
    heads, width = k.shape[-2:]
    group = q.shape[1] // heads
    grad, out, lse = (t.contiguous() for t in (grad, out, lse))
    if grad.data_ptr() & 15:
        grad = grad.clone()
    # (queries, too, are loaded 16 bytes at a time, straight to LDS)
    q, (_, q_token, q_head) = _cache_rows(q)
    k, (_, k_row, k_head) = _cache_rows(k)
    v, (_, v_row, v_head) = _cache_rows(v)
    if blocks.stride(2) != 1:
        blocks = blocks.contiguous()
    dq = grad.new_empty(q.shape) if queries else None
    dk, dv = (grad.new_empty(k.shape), grad.new_empty(v.shape)) if keys else (None, None)
    top, lib, code = blocks.shape[2], _lib.lib(), BLOCK_VALUE_CODES[q.dtype]
    lists = blocks.shape[1]
    if q.shape[0] * lists * top > _INT32_MAX:
        raise ValueError("selected blocks of all queries exceed the int32 range")
    described = _described(seqs, q.shape[0], k)
    need = lib.fs_block_attention_grad_workspace_bytes(code, described, heads, group, width, lists, top)
    ws = _lib.workspace(need, q.device)
    rc = lib.fs_block_attention_grad(
        code, described, heads, group, width, lists, top, _lib.ptr(grad), _lib.ptr(q), q_token, q_head,
        _lib.ptr(k) or 16, k_row, k_head, _lib.ptr(v) or 16, v_row, v_head, _lib.ptr(blocks), blocks.stride(0),
        blocks.stride(1) if lists > 1 else 0, scale, _lib.ptr(out), _lib.ptr(lse), _lib.ptr(dq), _lib.ptr(dk),
        _lib.ptr(dv), ws.data_ptr(), need, _lib.stream_handle(q.device))
    if rc:
        _lib.check(rc, "fs_block_attention_grad")
    return dq, dk, dv


class _BlockAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, blocks, seqs, scale):
        out, lse = _attention(q, k, v, blocks, seqs, scale, want_lse=True)
        # the backward pass reads the lengths again: saved with the others, so that it
        # raises where they have been overwritten since
        ctx.save_for_backward(q, k, v, blocks, out, lse, seqs.q_offsets, seqs.k_offsets)
        ctx.seqs, ctx.scale = seqs, scale
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _):
        q, k, v, blocks, out, lse, _, _ = ctx.saved_tensors
        of_q, of_k, of_v = ctx.needs_input_grad[:3]
        dq, dk, dv = _attention_grad(grad, q, k, v, blocks, ctx.seqs, ctx.scale, out, lse, of_q, of_k or of_v)
        return dq, dk if of_k else None, dv if of_v else None, None, None, None


def flagsparse_block_attention(q, k, v, blocks, seqs, scale=None, out=None, return_lse=False):
    """Attention of each query over the keys of its selected blocks: q's shape.

    q is (T, heads * group, width); k and v are (rows, heads, width), or (pages,
    page rows, heads, width) with pages.  blocks, (T, heads, top) int32, or
    (T, 1, top) for all heads alike, names blocks of the query's sequence: one
    named twice counts once, a negative one or one behind the query's own not at
    all.  Within its blocks a query sees the keys up to its own position; one that
    sees none gets zeros, one whose scores are all minus infinity not-a-numbers.
    scale is width ** -0.5 unless given.  With return_lse also the logarithm of the
    sum of the exponentials, (T, heads * group) float32, minus infinity for both; it
    carries no gradient.

    Differentiable in q, k and v of packed rows.
    """
    heads, group, width = _check_attention(q, k, v, blocks, seqs)
    scale = _scale_of(scale, width)
    if (q.requires_grad or k.requires_grad or v.requires_grad) and recording():
        if out is not None:
            raise ValueError("out cannot be given where a gradient is recorded")
        if seqs.pages is not None:
            raise ValueError("keys and values of a cache have no gradient: detach them, and q")
        _check_gradient(group, width, q.dtype)
        result, lse = _BlockAttention.apply(q, k, v, blocks, seqs, scale)
    else:
        if out is not None:
            check_out(out, q.device, q.shape, q.dtype)
        result, lse = _attention(q, k, v, blocks, seqs, scale, out, return_lse)
    return (result, lse) if return_lse else result


def flagsparse_block_attention_grad(grad, q, k, v, blocks, seqs, out, lse, scale=None):
    """Gradients of ``flagsparse_block_attention`` in q, k and v, of packed rows.

    grad has q's shape; out and lse are the forward call's results.  Rows of no
    sequence get zeros.  Rows of more than 256 bytes take groups of up to 96 heads.
    Records no graph.
    """
    heads, group, width = _check_attention(q, k, v, blocks, seqs)
    if seqs.pages is not None:
        raise ValueError("keys and values of a cache have no gradient")
    _check_gradient(group, width, q.dtype)
    for t, what in ((grad, "grad"), (out, "out")):
        _check_values(t, what, seqs, 3)
        if t.dtype != q.dtype:
            raise TypeError(f"{what} dtype must match q dtype")
        if t.shape != q.shape:
            raise ValueError(f"{what} must have q's shape {tuple(q.shape)}, got {tuple(t.shape)}")
    if not isinstance(lse, torch.Tensor):
        raise TypeError("lse must be a torch.Tensor")
    if lse.dtype != torch.float32:
        raise TypeError("lse dtype must be torch.float32")
    if lse.device != q.device:
        raise ValueError("lse must be on the same CUDA device as the queries")
    if lse.shape != q.shape[:2]:
        raise ValueError(f"lse must have shape {tuple(q.shape[:2])}, got {tuple(lse.shape)}")
    return _attention_grad(grad, q, k, v, blocks, seqs, _scale_of(scale, width), out, lse)


__all__ = [
    "BLOCK_SIZES",
    "MAX_SELECTED_BLOCKS",
    "PreparedBlockSequences",
    "prepare_block_sequences",
    "flagsparse_block_means",
    "flagsparse_block_select",
    "flagsparse_block_attention",
    "flagsparse_block_attention_grad",
]
