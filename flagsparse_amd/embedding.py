"""Embedding lookup with scaling, and its gradient by sorted tokens.

    out[t] = scale * table[tokens[t]]
    grad_table[v] = scale * sum over the t with tokens[t] = v of grad[t]

Products with a selection matrix of one entry a row and with its transpose
(csrc/embedding.hip).  Values: float16, bfloat16, float32 or float64; 16-bit
and 32-bit values are scaled and summed in float32 and rounded once.  Tokens:
int32 or int64 of any shape.  A token outside [0, rows of the table) reads
nothing: its result row is zero and its gradient goes nowhere (a process that
holds a part of the vocabulary subtracts its first row from the tokens).
Nothing synchronises, and sums run in a fixed order.  ``out`` may share memory
with an operand.

The reference has no counterpart; names, checks and errors follow its other
operators (sparse_operations/spmm_coo.py:335-395, 619-625).
"""

import torch

from . import _lib
from ._common import SUPPORTED_INDEX_DTYPES
from ._rows import (
    ROW_DTYPE_MESSAGE,
    ROW_VALUE_CODES,
    check_out,
    done,
    into,
    launch,
    recording,
    refuse_tangent,
    row_major,
    tangents,
)


def _check_tokens(tokens, values, what):
    if not (isinstance(tokens, torch.Tensor) and isinstance(values, torch.Tensor)):
        raise TypeError(f"{what} and tokens must be torch.Tensor")
    if values.dtype not in ROW_VALUE_CODES:
        raise TypeError(f"{what} dtype must be one of: {ROW_DTYPE_MESSAGE}")
    if tokens.dtype not in SUPPORTED_INDEX_DTYPES:
        raise TypeError("tokens dtype must be torch.int32 or torch.int64")
    if not (values.is_cuda and tokens.is_cuda):
        raise ValueError(f"{what} and tokens must be CUDA tensors")
    if values.device != tokens.device:
        raise ValueError(f"{what} and tokens must be on the same CUDA device")
    if tangents():
        refuse_tangent(values, what)


def _normalize_padding(padding_idx, n_rows):
    if padding_idx is None:
        return -1
    padding_idx = int(padding_idx)
    if not -n_rows <= padding_idx < n_rows:
        raise ValueError(f"padding_idx must be within the table's {n_rows} rows, got {padding_idx}")
    return padding_idx % n_rows


def _lookup(table, tokens, scale, out=None):
    n_rows, width = table.shape
    table, ld = row_major(table, width)
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    result = table.new_empty((*tokens.shape, width)) if out is None else into(out, table, tokens)
    launch(_lib.lib().fs_embedding, table.device, ROW_VALUE_CODES[table.dtype], _lib.INDEX_TYPE_CODES[tokens.dtype],
           tokens.numel(), n_rows, width, table.data_ptr(), ld, tokens.data_ptr(), scale, result.data_ptr())
    return result if out is None else done(out, result)


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, tokens, scale, padding_idx):
        ctx.save_for_backward(tokens)
        ctx.n_rows, ctx.scale, ctx.padding_idx = table.shape[0], scale, padding_idx
        return _lookup(table, tokens, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (tokens,) = ctx.saved_tensors
        return flagsparse_embedding_grad(grad, tokens, ctx.n_rows, ctx.scale, ctx.padding_idx), None, None, None


def flagsparse_embedding(table, tokens, scale=1.0, padding_idx=None, out=None):
    """scale * table[tokens]: tokens.shape + (width,), in the table's type.

    table is (rows, width).  padding_idx names a row whose gradient is zero
    (the lookup reads it as any other).  Differentiable once in `table`; `out`
    cannot be given then.
    """
    _check_tokens(tokens, table, "table")
    if table.ndim != 2:
        raise ValueError("table must be a 2D tensor: (rows, width)")
    scale = float(scale)
    if padding_idx is not None:
        padding_idx = _normalize_padding(padding_idx, table.shape[0])
    if table.requires_grad and recording():
        if out is not None:
            raise ValueError("out cannot be given where a gradient is recorded")
        return _Embedding.apply(table, tokens, scale, padding_idx)
    if out is not None:
        check_out(out, table.device, (*tokens.shape, table.shape[1]), table.dtype)
    return _lookup(table, tokens, scale, out)


def flagsparse_embedding_grad(grad, tokens, num_rows, scale=1.0, padding_idx=None, dtype=None, out=None):
    """Gradient of ``flagsparse_embedding`` in its table: (num_rows, width).

    grad is tokens.shape + (width,).  dtype is the result's: grad's own, or
    float32 for 16-bit grad.  Rows that no token names, and padding_idx, are
    zero.  Records no graph.
    """
    _check_tokens(tokens, grad, "grad")
    if grad.ndim != tokens.ndim + 1 or grad.shape[:-1] != tokens.shape:
        raise ValueError("grad must have the shape of tokens plus a width")
    num_rows = int(num_rows)
    if num_rows < 0:
        raise ValueError("num_rows must be non-negative")
    padding = _normalize_padding(padding_idx, num_rows)
    dtype = grad.dtype if dtype is None else dtype
    if dtype != grad.dtype and not (dtype == torch.float32 and grad.element_size() == 2):
        raise TypeError("dtype must be grad's, or torch.float32 for 16-bit grad")
    n, width = tokens.numel(), grad.shape[-1]
    if out is not None:
        check_out(out, grad.device, (num_rows, width), dtype)
    grad, ld = row_major(grad.reshape(n, width), width)
    tokens = tokens.contiguous()
    result = grad.new_empty((num_rows, width), dtype=dtype) if out is None else into(out, grad, tokens)
    code = ROW_VALUE_CODES[grad.dtype]
    lib = _lib.lib()
    ws = _lib.workspace(lib.fs_embedding_grad_workspace_bytes(code, n, num_rows, width), grad.device)
    launch(lib.fs_embedding_grad, grad.device, code, ROW_VALUE_CODES[dtype], _lib.INDEX_TYPE_CODES[tokens.dtype], n,
           num_rows, width, grad.data_ptr(), ld, tokens.data_ptr(), float(scale), padding, result.data_ptr(),
           ws.data_ptr(), ws.numel())
    return result if out is None else done(out, result)


__all__ = ["flagsparse_embedding", "flagsparse_embedding_grad"]
