"""Checks and layouts that the row operators share (embedding.py, expert.py)."""

import torch
from torch.autograd import forward_ad

from . import _lib

ROW_VALUE_CODES = {
    torch.float16: _lib.FS_F16,
    torch.bfloat16: _lib.FS_BF16,
    torch.float32: _lib.FS_F32,
    torch.float64: _lib.FS_F64,
}
ROW_DTYPE_MESSAGE = "float16, bfloat16, float32, float64"


def row_major(t, width):
    """(t, stride of its rows) of a 2D tensor whose rows are contiguous; a copy
    where they are not, or where rows overlap."""
    if t.is_contiguous():
        return t, width
    if t.stride(1) == 1 and t.stride(0) >= width:
        return t, t.stride(0)
    return t.contiguous(), width


recording = torch.is_grad_enabled


def tangents():
    """Whether operands may have forward-mode tangents."""
    return forward_ad._current_level >= 0


def refuse_tangent(t, what):
    """The kernels would drop a forward-mode tangent without a word."""
    if forward_ad.unpack_dual(t).tangent is not None:
        raise NotImplementedError(f"{what} has a forward-mode tangent, which this operator does not propagate")


def launch(function, device, *args):
    """One call of a C entry point whose last argument is the stream."""
    rc = function(*args, _lib.stream_handle(device))
    if rc:
        _lib.check(rc, function.__name__)


def _span(t):
    """Addresses from a tensor's first byte to behind its last."""
    if t.numel() == 0:
        return 0, 0
    start = t.data_ptr()
    last = sum((n - 1) * stride for n, stride in zip(t.shape, t.stride()))
    return start, start + (last + 1) * t.element_size()


def into(out, *operands):
    """The tensor that a kernel writes: ``out`` itself where it is contiguous and
    shares no memory with an operand, which other workgroups would still read; a
    new one otherwise (``done`` copies it)."""
    if out.is_contiguous():
        first, end = _span(out)
        spans = (_span(t) for t in operands if t is not None)
        if not any(first < b and a < end for a, b in spans):
            return out
    return out.new_empty(out.shape)


def done(out, result):
    """``out``, with the result in it.  Autograd learns of the write, so a backward
    pass that still needs what ``out`` held raises."""
    if result is out:
        torch.autograd.graph.increment_version(out)
    else:
        out.copy_(result)
    return out


def check_out(out, device, shape, dtype):
    """Same checks and messages as the sparse products' (spmm_coo.py:619-625)."""
    if not isinstance(out, torch.Tensor):
        raise TypeError("out must be a torch.Tensor")
    if not out.is_cuda:
        raise ValueError("out must be a CUDA tensor")
    if out.device != device:
        raise ValueError("out must be on the same CUDA device as the inputs")
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype:
        raise ValueError("out shape/dtype must match result")
    if out.requires_grad and recording():  # (its graph would be that of the values it held before)
        raise ValueError("out cannot be given where a gradient is recorded")
