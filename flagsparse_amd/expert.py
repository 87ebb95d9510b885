"""Tokens routed to experts: rows sorted by expert, the experts' products, and
the rows back with weights applied, each with its gradient.

``prepare_expert_route`` sorts the slots of T tokens, k slots a token, by the
expert each names; equal experts keep slot order.  A slot whose expert is
outside [0, num_experts) belongs to none (over capacity, or an expert that
another process holds: subtract the first expert held here): its place is
behind all others, its row is zero and it adds nothing to a token.  Places run
from 0 to T k whatever the experts are, so no shape depends on the data and
nothing synchronises.

    dispatch   rows[inverse[t, j]] = x[t]
    product    y[r] = rows[r] op(W[e]), e the expert of place r
    combine    out[t] = sum_j weights[t, j] y[inverse[t, j]]

Products with the routing matrix, with a block-diagonal matrix and with the
routing matrix's transpose (csrc/select_sort.hip, expert_rows.hip,
expert_product.hip).  Values: float16, bfloat16, float32 (float64 too but for
the product); sums run in 32 bits (64 for float64), in a fixed order, and are
rounded once.  Routing weights are float32 (float64 with float64 rows).  The
forward calls are differentiable once; the gradients called by name record no
graph.  ``out`` may share memory with an operand.

The reference has no counterpart; names, checks and errors follow its other
operators (sparse_operations/spmm_coo.py:335-395, 619-625).
"""

import torch

from . import _lib
from ._common import _INDEX_LIMIT_INT32, SUPPORTED_INDEX_DTYPES
from ._rows import (
    ROW_DTYPE_MESSAGE,
    ROW_VALUE_CODES,
    check_out,
    done,
    into,
    recording,
    refuse_tangent,
    row_major,
    tangents,
)
from .spmm_csr import _normalize_spmm_op, _spmm_op_transposes

MAX_EXPERTS = 1023


class PreparedExpertRoute:
    """Slots of tokens sorted by expert (``prepare_expert_route``).

    order     int32 (T k,): slot t k + j at each place
    inverse   int32 (T, k): place of each slot
    offsets   int32 (num_experts + 1,): first place of each expert; the last is
              the number of slots that name one

    It may be dropped while calls that use it are queued, on any stream; calls on
    other streams than its own have to be ordered behind its preparation.
    """

    __slots__ = ("n_tokens", "slots", "num_experts", "n_rows", "device", "_places", "_inverse_ptr", "_offsets_ptr",
                 "_stream")

    def __init__(self, n_tokens, slots, num_experts, places, stream):
        n = n_tokens * slots
        self.n_tokens, self.slots, self.num_experts, self.n_rows = n_tokens, slots, num_experts, n
        self.device = places.device
        # one int32 tensor: order, inverse, offsets and the sort's scratch (views of it cost more than the sort
        # of a decode step)
        self._places = places
        start = places.data_ptr()
        self._inverse_ptr, self._offsets_ptr = start + 4 * n, start + 8 * n
        self._stream = stream  # the handle of the one that writes the places

    @property
    def order(self):
        return self._places[: self.n_rows]

    @property
    def inverse(self):
        return self._places.as_strided((self.n_tokens, self.slots), (self.slots, 1), self.n_rows)

    @property
    def offsets(self):
        return self._places[2 * self.n_rows : 2 * self.n_rows + self.num_experts + 1]


def prepare_expert_route(experts, num_experts):
    """Sort the slots of ``experts``, (T, k) int32 or int64, by expert."""
    if not isinstance(experts, torch.Tensor):
        raise TypeError("experts must be a torch.Tensor")
    if experts.ndim != 2:
        raise ValueError("experts must be a 2D tensor: (tokens, slots)")
    if experts.dtype not in SUPPORTED_INDEX_DTYPES:
        raise TypeError("experts dtype must be torch.int32 or torch.int64")
    if not experts.is_cuda:
        raise ValueError("experts must be a CUDA tensor")
    num_experts = int(num_experts)
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"num_experts must be in 1..{MAX_EXPERTS}, got {num_experts}")
    n_tokens, slots = experts.shape
    if slots < 1:
        raise ValueError("experts must have at least one slot a token")
    n = n_tokens * slots
    if n > _INDEX_LIMIT_INT32:
        raise ValueError("tokens * slots exceeds the int32 range")
    experts = experts.contiguous()
    device = experts.device
    lib = _lib.lib()
    need = lib.fs_expert_route_workspace_bytes(n, num_experts)
    scratch = (2 * n + num_experts + 64) // 64 * 64  # 256-byte boundary behind the places
    places = torch.empty(scratch + (need + 3) // 4, dtype=torch.int32, device=device)
    stream = _lib.stream_handle(device)
    route = PreparedExpertRoute(n_tokens, slots, num_experts, places, stream)
    start = places.data_ptr()
    rc = lib.fs_expert_route(_lib.INDEX_TYPE_CODES[experts.dtype], n, num_experts, experts.data_ptr(), start,
                             route._inverse_ptr, route._offsets_ptr, start + 4 * scratch, need, stream)
    if rc:
        _lib.check(rc, "fs_expert_route")
    return route


def _check_rows(rows, what, route, n_rows):
    if not isinstance(route, PreparedExpertRoute):
        raise TypeError("route must be a PreparedExpertRoute")
    if not isinstance(rows, torch.Tensor):
        raise TypeError(f"{what} must be a torch.Tensor")
    if rows.dtype not in ROW_VALUE_CODES:
        raise TypeError(f"{what} dtype must be one of: {ROW_DTYPE_MESSAGE}")
    if not rows.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    if rows.device != route.device:
        raise ValueError(f"{what} must be on the same CUDA device as the route")
    if rows.ndim != 2 or rows.shape[0] != n_rows:
        raise ValueError(f"{what} must be a 2D tensor with {n_rows} rows, got shape {tuple(rows.shape)}")
    if tangents():
        refuse_tangent(rows, what)


def _check_weights(weights, rows, route):
    wide = torch.float64 if rows.dtype == torch.float64 else torch.float32
    if not isinstance(weights, torch.Tensor):
        raise TypeError("weights must be a torch.Tensor")
    if weights.dtype != wide:
        raise TypeError(f"weights dtype must be {wide} for {rows.dtype} rows")
    if weights.device != route.device:
        raise ValueError("weights must be on the same CUDA device as the route")
    if weights.shape != (route.n_tokens, route.slots):
        raise ValueError(f"weights must have shape {(route.n_tokens, route.slots)}, got {tuple(weights.shape)}")
    if tangents():
        refuse_tangent(weights, "weights")


def _launch(function, route, *args):
    """One call that reads a route's places.  A dropped route's memory waits for calls
    still queued on other streams than its own: its next owner would overwrite the
    places that they store to."""
    stream = _lib.stream_handle(route.device)
    if stream != route._stream:
        route._places.record_stream(torch.cuda.current_stream(route.device))
    rc = function(*args, stream)
    if rc:
        _lib.check(rc, function.__name__)


def _dispatch(x, route, out=None):
    width = x.shape[1]
    x, ld = row_major(x, width)
    result = x.new_empty((route.n_rows, width)) if out is None else into(out, x)
    _launch(_lib.lib().fs_expert_dispatch, route, ROW_VALUE_CODES[x.dtype], route.n_tokens, route.slots, width,
           route.num_experts, x.data_ptr(), ld, route._inverse_ptr, route._offsets_ptr, result.data_ptr())
    return result if out is None else done(out, result)


def _combine(rows, route, weights, out=None):
    width = rows.shape[1]
    rows, ld = row_major(rows, width)
    if weights is not None and not weights.is_contiguous():
        weights = weights.contiguous()
    result = rows.new_empty((route.n_tokens, width)) if out is None else into(out, rows, weights)
    _launch(_lib.lib().fs_expert_combine, route, ROW_VALUE_CODES[rows.dtype], route.n_tokens, route.slots, width,
           route.num_experts, rows.data_ptr(), ld, route._inverse_ptr, route._offsets_ptr,
           None if weights is None else weights.data_ptr(), result.data_ptr())
    return result if out is None else done(out, result)


def _combine_grad(grad, rows, route, weights):
    """(gradient of the rows, which needs the weights, gradient of the weights, which
    needs the rows): None for one whose operand is None."""
    width = grad.shape[1]
    grad, ldg = row_major(grad, width)
    grad_rows = grad_weights = None
    ldr = width
    if weights is not None:
        weights = weights.contiguous()
        grad_rows = grad.new_empty((route.n_rows, width))
    if rows is not None:
        rows, ldr = row_major(rows, width)
        wide = torch.float64 if rows.dtype == torch.float64 else torch.float32
        grad_weights = grad.new_empty((route.n_tokens, route.slots), dtype=wide)
    address = [None if t is None else t.data_ptr() for t in (rows, weights, grad_rows, grad_weights)]
    _launch(_lib.lib().fs_expert_combine_grad, route, ROW_VALUE_CODES[grad.dtype], route.n_tokens, route.slots,
           width, route.num_experts, grad.data_ptr(), ldg, address[0], ldr, route._inverse_ptr, route._offsets_ptr,
           *address[1:])
    return grad_rows, grad_weights


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, route):
        ctx.route = route
        return _dispatch(x, route)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return _combine(grad, ctx.route, None), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, route, weights):
        ctx.route, ctx.weighted = route, weights is not None
        # (each gradient reads the other operand only)
        ctx.save_for_backward(rows if ctx.needs_input_grad[2] else None, weights if ctx.needs_input_grad[0] else None)
        return _combine(rows, route, weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        if not ctx.weighted:
            return _dispatch(grad, ctx.route), None, None
        rows, weights = ctx.saved_tensors
        grad_rows, grad_weights = _combine_grad(grad, rows, ctx.route, weights)
        return grad_rows, None, grad_weights


def flagsparse_expert_dispatch(x, route, out=None):
    """Rows of ``x``, (T, width), in expert order: (T k, width).

    Differentiable in ``x``.
    """
    n_tokens = route.n_tokens if isinstance(route, PreparedExpertRoute) else 0
    _check_rows(x, "x", route, n_tokens)
    if x.requires_grad and recording():
        if out is not None:
            raise ValueError("out cannot be given where a gradient is recorded")
        return _Dispatch.apply(x, route)
    if out is not None:
        check_out(out, x.device, (route.n_rows, x.shape[1]), x.dtype)
    return _dispatch(x, route, out)


def flagsparse_expert_dispatch_grad(grad, route, out=None):
    """Gradient of ``flagsparse_expert_dispatch`` in x: a token's routed rows of ``grad`` summed, (T, width)."""
    n_rows = route.n_rows if isinstance(route, PreparedExpertRoute) else 0
    _check_rows(grad, "grad", route, n_rows)
    if out is not None:
        check_out(out, grad.device, (route.n_tokens, grad.shape[1]), grad.dtype)
    return _combine(grad, route, None, out)


def flagsparse_expert_combine(rows, route, weights=None, out=None):
    """Tokens' rows back from expert order, weighted and summed: (T, width).

    rows is (T k, width), weights (T, k), or None for ones.  Differentiable in
    both.
    """
    n_rows = route.n_rows if isinstance(route, PreparedExpertRoute) else 0
    _check_rows(rows, "rows", route, n_rows)
    if weights is not None:
        _check_weights(weights, rows, route)
    if (rows.requires_grad or (weights is not None and weights.requires_grad)) and recording():
        if out is not None:
            raise ValueError("out cannot be given where a gradient is recorded")
        return _Combine.apply(rows, route, weights)
    if out is not None:
        check_out(out, rows.device, (route.n_tokens, rows.shape[1]), rows.dtype)
    return _combine(rows, route, weights, out)


def flagsparse_expert_combine_grad(grad, rows, route, weights):
    """Gradients of ``flagsparse_expert_combine`` in its rows and weights, in one pass.

    grad is (T, width).  Slots of no expert get zeros in both.
    """
    n_rows = route.n_rows if isinstance(route, PreparedExpertRoute) else 0
    _check_rows(rows, "rows", route, n_rows)
    _check_rows(grad, "grad", route, route.n_tokens)
    if grad.dtype != rows.dtype:
        raise TypeError("grad dtype must match rows dtype")
    if grad.shape[1] != rows.shape[1]:
        raise ValueError(f"grad must have width {rows.shape[1]}, got {grad.shape[1]}")
    _check_weights(weights, rows, route)
    return _combine_grad(grad, rows, route, weights)


PRODUCT_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


def _check_product(rows, matrices, route, op):
    """(trans, inner, outer) of a product's arguments."""
    n_rows = route.n_rows if isinstance(route, PreparedExpertRoute) else 0
    _check_rows(rows, "rows", route, n_rows)
    if rows.dtype not in PRODUCT_DTYPES:
        raise TypeError("rows dtype must be one of: float16, bfloat16, float32")
    if not isinstance(matrices, torch.Tensor):
        raise TypeError("matrices must be a torch.Tensor")
    if matrices.dtype != rows.dtype:
        raise TypeError("matrices dtype must match rows dtype")
    if matrices.device != route.device:
        raise ValueError("matrices must be on the same CUDA device as the route")
    if matrices.ndim != 3 or matrices.shape[0] != route.num_experts:
        raise ValueError(f"matrices must be a 3D tensor with {route.num_experts} matrices, got shape "
                         f"{tuple(matrices.shape)}")
    if tangents():
        refuse_tangent(matrices, "matrices")
    trans = _spmm_op_transposes(_normalize_spmm_op(op))
    inner, outer = matrices.shape[2 if trans else 1], matrices.shape[1 if trans else 2]
    if rows.shape[1] != inner:
        raise ValueError(f"rows must have width {inner}, got {rows.shape[1]}")
    return trans, inner, outer


def _dense_matrices(matrices, trans):
    """(matrices, trans) of a contiguous tensor: a transposed view is taken as it lies."""
    if matrices.is_contiguous():
        return matrices, trans
    flipped = matrices.transpose(1, 2)
    if flipped.is_contiguous():
        return flipped, not trans
    return matrices.contiguous(), trans


def _product(rows, matrices, route, trans, inner, outer, out=None):
    rows, ld = row_major(rows, inner)
    matrices, trans = _dense_matrices(matrices, trans)
    result = rows.new_empty((route.n_rows, outer)) if out is None else into(out, rows, matrices)
    lib = _lib.lib()
    sizes = (ROW_VALUE_CODES[rows.dtype], int(trans), route.n_rows, route.num_experts, inner, outer)
    need = lib.fs_expert_product_workspace_bytes(*sizes)
    ws = _lib.workspace(need, rows.device) if need else None
    _launch(lib.fs_expert_product, route, *sizes, rows.data_ptr(), ld, matrices.data_ptr(), route._offsets_ptr,
           result.data_ptr(), _lib.ptr(ws), need)
    return result if out is None else done(out, result)


def _product_grad_matrices(grad, rows, route, trans, inner, outer):
    grad, ldg = row_major(grad, outer)
    rows, ldr = row_major(rows, inner)
    shape = (route.num_experts, outer, inner) if trans else (route.num_experts, inner, outer)
    result = rows.new_empty(shape)
    lib = _lib.lib()
    sizes = (ROW_VALUE_CODES[rows.dtype], int(trans), route.n_rows, route.num_experts, inner, outer)
    need = lib.fs_expert_product_grad_matrices_workspace_bytes(*sizes)
    ws = _lib.workspace(need, rows.device) if need else None
    _launch(lib.fs_expert_product_grad_matrices, route, *sizes, grad.data_ptr(), ldg, rows.data_ptr(), ldr,
           route._offsets_ptr, result.data_ptr(), _lib.ptr(ws), need)
    return result


class _Product(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, matrices, route, trans, inner, outer):
        # (each gradient reads the other operand only)
        ctx.save_for_backward(rows if ctx.needs_input_grad[1] else None, matrices if ctx.needs_input_grad[0] else None)
        ctx.route, ctx.sizes = route, (trans, inner, outer)
        return _product(rows, matrices, route, trans, inner, outer)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        rows, matrices = ctx.saved_tensors
        trans, inner, outer = ctx.sizes
        grad_rows = grad_matrices = None
        if ctx.needs_input_grad[0]:
            grad_rows = _product(grad, matrices, ctx.route, not trans, outer, inner)
        if ctx.needs_input_grad[1]:
            grad_matrices = _product_grad_matrices(grad, rows, ctx.route, trans, inner, outer)
        return grad_rows, grad_matrices, None, None, None, None


def flagsparse_expert_product(rows, matrices, route, op="non", out=None):
    """Each row times its expert's matrix: (T k, outer).

    rows is (T k, inner) in expert order; matrices is (num_experts, inner,
    outer), or (num_experts, outer, inner) with op="trans" ("conj" is the same
    for these real types).  Rows of no expert are zero.  Differentiable in both.
    """
    trans, inner, outer = _check_product(rows, matrices, route, op)
    if (rows.requires_grad or matrices.requires_grad) and recording():
        if out is not None:
            raise ValueError("out cannot be given where a gradient is recorded")
        return _Product.apply(rows, matrices, route, trans, inner, outer)
    if out is not None:
        check_out(out, rows.device, (route.n_rows, outer), rows.dtype)
    return _product(rows, matrices, route, trans, inner, outer, out)


def flagsparse_expert_product_grad(grad, rows, matrices, route, op="non"):
    """Gradients of ``flagsparse_expert_product`` in its rows and its matrices.

    grad is (T k, outer).  Rows of no expert get zeros, as do the matrices of
    experts without rows.
    """
    trans, inner, outer = _check_product(rows, matrices, route, op)
    _check_rows(grad, "grad", route, route.n_rows)
    if grad.dtype != rows.dtype:
        raise TypeError("grad dtype must match rows dtype")
    if grad.shape[1] != outer:
        raise ValueError(f"grad must have width {outer}, got {grad.shape[1]}")
    return (_product(grad, matrices, route, not trans, outer, inner),
            _product_grad_matrices(grad, rows, route, trans, inner, outer))


__all__ = [
    "MAX_EXPERTS",
    "PreparedExpertRoute",
    "prepare_expert_route",
    "flagsparse_expert_dispatch",
    "flagsparse_expert_dispatch_grad",
    "flagsparse_expert_combine",
    "flagsparse_expert_combine_grad",
    "flagsparse_expert_product",
    "flagsparse_expert_product_grad",
]
