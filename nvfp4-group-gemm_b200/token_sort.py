"""Tokens sorted by expert and back, with weights applied, and the gradients of both.

    r = moe.route(topk_ids, num_experts)
    rows = dispatch_tokens(x, r)                 # [r.rows, H], every expert's rows together
    ...                                          # the experts
    out = combine_tokens(rows, r, topk_weights)  # [tokens, H]

bf16, fp16 and fp32, any width and row stride, differentiable in ``x``, the rows and the
weights (with weights: once). Weights of any floating-point type are converted to fp32 first
(fp64 ones lose bits by that). Sums are fp32 in slot order, rounded once: results do not depend on
timing.
The ``*_backward`` functions are the gradients by themselves, for training loops that do not go
through autograd.

Capturing a backward pass in a CUDA graph follows torch's rule: while an eager graph of the same
leaves is alive, its gradient nodes belong to the stream it was made on, and the capture fails
with an error. Drop such graphs first, or capture the ``*_backward`` functions, which have no
such nodes. The reference has no counterpart of this module.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _native
from .int8 import _OUT_DTYPES, _launch_on, _within


def _check_routing(routing) -> tuple:
    """``(tokens, topk, rows, dest, src_rows)`` of a Routing, checked against one another."""
    tokens, topk, rows = routing.tokens, routing.topk, routing.rows
    dest, src = routing.dest, routing.src_rows
    if tokens * topk > _native.MAX_PAIRS:
        raise ValueError(f"{tokens * topk} pairs, at most {_native.MAX_PAIRS}")
    if dest.dtype != torch.int32 or dest.numel() < tokens * topk or not dest.is_contiguous():
        raise ValueError(f"routing.dest must be contiguous int32 with {tokens * topk} entries")
    if src.dtype != torch.int32 or src.numel() < rows or not src.is_contiguous():
        raise ValueError(f"routing.src_rows must be contiguous int32 with >= {rows} entries")
    return tokens, topk, rows, dest, src


def _check_rows(t: torch.Tensor, rows: int, name: str, cols: int | None = None) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype not in _OUT_DTYPES or t.dim() != 2:
        raise ValueError(f"{name} must be a 2-D CUDA bf16, fp16 or fp32 tensor")
    have = t.shape
    if have[1] > _native.MAX_ROW_COLUMNS:
        raise ValueError(f"{name} has {have[1]} columns, at most {_native.MAX_ROW_COLUMNS}")
    if have[0] != rows or have[1] < 1 or (cols is not None and have[1] != cols):
        want = f"[{rows}, {'cols' if cols is None else cols}]"
        raise ValueError(f"{name} must be {want}, got {list(t.shape)}")


def _rows_of(t: torch.Tensor) -> tuple:
    """``(tensor, row stride)``: ``t``, or a copy where its rows overlap (expanded tensors) or are
    not contiguous."""
    rows, cols = t.shape
    ld, inner = t.stride()
    if inner == 1 and ld >= cols:
        return t, ld
    if rows <= 1 and (inner == 1 or cols == 1):
        return t, cols
    return t.contiguous(), cols


def _fp32(weights):
    if weights is None or (weights.dtype == torch.float32 and weights.is_contiguous()):
        return weights
    return weights.to(torch.float32).contiguous()


def _ptr(t):
    return t.data_ptr() if t is not None else None


# The launches, on checked arguments; `sizes` is (tokens, topk, rows) of the routing.
def _launch_dispatch(x, dest, src, sizes, raw_stream):
    tokens, topk, rows = sizes
    x, ld = _rows_of(x)
    cols = x.shape[1]
    y = x.new_empty((rows, cols))
    lib = _native.load_library()
    _native.check(lib.nvfp4_moe_dispatch_tokens(
        x.data_ptr(), ld, _OUT_DTYPES[x.dtype], dest.data_ptr(), src.data_ptr(), tokens, topk, cols,
        rows, y.data_ptr(), cols, raw_stream), lib)
    return y


def _launch_combine(y, dest, weights, sizes, raw_stream):
    tokens, topk, rows = sizes
    y, ld = _rows_of(y)
    w = _fp32(weights)
    cols = y.shape[1]
    out = y.new_empty((tokens, cols))
    lib = _native.load_library()
    _native.check(lib.nvfp4_moe_combine_tokens(
        y.data_ptr(), ld, _OUT_DTYPES[y.dtype], dest.data_ptr(), _ptr(w), tokens, topk, cols, rows,
        out.data_ptr(), cols, raw_stream), lib)
    return out


def _launch_combine_backward(g, y, dest, src, weights, sizes, want_y, raw_stream):
    """Gradients of the rows (or None) and, where ``y`` is given, of the weights."""
    tokens, topk, rows = sizes
    g, ldg = _rows_of(g)
    y, ldy = _rows_of(y) if y is not None else (None, 0)
    w = _fp32(weights)
    cols = g.shape[1]
    gy = g.new_empty((rows, cols)) if want_y else None
    gw = g.new_empty((tokens, topk), dtype=torch.float32) if y is not None else None
    lib = _native.load_library()
    _native.check(lib.nvfp4_moe_combine_tokens_backward(
        g.data_ptr(), ldg, _ptr(y), ldy, _OUT_DTYPES[g.dtype], dest.data_ptr(), src.data_ptr(),
        _ptr(w), tokens, topk, cols, rows, _ptr(gy), cols, _ptr(gw), raw_stream), lib)
    return gy, gw


def _check_weights(weights, tokens, topk):
    if tuple(weights.shape) != (tokens, topk) or not weights.is_floating_point():
        raise ValueError(f"weights must be a floating-point tensor [{tokens}, {topk}]")


def _dispatch(x, routing, stream):
    tokens, topk, rows, dest, src = _check_routing(routing)
    _check_rows(x, tokens, "x")
    raw, where = _launch_on((x, dest, src), stream)
    return _within(where, _launch_dispatch, x, dest, src, (tokens, topk, rows), raw)


def _combine(y, routing, weights, stream):
    tokens, topk, rows, dest, _ = _check_routing(routing)
    _check_rows(y, rows, "y")
    if weights is not None:
        _check_weights(weights, tokens, topk)
    raw, where = _launch_on((y, dest, weights), stream)
    return _within(where, _launch_combine, y, dest, weights, (tokens, topk, rows), raw)


def dispatch_tokens_backward(grad_y: torch.Tensor, routing,
                             stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """Gradient of :func:`dispatch_tokens`: ``grad_x[t] = sum_j grad_y[dest[t, j]]``."""
    return _combine(grad_y, routing, None, stream)


def combine_tokens_backward(grad_out: torch.Tensor, y: torch.Tensor | None, routing,
                            weights: torch.Tensor | None = None, want_y: bool = True,
                            want_weights: bool = True,
                            stream: torch.cuda.Stream | None = None) -> tuple:
    """Gradients of :func:`combine_tokens`: ``(grad_y, grad_weights)``, None for one not wanted.

    ``grad_y[dest[t, j]] = weights[t, j] * grad_out[t]`` (zeros on padding rows) in the type of
    ``grad_out``; ``grad_weights[t, j] = <grad_out[t], y[dest[t, j]]>`` in fp32 (0 for dropped
    pairs; ``y`` is needed for it).
    """
    tokens, topk, rows, dest, src = _check_routing(routing)
    _check_rows(grad_out, tokens, "grad_out")
    if want_weights:
        if y is None:
            raise ValueError("the gradient of the weights needs y")
        _check_rows(y, rows, "y", int(grad_out.shape[1]))
        if y.dtype != grad_out.dtype:
            raise ValueError(f"y is {y.dtype}, grad_out is {grad_out.dtype}")
    if weights is not None:
        _check_weights(weights, tokens, topk)
    y = y if want_weights else None
    raw, where = _launch_on((grad_out, dest, src, weights, y), stream)
    return _within(where, _launch_combine_backward, grad_out, y, dest, src, weights,
                   (tokens, topk, rows), want_y, raw)


class _Kept:
    """A Routing's parts that the gradients need."""

    def __init__(self, sizes, dest, src_rows):
        self.tokens, self.topk, self.rows = sizes
        self.dest, self.src_rows = dest, src_rows


# The backward passes run on the device and stream of their forward pass (autograd sees to it),
# with gradients of the outputs' shape, type and device.
class _DispatchTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, routing):
        dest, src = routing.dest, routing.src_rows
        ctx.sizes = routing.tokens, routing.topk, routing.rows
        ctx.save_for_backward(dest, src)
        return _dispatch(x, routing, None)

    @staticmethod
    def backward(ctx, grad_y):
        dest, src = ctx.saved_tensors
        if torch.is_grad_enabled():  # the gradient of the gradient: the same two operators again
            return combine_tokens(grad_y, _Kept(ctx.sizes, dest, src)), None
        raw = torch._C._cuda_getCurrentRawStream(grad_y.get_device())
        return _launch_combine(grad_y, dest, None, ctx.sizes, raw), None


def _combine_gradients(ctx, grad_out):
    dest, src, weights, y = ctx.saved_tensors
    raw = torch._C._cuda_getCurrentRawStream(grad_out.get_device())
    gy, gw = _launch_combine_backward(grad_out, y, dest, src, weights, ctx.sizes,
                                      ctx.needs_input_grad[0], raw)
    if gw is not None and gw.dtype != weights.dtype:
        gw = gw.to(weights.dtype)
    return gy, gw, None


class _CombineTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, routing):
        want_w = weights is not None and ctx.needs_input_grad[1]
        ctx.sizes = routing.tokens, routing.topk, routing.rows
        ctx.save_for_backward(routing.dest, routing.src_rows, weights, y if want_w else None)
        return _combine(y, routing, weights, None)

    @staticmethod
    def backward(ctx, grad_out):
        if torch.is_grad_enabled():
            dest, src, weights, _ = ctx.saved_tensors
            if weights is None:
                return dispatch_tokens(grad_out, _Kept(ctx.sizes, dest, src)), None, None
            return once_differentiable(_combine_gradients)(ctx, grad_out)
        return _combine_gradients(ctx, grad_out)


def dispatch_tokens(x: torch.Tensor, routing,
                    stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """Tokens in expert order: ``[routing.rows, H]`` with ``y[routing.dest[t, j]] = x[t]`` and
    zeros on every expert's padding rows; differentiable in ``x`` (bf16, fp16 or fp32)."""
    if stream is None:
        return _DispatchTokens.apply(x, routing)
    _launch_on((x, routing.dest, routing.src_rows), stream)
    with torch.cuda.stream(stream):  # the backward pass runs on the stream of the forward pass
        return _DispatchTokens.apply(x, routing)


def combine_tokens(y: torch.Tensor, routing, weights: torch.Tensor | None = None,
                   stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """``out[t] = sum_j weights[t, j] * y[routing.dest[t, j]]`` (``weights`` None: ones), ``y``
    bf16, fp16 or fp32 ``[routing.rows, H]``, the result in its type; dropped pairs add nothing.
    Weights are taken in fp32 whatever their type, products and sums are fp32. Differentiable in ``y`` and ``weights``. (:func:`moe.combine` is
    the inference form from fp16 rows to bf16.)"""
    if stream is None:
        return _CombineTokens.apply(y, weights, routing)
    _launch_on((y, routing.dest, routing.src_rows, weights), stream)
    with torch.cuda.stream(stream):
        return _CombineTokens.apply(y, weights, routing)
