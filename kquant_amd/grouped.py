"""Matrix products grouped by expert over dense 16-bit weights, with gradients.

``grouped_linear`` multiplies rows that are sorted by expert (the order of
``kq_route_sort``) with each expert's dense matrix in one launch, and is
differentiable in the rows and in the weights.  It is the product that the
unquantized experts need (``moe.reconstruct_source`` gives their bf16
matrices): a teacher's forward pass for calibration rows, and the training or
recovery of experts; ``moe.grouped_expert_forward`` is the fused inference path
over MXFP4 weights.

Group sizes are device data throughout: nothing is read back to the host, so
the calls can be captured into a graph and replayed with other offsets.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _native as N

MAX_GROUPS = 4096
MAX_STRIDE = 1 << 22  # elements from row to row


def _rows(t: torch.Tensor, most: int | None = None) -> torch.Tensor:
    """``t`` [rows, columns] with unit column stride, a row stride that is a
    multiple of 8 and no more than ``most``, and 16-byte aligned rows (copied
    where it is not)."""
    near = most is None or t.stride(0) <= most
    if near and t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1] and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _forward(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    rows, (groups, n, k) = x.shape[0], weight.shape
    y = torch.empty(rows, n, dtype=x.dtype, device=x.device)
    N.call("kq_grouped_linear", N.DTYPE_CODES[x.dtype], N.ptr(x), x.stride(0), rows, N.ptr(offsets), groups,
           N.ptr(weight), n, k, N.ptr(y), n, N.stream(x.device))
    return y


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, offsets):
        with N.on_device(x.device):
            x, weight = _rows(x, MAX_STRIDE), N.aligned(weight)
            ctx.save_for_backward(x, weight, offsets)
            return _forward(x, weight, offsets)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, offsets = ctx.saved_tensors
        rows, (groups, n, k) = x.shape[0], weight.shape
        code = N.DTYPE_CODES[x.dtype]
        dx = dw = None
        with N.on_device(x.device):
            dy = _rows(dy, MAX_STRIDE)
            if ctx.needs_input_grad[0]:
                dx = torch.empty(rows, k, dtype=x.dtype, device=x.device)
                N.call("kq_grouped_linear_dx", code, N.ptr(dy), dy.stride(0), rows, N.ptr(offsets), groups,
                       N.ptr(weight), n, k, N.ptr(dx), k, N.stream(x.device))
            if ctx.needs_input_grad[1]:
                dw = torch.empty_like(weight)
                N.call("kq_grouped_linear_dw", code, N.ptr(dy), dy.stride(0), N.ptr(x), x.stride(0), rows,
                       N.ptr(offsets), groups, n, k, N.ptr(dw), N.stream(x.device))
        return dx, dw, None


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """``y[r] = weight[g] @ x[r]`` for the rows r in [offsets[g], offsets[g + 1]).

    x [rows, K] and weight [groups, N, K] are bf16 or fp16, both the same; N
    and K are multiples of 8.  offsets (int64 or int32 [groups + 1], not
    decreasing, on x's device) may leave groups empty and rows in front of the
    first or behind the last group: those rows of y and of x's gradient are
    zero.  Products accumulate in fp32 and are rounded once, to x's type.
    Offsets outside [0, rows] are taken as the nearest of the two; where they
    decrease, results are undefined, but nothing outside them is touched.  x and y's
    gradient may have any strides (copied unless rows are contiguous, 16-byte
    aligned and at most 2^22 elements apart, a multiple of 8); a weight whose
    matrices are not contiguous, a transposed one among them, is copied whole in
    every call.

    Differentiable once, in x and weight; an empty group's weight gradient is
    zero.  Results do not change from call to call (no atomics).  Captured into
    a graph, forward and backward go into one capture, made while no eager graph
    of the same leaves lives.
    """

    if x.dtype not in (torch.bfloat16, torch.float16) or weight.dtype != x.dtype:
        raise TypeError(f"x and weight must both be bfloat16 or both float16, got {x.dtype} and {weight.dtype}")
    if offsets.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"offsets must be int64 or int32, got {offsets.dtype}")
    if x.ndim != 2 or weight.ndim != 3:
        raise ValueError("x must be [rows, K] and weight [groups, N, K]")
    groups, n, k = weight.shape
    if x.shape[1] != k:
        raise ValueError(f"x has {x.shape[1]} columns, weight expects K={k}")
    if not 1 <= groups <= MAX_GROUPS:
        raise ValueError(f"groups={groups} must be between 1 and {MAX_GROUPS}")
    if n == 0 or k == 0 or n % 8 or k % 8:
        raise ValueError(f"N={n} and K={k} must be positive multiples of 8")
    if tuple(offsets.shape) != (groups + 1,):
        raise ValueError(f"offsets shape {tuple(offsets.shape)} != {(groups + 1,)}")
    if not (x.device == weight.device == offsets.device):
        raise ValueError("x, weight and offsets must be on one device")
    host = None if x.is_cuda else x.device
    if host is not None:
        gpu = N.require_gpu()
        x, weight, offsets = x.to(gpu), weight.to(gpu), offsets.to(gpu)
    else:
        N.check_capture(x, weight)
    offsets = N.aligned(offsets if offsets.dtype == torch.int64 else offsets.to(torch.int64), 8)
    y = _GroupedLinear.apply(x, weight, offsets)
    N.note_leaves(y)
    return y if host is None else y.to(host)
