"""Dequant-fused block-scaled linear layers (bf16 activations x MX weights).

``mxfp8_linear`` / ``mxfp4_linear`` compute ``source @ dequant(weight).T`` with
fp32 accumulation in one HIP kernel (``kq_mx_linear``).  They replace the
dequantize-then-matmul fp32 oracle of kquant's closures
(scripts/closure_mxfp8_mlp.py:146-160, kquant/pack/qsrt_validation.py:249-258)
and the external ``mxfp8_linear.mm`` kernel call
(scripts/closure_mxfp8_mlp.py:172-177) with an A16 kernel: activations stay
bf16, weights are expanded exactly to bf16 inside the kernel.

fp32 sources take ``kq_mx_linear_f32``: the source is split exactly into
three bf16 terms and all three products accumulate in fp32 in one launch, so
the result has fp32-GEMM accuracy, as the reference's fp32 ``F.linear``
(kquant/pack/qsrt_validation.py:240-258) does.

``mxfp8_linear_mm`` is the production form of the MXFP8 linear
(scripts/closure_mxfp8_mlp.py:163-187): the input rows are quantized to
MXFP8 with the ``mxfp8_quantize`` rule (``block_fp8_linear.quantize_input``,
:155) and both MXFP8 operands are multiplied as they are on the block-scaled
fp8 matrix cores (``kq_mx_linear_mm``); ``mxfp8_linear_mx`` takes input rows
that are already quantized (``kq_mx_linear_mx``).  Its oracle is
``_reference_from_packed`` (:146-160): dequantize both operands, fp32 product.

``int8_linear`` is the linear over 8-bit integers with a scale of each token and
each channel (``kq_int8_linear``), with the same epilogue.
"""

from __future__ import annotations

import torch

from . import _native as N
from .int8 import (INT8_K_ALIGN, _check_no_gradient, _check_source_scale, _check_weight, _pad_k as _pad_codes, _quantize,
                   _row_stride, _row_view)


def _check_epilogue(source, bias, activation, residual, lead, n: int, f32: bool, out_dtype: torch.dtype) -> None:
    if activation not in N.LIN_ACTIVATIONS:
        raise ValueError(f"activation must be None, relu, silu, gelu or gelu_tanh, got {activation!r}")
    if f32 and out_dtype != torch.float32:
        raise TypeError("a float32 source with an epilogue gives a float32 result")
    if bias is not None:
        if bias.dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"bias must be bfloat16 or float32, got {bias.dtype}")
        if tuple(bias.shape) != (n,):
            raise ValueError(f"bias shape {tuple(bias.shape)} != {(n,)}")
    if residual is not None:
        if residual.dtype != out_dtype:
            raise TypeError(f"residual must have the result's type {out_dtype}, got {residual.dtype}")
        if tuple(residual.shape) != (*lead, n):
            raise ValueError(f"residual shape {tuple(residual.shape)} != {(*lead, n)}")
    if N.carries_gradient(source, bias, residual):
        raise RuntimeError("a linear with bias, activation or residual carries no gradient: detach its inputs, or call it "
                           "under torch.no_grad() where none has a tangent")


def _linear(fmt: int, source: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor,
            out_dtype: torch.dtype | None, bias: torch.Tensor | None = None, activation: str | None = None,
            residual: torch.Tensor | None = None) -> torch.Tensor:
    if out_dtype is None:
        out_dtype = torch.float32 if source.dtype == torch.float32 else torch.bfloat16
    if source.ndim < 1:
        raise ValueError("source must have a feature dimension")
    if scale.dtype != torch.uint8:
        raise TypeError(f"scales must be uint8 E8M0, got {scale.dtype}")
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("out_dtype must be bfloat16 or float32")
    k = source.shape[-1]
    n = weight.shape[0]
    packed_k = k if fmt == N.FMT_MXFP8_E4M3 else k // 2
    if weight.ndim != 2 or weight.shape[1] != packed_k:
        raise ValueError(f"weight shape {tuple(weight.shape)} does not match K={k}")
    if tuple(scale.shape) != (n, k // 32):
        raise ValueError(f"scale shape {tuple(scale.shape)} != {(n, k // 32)}")
    if k % 64:
        raise ValueError(f"K={k} must be a multiple of 64")
    lead = source.shape[:-1]
    a = source.reshape(-1, k)
    exact_f32 = a.dtype == torch.float32
    if not exact_f32 and a.dtype != torch.bfloat16:
        a = a.to(torch.bfloat16)
    epilogue = bias is not None or activation is not None or residual is not None
    if epilogue:
        _check_epilogue(source, bias, activation, residual, lead, n, exact_f32, out_dtype)
        residual = None if residual is None else residual.reshape(-1, n)
    (a, w, s, bias, residual), gpu, host = N.to_gpu([a, weight.view(torch.uint8), scale, bias, residual])
    a, w, s = N.aligned(a), N.aligned(w), N.aligned(s)
    m = a.shape[0]
    if epilogue:
        return _linear_epilogue(fmt, a, w, s, out_dtype, bias, activation, residual, lead, gpu, host)
    if exact_f32:
        out = torch.empty(m, n, dtype=torch.float32, device=gpu)
        ws = torch.empty(max(int(N.library().kq_mx_linear_f32_split_workspace_size(m, n, k)), 16),
                         dtype=torch.uint8, device=gpu)
        N.call("kq_mx_linear_f32", fmt, N.ptr(a), k, N.ptr(w), N.ptr(s), m, n, k, N.ptr(out), n,
               N.ptr(ws), ws.numel(), N.stream(gpu))
        out = out.to(out_dtype)
    else:
        out = torch.empty(m, n, dtype=out_dtype, device=gpu)
        need = int(N.library().kq_mx_linear_workspace_size(m, n, k))
        ws = torch.empty(need, dtype=torch.uint8, device=gpu) if need > 0 else None  # a K split's planes
        N.call("kq_mx_linear_ws", fmt, N.ptr(a), k, N.ptr(w), N.ptr(s), m, n, k,
               N.DTYPE_CODES[out_dtype], N.ptr(out), n, N.ptr(ws), max(need, 0), N.stream(gpu))
    out = out.reshape(*lead, n)
    return out if host is None else out.to(host)


def _linear_epilogue(fmt, a, w, s, out_dtype, bias, activation, residual, lead, gpu, host) -> torch.Tensor:
    m, k = a.shape
    n = w.shape[0]
    f32 = a.dtype == torch.float32
    if bias is not None:
        bias = bias.contiguous()
    if residual is not None and (residual.stride(1) != 1 or residual.stride(0) < n):
        residual = residual.contiguous()
    with N.on_device(gpu):
        size = N.library().kq_mx_linear_f32_split_workspace_size if f32 else N.library().kq_mx_linear_workspace_size
        need = max(int(size(m, n, k)), 0)
        ws = torch.empty(need, dtype=torch.uint8, device=gpu) if need else None
        out = torch.empty(m, n, dtype=out_dtype, device=gpu)
        N.call("kq_mx_linear_epilogue", fmt, N.DTYPE_CODES[a.dtype], N.ptr(a), k, N.ptr(w), N.ptr(s), m, n, k,
               N.LIN_ACTIVATIONS[activation], N.ptr(bias), N.DT_BF16 if bias is None else N.DTYPE_CODES[bias.dtype],
               N.ptr(residual), n if residual is None else residual.stride(0), N.DTYPE_CODES[out_dtype], N.ptr(out), n,
               N.ptr(ws), need, N.stream(gpu))
    out = out.reshape(*lead, n)
    return out if host is None else out.to(host)


def mxfp8_linear(source: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, *,
                 bias: torch.Tensor | None = None, activation: str | None = None,
                 residual: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``source [..., K] @ dequant(weight E4M3 [N, K], scale [N, K/32]).T``.

    Output dtype defaults to fp32 for fp32 sources and bf16 otherwise.

    ``bias`` [N] (bf16 or fp32), ``activation`` ("relu", "silu", "gelu", its
    tanh form "gelu_tanh", or None) and ``residual`` (of the result's shape and
    type) are applied in the kernel's epilogue on the fp32 sums, which are then
    rounded once: ``activation(source @ W.T + bias) + residual``.  The result
    carries no gradient: with any of the three, a source, bias or residual that
    requires one (while autograd records) or has a tangent is refused (a skip
    connection inside the call would leave the graph unseen).
    """
    if weight.dtype not in (torch.float8_e4m3fn, torch.uint8):
        raise TypeError(f"MXFP8 weight must be float8_e4m3fn, got {weight.dtype}")
    return _linear(N.FMT_MXFP8_E4M3, source, weight, scale, out_dtype, bias, activation, residual)


def mxfp4_linear(source: torch.Tensor, packed: torch.Tensor, scale: torch.Tensor, *,
                 bias: torch.Tensor | None = None, activation: str | None = None,
                 residual: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``source [..., K] @ dequant(packed [N, K/2], scale [N, K/32]).T``.

    Output dtype defaults to fp32 for fp32 sources and bf16 otherwise; bias,
    activation and residual as in ``mxfp8_linear``.
    """
    if packed.dtype != torch.uint8:
        raise TypeError(f"expected uint8, got {packed.dtype}")
    return _linear(N.FMT_MXFP4_E2M1, source, packed, scale, out_dtype, bias, activation, residual)


MX_LINEAR_K_ALIGN = 128  # the MXFP8 x MXFP8 kernel's K granule


def _pad_k(t: torch.Tensor, width: int, value: int = 0) -> torch.Tensor:
    """Zero-pad the last dimension (the reference pads the source to the packed
    weight's padded_in_features, scripts/closure_mxfp8_mlp.py:136-143)."""
    if t.shape[-1] == width:
        return t
    return torch.nn.functional.pad(t, (0, width - t.shape[-1]), value=value)


def _mx_weight(weight: torch.Tensor, scale: torch.Tensor, k: int):
    if weight.dtype not in (torch.float8_e4m3fn, torch.uint8):
        raise TypeError(f"MXFP8 weight must be float8_e4m3fn, got {weight.dtype}")
    if scale.dtype != torch.uint8:
        raise TypeError(f"scales must be uint8 E8M0, got {scale.dtype}")
    if weight.ndim != 2 or weight.shape[1] != k:
        raise ValueError(f"weight shape {tuple(weight.shape)} does not match K={k}")
    if tuple(scale.shape) != (weight.shape[0], k // 32):
        raise ValueError(f"scale shape {tuple(scale.shape)} != {(weight.shape[0], k // 32)}")
    kp = -(-k // MX_LINEAR_K_ALIGN) * MX_LINEAR_K_ALIGN
    # padded weight columns are zero codes, so they add nothing whatever their scale
    return _pad_k(weight.view(torch.uint8), kp), _pad_k(scale, kp // 32, 127), kp


def mxfp8_linear_mm(source: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, *,
                    out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``mxfp8_linear.mm(source, packed)`` of the reference's production MXFP8
    linear: ``source [..., K]`` (bf16, fp16 or fp32) is quantized per row to
    MXFP8 (the ``mxfp8_quantize`` rule, 32-element blocks along K), then
    multiplied by the MXFP8 weight (E4M3 [N, K], scale [N, K/32]) on the
    block-scaled fp8 matrix cores with fp32 accumulation.  Equals
    ``dequant(quantize(source)) @ dequant(weight).T`` (the reference's
    operand-exact oracle) up to the matrix cores' summation.  K is padded to
    a multiple of 128 with zeros when needed (a per-call copy of the weight;
    pad it once to skip that)."""
    if source.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError("source must be bfloat16, float16 or float32")
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("out_dtype must be bfloat16 or float32")
    k = source.shape[-1]
    if k % 32:
        raise ValueError(f"K={k} must be a multiple of 32 (the MX block)")
    lead = source.shape[:-1]
    (a, w, s), gpu, host = N.to_gpu([source.reshape(-1, k), weight.view(torch.uint8), scale])
    w, s, kp = _mx_weight(w, s, k)
    a = _pad_k(a, kp)
    a = a if a.stride(-1) == 1 and a.stride(0) % 8 == 0 else a.contiguous()
    a, w, s = N.aligned(a), N.aligned(w), N.aligned(s, 4)
    m, n = a.shape[0], w.shape[0]
    out = torch.empty(m, n, dtype=out_dtype, device=gpu)
    ws = torch.empty(max(int(N.library().kq_mx_linear_mm_workspace_size(m, n, kp)), 256), dtype=torch.uint8,
                     device=gpu)
    N.call("kq_mx_linear_mm", N.FMT_MXFP8_E4M3, N.ptr(a), N.DTYPE_CODES[a.dtype], a.stride(0), N.ptr(w), N.ptr(s),
           m, n, kp, N.DTYPE_CODES[out_dtype], N.ptr(out), n, N.ptr(ws), ws.numel(), N.stream(gpu))
    out = out.reshape(*lead, n)
    return out if host is None else out.to(host)


def mxfp8_linear_mx(source_q: torch.Tensor, source_scale: torch.Tensor, weight: torch.Tensor,
                    scale: torch.Tensor, *, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``dequant(source_q, source_scale) @ dequant(weight, scale).T`` for input
    rows already in MXFP8 (E4M3 [M, K], E8M0 [M, K/32], e.g. from
    ``mxfp8_quantize``), on the block-scaled fp8 matrix cores."""
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("out_dtype must be bfloat16 or float32")
    if source_q.ndim != 2:
        raise ValueError("source_q must be [M, K]")
    k = source_q.shape[1]
    if k % 32:
        raise ValueError(f"K={k} must be a multiple of 32 (the MX block)")
    if source_scale.dtype != torch.uint8 or tuple(source_scale.shape) != (source_q.shape[0], k // 32):
        raise ValueError(f"source_scale must be uint8 [{source_q.shape[0]}, {k // 32}]")
    (aq, as_, w, s), gpu, host = N.to_gpu([source_q.view(torch.uint8), source_scale, weight.view(torch.uint8), scale])
    w, s, kp = _mx_weight(w, s, k)
    aq, as_ = _pad_k(aq, kp).contiguous(), _pad_k(as_, kp // 32, 127).contiguous()
    aq, as_, w, s = N.aligned(aq), N.aligned(as_, 4), N.aligned(w), N.aligned(s, 4)
    m, n = aq.shape[0], w.shape[0]
    out = torch.empty(m, n, dtype=out_dtype, device=gpu)
    ws = torch.empty(max(int(N.library().kq_mx_linear_mx_workspace_size(m, n, kp)), 256), dtype=torch.uint8,
                     device=gpu)
    N.call("kq_mx_linear_mx", N.FMT_MXFP8_E4M3, N.ptr(aq), N.ptr(as_), kp, N.FMT_MXFP8_E4M3, N.ptr(w), N.ptr(s),
           m, n, kp, N.DTYPE_CODES[out_dtype], N.ptr(out), n, N.ptr(ws), ws.numel(), N.stream(gpu))
    return out if host is None else out.to(host)


def int8_linear(source: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, *,
                source_scale: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                activation: str | None = None, residual: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``activation(dequant(source) @ dequant(weight).T + bias) + residual`` over
    8-bit integers: weight int8 [N, K] with fp32 scales [N] (or [N, 1]), source
    either int8 codes [..., K] with ``source_scale`` [...] (``int8_quantize``,
    once for all layers that read the rows) or bf16, fp16 or fp32 rows, which are
    quantized in the call by the same rule.

    The integer sums are exact; scaling (by the row's scale, then the channel's), bias [N] (bf16 or fp32), activation
    ("relu", "silu", "gelu", "gelu_tanh") and residual (of the result's shape and
    type) are fp32, rounded once.  The result is bf16, fp16 or fp32: ``out_dtype``,
    else the source's type, else (codes) bf16.  A row whose source holds an
    infinity or a NaN is NaN.  K is at most 131056; a K that is no multiple of 16
    is padded with zeros (a copy of the weight in every call: pad it once to skip
    that).  Results do not change from call to call.  They carry no gradient: a
    source, bias, residual or scale that requires one (while autograd records) or has a
    tangent is refused.
    """
    source_scale = _check_source_scale(source, source_scale)
    if source.ndim < 1:
        raise ValueError("source must have a feature dimension")
    k = source.shape[-1]
    scale = _check_weight(weight, scale, 2, k)
    if out_dtype is None:
        out_dtype = torch.bfloat16 if source.dtype == torch.int8 else source.dtype
    if out_dtype not in N.DTYPE_CODES:
        raise TypeError("out_dtype must be bfloat16, float16 or float32")
    n, lead = weight.shape[0], source.shape[:-1]
    _check_epilogue(source, bias, activation, residual, lead, n, False, out_dtype)
    _check_no_gradient("int8_linear", scale, source_scale)
    (a, w, s, sx, bias, residual), gpu, host = N.to_gpu((source, weight, scale, source_scale, bias, residual))
    a, s = _row_view(a), N.aligned(s, 4)
    kp = -(-k // INT8_K_ALIGN) * INT8_K_ALIGN
    w = N.aligned(_pad_codes(w, kp))
    m = a.shape[0]
    with N.on_device(gpu):
        ws, need = None, 0
        if sx is not None:
            sx = N.aligned(sx if sx.ndim == 1 else sx.reshape(-1), 4)
            a = _pad_codes(a, kp)
            if a.data_ptr() % 16 or _row_stride(a) % 16 or _row_stride(a) > 1 << 22:
                a = a.clone(memory_format=torch.contiguous_format)
        elif kp != k:
            a, sx = _quantize(a, kp)
        code = N.DT_I8 if sx is not None else N.DTYPE_CODES[a.dtype]
        if sx is None or m > 16:
            need = N.library().kq_int8_linear_workspace_size(code, m, n, kp)
            if need > 0:
                ws = torch.empty(need, dtype=torch.uint8, device=gpu)
        if bias is not None:
            bias = bias.contiguous()
        if residual is not None:
            residual = _row_view(residual if residual.ndim == 2 else residual.reshape(m, n))
        out = torch.empty(m, n, dtype=out_dtype, device=gpu)
        N.call("kq_int8_linear", code, a.data_ptr(), _row_stride(a), N.ptr(sx), w.data_ptr(), s.data_ptr(), m, n, kp,
               N.LIN_ACTIVATIONS[activation], N.ptr(bias), 0 if bias is None else N.DTYPE_CODES[bias.dtype],
               N.ptr(residual), n if residual is None else _row_stride(residual), N.DTYPE_CODES[out_dtype],
               out.data_ptr(), n, N.ptr(ws), need, N.stream(gpu))
    if source.ndim != 2:
        out = out.reshape(*lead, n)
    return out if host is None else out.to(host)
