"""8-bit integers with one fp32 scale a row (symmetric, per token or per channel).

The codec of ``linear.int8_linear`` and ``grouped.int8_grouped_linear``: the
layout in which W8A8 checkpoints keep their weights ([out, in] codes, a scale of
each output channel) and in which a product takes its tokens.
"""

from __future__ import annotations

import torch

from . import _native as N

INT8_MAX_K = (1 << 17) - 16  # int32 sums of products up to 2^14
INT8_K_ALIGN = 16            # the products' K granule


def _row_view(x: torch.Tensor) -> torch.Tensor:
    """[..., K] as [rows, K] with unit column stride and rows that do not overlap (copied where they do)."""
    a = x if x.ndim == 2 else x.reshape(-1, x.shape[-1])
    if a.stride(1) != 1 or (a.shape[0] > 1 and a.stride(0) < a.shape[1]):
        a = a.contiguous()
    return a


def _row_stride(a: torch.Tensor) -> int:
    return max(a.stride(0), a.shape[1])


def _quantize(a: torch.Tensor, width: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes [rows, width] (zeros past K) and scales of GPU rows ``a`` [rows, K]."""
    rows, k = a.shape
    make = torch.empty if width == k else torch.zeros
    q = make(rows, width, dtype=torch.int8, device=a.device)
    scale = torch.empty(rows, dtype=torch.float32, device=a.device)
    if rows:
        N.call("kq_int8_quantize", N.DTYPE_CODES[a.dtype], N.ptr(a), _row_stride(a), rows, k, N.ptr(q), width,
               N.ptr(scale), N.stream(a.device))
    return q, scale


def int8_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes (int8 [..., K]) and scales (fp32 [...]) of the rows of x [..., K],
    bf16, fp16 or fp32:

        scale = max(max |x| * fp32(1 / 127), 2^-126),  q = round(x / scale)

    with the product rounded to fp32 (at most one fp32 step below max |x| / 127 rounded once) and the exact quotient
    rounded to nearest, ties to even, so the codes do not depend on how the division is carried out.  A row with an infinity or a
    NaN has scale NaN and codes 0: whatever it is multiplied with is NaN, and no
    other row is.  A row of zeros has codes 0.  The results carry no gradient.
    """

    if x.dtype not in N.DTYPE_CODES:
        raise TypeError(f"x must be bfloat16, float16 or float32, got {x.dtype}")
    if x.ndim < 1 or x.shape[-1] == 0:
        raise ValueError("x must have a feature dimension")
    (a,), gpu, host = N.to_gpu([x])
    a = _row_view(a)
    with N.on_device(gpu):
        q, scale = _quantize(a, a.shape[1])
    if x.ndim != 2:
        q, scale = q.reshape(x.shape), scale.reshape(x.shape[:-1])
    return (q, scale) if host is None else (q.to(host), scale.to(host))


def int8_dequantize(q: torch.Tensor, scale: torch.Tensor, *, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``q * scale`` of codes [..., K] and their rows' scales [...], rounded once to ``dtype``.

    Differentiable in the scales.  On the GPU, in bf16, fp16 or fp32 and without a derivative, one kernel; else
    elementwise torch operations with the same results, on the tensors' own device.
    """

    if q.dtype != torch.int8 or scale.dtype != torch.float32:
        raise TypeError(f"expected int8 codes and float32 scales, got {q.dtype} and {scale.dtype}")
    if q.ndim < 1 or tuple(scale.shape) != tuple(q.shape[:-1]):
        raise ValueError(f"scale shape {tuple(scale.shape)} != {tuple(q.shape[:-1])}")
    if (q.is_cuda and scale.device == q.device and dtype in N.DTYPE_CODES and q.shape[-1] and not N.carries_gradient(scale)
            and not any(map(torch._C._functorch.is_functorch_wrapped_tensor, (q, scale)))):
        a = _row_view(q)
        with N.on_device(q.device):
            out = torch.empty(a.shape, dtype=dtype, device=q.device)
            N.call("kq_int8_dequantize", N.ptr(a), _row_stride(a), N.ptr(N.aligned(scale.reshape(-1), 4)), *a.shape,
                   N.DTYPE_CODES[dtype], N.ptr(out), a.shape[1], N.stream(q.device))
        return out.reshape(q.shape)
    s, codes = scale.unsqueeze(-1), q.float()
    if dtype == torch.float64:
        return q.double() * s.double()
    values = codes * s
    if dtype not in (torch.bfloat16, torch.float16):
        return values.to(dtype)
    # Rounded to fp32 and then to 16 bits a product can end on the far side of a border between two results that its
    # fp32 value lies on.  A product that is not an fp32 number is therefore taken as the neighbour with an odd last bit,
    # which no border has.  (What lies below fp32's normal numbers is exact: no rest.)
    v = values.detach()
    rest = codes.double() * s.detach().double() - v.double()
    beyond = torch.nextafter(v, torch.where(rest > 0, torch.inf, -torch.inf).to(v.dtype))
    half = torch.frexp(v).mantissa * 2.0 ** 23  # of an odd last bit: no whole number
    even = (half == torch.floor(half)) & (rest != 0) & torch.isfinite(v)
    return (values + torch.where(even, beyond - v, 0.0)).to(dtype)


def _pad_k(q: torch.Tensor, width: int) -> torch.Tensor:
    return q if q.shape[-1] == width else torch.nn.functional.pad(q, (0, width - q.shape[-1]))


def _check_weight(weight: torch.Tensor, scale: torch.Tensor, dims: int, k: int) -> torch.Tensor:
    """The scales without a trailing dimension of one."""
    names = "[groups, N, K]" if dims == 3 else "[N, K]"
    if weight.dtype != torch.int8:
        raise TypeError(f"weight must be int8, got {weight.dtype}")
    if scale.dtype != torch.float32:
        raise TypeError(f"scales must be float32, got {scale.dtype}")
    if weight.ndim != dims or weight.shape[-1] != k:
        raise ValueError(f"weight shape {tuple(weight.shape)} is not {names} with K={k}")
    if scale.ndim == dims and scale.shape[-1] == 1:
        scale = scale.squeeze(-1)
    if tuple(scale.shape) != tuple(weight.shape[:-1]):
        raise ValueError(f"scale shape {tuple(scale.shape)} != {tuple(weight.shape[:-1])}")
    if not 0 < k <= INT8_MAX_K:
        raise ValueError(f"K={k} must be between 1 and {INT8_MAX_K}")
    return scale


def _check_no_gradient(name: str, *tensors: torch.Tensor | None) -> None:
    if N.carries_gradient(*tensors):
        raise RuntimeError(f"{name} carries no gradient: detach its arguments, or call it under "
                           "torch.no_grad() where none has a tangent")


def _check_source_scale(source: torch.Tensor, scale: torch.Tensor | None) -> torch.Tensor | None:
    if source.dtype == torch.int8:
        if scale is None:
            raise ValueError("int8 rows need their scales")
        if scale.dtype != torch.float32:
            raise TypeError(f"scales must be float32, got {scale.dtype}")
        if scale.ndim == source.ndim and scale.shape[-1] == 1:
            scale = scale.squeeze(-1)
        if tuple(scale.shape) != tuple(source.shape[:-1]):
            raise ValueError(f"scales of the rows have shape {tuple(scale.shape)}, not {tuple(source.shape[:-1])}")
        return scale
    if source.dtype not in N.DTYPE_CODES:
        raise TypeError(f"rows must be int8, bfloat16, float16 or float32, got {source.dtype}")
    if scale is not None:
        raise ValueError("scales of the rows belong to int8 rows")
    return None
