"""Sampling the next token from logits and given uniform numbers.

The step behind a vocabulary head (``linear.mxfp8_linear``, ``mxfp4_linear``,
``int8_linear``): the counterpart of ``loss.linear_cross_entropy``, which scores
tokens that are given.
"""

from __future__ import annotations

import math

import torch

from . import _native as N

MAX_VOCAB = 1 << 18


def _flat(v: torch.Tensor) -> torch.Tensor:
    return N.aligned(v if v.ndim == 1 else v.reshape(-1), 4)


def _setting(name: str, value, lead, default: float, check) -> tuple[torch.Tensor | None, float]:
    """(one value a row or None, one for all)."""
    if value is None:
        return None, default
    if isinstance(value, torch.Tensor) and value.ndim > 0:
        want = "int32 or int64" if name == "top_k" else "float32"
        if value.dtype not in ((torch.int32, torch.int64) if name == "top_k" else (torch.float32,)):
            raise TypeError(f"{name} of each row must be {want}, got {value.dtype}")
        if tuple(value.shape) != tuple(lead):
            raise ValueError(f"{name} has shape {tuple(value.shape)}, the rows {tuple(lead)}")
        return value, default
    if isinstance(value, torch.Tensor):
        raise TypeError(f"{name} must be a number or a tensor with a value for each row")
    if not check(value):
        raise ValueError(f"{name}={value!r} is out of range")
    return None, value


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, *, temperature: float | torch.Tensor = 1.0,
                  top_k: int | torch.Tensor | None = None, top_p: float | torch.Tensor | None = None,
                  min_p: float | torch.Tensor | None = None, return_logprobs: bool = False):
    """One token (int64 [...]) for each row of logits [..., V] (bf16, fp16 or
    fp32, V at most 262144), drawn with the row's number in ``uniform`` (fp32
    [...], in [0, 1)).

    With w_i = exp((logits_i - max) / temperature) and the tokens in the order of
    descending logits, ties by ascending index:

      top_k   keeps the first top_k tokens (None, 0 or fewer: all)
      top_p   of those the shortest prefix whose weight reaches top_p of theirs:
              a token stays while the weight before it is below that (1: all)
      min_p   of those the tokens with w_i >= min_p (None or 0: all)

    The first token always stays.  The token drawn is the first kept one, by
    index, up to and with which the kept weight exceeds uniform times the total;
    a number from 1 up draws the last kept token, one below 0 the first.  A
    temperature of 0 takes the largest logit.  Each setting is a number or a
    tensor [...] with a row's own (fp32; top_k int32 or int64), where a top_k of 0
    or fewer and a top_p of 1 or more keep all, a top_p of 0 or less and a min_p
    of 1 or more the first token and its equals at most, and a temperature that is
    not above 0 takes the largest logit.

    Logits of -inf are never drawn; logits of +inf share the draw among them.  A
    row with a NaN, or with nothing above -inf, gives -1.

    Weights are exact multiples of 2^-45, summed as integers, so the result
    depends on the row and its settings alone: not on the batch, the call or the
    order of sums.  Weights below 2^-46 of the largest count as 0.

    ``return_logprobs`` returns also the natural logarithm of the probability
    with which each token was drawn, among those kept (fp32 [...]; NaN where the
    token is -1); they carry no gradient: logits that require one
    (while autograd records) or have a tangent are refused then.
    """

    if logits.dtype not in N.DTYPE_CODES:
        raise TypeError(f"logits must be bfloat16, float16 or float32, got {logits.dtype}")
    if uniform.dtype != torch.float32:
        raise TypeError(f"uniform must be float32, got {uniform.dtype}")
    if logits.ndim < 1 or not 0 < logits.shape[-1] <= MAX_VOCAB:
        raise ValueError(f"logits must be [..., V] with V between 1 and {MAX_VOCAB}, got {tuple(logits.shape)}")
    if return_logprobs and N.carries_gradient(logits):
        raise RuntimeError("sample_tokens carries no gradient: detach the logits, or call it under "
                           "torch.no_grad() where they have no tangent")
    vocab, lead = logits.shape[-1], logits.shape[:-1]
    if tuple(uniform.shape) != tuple(lead):
        raise ValueError(f"uniform has shape {tuple(uniform.shape)}, the rows {tuple(lead)}")
    t_rows, t = _setting("temperature", temperature, lead, 1.0, lambda v: v >= 0 and math.isfinite(v))
    k_rows, k = _setting("top_k", top_k, lead, 0, lambda v: v == int(v))
    p_rows, p = _setting("top_p", top_p, lead, 1.0, lambda v: 0 < v <= 1)
    m_rows, m = _setting("min_p", min_p, lead, 0.0, lambda v: 0 <= v <= 1)
    k = max(0, min(int(k), MAX_VOCAB))
    if temperature is None:
        raise TypeError("temperature must be a number or a tensor with a value for each row")
    (z, u, t_rows, k_rows, p_rows, m_rows), gpu, host = N.to_gpu((logits, uniform, t_rows, k_rows, p_rows, m_rows))
    if z.ndim != 2:
        z = z.reshape(-1, vocab)
    rows, ld = z.shape[0], z.stride(0)
    if z.stride(1) != 1 or ld < vocab:
        if rows > 1 or z.stride(1) != 1:
            z = z.contiguous()
        ld = vocab
    with N.on_device(gpu):
        u = _flat(u)
        if k_rows is not None:
            k_rows = _flat(k_rows if k_rows.dtype == torch.int32 else k_rows.clamp(0, MAX_VOCAB).to(torch.int32))
        t_rows, p_rows, m_rows = (None if v is None else _flat(v) for v in (t_rows, p_rows, m_rows))
        filters = k_rows is not None or k > 0 or p_rows is not None or p < 1
        need = N.library().kq_sample_tokens_workspace_size(rows, vocab, filters)
        ws = torch.empty(need, dtype=torch.uint8, device=gpu) if need > 0 else None
        tokens = torch.empty(rows, dtype=torch.int64, device=gpu)  # (a torch.Size would cost a microsecond)
        logprobs = torch.empty(rows, dtype=torch.float32, device=gpu) if return_logprobs else None
        N.call("kq_sample_tokens", N.DTYPE_CODES[z.dtype], z.data_ptr(), ld, rows, vocab, u.data_ptr(), N.ptr(t_rows), t,
               N.ptr(k_rows), k, N.ptr(p_rows), p, N.ptr(m_rows), m, tokens.data_ptr(), N.ptr(logprobs), N.ptr(ws),
               max(need, 0), N.stream(gpu))
    if len(lead) != 1:
        tokens, logprobs = tokens.reshape(lead), None if logprobs is None else logprobs.reshape(lead)
    if host is not None:
        tokens, logprobs = tokens.to(host), None if logprobs is None else logprobs.to(host)
    return (tokens, logprobs) if return_logprobs else tokens
