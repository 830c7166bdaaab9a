"""Softmax cross entropy of a vocabulary head, without keeping its logits.

``linear_cross_entropy`` is the loss of ``hidden @ head.T`` against target ids,
for a dense bf16 head or an MXFP8 / MXFP4 one: the perplexity of a quantized
model, and with its gradients the training of a head or the recovery of the
layers below a frozen quantized one.  No [tokens, vocabulary] array reaches
memory in the forward pass; the backward pass works through the vocabulary in
pieces of at most 1 GiB.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _native as N
from .grouped import _rows

_REDUCTIONS = {"none": N.LOSS_NONE, "mean": N.LOSS_MEAN, "sum": N.LOSS_SUM}


def _workspace(fmt: int, tokens: int, vocab: int, k: int, backward: int, device: torch.device) -> torch.Tensor:
    nbytes = int(N.library().kq_linear_cross_entropy_workspace_size(fmt, tokens, vocab, k, backward))
    if nbytes < 0:
        raise ValueError("at most 2^20 tokens, 2^24 vocabulary rows and K = 2^16")
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, scale, target, fmt, ignore_index, reduction):
        tokens, k = hidden.shape
        vocab = weight.shape[0]
        with N.on_device(hidden.device):
            hidden = _rows(hidden)
            losses = torch.empty(tokens, dtype=torch.float32, device=hidden.device)
            lse = torch.empty_like(losses)
            sums = None if reduction == N.LOSS_NONE else torch.empty(2, dtype=torch.float32, device=hidden.device)
            ws = _workspace(fmt, tokens, vocab, k, 0, hidden.device)
            N.call("kq_linear_cross_entropy", fmt, N.ptr(hidden), hidden.stride(0), tokens, N.ptr(weight), N.ptr(scale),
                   vocab, k, N.ptr(target), ignore_index, N.ptr(losses), N.ptr(lse), N.ptr(sums), N.ptr(ws), ws.numel(),
                   N.stream(hidden.device))
        ctx.save_for_backward(hidden, weight, scale, target, lse)
        ctx.args = fmt, ignore_index, reduction
        if reduction == N.LOSS_NONE:
            return losses
        # a tensor of its own over sums' memory: a view made in here could not be changed in place (loss /= steps)
        at = 1 if reduction == N.LOSS_MEAN else 0
        return sums.new_empty(0).set_(sums.untyped_storage(), at, (), ())

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        hidden, weight, scale, target, lse = ctx.saved_tensors
        fmt, ignore_index, reduction = ctx.args
        tokens, k = hidden.shape
        vocab = weight.shape[0]
        dh = dw = None
        with N.on_device(hidden.device):
            grad = grad.to(torch.float32).contiguous()
            if ctx.needs_input_grad[0]:
                dh = torch.empty(tokens, k, dtype=torch.bfloat16, device=hidden.device)
            if ctx.needs_input_grad[1]:
                dw = torch.empty_like(weight)
            ws = _workspace(fmt, tokens, vocab, k, 1, hidden.device)
            N.call("kq_linear_cross_entropy_backward", fmt, N.ptr(hidden), hidden.stride(0), tokens, N.ptr(weight),
                   N.ptr(scale), vocab, k, N.ptr(target), ignore_index, N.ptr(lse), N.ptr(grad), reduction, N.ptr(dh), k,
                   N.ptr(dw), N.ptr(ws), ws.numel(), N.stream(hidden.device))
        return dh, dw, None, None, None, None, None


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor,
                         scale: torch.Tensor | None = None, *, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """Cross entropy (fp32) of the logits ``hidden @ weight.T`` at ``target``.

    hidden bf16 [..., K]; target int64 [...].  The head is bf16 [V, K] (K a
    multiple of 8), or block-scaled with E8M0 ``scale`` uint8 [V, K / 32] (K a
    multiple of 64): MXFP8 E4M3 [V, K] (``float8_e4m3fn`` or its bytes) or MXFP4
    packed uint8 [V, K / 2].  ``reduction`` is "mean" (over the counted tokens;
    NaN if there are none), "sum" or "none" (a loss per token, in target's
    shape).  Tokens whose target is ``ignore_index`` count nowhere: their loss
    and gradient are 0 whatever their row holds.  Another target outside [0, V)
    gives a NaN loss.

    hidden may have any strides (copied unless its rows are contiguous, 16-byte
    aligned and a multiple of 8 elements apart); a head that is not contiguous,
    such as the transpose of one stored [K, V], is copied whole in every call.

    Differentiable once, in hidden and in a bf16 weight; a block-scaled head is
    frozen.  The logits and all sums are fp32; the gradients are bf16, their
    softmax terms rounded to bf16 as operands of the gradients' products.
    Results do not change from call to call (no atomics).  Captured into a graph,
    forward and backward go into one capture, made while no eager graph of the
    same leaves lives.
    """

    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    if hidden.dtype != torch.bfloat16:
        raise TypeError(f"hidden must be bfloat16, got {hidden.dtype}")
    if target.dtype != torch.int64:
        raise TypeError(f"target must be int64, got {target.dtype}")
    if hidden.ndim < 1 or weight.ndim != 2:
        raise ValueError("hidden must be [..., K] and weight [V, K]")
    k = hidden.shape[-1]
    if tuple(target.shape) != tuple(hidden.shape[:-1]):
        raise ValueError(f"target shape {tuple(target.shape)} != {tuple(hidden.shape[:-1])}")
    if scale is None:
        if weight.dtype != torch.bfloat16:
            raise TypeError(f"a head without scales must be bfloat16, got {weight.dtype}")
        fmt, granule, packed_k = N.FMT_BF16, 8, k
    else:
        if weight.dtype not in (torch.float8_e4m3fn, torch.uint8):
            raise TypeError(f"a block-scaled head must be float8_e4m3fn or uint8, got {weight.dtype}")
        if scale.dtype != torch.uint8:
            raise TypeError(f"scales must be uint8 E8M0, got {scale.dtype}")
        packed = weight.dtype == torch.uint8 and weight.shape[1] * 2 == k
        fmt, granule, packed_k = (N.FMT_MXFP4_E2M1, 64, k // 2) if packed else (N.FMT_MXFP8_E4M3, 64, k)
    if k == 0 or k % granule:
        raise ValueError(f"K={k} must be a positive multiple of {granule}")
    vocab = weight.shape[0]
    if vocab == 0 or weight.shape[1] != packed_k:
        raise ValueError(f"weight shape {tuple(weight.shape)} does not match K={k}")
    if scale is not None and tuple(scale.shape) != (vocab, k // 32):
        raise ValueError(f"scale shape {tuple(scale.shape)} != {(vocab, k // 32)}")
    tensors = [t for t in (hidden, weight, target, scale) if t is not None]
    if any(t.device != hidden.device for t in tensors):
        raise ValueError("hidden, weight, target and scale must be on one device")
    host = None if hidden.is_cuda else hidden.device
    if host is None:
        N.check_capture(hidden, weight)
    h, t = hidden if hidden.ndim == 2 else hidden.reshape(-1, k), target.reshape(-1)
    if host is not None:
        gpu = N.require_gpu()
        h, weight, t = h.to(gpu), weight.to(gpu), t.to(gpu)
        scale = None if scale is None else scale.to(gpu)
    if scale is not None:
        weight, scale = weight.view(torch.uint8), N.aligned(scale)
    weight, t = N.aligned(weight), N.aligned(t, 8)
    loss = _LinearCrossEntropy.apply(h, weight, scale, t, fmt, int(ignore_index), _REDUCTIONS[reduction])
    N.note_leaves(loss)
    if reduction == "none":
        loss = loss.reshape(target.shape)
    return loss if host is None else loss.to(host)
