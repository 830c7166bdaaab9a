"""The router, the products grouped by expert, the dense linear with its epilogue
and the head loss as they are used one after another: a layer scored through a
quantized head, calibration rows for the experts' down product, and a training
step of the experts and the head.

Every stage is compared with its formula in float64 on the rows that it was
given, within its own tolerance; the scores also with the whole layer in
float64, within the stages' errors carried through absolute values."""

from __future__ import annotations

import math

import pytest
import torch

from kquant_amd import _native as N
from kquant_amd import candidate_hessian, linear, mxfp8
from kquant_amd.grouped import grouped_linear
from kquant_amd.loss import linear_cross_entropy
from kquant_amd.tp_simulator import kimi_topk, swiglu

from .test_gpu_grouped import close
from .test_gpu_linear_epilogue import activate
from .test_gpu_linear_epilogue import check as check_linear
from .test_gpu_loss import check_sum, formula, near

pytestmark = pytest.mark.gpu
U24, U8 = 2.0 ** -24, 2.0 ** -8
TOKENS, HIDDEN, INTER, EXPERTS, TOPK, VOCAB = 301, 256, 136, 6, 2, 777


def route(logits, gpu):
    """Gates, tokens and offsets of the (token, expert) pairs in expert order."""
    gates, ids = kimi_topk(logits, torch.zeros(EXPERTS, device=gpu), TOPK)
    pairs = ids.numel()
    need = max(int(N.library().kq_route_sort_workspace_size(TOKENS, TOPK, EXPERTS)), 256)
    ws = torch.empty(need, dtype=torch.uint8, device=gpu)
    offsets = torch.empty(EXPERTS + 1, dtype=torch.int64, device=gpu)
    rows = torch.empty(pairs, dtype=torch.int32, device=gpu)
    sorted_gates = torch.empty(pairs, dtype=torch.float32, device=gpu)
    N.call("kq_route_sort", N.ptr(ids), TOKENS, TOPK, EXPERTS, N.ptr(gates), N.ptr(offsets), N.ptr(rows), None,
           N.ptr(sorted_gates), N.ptr(ws), need, N.stream(gpu))
    return sorted_gates, rows.long(), offsets


def model(gpu):
    g = torch.Generator(device=gpu).manual_seed(5)

    def weight(*shape):
        return (torch.randn(*shape, generator=g, device=gpu) / math.sqrt(shape[-1])).to(torch.bfloat16)

    h = torch.randn(TOKENS, HIDDEN, generator=g, device=gpu).to(torch.bfloat16)
    logits = torch.randn(TOKENS, EXPERTS, generator=g, device=gpu)
    logits[:, 4] = -50.0  # an expert that no token takes
    target = torch.randint(0, VOCAB, (TOKENS,), generator=g, device=gpu)
    target[::7] = -100
    experts = weight(EXPERTS, INTER, HIDDEN), weight(EXPERTS, INTER, HIDDEN), weight(EXPERTS, HIDDEN, INTER)
    return h, logits, target, experts, 3 * weight(VOCAB, HIDDEN), weight(HIDDEN, HIDDEN)


def check_grouped(y, x, w, offsets):
    starts = offsets.tolist()
    assert starts[0] == 0 and starts[-1] == x.shape[0]
    for e in range(EXPERTS):
        close(y[starts[e]:starts[e + 1]], x[starts[e]:starts[e + 1]], w[e], w.shape[2])


class Carried:
    """A value in float64 and a bound on the distance of the computed one from it."""

    def __init__(self, value, err):
        self.value, self.err = value, err

    def rounded(self):
        return Carried(self.value, self.err + U8 * (self.value.abs() + self.err))

    def times(self, w, length):
        """The product with exact bf16 rows w, summed in fp32."""
        w = w.double()
        size = (self.value.abs() + self.err) @ w.abs().T
        return Carried(self.value @ w.T, self.err @ w.abs().T + length * U24 * size)


def test_scoring(gpu):
    h, logits, target, (w1, w3, w2), head, dense = model(gpu)
    gates, rows, offsets = route(logits, gpu)
    x = h[rows]
    gate, up = grouped_linear(x, w1, offsets), grouped_linear(x, w3, offsets)
    act = swiglu(gate, up)
    down = grouped_linear(act, w2, offsets)
    out = h.float().index_add(0, rows, gates[:, None] * down.float()).to(torch.bfloat16)
    q, s = mxfp8.mxfp8_quantize(dense)
    bias = torch.linspace(-1, 1, HIDDEN, device=gpu)
    top = linear.mxfp8_linear(out, q, s, bias=bias, activation="gelu_tanh", residual=out)
    hq, hs = mxfp8.mxfp8_quantize(head)
    losses = linear_cross_entropy(top, hq, target, hs, reduction="none")

    values, head_values = mxfp8.mxfp8_dequantize(q, s).double(), mxfp8.mxfp8_dequantize(hq, hs).double()
    check_grouped(gate, x, w1, offsets)
    check_grouped(up, x, w3, offsets)
    check_grouped(down, act, w2, offsets)
    check_linear(top, out, values, bias, "gelu_tanh", out, torch.bfloat16)
    want, tol, _, _ = formula(top, head_values, target)
    near(losses, want, tol)

    # the whole layer
    cd = []
    starts = offsets.tolist()
    for e in range(EXPERTS):
        xe = Carried(x[starts[e]:starts[e + 1]].double(), 0.0 * x[starts[e]:starts[e + 1]].double())
        g, u = xe.times(w1[e], HIDDEN).rounded(), xe.times(w3[e], HIDDEN).rounded()
        silu = activate(g.value, "silu")
        serr = 1.1 * g.err + 16 * U24 * (silu.abs() + g.err)  # |silu'| < 1.1
        a = Carried(silu * u.value, silu.abs() * u.err + serr * (u.value.abs() + u.err)).rounded()
        d = a.times(w2[e], INTER).rounded()
        cd.append((d.value, d.err))
    value, err = torch.cat([v for v, _ in cd]), torch.cat([e for _, e in cd])
    gd = gates.double()[:, None]
    value = h.double().index_add(0, rows, gd * value)
    size = h.double().abs().index_add(0, rows, gd * torch.cat([v.abs() + e for v, e in cd]))
    err = torch.zeros_like(value).index_add(0, rows, gd * err) + 2 * TOPK * U24 * size
    o = Carried(value, err).rounded()
    z = o.times(values, HIDDEN)
    zv = z.value + bias.double()
    act_v = activate(zv, "gelu_tanh")
    t = Carried(act_v + o.value, 1.13 * (z.err + U24 * (zv.abs() + z.err)) + 20 * U24 * (zv.abs() + z.err) + o.err +
                U24 * (act_v + o.value).abs()).rounded()
    lz = t.times(head_values, HIDDEN)
    counted = target != -100
    column = target.clamp(min=0)[:, None]
    whole = (torch.logsumexp(lz.value, 1) - lz.value.gather(1, column)[:, 0]) * counted
    near(losses, whole, 2 * lz.err.amax(1) + tol)

    # calibration of the down product from its own rows
    hess, denom = candidate_hessian.expert_hessians_from_rows(act, offsets, gates, square_weights=True)
    for e in range(EXPERTS):
        a, g2 = act[starts[e]:starts[e + 1]].double(), gates[starts[e]:starts[e + 1]].double() ** 2
        if len(g2):
            exact = a.T @ (g2[:, None] * a)
            size = a.abs().T @ (g2[:, None] * a.abs())
            got = hess[e].double() * denom[e].double()
            # each operand may be weighted and rounded to bf16 once; fp32 sums
            assert ((got - exact).abs() <= (2 * U8 + (len(g2) + 16) * U24) * size).all()


def test_training(gpu):
    """Gradients of the experts, the head and the layer's input, each stage against its formula."""
    h, logits, target, experts, head, _ = model(gpu)
    gates, rows, offsets = route(logits, gpu)
    starts = offsets.tolist()
    h = h.requires_grad_()
    w1, w3, w2 = (w.requires_grad_() for w in experts)
    head = head.requires_grad_()
    x = h[rows]
    gate, up = grouped_linear(x, w1, offsets), grouped_linear(x, w3, offsets)
    act = (torch.nn.functional.silu(gate.float()) * up.float()).to(torch.bfloat16)
    down = grouped_linear(act, w2, offsets)
    out = h.float().index_add(0, rows, gates[:, None] * down.float()).to(torch.bfloat16)
    kept = x, gate, up, act, down, out
    for t in kept:
        t.retain_grad()
    loss = linear_cross_entropy(out, head, target)
    loss.backward()
    count = int((target != -100).sum())
    losses, tol, d, dtol = formula(out.detach(), head.detach(), target)
    near(loss.detach()[None], losses.sum()[None] / count, tol.sum()[None] / count + 4 * U24 * (1 + losses.sum() / count))
    d, dtol = d / count, dtol / count + 4 * U24 * d.abs() / count
    check_sum(out.grad, d, dtol, head.detach())
    check_sum(head.grad, d.T, dtol.T, torch.where((target != -100)[:, None], out.detach(), torch.zeros_like(out)))
    for e in range(EXPERTS):
        a, b = starts[e], starts[e + 1]
        for y, rows_in, w in ((down, act, w2), (gate, x, w1), (up, x, w3)):
            close(w.grad[e], y.grad[a:b].T, rows_in.detach()[a:b].T, b - a)
        close(act.grad[a:b], down.grad[a:b], w2.detach()[e].T, HIDDEN)
    # x takes the gradients of both products, added in bf16
    for e in range(EXPERTS):
        a, b = starts[e], starts[e + 1]
        parts = [(y.grad[a:b].double(), w.detach()[e].double()) for y, w in ((gate, w1), (up, w3))]
        terms = [p @ w for p, w in parts]
        each = [INTER * U24 * (p.abs() @ w.abs()) + U8 * t.abs() for (p, w), t in zip(parts, terms)]
        err = sum(e * (1 + U8) for e in each)
        want = sum(terms)
        assert ((x.grad[a:b].double() - want).abs() <= err + U8 * (want.abs() + err)).all()
    assert h.grad.isfinite().all() and h.grad.any()
