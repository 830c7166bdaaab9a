"""Softmax cross entropy of a vocabulary head against its formulas in float64.

Tolerances.  With B[t][v] = sum_k |h| |w| and E = K 2^-24 B an fp32 logit's
distance from the exact one (exact products, each of at most K additions
rounds by half a step of a partial sum), a loss is within 2 max_v E, plus what
the exponentials add: the argument z - m is rounded twice and exp2 and log2
are within two steps (8 2^-24 (1 + |z - m|) relative to a term, terms of
|z - m| > 30 being nothing next to the sum), sums of at most 400 additions in a
row, and the roundings of lse and the loss themselves.  A gradient's term d is
off by p times that, plus half a bf16 step; its fp32 sum and the result's
rounding come on top."""

from __future__ import annotations

import math

import pytest
import torch

from kquant_amd import _native as N
from kquant_amd import mxfp4, mxfp8
from kquant_amd.io import mxfp4 as mxfp4_io
from kquant_amd.loss import linear_cross_entropy

pytestmark = pytest.mark.gpu
U24, U8 = 2.0 ** -24, 2.0 ** -8


def formula(h, w, target, ignore=-100):
    """losses, their tolerance, and d per unit upstream gradient with its tolerance, in 64 bits."""
    h, w = h.double(), w.double()
    counted = target != ignore
    h = torch.where(counted[:, None], h, torch.zeros_like(h))
    column = torch.where(counted, target, torch.zeros_like(target))[:, None]
    z = h @ w.T
    err = h.shape[1] * U24 * (h.abs() @ w.abs().T).amax(1)
    lse = torch.logsumexp(z, 1)
    losses = torch.where(counted, lse - z.gather(1, column)[:, 0], torch.zeros_like(lse))
    rel = 2 * err + U24 * (8 * 31 + 400)
    tol = rel + U24 * 4 * (lse.abs() + z.abs().amax(1) + losses.abs())
    d = torch.exp(z - lse[:, None])
    dtol = d * (tol + rel)[:, None]
    d.scatter_add_(1, column, -torch.ones_like(column, dtype=d.dtype))
    d, dtol = d * counted[:, None], (dtol + 4 * U24) * counted[:, None]
    return losses, tol, d, dtol


def check_sum(got, d, dtol, other):
    """got bf16 [m, n] against d [m, l] @ other [l, n], d an operand rounded to bf16."""
    other = other.double()
    want = d @ other
    size = d.abs() @ other.abs()
    tol = dtol @ other.abs() * (1 + U8) + U8 * size + d.shape[1] * U24 * size * (1 + U8)
    tol = tol + U8 * (want.abs() + tol) + 2.0 ** -126 * (1 + other.abs().sum(0)[None])
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside, first at {bad.nonzero()[0].tolist()}"


def near(got, want, tol):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} outside, first {bad.nonzero()[0].tolist()}"


def inputs(tokens, vocab, k, gpu, seed=0, ignored=0.2, spread=3.0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    h = torch.randn(tokens, k, generator=g, device=gpu).to(torch.bfloat16)
    w = (torch.randn(vocab, k, generator=g, device=gpu) * (spread / math.sqrt(k))).to(torch.bfloat16)
    target = torch.randint(0, vocab, (tokens,), generator=g, device=gpu)
    target[torch.rand(tokens, generator=g, device=gpu) < ignored] = -100
    return h, w, target


def check(h, w, target, values=None, scale=None, reduction="mean", up=None):
    """values: the head in float64 (w itself by default)."""
    values = w if values is None else values
    losses, tol, d, dtol = formula(h, values, target)
    counted = int((target != -100).sum())
    dense = scale is None
    h = h.detach().requires_grad_()
    w = w.detach().requires_grad_() if dense else w
    got = linear_cross_entropy(h, w, target, scale, reduction=reduction)
    assert got.dtype == torch.float32
    if reduction == "none":
        near(got.detach(), losses, tol)
        up = torch.ones_like(got) if up is None else up
        g = up.double()
    else:
        total, ttol = losses.sum(), tol[target != -100].sum()
        share = 1 / counted if reduction == "mean" else 1.0
        near(got.detach()[None], total[None] * share, (ttol * share + 2 * U24 * (total.abs() * share + 1))[None])
        up = torch.ones_like(got) if up is None else up
        g = (up.double() * share).expand(h.shape[0])
    grads = torch.autograd.grad(got, (h, w) if dense else (h,), up)
    d = d * g[:, None]
    dtol = dtol * g.abs()[:, None] + 4 * U24 * d.abs()
    check_sum(grads[0], d, dtol, values)
    if dense:
        check_sum(grads[1], d.T, dtol.T, torch.where((target != -100)[:, None], h.detach(), torch.zeros_like(h)))
    return (got.detach(), *grads)


@pytest.mark.parametrize("tokens", [1, 5, 32, 33, 64, 65, 300])
@pytest.mark.parametrize("vocab,k", [(1, 8), (7, 72), (256, 64), (257, 264), (1000, 520)])
def test_sizes(gpu, tokens, vocab, k):
    h, w, target = inputs(tokens, vocab, k, gpu, seed=tokens)
    target[-1] = vocab - 1
    check(h, w, target)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("ignored", [0.0, 0.5, 0.97])
def test_reductions(gpu, reduction, ignored):
    h, w, target = inputs(150, 777, 136, gpu, ignored=ignored)
    target[3] = 5
    up = torch.randn(150, device=gpu) if reduction == "none" else torch.tensor(-2.5, device=gpu)
    check(h, w, target, reduction=reduction, up=up)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("tokens,vocab,k", [(1, 100, 64), (5, 1003, 256), (40, 513, 192), (300, 2049, 448)])
def test_block_scaled_heads(gpu, fmt, tokens, vocab, k):
    h, w, target = inputs(tokens, vocab, k, gpu)
    target[0] = vocab - 1
    if fmt == "mxfp8":
        q, s = mxfp8.mxfp8_quantize(w)
        values = mxfp8.mxfp8_dequantize(q, s)
    else:
        q, s = mxfp4.mxfp4_quantize(w)
        values = mxfp4_io.dequant(q, s)
    check(h, q, target, values=values, scale=s)
    if fmt == "mxfp8":
        again = linear_cross_entropy(h, q.view(torch.uint8), target, s)
        assert torch.equal(again, linear_cross_entropy(h, q, target, s))


def test_large_logits(gpu):
    """Logits of some hundreds, a certain target and an impossible one: no overflow, and losses near 0 and far from it."""
    h, w, target = inputs(40, 300, 64, gpu, spread=150.0, ignored=0.0)
    z = h.float() @ w.float().T
    target[:20] = z.argmax(1)[:20]
    target[20:] = z.argmin(1)[20:]
    check(h, w, target, reduction="none")


def test_ignored_rows_reach_nothing(gpu):
    """NaN and Inf in ignored rows change no loss and no gradient; their own gradient is zero."""
    h, w, target = inputs(90, 500, 72, gpu, ignored=0.4)
    target[0] = 3
    want = check(h, w, target)
    bad = h.clone()
    gone = target == -100
    bad[gone] = float("nan")
    bad[gone.nonzero()[0]] = float("inf")
    x, y = bad.requires_grad_(), w.clone().requires_grad_()
    loss = linear_cross_entropy(x, y, target)
    dh, dw = torch.autograd.grad(loss, (x, y))
    assert torch.equal(loss.detach(), want[0]) and torch.equal(dh, want[1]) and torch.equal(dw, want[2])
    assert not dh[gone].any()


def test_nothing_counted(gpu):
    h, w, target = inputs(70, 300, 64, gpu)
    target[:] = 9
    for reduction, value in (("mean", math.nan), ("sum", 0.0)):
        x, y = h.clone().requires_grad_(), w.clone().requires_grad_()
        loss = linear_cross_entropy(x, y, target, ignore_index=9, reduction=reduction)
        assert torch.equal(loss.detach().cpu(), torch.tensor(value)) or (loss.isnan() and math.isnan(value))
        for grad in torch.autograd.grad(loss, (x, y)):
            assert not grad.any()
    x, y = h[:0].clone().requires_grad_(), w.clone().requires_grad_()
    loss = linear_cross_entropy(x, y, target[:0], reduction="none")
    dh, dw = torch.autograd.grad(loss, (x, y), torch.empty(0, device=gpu))
    assert loss.shape == (0,) and dh.shape == (0, 64) and not dw.any()


def test_target_outside_the_vocabulary(gpu):
    for tokens in (6, 80):
        h, w, target = inputs(tokens, 100, 64, gpu, ignored=0.0)
        clean = linear_cross_entropy(h, w, target, reduction="none")
        target[2], target[4] = 100, -1
        losses = linear_cross_entropy(h, w, target, reduction="none")
        assert losses[[2, 4]].isnan().all()
        rest = [i for i in range(tokens) if i not in (2, 4)]
        assert torch.equal(losses[rest], clean[rest])


def test_nonfinite_logits(gpu):
    """A row of NaN makes its own loss NaN; a head row of -inf logits takes no part in the others."""
    for tokens in (6, 80):
        h, w, target = inputs(tokens, 300, 64, gpu, ignored=0.0)
        h[1] = float("nan")
        losses = linear_cross_entropy(h, w, target, reduction="none")
        assert losses[1].isnan() and not losses[2:].isnan().any()
        h, w, target = inputs(tokens, 300, 64, gpu, ignored=0.0)
        h[:, 0], w[:, 0] = 1.0, 0.0
        target[target == 7] = 8
        w[7] = 0.0
        w[7, 0] = float("-inf")
        losses = linear_cross_entropy(h, w, target, reduction="none")
        keep = [v for v in range(300) if v != 7]
        moved = torch.where(target > 7, target - 1, target)
        want, tol, _, _ = formula(h, w[keep], moved)
        near(losses, want, tol)


def test_vocabulary_pieces(gpu):
    """More tokens x vocabulary than one piece of the backward pass holds, and dh summed over pieces."""
    tokens, vocab, k = 9000, 70001, 64
    h, w, target = inputs(tokens, vocab, k, gpu, ignored=0.1)
    x, y = h.clone().requires_grad_(), w.clone().requires_grad_()
    loss = linear_cross_entropy(x, y, target, reduction="sum")
    dh, dw = torch.autograd.grad(loss, (x, y))
    some = torch.arange(0, tokens, 150, device=gpu)
    losses, tol, d, dtol = formula(h[some], w, target[some])
    check_sum(dh[some], d, dtol, w)
    near(linear_cross_entropy(h, w, target, reduction="none")[some], losses, tol)
    del d, dtol
    lse = torch.logsumexp((h.double() @ w.double().T), 1)
    cols = torch.tensor([0, 1, 255, 256, 30000, 59391, 59392, vocab - 1], device=gpu)
    hd = torch.where((target != -100)[:, None], h, torch.zeros_like(h)).double()
    z = h.double() @ w[cols].double().T
    counted = (target != -100)[:, None]
    p = torch.exp(z - lse[:, None]) * counted
    d = p - (target[:, None] == cols[None]).double()
    err = k * U24 * (h.double().abs() @ w.double().abs().T).amax(1)
    dtol = p * (4 * err[:, None] + U24 * 1400) + 4 * U24 * counted
    check_sum(dw[cols], d.T, dtol.T, hd)


def test_shapes_and_strides(gpu):
    """[batch, length, K] states as a slice of a wider buffer, a strided target."""
    h, w, target = inputs(60, 321, 64, gpu)
    wide = torch.full((4, 15, 100), float("nan"), dtype=torch.bfloat16, device=gpu)
    wide[..., 8:72] = h.reshape(4, 15, 64)
    strided = torch.stack([target.reshape(4, 15), torch.zeros(4, 15, dtype=torch.int64, device=gpu)], -1)[..., 0]
    x = wide.requires_grad_()
    losses = linear_cross_entropy(x[..., 8:72], w, strided, reduction="none")
    assert losses.shape == (4, 15)
    (dx,) = torch.autograd.grad(losses.sum(), x)
    want = check(h, w, target, reduction="sum")
    assert torch.equal(losses.reshape(-1).detach(), linear_cross_entropy(h, w, target, reduction="none"))
    assert torch.equal(dx[..., 8:72].reshape(60, 64), want[1]) and not dx[..., :8].any() and not dx[..., 72:].any()


def test_gradient_against_differences(gpu):
    """Central differences along a direction: the truncation is at most a sixth
    of the third derivative, itself at most the cube of the spread of the
    logits' change."""
    g = torch.Generator(device=gpu).manual_seed(3)
    h = (torch.randint(-8, 9, (50, 64), generator=g, device=gpu) / 8).to(torch.bfloat16)
    w = (torch.randint(-8, 9, (200, 64), generator=g, device=gpu) / 16).to(torch.bfloat16)
    target = torch.randint(0, 200, (50,), generator=g, device=gpu)
    x, y = h.clone().requires_grad_(), w.clone().requires_grad_()
    dh, dw = torch.autograd.grad(linear_cross_entropy(x, y, target, reduction="sum"), (x, y))
    for leaf, grad, which in ((h, dh, 0), (w, dw, 1)):
        e = (torch.randint(-1, 2, leaf.shape, generator=g, device=gpu) / 64).to(torch.bfloat16)
        hi, lo = (leaf.float() + e.float()).to(torch.bfloat16), (leaf.float() - e.float()).to(torch.bfloat16)
        assert torch.equal(hi.float() - lo.float(), 2 * e.float())
        at = [linear_cross_entropy(*((t, w) if which == 0 else (h, t)), target, reduction="none").double() for t in (hi, lo)]
        dz = e.double() @ w.double().T if which == 0 else h.double() @ e.double().T
        spread = dz.amax(1) - dz.amin(1)
        _, tol, d, dtol = formula(h, w, target)
        rounded = ((dtol + U8 * d.abs()) * dz.abs()).sum() + U8 * (grad.double().abs() * e.double().abs()).sum()
        got, want = ((at[0] - at[1]) / 2).sum(), (grad.double() * e.double()).sum()
        assert (got - want).abs() <= (spread ** 3 / 6).sum() + 2 * tol.sum() + 2 * rounded


@pytest.mark.parametrize("tokens", [9, 200])
def test_repeated_and_captured(gpu, tokens):
    h, w, target = inputs(tokens, 700, 136, gpu)
    target[0] = 1

    def step(h, w, target):
        loss = linear_cross_entropy(h, w, target)
        return (loss.detach(), *torch.autograd.grad(loss, (h, w)))

    x, y = h.clone().requires_grad_(), w.clone().requires_grad_()
    for a, b in zip(step(x, y, target), step(x, y, target)):
        assert torch.equal(a, b)
    sx, sy, st = h.clone().requires_grad_(), w.clone().requires_grad_(), target.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(sx, sy, st)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(sx, sy, st)
    for seed in range(3):
        nh, _, nt = inputs(tokens, 700, 136, gpu, seed=10 + seed, ignored=0.4 * seed)
        nt[-1] = 0
        with torch.no_grad():
            sx.copy_(nh)
            st.copy_(nt)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step(nh.requires_grad_(), y, nt)):
            assert torch.equal(a, b)


def test_streams(gpu):
    h, w, target = inputs(300, 900, 136, gpu)
    _, _, other = inputs(300, 900, 136, gpu, seed=4)
    want = [linear_cross_entropy(h, w, t, reduction="none") for t in (target, other)]
    torch.cuda.synchronize()
    got = []
    for t in (target, other):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got.append(linear_cross_entropy(h, w, t, reduction="none"))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_cpu_tensors(gpu):
    h, w, target = inputs(50, 200, 64, gpu)
    x, y = h.cpu().requires_grad_(), w.cpu().requires_grad_()
    loss = linear_cross_entropy(x, y, target.cpu())
    grads = torch.autograd.grad(loss, (x, y))
    gx, gy = h.clone().requires_grad_(), w.clone().requires_grad_()
    want = linear_cross_entropy(gx, gy, target)
    assert loss.device.type == "cpu" and torch.equal(loss.detach(), want.detach().cpu())
    for a, b in zip(grads, torch.autograd.grad(want, (gx, gy))):
        assert torch.equal(a, b.cpu())


@pytest.mark.parametrize("tokens,k", [(3, 128), (3, 192), (40, 256), (70, 128)])
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_block_scaled_ignored_captured_and_offset(gpu, fmt, tokens, k):
    """A block-scaled head: NaN in ignored rows, a target outside, scales that begin at odd bytes, and replays."""
    h, w, target = inputs(tokens, 333, k, gpu, ignored=0.3)
    target[0], target[1], target[2] = 332, -100, 333
    q, s = (mxfp8.mxfp8_quantize if fmt == "mxfp8" else mxfp4.mxfp4_quantize)(w)
    odd = torch.zeros(s.numel() + 1, dtype=torch.uint8, device=gpu)
    odd[1:] = s.reshape(-1)
    odd = odd[1:].reshape(s.shape)
    bad = h.clone()
    bad[target == -100] = float("nan")
    want = linear_cross_entropy(h, q, target, s, reduction="none")
    got = linear_cross_entropy(bad, q, target, odd, reduction="none")
    inside = target != 333
    assert got[2].isnan() and torch.equal(got[inside], want[inside]) and not got[target == -100].any()
    still, st = bad.clone(), target.clone()
    linear_cross_entropy(still, q, st, s, reduction="none")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = linear_cross_entropy(still, q, st, s, reduction="none")
    for seed in range(3):
        nh, _, nt = inputs(tokens, 333, k, gpu, seed=seed, ignored=0.3)
        still.copy_(nh)
        st.copy_(nt)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, linear_cross_entropy(nh, q, nt, s, reduction="none"))


@pytest.mark.parametrize("head", ["bf16", "mxfp8", "mxfp4"])
def test_head_past_2_gib(gpu, head):
    tokens, vocab, k = 6, 70_000, 32_768
    if head == "mxfp4":
        vocab = 140_000
    g = torch.Generator(device=gpu).manual_seed(0)
    h = torch.randn(tokens, k, generator=g, device=gpu).to(torch.bfloat16)
    q, s, z, err = [], [], [], []
    for r in range(0, vocab, 10_000):
        w = (torch.randn(10_000, k, generator=g, device=gpu) * (3 / math.sqrt(k))).to(torch.bfloat16)
        if head != "bf16":
            a, b = (mxfp8.mxfp8_quantize if head == "mxfp8" else mxfp4.mxfp4_quantize)(w)
            w = (mxfp8.mxfp8_dequantize if head == "mxfp8" else mxfp4_io.dequant)(a, b)
            q.append(a.view(torch.uint8))
            s.append(b)
        else:
            q.append(w)
        z.append(h.double() @ w.double().T)
        err.append((h.double().abs() @ w.double().abs().T).amax(1))
    q, s = torch.cat(q), torch.cat(s) if s else None
    z, err = torch.cat(z, 1), k * U24 * torch.stack(err).amax(0)
    assert q.numel() * q.element_size() > 1 << 31
    target = torch.tensor([0, vocab - 1, 65_535, 65_536, vocab - 300, -100], device=gpu)
    lse = torch.logsumexp(z, 1)
    want = lse - z.gather(1, target.clamp(min=0)[:, None])[:, 0]
    want[-1] = 0
    tol = 2 * err + U24 * (8 * 31 + 400) + U24 * 4 * (lse.abs() + z.abs().amax(1) + want.abs())
    near(linear_cross_entropy(h, q, target, s, reduction="none"), want, tol)


def test_infinite_upstream_of_no_token(gpu):
    h, w, target = inputs(5, 40, 64, gpu)
    h.requires_grad_()
    w.requires_grad_()
    for reduction in ("sum", "mean"):
        loss = linear_cross_entropy(h, w, torch.full_like(target, -100), reduction=reduction)
        dh, dw = torch.autograd.grad(loss, (h, w), torch.full_like(loss, float("inf")))
        assert not dh.any() and not dw.any()


def test_differentiable_once(gpu):
    h, w, target = inputs(5, 40, 64, gpu)
    target[0] = 1
    h.requires_grad_()
    up = torch.ones((), device=gpu, requires_grad=True)
    (dh,) = torch.autograd.grad(linear_cross_entropy(h, w, target), h, up, create_graph=True)
    with pytest.raises(RuntimeError):
        dh.float().sum().backward()


def test_capture_beside_a_living_graph(gpu):
    h, w, target = inputs(30, 100, 64, gpu)
    target[0] = 1
    x, y, flag = h.clone().requires_grad_(), w.clone().requires_grad_(), torch.ones(4, device=gpu)
    eager = linear_cross_entropy(x, y, target)
    want = torch.autograd.grad(eager, (x, y), retain_graph=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        flag.zero_()
        with pytest.raises(RuntimeError, match="still lives"):
            linear_cross_entropy(x, y, target)
    for a, b in zip(want, torch.autograd.grad(eager, (x, y))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("ignored", [0.0, 0.5, 0.9, 0.999])
def test_slices_follow_the_counted_tokens(gpu, ignored):
    """The hidden gradient's contraction, cut into the more slices the fewer tokens count; one captured graph for all."""
    h, w, target = inputs(1500, 6000, 136, gpu, ignored=ignored)
    target[700] = 5999
    want = check(h, w, target)
    sh, sw, st = h.clone().requires_grad_(), w.clone().requires_grad_(), torch.randint(0, 6000, (1500,), device=gpu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = linear_cross_entropy(sh, sw, st)
        grads = torch.autograd.grad(loss, (sh, sw))
    st.copy_(target)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((loss.detach(), *grads), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("tokens,vocab,k", [(5, 24601, 256), (16, 24601, 1152), (20, 8209, 256), (33, 8209, 384), (64, 8209, 256),
                                            (64, 8209, 192)])
def test_wide_block_scaled_heads_few_tokens(gpu, fmt, tokens, vocab, k):
    """Each cut of the one-pass kernel that wide heads take, with odd vocabularies."""
    h, w, target = inputs(tokens, vocab, k, gpu, ignored=0.2)
    target[0] = vocab - 1
    q, s = (mxfp8.mxfp8_quantize if fmt == "mxfp8" else mxfp4.mxfp4_quantize)(w)
    values = (mxfp8.mxfp8_dequantize if fmt == "mxfp8" else mxfp4_io.dequant)(q, s).double()
    check(h, q, target, values, s, reduction="none")


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_changed_in_place(gpu, reduction):
    """loss /= steps and loss += another one, as with F.cross_entropy's result."""
    h, w, target = inputs(80, 300, 64, gpu)
    x, y = h.clone().requires_grad_(), w.clone().requires_grad_()
    want = linear_cross_entropy(x, y, target, reduction=reduction)
    grads = torch.autograd.grad(want, (x, y), torch.full_like(want, 0.25))
    loss = linear_cross_entropy(x, y, target, reduction=reduction)
    loss /= 4
    assert torch.equal(loss.detach(), want.detach() / 4)
    loss += 1.0
    for a, b in zip(torch.autograd.grad(loss.sum(), (x, y)), grads):
        assert torch.equal(a, b)


def test_pieces_of_many_tokens(gpu):
    """More tokens than a piece of 1024 vocabulary rows has room for: pieces of 768 rows."""
    tokens, vocab, k = (1 << 19) + 9, 1300, 64
    h, w, target = inputs(tokens, vocab, k, gpu, ignored=0.1)
    target[-3:] = torch.tensor([767, 768, vocab - 1], device=gpu)
    x, y = h.clone().requires_grad_(), w.clone().requires_grad_()
    dh, dw = torch.autograd.grad(linear_cross_entropy(x, y, target, reduction="sum"), (x, y))
    some = torch.cat([torch.arange(0, tokens, 5003, device=gpu), torch.arange(tokens - 9, tokens, device=gpu)])
    losses, tol, d, dtol = formula(h[some], w, target[some])
    near(linear_cross_entropy(h, w, target, reduction="none")[some], losses, tol)
    check_sum(dh[some], d, dtol, w)
    _, _, d, dtol = formula(h, w, target)
    check_sum(dw, d.T, dtol.T, torch.where((target != -100)[:, None], h, torch.zeros_like(h)))


def exact_inputs(tokens, vocab, k, fmt, gpu):
    """Block-scaled heads and states whose logits are exact in fp32 in any order of the sums: multiples of 2^-9 below 2^7."""
    g = torch.Generator(device=gpu).manual_seed(tokens)
    h = torch.randint(-1, 2, (tokens, k), generator=g, device=gpu).to(torch.bfloat16)
    steps = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, -0.5, -1.0, -1.5, -2.0, -3.0], device=gpu)
    w = steps[torch.randint(0, 11, (vocab, k), generator=g, device=gpu)]
    w[:, :64] = w[:, :64].abs()  # sums over the vocabulary that do not cancel
    scale = torch.full((vocab, k // 32), 127 - 8, dtype=torch.uint8, device=gpu)
    if fmt == "mxfp8":
        q = w.to(torch.float8_e4m3fn)
    else:
        grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0], device=gpu)
        code = torch.bucketize(w.abs(), grid).to(torch.uint8) | ((w < 0).to(torch.uint8) << 3)
        q = code[:, 0::2] | (code[:, 1::2] << 4)
    values = w.double() / 256
    target = torch.randint(0, vocab, (tokens,), generator=g, device=gpu)
    target[::5] = -100
    return h, q, scale, values, target


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_pieces_of_block_scaled_heads(gpu, fmt):
    """A head expanded in two pieces of 8704 and 8296 rows, forward and backward, targets on both sides of the seam.

    The logits are exact, so that a loss is within what the exponentials and the roundings add (see above, E = 0)."""
    tokens, vocab, k = 70, 17_000, 32_768
    h, q, scale, values, target = exact_inputs(tokens, vocab, k, fmt, gpu)
    target[1:5] = torch.tensor([8703, 8704, vocab - 1, 0], device=gpu)
    size = N.library().kq_linear_cross_entropy_workspace_size
    head = N.FMT_MXFP8_E4M3 if fmt == "mxfp8" else N.FMT_MXFP4_E2M1
    assert size(head, tokens, vocab, k, 0) < vocab * k * 2  # not all of it at once
    counted = target != -100
    z = h.double() @ values.T
    assert z.abs().max() < 128
    lse = torch.logsumexp(z, 1)
    losses = (lse - z.gather(1, target.clamp(min=0)[:, None])[:, 0]) * counted
    rel = U24 * (8 * 31 + 400)
    tol = rel + U24 * 4 * (lse.abs() + z.abs().amax(1) + losses.abs())
    x = h.clone().requires_grad_()
    got = linear_cross_entropy(x, q, target, scale, reduction="none")
    near(got.detach(), losses, tol)
    (dh,) = torch.autograd.grad(got.sum(), x)
    d = torch.exp(z - lse[:, None])
    dtol = d * (tol + rel)[:, None] + 4 * U24
    d.scatter_add_(1, target.clamp(min=0)[:, None], -torch.ones(tokens, 1, dtype=torch.float64, device=gpu))
    check_sum(dh, d * counted[:, None], dtol * counted[:, None], values)
    assert (dh[counted].abs().amax(1) > 0).all() and not dh[~counted].any()


@pytest.mark.parametrize("head", ["bf16", "mxfp8", "mxfp4"])
@pytest.mark.parametrize("batch", [1, 4, 5])
def test_row_strides_of_states(gpu, head, batch):
    """States that stay a slice of a wider buffer (20, 80 and 100 rows, 104 apart), NaN beside them."""
    k, vocab = 64, 321
    h, w, target = inputs(20 * batch, vocab, k, gpu)
    if head == "bf16":
        q, s = w, None
    else:
        q, s = (mxfp8.mxfp8_quantize if head == "mxfp8" else mxfp4.mxfp4_quantize)(w)
    wide = torch.full((batch, 20, 104), float("nan"), dtype=torch.bfloat16, device=gpu)
    wide[..., 8:72] = h.reshape(batch, 20, k)
    view = wide[..., 8:72]
    assert view.reshape(-1, k).data_ptr() == view.data_ptr()
    x, y = view.detach().requires_grad_(), h.clone().requires_grad_()
    got = linear_cross_entropy(x, q, target.reshape(batch, 20), s, reduction="sum")
    want = linear_cross_entropy(y, q, target, s, reduction="sum")
    assert torch.equal(got.detach(), want.detach())
    (dx,), (dy,) = torch.autograd.grad(got, x), torch.autograd.grad(want, y)
    assert torch.equal(dx.reshape(-1, k), dy) and torch.isfinite(dy).all()


@pytest.mark.parametrize("tokens,vocab", [(70, 300), (300, 20_000)])
def test_row_strides_of_gradients(gpu, tokens, vocab):
    """The C entry point with rows of h and dh further apart than K: stored at once, and as a sum of slices; what lies
    between the rows and around them stays."""
    k, ldh, lddh = 136, 152, 168
    h, w, target = inputs(tokens, vocab, k, gpu)
    y = h.clone().requires_grad_()
    loss = linear_cross_entropy(y, w, target, reduction="sum")
    (want,) = torch.autograd.grad(loss, y)
    wide = torch.full((tokens, ldh), float("nan"), dtype=torch.bfloat16, device=gpu)
    wide[:, :k] = h
    out = torch.full((tokens + 2, lddh), 7.0, dtype=torch.bfloat16, device=gpu)
    losses, lse = (torch.empty(tokens, device=gpu) for _ in range(2))
    for backward in (0, 1):
        need = int(N.library().kq_linear_cross_entropy_workspace_size(N.FMT_BF16, tokens, vocab, k, backward))
        ws = torch.empty(need, dtype=torch.uint8, device=gpu)
        if backward:
            N.call("kq_linear_cross_entropy_backward", N.FMT_BF16, N.ptr(wide), ldh, tokens, N.ptr(w), None, vocab, k,
                   N.ptr(target), -100, N.ptr(lse), N.ptr(torch.ones(1, device=gpu)), N.LOSS_SUM, N.ptr(out[1:]), lddh, None,
                   N.ptr(ws), need, N.stream(gpu))
        else:
            N.call("kq_linear_cross_entropy", N.FMT_BF16, N.ptr(wide), ldh, tokens, N.ptr(w), None, vocab, k, N.ptr(target),
                   -100, N.ptr(losses), N.ptr(lse), None, N.ptr(ws), need, N.stream(gpu))
        torch.cuda.synchronize()
    assert torch.equal(losses, linear_cross_entropy(h, w, target, reduction="none"))
    assert torch.equal(out[1:-1, :k], want)
    assert (out[:, k:] == 7).all() and (out[0] == 7).all() and (out[-1] == 7).all()


def test_gradient_of_the_head_alone(gpu):
    """The C entry point with neither dh nor its row stride."""
    tokens, vocab, k = 70, 300, 136
    h, w, target = inputs(tokens, vocab, k, gpu)
    y = w.clone().requires_grad_()
    (want,) = torch.autograd.grad(linear_cross_entropy(h, y, target, reduction="sum"), y)
    lse = torch.logsumexp(h.float() @ w.float().T, 1)
    dw = torch.empty_like(w)
    need = int(N.library().kq_linear_cross_entropy_workspace_size(N.FMT_BF16, tokens, vocab, k, 1))
    ws = torch.empty(need, dtype=torch.uint8, device=gpu)
    N.call("kq_linear_cross_entropy_backward", N.FMT_BF16, N.ptr(h), k, tokens, N.ptr(w), None, vocab, k, N.ptr(target), -100,
           N.ptr(lse), N.ptr(torch.ones(1, device=gpu)), N.LOSS_SUM, None, 0, N.ptr(dw), N.ptr(ws), need, N.stream(gpu))
    torch.cuda.synchronize()
    _, _, d, dtol = formula(h, w, target)
    for got in (dw, want):
        check_sum(got, d.T, dtol.T, torch.where((target != -100)[:, None], h, torch.zeros_like(h)))
