"""Products grouped by expert and their gradients against float64 products.

Tolerances: a result is an fp32 sum of exact products, rounded once.  The sum
of L products is within L 2^-24 sum|a b| of the exact one (each addition rounds
by at most half a step of a partial sum, itself at most sum|a b|), the rounding
within eps / 2 of the value; half a step of the smallest subnormal is allowed
besides (fp16)."""

from __future__ import annotations

import pytest
import torch

from kquant_amd import _native as N
from kquant_amd import grouped
from kquant_amd.grouped import grouped_linear

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def close(got, a, b, length):
    """got [m, n] against a [m, l] b [n, l]^T in 64 bits."""
    a, b = a.double(), b.double()
    want = a @ b.T
    bound = a.abs() @ b.abs().T
    tol = length * 2.0 ** -24 * bound + torch.finfo(got.dtype).eps / 2 * (want.abs() + length * 2.0 ** -24 * bound)
    bad = (got.double() - want).abs() > tol + TINY[got.dtype]
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside, first at {bad.nonzero()[0].tolist()}"


def operands(rows, groups, n, k, dtype, gpu, seed=0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    x = torch.randn(rows, k, generator=g, device=gpu).to(dtype)
    w = (torch.randn(groups, n, k, generator=g, device=gpu) * 0.05).to(dtype)
    dy = torch.randn(rows, n, generator=g, device=gpu).to(dtype)
    return x, w, dy


def check(x, w, dy, starts, offsets=None):
    rows, (groups, n, k) = x.shape[0], w.shape
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    if offsets is None:
        offsets = torch.tensor(starts, device=x.device)
    y = grouped_linear(x, w, offsets)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert y.shape == (rows, n) and y.dtype == x.dtype and dx.shape == x.shape and dw.shape == w.shape
    x, w, y = x.detach(), w.detach(), y.detach()
    inside = torch.zeros(rows, dtype=torch.bool, device=x.device)
    for e in range(groups):
        a, b = starts[e], starts[e + 1]
        inside[a:b] = True
        close(y[a:b], x[a:b], w[e], k)
        close(dx[a:b], dy[a:b], w[e].T, n)
        close(dw[e], dy[a:b].T, x[a:b].T, b - a)
    assert not y[~inside].any() and not dx[~inside].any()
    return y, dx, dw


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,k", [(8, 8), (64, 72), (256, 256), (264, 520), (1416, 1032)])
def test_sizes(gpu, dtype, n, k):
    """Row counts on both sides of every row-tile height, empty groups, rows of no group."""
    counts = [0, 1, 31, 32, 33, 0, 64, 65, 127, 128, 129, 256, 257, 0]
    starts = [3]
    for c in counts:
        starts.append(starts[-1] + c)
    x, w, dy = operands(starts[-1] + 5, len(counts), n, k, dtype, gpu)
    check(x, w, dy, starts)


@pytest.mark.parametrize("rows", [1, 2, 17, 300])
def test_one_group(gpu, rows):
    x, w, dy = operands(rows, 1, 520, 328, torch.bfloat16, gpu)
    check(x, w, dy, [0, rows])


def test_many_groups(gpu):
    """More groups than threads, most of them empty or one row."""
    groups = 1000
    starts = [0]
    for e in range(groups):
        starts.append(starts[-1] + (e % 3 == 0) + (40 if e == 777 else 0))
    x, w, dy = operands(starts[-1], groups, 72, 40, torch.bfloat16, gpu)
    check(x, w, dy, starts)


def test_no_rows_and_all_groups_empty(gpu):
    x, w, dy = operands(0, 3, 24, 16, torch.bfloat16, gpu)
    check(x, w, dy, [0, 0, 0, 0])
    x, w, dy = operands(9, 3, 24, 16, torch.bfloat16, gpu)
    check(x, w, dy, [4, 4, 4, 4])


def test_strided_rows_and_int32_offsets(gpu):
    """x as a column slice of a wider buffer (row stride kept), dy transposed and misaligned (copied)."""
    x, w, _ = operands(100, 4, 48, 64, torch.bfloat16, gpu)
    wide = torch.full((100, 200), float("nan"), dtype=torch.bfloat16, device=gpu)
    wide[:, 8:72] = x
    dy = torch.randn(48, 100, device=gpu).to(torch.bfloat16).T
    starts = [0, 10, 10, 70, 100]
    check(wide[:, 8:72], w, dy, starts, torch.tensor(starts, dtype=torch.int32, device=gpu))
    check(wide[:, 8:72], w, torch.ones(1, 1, dtype=torch.bfloat16, device=gpu).expand(100, 48), starts)


def test_neighbours_stay_apart(gpu):
    """NaN and Inf in the rows behind and between the groups reach no other group's results."""
    n, k = 264, 136
    starts, real = [2, 35, 35, 200], [(2, 35), (35, 200)]
    x, w, dy = operands(260, 3, n, k, torch.bfloat16, gpu)
    clean = check(x, w, dy, starts)
    x2, dy2 = x.clone(), dy.clone()
    for t in (x2, dy2):
        t[:2] = float("nan")
        t[200:] = float("inf")
    w2 = w.clone()
    w2[1] = float("nan")  # the empty group's weight
    got = [t.detach() for t in _all(x2, w2, dy2, torch.tensor(starts, device=gpu))]
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1]) and torch.equal(got[2], clean[2])
    x2[40, 7] = float("nan")  # a row of the last group: its own row of y, and its group's dw column
    got = [t.detach() for t in _all(x2, w2, dy2, torch.tensor(starts, device=gpu))]
    assert got[0][40].isnan().all() and not got[0][2:40].isnan().any() and not got[0][41:200].isnan().any()
    assert not got[2][0].isnan().any() and got[2][2][:, 7].isnan().all() and not got[2][2][:, 8:].isnan().any()


def _all(x, w, dy, offsets):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    y = grouped_linear(x, w, offsets)
    return (y.detach(), *torch.autograd.grad(y, (x, w), dy))


def test_bad_offsets_stay_inside(gpu):
    """Offsets past the rows or negative are clamped: no access outside, the rest as ever."""
    x, w, dy = operands(50, 3, 16, 24, torch.bfloat16, gpu)
    want = _all(x, w, dy, torch.tensor([0, 20, 30, 50], device=gpu))
    got = _all(x, w, dy, torch.tensor([-5, 20, 30, 10 ** 12], device=gpu))
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    for bad in ([50, 20, 0, 10], [-(2 ** 62), 2 ** 62, -3, 7]):
        for t in _all(x, w, dy, torch.tensor(bad, device=gpu)):
            assert t.shape  # runs, and stays inside its buffers
    torch.cuda.synchronize()


def test_gradient_against_differences(gpu):
    """Central differences of a weighted sum of y, in a direction of each leaf.

    y is linear in x and in w: the difference over a step of 1 is exact but for
    the roundings of y, each below eps / 2 |y|, and those of the gradient."""
    x, w, dy = operands(70, 3, 40, 48, torch.float16, gpu)
    offsets = torch.tensor([0, 30, 31, 70], device=gpu)
    _, dx, dw = _all(x, w, dy, offsets)
    g = torch.Generator(device=gpu).manual_seed(5)
    eps = torch.finfo(torch.float16).eps
    for leaf, grad, which in ((x, dx, 0), (w, dw, 1)):
        step = torch.randint(-1, 2, leaf.shape, generator=g, device=gpu).to(leaf.dtype) * 2.0 ** -4
        hi, lo = leaf + step, leaf - step
        ys = [grouped_linear(*((t, w) if which == 0 else (x, t)), offsets).double() for t in (hi, lo)]
        moved = (hi.double() - lo.double())
        got = ((ys[0] - ys[1]) * dy.double()).sum()
        want = (moved * grad.double()).sum()
        tol = eps / 2 * ((ys[0].abs() + ys[1].abs()) * dy.double().abs()).sum() + eps * (moved.abs() * grad.double().abs()).sum()
        assert (got - want).abs() <= 2 * tol


def test_repeated_and_captured(gpu):
    """Bitwise the same from call to call; a captured forward and backward replays with new offsets and rows."""
    x, w, dy = operands(300, 5, 136, 200, torch.bfloat16, gpu)
    offsets = torch.tensor([0, 10, 150, 150, 290, 300], device=gpu)
    first = _all(x, w, dy, offsets)
    for a, b in zip(first, _all(x, w, dy, offsets)):
        assert torch.equal(a, b)
    sx, sw, so = x.clone().requires_grad_(), w.clone().requires_grad_(), offsets.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = grouped_linear(sx, sw, so)
        torch.autograd.grad(y, (sx, sw), dy)
    torch.cuda.current_stream().wait_stream(side)
    del y  # no eager graph of the leaves lives on
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = grouped_linear(sx, sw, so)
        dx, dw = torch.autograd.grad(y, (sx, sw), dy)
    for i in range(3):
        nx = torch.randn(300, 200, device=gpu).to(torch.bfloat16)
        no = torch.tensor([[0, 10, 150, 150, 290, 300], [5, 5, 5, 100, 260, 299], [0, 0, 0, 0, 0, 300]][i], device=gpu)
        with torch.no_grad():
            sx.copy_(nx)
            so.copy_(no)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((y, dx, dw), _all(nx, w, dy, no)):
            assert torch.equal(a.detach(), b)


def test_streams(gpu):
    """Two calls at once on two streams."""
    x, w, dy = operands(700, 4, 264, 264, torch.bfloat16, gpu)
    o1, o2 = torch.tensor([0, 100, 300, 600, 700], device=gpu), torch.tensor([0, 400, 400, 500, 690], device=gpu)
    want1, want2 = _all(x, w, dy, o1), _all(x, w, dy, o2)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s1):
        got1 = _all(x, w, dy, o1)
    with torch.cuda.stream(s2):
        got2 = _all(x, w, dy, o2)
    torch.cuda.synchronize()
    for a, b in zip(want1 + want2, got1 + got2):
        assert torch.equal(a, b)


def test_cpu_tensors(gpu):
    """Host tensors come back on the host, gradients too."""
    x, w, dy = operands(40, 3, 24, 32, torch.bfloat16, gpu)
    offsets = torch.tensor([0, 11, 30, 40])
    want = _all(x, w, dy, offsets.to(gpu))
    got = _all(x.cpu(), w.cpu(), dy.cpu(), offsets)
    for a, b in zip(want, got):
        assert b.device.type == "cpu" and torch.equal(a.cpu(), b)


def test_large_offsets(gpu):
    """Rows and weights past 2^31 elements."""
    rows, k, n = 300_000, 7200, 16
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device=gpu)
    x[-3:] = torch.randn(3, k, device=gpu).to(torch.bfloat16)
    w = (torch.randn(2, n, k, device=gpu) * 0.05).to(torch.bfloat16)
    y = grouped_linear(x, w, torch.tensor([0, rows - 2, rows], device=gpu))
    close(y[-2:], x[-2:], w[1], k)
    close(y[-3:-2], x[-3:-2], w[0], k)
    del x, y
    groups, n, k = 40, 8192, 7168
    w = torch.zeros(groups, n, k, dtype=torch.bfloat16, device=gpu)
    w[-1] = (torch.randn(n, k, device=gpu) * 0.05).to(torch.bfloat16)
    x = torch.randn(2, k, device=gpu).to(torch.bfloat16)
    starts = [0] * groups + [2]
    y = grouped_linear(x, w, torch.tensor(starts, device=gpu))
    close(y, x, w[-1], k)
    assert grouped.MAX_GROUPS >= groups


def test_more_tiles_than_a_table_holds(gpu):
    """More than 256 output tiles for each compute unit, in all three products."""
    groups, n, k = 4096, 1032, 1032
    rows = 3 * groups
    g = torch.Generator(device=gpu).manual_seed(1)
    sizes = torch.randint(0, 6, (groups,), generator=g, device=gpu)
    sizes[0], sizes[-1] = 2, 1
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device=gpu), sizes.cumsum(0)]).clamp(max=rows)
    starts = offsets.tolist()
    x = torch.randn(rows, k, generator=g, device=gpu).to(torch.bfloat16)
    dy = torch.randn(rows, n, generator=g, device=gpu).to(torch.bfloat16)
    w = torch.randn(groups, n, k, dtype=torch.bfloat16, generator=g, device=gpu).requires_grad_()
    (dw,) = torch.autograd.grad(grouped_linear(x, w, offsets), w, dy)
    for e in [0, 1, 2, 777, 2047, 2048, 3333, groups - 2, groups - 1]:
        a, b = starts[e], starts[e + 1]
        close(dw[e], dy[a:b].T, x[a:b].T, b - a)
    empty = (offsets[1:] == offsets[:-1]).nonzero()[:, 0]
    assert empty.numel() > 0 and not dw[empty].any()
    del w, dw
    n, k = 6152, 64  # 25 column tiles of a row tile for each group
    w = torch.randn(groups, n, k, dtype=torch.bfloat16, generator=g, device=gpu)
    x = torch.randn(rows, k, generator=g, device=gpu).to(torch.bfloat16).requires_grad_()
    dy = torch.randn(rows, n, generator=g, device=gpu).to(torch.bfloat16)
    y = grouped_linear(x, w, offsets)
    (dx,) = torch.autograd.grad(y, x, dy)
    for e in [0, 1, 2, 777, 2047, 2048, 3333, groups - 2, groups - 1]:
        a, b = starts[e], starts[e + 1]
        close(y[a:b].detach(), x[a:b].detach(), w[e], k)
        close(dx[a:b], dy[a:b], w[e].T, n)


def test_differentiable_once(gpu):
    x, w, dy = operands(20, 2, 16, 24, torch.bfloat16, gpu)
    x.requires_grad_()
    (dx,) = torch.autograd.grad(grouped_linear(x, w, torch.tensor([0, 5, 20], device=gpu)), x, dy.requires_grad_(),
                                create_graph=True)
    with pytest.raises(RuntimeError):
        dx.float().sum().backward()


def test_views_of_weights_and_gradients(gpu):
    """Transposed and sliced weights, an expanded upstream gradient."""
    x, w, _ = operands(70, 3, 40, 48, torch.bfloat16, gpu)
    offsets = torch.tensor([0, 30, 30, 65], device=gpu)
    leaf = w.transpose(1, 2).contiguous().requires_grad_()  # [groups, K, N]
    y = grouped_linear(x, leaf.transpose(1, 2), offsets)
    up = torch.ones(1, 1, dtype=torch.bfloat16, device=gpu).expand_as(y)
    (dleaf,) = torch.autograd.grad(y, leaf, up)
    want = _all(x, w, up.contiguous(), offsets)
    assert torch.equal(y.detach(), want[0]) and torch.equal(dleaf, want[2].transpose(1, 2))
    wide = torch.randn(5, 40, 48, device=gpu).to(torch.bfloat16).requires_grad_()
    (dwide,) = torch.autograd.grad(grouped_linear(x, wide[1:4], offsets), wide, up)
    assert not dwide[0].any() and not dwide[4].any() and torch.equal(dwide[1:4], want[2])


def test_capture_beside_a_living_graph(gpu):
    """Refused before anything of it is captured; once that graph is gone, it goes through."""
    x, w, dy = operands(64, 3, 64, 64, torch.bfloat16, gpu)
    offsets = torch.tensor([0, 9, 40, 64], device=gpu)
    want = _all(x, w, dy, offsets)
    sx, sw, flag = x.clone().requires_grad_(), w.clone().requires_grad_(), torch.ones(4, device=gpu)
    eager = grouped_linear(sx, sw, offsets)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        flag.zero_()
        with pytest.raises(RuntimeError, match="still lives"):
            grouped_linear(sx, sw, offsets)
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = grouped_linear(sx, sw, offsets)
        dx, dw = torch.autograd.grad(y, (sx, sw), dy)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((y, dx, dw), want):
            assert torch.equal(a.detach(), b)


def test_rows_far_apart(gpu):
    """Every so many rows of a long buffer, past the row stride that the kernels take, forward and backward."""
    x, w, dy = operands(5, 2, 40, 64, torch.bfloat16, gpu)
    starts = [0, 2, 5]
    want = check(x, w, dy, starts)
    stride = grouped.MAX_STRIDE + 64
    far = torch.zeros(4 * stride + 64, dtype=torch.bfloat16, device=gpu)
    fx, fdy = far.as_strided((5, 64), (stride, 1)), far.clone().as_strided((5, 40), (stride, 1))
    fx.copy_(x)
    fdy.copy_(dy)
    for a, b in zip(_all(fx, w, fdy, torch.tensor(starts, device=gpu)), want):
        assert torch.equal(a, b)


def test_overlapping_groups_of_many_tiles(gpu):
    """Decreasing offsets: 2048 groups of all rows, 2^32 tiles and more by their sizes alone.  All weights are the same,
    so that each row's result is known whichever group wrote it last."""
    rows, groups, n, k = (1 << 29) + (1 << 20), 4096, 8, 8
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device=gpu)
    at = [0, 1, 255, 256, 1 << 20, rows // 2, rows - 257, rows - 1]
    for r in at:
        x[r] = torch.randn(k, device=gpu).to(torch.bfloat16)
    w = torch.randn(1, n, k, device=gpu).to(torch.bfloat16).expand(groups, n, k).contiguous()
    offsets = torch.zeros(groups + 1, dtype=torch.int64, device=gpu)
    offsets[1::2] = rows
    offsets[-1] = rows
    with torch.no_grad():
        y = grouped_linear(x, w, offsets)
    close(torch.stack([y[r] for r in at]), torch.stack([x[r] for r in at]), w[0], k)
    for r in at:
        y[r] = 0
    for r in range(0, rows, 1 << 26):
        assert not y[r:r + (1 << 26)].any()


def test_capture_of_views_beside_a_living_graph(gpu):
    """Weights kept as [groups N, K]: refused while an eager graph lives, captured once it is gone."""
    x, w, dy = operands(64, 3, 64, 64, torch.bfloat16, gpu)
    offsets = torch.tensor([0, 9, 40, 64], device=gpu)
    want = _all(x, w, dy, offsets)
    leaf, flag = w.reshape(192, 64).clone().requires_grad_(), torch.ones(4, device=gpu)
    eager = grouped_linear(x, leaf.view(3, 64, 64), offsets)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        flag.zero_()
        with pytest.raises(RuntimeError, match="still lives"):
            grouped_linear(x, leaf.view(3, 64, 64), offsets)
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = grouped_linear(x, leaf.view(3, 64, 64), offsets)
        (dw,) = torch.autograd.grad(y, leaf, dy)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.detach(), want[0]) and torch.equal(dw.view(3, 64, 64), want[2])


@pytest.mark.parametrize("offsets", [[50, 20, 0, 10], [-(2 ** 62), 2 ** 62, -3, 7], [0, 50, 0, 50], [60, 70, 80, 90],
                                     [-9, -8, -7, -6], [0, 20, 30, 50]], ids=str)
def test_nothing_outside_the_results_is_written(gpu, offsets):
    """Offsets of any values: what lies before, behind and between the rows of each result stays."""
    rows, groups, n, k = 50, 3, 40, 72
    x, w, dy = operands(rows, groups, n, k, torch.bfloat16, gpu)
    at = torch.tensor(offsets, dtype=torch.int64, device=gpu)
    st, code = N.stream(gpu), N.DT_BF16
    ldy, ldx, edge = n + 16, k + 24, 300
    for width, ld, name in ((n, ldy, "kq_grouped_linear"), (k, ldx, "kq_grouped_linear_dx")):
        out = torch.full((rows + 2 * edge, ld), 7.0, dtype=torch.bfloat16, device=gpu)
        source = x if name == "kq_grouped_linear" else dy
        N.call(name, code, N.ptr(source), source.stride(0), rows, N.ptr(at), groups, N.ptr(w), n, k, N.ptr(out[edge:]), ld, st)
        torch.cuda.synchronize()
        assert (out[:edge] == 7).all() and (out[-edge:] == 7).all() and (out[:, width:] == 7).all(), name
    out = torch.full((groups + 2, n, k), 7.0, dtype=torch.bfloat16, device=gpu)
    N.call("kq_grouped_linear_dw", code, N.ptr(dy), n, N.ptr(x), k, rows, N.ptr(at), groups, n, k, N.ptr(out[1:]), st)
    torch.cuda.synchronize()
    assert (out[0] == 7).all() and (out[-1] == 7).all()
