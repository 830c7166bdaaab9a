"""The linear's epilogue (bias, activation, residual) on every path a shape takes.

Tolerance.  The product is an fp32 sum of K exact products (three per k for
fp32 rows): within L 2^-24 sum|a||w| of the exact one.  No activation is
steeper than 1.13.  The sigmoid and the exponential are within a few fp32
steps, their arguments' roundings within 4 steps of an argument whose effect is
damped by the sigmoid's slope: 16 2^-24 |x| covers them; the exact GELU's erf
is within 1.5e-7, halved and times |x|.  Two fp32 additions and the result's
rounding come on top."""

from __future__ import annotations

import math

import pytest
import torch

from kquant_amd import _native as N
from kquant_amd import linear, mxfp4, mxfp8
from kquant_amd.io import mxfp4 as mxfp4_io

pytestmark = pytest.mark.gpu
U24 = 2.0 ** -24
KINDS = [None, "relu", "silu", "gelu", "gelu_tanh"]


def quantized(w, fmt):
    if fmt == "mxfp8":
        q, s = mxfp8.mxfp8_quantize(w)
        return q, s, mxfp8.mxfp8_dequantize(q, s).double(), linear.mxfp8_linear
    q, s = mxfp4.mxfp4_quantize(w)
    return q, s, mxfp4_io.dequant(q, s).double(), linear.mxfp4_linear


def activate(x, kind):
    if kind == "relu":
        return x.clamp(min=0)
    if kind == "silu":
        return x * torch.sigmoid(x)
    if kind == "gelu":
        return x * torch.special.ndtr(x)
    if kind == "gelu_tanh":
        return x * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))
    return x


def check(got, x, values, bias, kind, residual, dtype):
    a = x.double()
    length = x.shape[-1] * (3 if x.dtype == torch.float32 else 1)
    z, err = a @ values.T, length * U24 * (a.abs() @ values.abs().T)
    if bias is not None:
        z = z + bias.double()
        err = err + U24 * (z.abs() + err)
    want = activate(z, kind)
    err = 1.13 * err + (16 * U24 + (0.8e-7 if kind == "gelu" else 0)) * (z.abs() + err) if kind else err
    if residual is not None:
        want = want + residual.double()
        err = err + U24 * (want.abs() + err)
    tol = err + torch.finfo(dtype).eps / 2 * (want.abs() + err)
    assert got.dtype == dtype and got.shape == want.shape
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside, first at {bad.nonzero()[0].tolist()}"


def inputs(m, n, k, dtype, gpu, seed=0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    x = torch.randn(m, k, generator=g, device=gpu).to(dtype)
    w = (torch.randn(n, k, generator=g, device=gpu) * (2 / math.sqrt(k))).to(torch.bfloat16)
    bias = torch.randn(n, generator=g, device=gpu)
    residual = torch.randn(m, n, generator=g, device=gpu).to(dtype)
    return x, w, bias, residual


# the one-pass kernel, the K split, whole direct-load tiles, register-staged tiles (K % 128 != 0), each ragged
SHAPES = [(1, 264, 256), (20, 264, 192), (33, 129, 512), (100, 520, 2048), (300, 777, 192), (257, 300, 64),
          (4100, 4100, 256)]


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("kind", KINDS)
def test_paths(gpu, fmt, shape, kind):
    m, n, k = shape
    x, w, bias, residual = inputs(m, n, k, torch.bfloat16, gpu)
    q, s, values, f = quantized(w, fmt)
    check(f(x, q, s, bias=bias, activation=kind, residual=residual), x, values, bias, kind, residual, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("parts", ["bias", "activation", "residual", "bias16"])
def test_parts(gpu, dtype, m, parts):
    """Each part alone; fp32 rows; a bf16 bias; fp32 results of bf16 rows."""
    x, w, bias, residual = inputs(m, 300, 384, dtype, gpu)
    q, s, values, f = quantized(w, "mxfp8")
    bias = bias.to(torch.bfloat16) if parts == "bias16" else bias if parts == "bias" else None
    kind = "silu" if parts == "activation" else None
    residual = residual.float() if parts == "residual" else None
    check(f(x, q, s, bias=bias, activation=kind, residual=residual, out_dtype=torch.float32), x, values, bias, kind,
          residual, torch.float32)


def test_without_parts_is_the_plain_linear(gpu):
    for m in (1, 70, 300):
        x, w, _, _ = inputs(m, 300, 384, torch.bfloat16, gpu)
        q, s, _, f = quantized(w, "mxfp4")
        zero = torch.zeros(300, device=gpu)
        assert torch.equal(f(x, q, s), f(x, q, s, bias=zero))


def test_saturated_and_nonfinite(gpu):
    """Inf and NaN go through as the functions have them; ReLU keeps NaN."""
    x, w, bias, residual = inputs(6, 64, 64, torch.bfloat16, gpu)
    w[:, 0] = 1.0
    q, s, values, f = quantized(w, "mxfp8")
    x[:, 1:] = 0
    x[:, 0] = torch.tensor([float("inf"), float("-inf"), float("nan"), 100.0, -100.0, 0.0], device=gpu)
    for kind, want in (("relu", [math.inf, 0, math.nan, 100, 0, 0]), ("silu", [math.inf, math.nan, math.nan, 100, 0, 0]),
                       ("gelu", [math.inf, math.nan, math.nan, 100, 0, 0]),
                       ("gelu_tanh", [math.inf, math.nan, math.nan, 100, 0, 0])):
        assert (values[:, 0] == 1).all()
        got = f(x[:, :], q, s, activation=kind)
        # 0 x inf elsewhere in the row cannot occur: the other columns of x are zeros and the weights finite
        for row, v in enumerate(want):
            col = got[row].float()
            assert col.isnan().all() if math.isnan(v) else (col == v).all(), (kind, row, col[:4])


def test_strided_residual_leading_axes_and_host(gpu):
    x, w, bias, _ = inputs(24, 72, 128, torch.bfloat16, gpu)
    q, s, values, f = quantized(w, "mxfp8")
    wide = torch.randn(2, 12, 100, device=gpu).to(torch.bfloat16)
    res = wide[..., 7:79]
    got = f(x.reshape(2, 12, 128), q, s, bias=bias, activation="gelu", residual=res)
    assert got.shape == (2, 12, 72)
    check(got.reshape(24, 72), x, values, bias, "gelu", res.reshape(24, 72), torch.bfloat16)
    turned = torch.randn(72, 24, device=gpu).to(torch.bfloat16).T
    check(f(x, q, s, residual=turned), x, values, None, None, turned, torch.bfloat16)
    host = f(x.cpu(), q.cpu(), s.cpu(), bias=bias.cpu(), activation="gelu", residual=res.reshape(24, 72).cpu())
    assert host.device.type == "cpu" and torch.equal(host, got.reshape(24, 72).cpu())


@pytest.mark.parametrize("m,n,k", [(3, 264, 256), (100, 520, 2048), (300, 777, 192), (4100, 4100, 256)])
def test_residual_in_place(gpu, m, n, k):
    """The C entry point adds to its own output buffer."""
    x, w, bias, residual = inputs(m, n, k, torch.bfloat16, gpu)
    q, s, _, f = quantized(w, "mxfp8")
    want = f(x, q, s, bias=bias, activation="silu", residual=residual)
    out = residual.clone()
    need = int(N.library().kq_mx_linear_workspace_size(m, n, k))
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=gpu)
    N.call("kq_mx_linear_epilogue", N.FMT_MXFP8_E4M3, N.DT_BF16, N.ptr(x), k, N.ptr(q), N.ptr(s), m, n, k, 2,
           N.ptr(bias), N.DT_F32, N.ptr(out), n, N.DT_BF16, N.ptr(out), n, N.ptr(ws), need, N.stream(gpu))
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("m", [1, 100, 300])
def test_captured(gpu, m):
    x, w, bias, residual = inputs(m, 520, 2048, torch.bfloat16, gpu)
    q, s, _, f = quantized(w, "mxfp8")
    f(x, q, s, bias=bias, activation="gelu", residual=residual)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f(x, q, s, bias=bias, activation="gelu", residual=residual)
    for seed in range(3):
        x.copy_(inputs(m, 520, 2048, torch.bfloat16, gpu, seed=seed + 1)[0])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, f(x, q, s, bias=bias, activation="gelu", residual=residual))


@pytest.mark.parametrize("shift,pad", [(0, 0), (0, 1), (0, 2), (0, 4), (1, 0), (2, 0), (4, 8)])
@pytest.mark.parametrize("m,n,k", [(1, 264, 256), (100, 520, 2048), (300, 776, 192), (4100, 4100, 256)])
def test_any_alignment_of_results_and_residuals(gpu, m, n, k, shift, pad):
    """Results and residuals at any element, with any row stride; what lies between the rows stays."""
    x, w, bias, residual = inputs(m, n, k, torch.bfloat16, gpu)
    q, s, _, f = quantized(w, "mxfp8")
    want = f(x, q, s, bias=bias, activation="relu", residual=residual)
    ld = n + pad
    need = int(N.library().kq_mx_linear_workspace_size(m, n, k))
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=gpu)
    for which in ("c", "r"):
        ldc, ldr = (ld, n) if which == "c" else (n, ld)
        out = torch.full((m * ldc + 16,), 7.0, dtype=torch.bfloat16, device=gpu)
        res = torch.full((m * ldr + 16,), 7.0, dtype=torch.bfloat16, device=gpu)
        c0, r0 = (shift, 0) if which == "c" else (0, shift)
        res[r0:r0 + m * ldr].view(m, ldr)[:, :n] = residual
        N.call("kq_mx_linear_epilogue", N.FMT_MXFP8_E4M3, N.DT_BF16, N.ptr(x), k, N.ptr(q), N.ptr(s), m, n, k, 1,
               N.ptr(bias), N.DT_F32, N.ptr(res[r0:]), ldr, N.DT_BF16, N.ptr(out[c0:]), ldc, N.ptr(ws), need,
               N.stream(gpu))
        torch.cuda.synchronize()
        body = out[c0:c0 + m * ldc].view(m, ldc)
        assert torch.equal(body[:, :n], want)
        assert (body[:, n:] == 7).all() and (out[:c0] == 7).all() and (out[c0 + m * ldc:] == 7).all()


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("m,n,k", [(1, 24601, 128), (16, 24601, 256), (17, 8209, 256), (32, 8209, 128), (40, 8209, 256),
                                   (64, 8209, 192)])
def test_wide_outputs_of_few_rows(gpu, fmt, dtype, m, n, k):
    """Several blocks of weight rows a workgroup, so that a thread has more than one sum."""
    x, w, bias, residual = inputs(m, n, k, dtype, gpu)
    q, s, values, f = quantized(w, fmt)
    check(f(x, q, s, bias=bias, activation="silu", residual=residual), x, values, bias, "silu", residual, dtype)


# the one-pass kernel, the K split, register-staged and whole direct-load tiles
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("shape", [(1, 264, 256), (20, 264, 192), (100, 520, 2048), (300, 777, 192), (1030, 4100, 128)], ids=str)
@pytest.mark.parametrize("kind", KINDS)
def test_paths_of_f32_rows(gpu, fmt, shape, kind):
    m, n, k = shape
    x, w, bias, residual = inputs(m, n, k, torch.float32, gpu)
    q, s, values, f = quantized(w, fmt)
    check(f(x, q, s, bias=bias, activation=kind, residual=residual), x, values, bias, kind, residual, torch.float32)


@pytest.mark.parametrize("kind", KINDS)
def test_f32_results_of_bf16_rows(gpu, kind):
    for m, n, k in ((5, 264, 256), (100, 520, 2048), (300, 777, 192), (1030, 4100, 128)):
        x, w, bias, residual = inputs(m, n, k, torch.bfloat16, gpu)
        q, s, values, f = quantized(w, "mxfp4")
        check(f(x, q, s, bias=bias, activation=kind, residual=residual.float(), out_dtype=torch.float32), x, values, bias, kind,
              residual.float(), torch.float32)
