"""8-bit integers: quantized rows, the dense linear and the products grouped by
expert, against their definitions in float64.

Tolerances.  Codes and int32 sums are exact.  A scale is one fp32 product,
rounded once.  A product's sum is rounded to fp32 (2^-24) and multiplied
by two scales (2^-24 each): 3.01 2^-24 of the value.  The epilogue's steps are
those of tests/test_gpu_linear_epilogue.py: a bias addition (2^-24), activations
no steeper than 1.13 and within 16 2^-24 |x| (the exact GELU 0.8e-7 more), the
residual's addition, the result's rounding, and half a step of fp16's smallest
subnormal."""

from __future__ import annotations

import pytest
import torch

from kquant_amd import _native as N
from kquant_amd.grouped import int8_grouped_linear
from kquant_amd.int8 import int8_dequantize, int8_quantize
from kquant_amd.linear import int8_linear

from .test_gpu_linear_epilogue import KINDS, activate

pytestmark = pytest.mark.gpu
U24 = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def codes64(x):
    """(codes, scales) by definition, on the device of x; non-finite rows: 0 and NaN."""
    x = x.double()
    finite = torch.isfinite(x).all(-1)
    top = torch.where(finite, torch.nan_to_num(x).abs().amax(-1), torch.ones((), dtype=torch.float64, device=x.device))
    part = torch.tensor(1.0, dtype=torch.float32) / 127  # the fp32 number nearest to a 127th
    scale = (top * float(part)).float().double().clamp(min=2.0 ** -126)  # (48 bits: exact before its rounding)
    q = torch.round(torch.nan_to_num(x) / scale[..., None])
    q = torch.where(finite[..., None], q, torch.zeros_like(q))
    return q, torch.where(finite, scale, torch.full_like(scale, float("nan")))


def check_codes(q, scale, x):
    want, s = codes64(x)
    assert q.dtype == torch.int8 and scale.dtype == torch.float32 and q.shape == x.shape and scale.shape == x.shape[:-1]
    assert torch.equal(q.double(), want)
    assert torch.equal(torch.isnan(scale), torch.isnan(s))
    fine = ~torch.isnan(s)
    assert torch.equal(scale[fine].double(), s[fine])  # one product, rounded once


def rows(m, k, dtype, gpu, seed=0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    spread = torch.exp(0.5 * torch.randn(k, generator=g, device=gpu))
    return (torch.randn(m, k, generator=g, device=gpu) * spread).to(dtype)


def weights(n, k, gpu, seed=1, lead=()):
    g = torch.Generator(device=gpu).manual_seed(seed)
    w = torch.randint(-128, 128, (*lead, n, k), generator=g, device=gpu, dtype=torch.int8)
    return w, torch.exp(torch.randn(*lead, n, generator=g, device=gpu)) * 1e-3


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("k", [1, 7, 8, 16, 33, 127, 512, 1033, 2048, 2049, 7168, 8200, 40001])
def test_quantize(gpu, dtype, k):
    x = rows(5, k, dtype, gpu, k)
    x[1] = 0
    x[2] *= 1e-3
    check_codes(*int8_quantize(x), x)
    q, s = int8_quantize(x)
    assert torch.equal(int8_dequantize(q, s), q.float() * s[:, None])


def test_quantize_many_rows(gpu):
    for m, k in ((1, 7168), (1000, 96), (4097, 257), (300, 3000)):
        x = rows(m, k, torch.bfloat16, gpu, m)
        check_codes(*int8_quantize(x), x)


def test_quantize_more_rows_than_a_launch(gpu):
    x = torch.randn((1 << 26) + 5, device=gpu, dtype=torch.float16)[:, None]
    q, scale = int8_quantize(x)
    assert torch.equal(q, 127 * torch.sign(x).to(torch.int8))
    assert torch.equal(scale, torch.clamp(x[:, 0].float().abs() * (1.0 / 127.0), min=2.0 ** -126))


def test_quantize_ties_and_borders(gpu):
    """Quotients that are halves, and the fp32 numbers next to them."""
    half = torch.arange(-126, 127, device=gpu).float() + 0.5
    for s in (1.0, 2.0 ** -20, 3.0, 1.0 + 2.0 ** -23, 0.1, 2.0 ** -126 * 1.5):
        scale = torch.tensor(s, device=gpu)
        at = half * scale
        x = torch.cat([(127 * scale).reshape(1), at, torch.nextafter(at, at + 1), torch.nextafter(at, at - 1)])
        check_codes(*int8_quantize(x[None]), x[None])


@pytest.mark.parametrize("k", [40, 5000])
def test_quantize_special_rows(gpu, k):
    x = rows(9, k, torch.float32, gpu, 3)
    x[0, 3] = float("inf")
    x[1, k - 1] = float("nan")
    x[2] = torch.finfo(torch.float32).max * torch.sign(x[2])
    x[3] = 2.0 ** -149  # quotients of 2^-23: codes 0 under the smallest scale
    x[4] = x[4] * 2.0 ** -130
    x[5] = -float("inf")
    x[6] = 0.0
    x[7] = 2.0 ** -120
    check_codes(*int8_quantize(x), x)


def test_quantize_strides(gpu):
    base = rows(40, 400, torch.bfloat16, gpu, 5)
    for x in (base[:, 3:300], base[::2, :256], base.T, base[:, 8:264], base[7], base.reshape(4, 10, 400),
              base[:1].expand(6, 400), base[:, ::2], base[:0]):
        check_codes(*int8_quantize(x), x)


def check(got, q, sx, w, sw, bias, kind, residual, dtype):
    z = (q.double() @ w.double().T) * sx.double()[:, None] * sw.double()
    err = 3.01 * U24 * z.abs() + 2.0 ** -149
    if bias is not None:
        z = z + bias.double()
        err = err + U24 * (z.abs() + err)
    want = activate(z, kind)
    err = 1.13 * err + (16 * U24 + (0.8e-7 if kind == "gelu" else 0)) * (z.abs() + err) if kind else err
    if residual is not None:
        want = want + residual.double()
        err = err + U24 * (want.abs() + err)
    tol = err + torch.finfo(dtype).eps / 2 * (want.abs() + err) + TINY[dtype]
    assert got.dtype == dtype and got.shape == want.shape
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside, first at {bad.nonzero()[0].tolist()}"


# fused few rows (one and three weight blocks, and past the size that is fused), few rows (one to four blocks), the
# same with 32 and 64 rows, slices of k, tiles of every height, each ragged
SHAPES = [(1, 24600, 144), (2, 24577, 400), (4, 129, 8192), (2, 129, 8208), (3, 40100, 3056), (6, 12300, 80), (13, 41000, 80),
          (7, 41000, 48), (1187, 74, 4192), (83, 70, 4096), (300, 384, 7168), (65, 24, 1040), (520, 8, 16384 + 48), (20, 8200, 144), (50, 8200, 144), (1, 264, 256), (3, 77, 144), (4, 129, 7168), (5, 129, 512), (16, 1000, 208), (17, 264, 192), (33, 129, 512),
          (64, 40, 1040), (65, 264, 128), (100, 520, 2048), (130, 1033, 16), (300, 777, 192), (257, 300, 64),
          (700, 512, 272), (4100, 4104, 256)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_linear(gpu, shape, dtype):
    m, n, k = shape
    x, (w, sw) = rows(m, k, dtype, gpu, m), weights(n, k, gpu, n)
    q, sx = int8_quantize(x)
    y = int8_linear(x, w, sw)
    check(y, q, sx, w, sw, None, None, None, dtype)
    # the rows quantized before give the same bits
    assert torch.equal(int8_linear(q, w, sw, source_scale=sx, out_dtype=dtype), y)
    assert torch.equal(int8_linear(x, w, sw), y)


@pytest.mark.parametrize("shape", [(1, 264, 256), (4, 129, 144), (16, 264, 256), (40, 77, 400), (300, 776, 192), (300, 777, 192),
                                   (131, 1024, 128), (100, 72, 2064)], ids=str)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_epilogue(gpu, shape, kind, dtype):
    m, n, k = shape
    x, (w, sw) = rows(m, k, dtype, gpu, m), weights(n, k, gpu, n)
    g = torch.Generator(device=gpu).manual_seed(9)
    bias = torch.randn(n, generator=g, device=gpu)
    residual = torch.randn(m, n, generator=g, device=gpu).to(dtype)
    q, sx = int8_quantize(x)
    y = int8_linear(x, w, sw, bias=bias, activation=kind, residual=residual)
    check(y, q, sx, w, sw, bias, kind, residual, dtype)
    bias = bias.to(torch.bfloat16)
    check(int8_linear(x, w, sw, bias=bias, activation=kind), q, sx, w, sw, bias, kind, None, dtype)
    check(int8_linear(x, w, sw, residual=residual), q, sx, w, sw, None, None, residual, dtype)


def test_linear_types(gpu):
    """Every result type of codes and of rows; scales with a trailing one; leading dimensions."""
    x, (w, sw) = rows(12, 96, torch.bfloat16, gpu), weights(40, 96, gpu)
    q, sx = int8_quantize(x)
    for out in DTYPES:
        check(int8_linear(q, w, sw[:, None], source_scale=sx[:, None], out_dtype=out), q, sx, w, sw, None, None, None, out)
        check(int8_linear(x, w, sw, out_dtype=out), q, sx, w, sw, None, None, None, out)
    assert int8_linear(q, w, sw, source_scale=sx).dtype == torch.bfloat16
    y = int8_linear(x.reshape(2, 3, 2, 96), w, sw)
    assert y.shape == (2, 3, 2, 40) and torch.equal(y.reshape(12, 40), int8_linear(x, w, sw))
    assert int8_linear(x[0], w, sw).shape == (40,)
    assert int8_linear(x[:0], w, sw).shape == (0, 40) and int8_linear(x, w[:0], sw[:0]).shape == (12, 0)
    assert torch.equal(int8_linear(x.cpu(), w.cpu(), sw.cpu()), int8_linear(x, w, sw).cpu())


@pytest.mark.parametrize("k", [1, 15, 17, 1033])
@pytest.mark.parametrize("m", [2, 30, 100])
def test_linear_odd_k(gpu, m, k):
    x, (w, sw) = rows(m, k, torch.float16, gpu), weights(24, k, gpu)
    q, sx = int8_quantize(x)
    check(int8_linear(x, w, sw), q, sx, w, sw, None, None, None, torch.float16)
    assert torch.equal(int8_linear(q, w, sw, source_scale=sx, out_dtype=torch.float16), int8_linear(x, w, sw))


def test_linear_largest_sums(gpu):
    """The largest K with the largest products: -128 x -128 everywhere is 2^31 - 2^18."""
    k = (1 << 17) - 16
    for m in (1, 100):
        q = torch.full((m, k), -128, dtype=torch.int8, device=gpu)
        w = torch.full((20, k), -128, dtype=torch.int8, device=gpu)
        one = torch.ones(m, device=gpu)
        y = int8_linear(q, w, torch.ones(20, device=gpu), source_scale=one, out_dtype=torch.float32)
        assert (y == float(k * 16384)).all()


@pytest.mark.parametrize("m", [3, 12, 100, 300])
def test_linear_special_rows(gpu, m):
    """A row with an infinity or NaN gives a row of NaN and touches no other; a row of zeros gives the bias."""
    x, (w, sw) = rows(m, 256, torch.bfloat16, gpu), weights(64, 256, gpu)
    clean = int8_linear(x, w, sw)
    bad = x.clone()
    bad[0, 5], bad[m - 1, 255] = float("inf"), float("nan")
    y = int8_linear(bad, w, sw)
    assert torch.isnan(y[0]).all() and torch.isnan(y[m - 1]).all() and torch.equal(y[1:m - 1], clean[1:m - 1])
    x[1] = 0
    bias = torch.arange(64, device=gpu).float()
    assert torch.equal(int8_linear(x, w, sw, bias=bias)[1].float(), bias)


@pytest.mark.parametrize("m", [2, 20, 300])
def test_linear_strides(gpu, m):
    base, (w, sw) = rows(m, 700, torch.bfloat16, gpu), weights(72, 320, gpu)
    wide = torch.zeros(m, 100, dtype=torch.bfloat16, device=gpu)
    for x in (base[:, :320], base[:, 1:321], base[:, 8:328], base[:, :640:2]):
        want = int8_linear(x.contiguous(), w, sw, residual=wide[:, :72].contiguous())
        assert torch.equal(int8_linear(x, w, sw, residual=wide[:, :72]), want)
        assert torch.equal(int8_linear(x, w, sw, residual=wide[:, 3:75]), want)
    q, sx = int8_quantize(base)
    for cut in (slice(0, 320), slice(1, 321), slice(16, 336)):
        want = int8_linear(q[:, cut].contiguous(), w, sw, source_scale=sx)
        assert torch.equal(int8_linear(q[:, cut], w, sw, source_scale=sx), want)
    assert torch.equal(int8_linear(q[:, :320], w.T.contiguous().T, sw, source_scale=sx), int8_linear(q[:, :320], w, sw, source_scale=sx))


def check_grouped(y, q, sx, w, sw, starts, dtype):
    inside = torch.zeros(q.shape[0], dtype=torch.bool, device=q.device)
    for e in range(w.shape[0]):
        a, b = starts[e], starts[e + 1]
        inside[a:b] = True
        if a < b:
            check(y[a:b], q[a:b], sx[a:b], w[e], sw[e], None, None, None, dtype)
    assert not y[~inside].any()


GROUPS = [([0, 1], 1, 8, 16), ([0, 3, 3, 40], 45, 264, 272), ([5, 5, 6, 70, 200, 333], 340, 520, 1040),
          ([0, 300, 300, 301, 900], 900, 1416, 144), ([0, 0, 0, 0], 5, 64, 32), ([2, 258, 514], 600, 256, 512)]


@pytest.mark.parametrize("case", GROUPS, ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_grouped(gpu, case, dtype):
    starts, m, n, k = case
    x, (w, sw) = rows(m, k, dtype, gpu, m), weights(n, k, gpu, n, (len(starts) - 1,))
    q, sx = int8_quantize(x)
    offsets = torch.tensor(starts, device=gpu)
    y = int8_grouped_linear(x, w, sw, offsets)
    check_grouped(y, q, sx, w, sw, starts, dtype)
    assert torch.equal(int8_grouped_linear(q, w, sw[..., None], offsets.int(), x_scale=sx, out_dtype=dtype), y)


def test_grouped_bounds(gpu):
    """Offsets outside the rows are taken as the nearest; a non-finite row is NaN alone; nothing behind y is written."""
    x, (w, sw) = rows(50, 64, torch.bfloat16, gpu), weights(16, 64, gpu, lead=(3,))
    x[20, 3] = float("nan")
    q, sx = int8_quantize(x)
    y = int8_grouped_linear(x, w, sw, torch.tensor([-9, 10, 30, 1 << 40], device=gpu))
    assert torch.isnan(y[20]).all()
    x[20], y[20] = 0, 0
    q, sx = int8_quantize(x)
    check_grouped(y, q, sx, w, sw, [0, 10, 30, 50], torch.bfloat16)
    assert int8_grouped_linear(x[:0], w, sw, torch.zeros(4, dtype=torch.int64, device=gpu)).shape == (0, 16)


def test_grouped_odd_k(gpu):
    x, (w, sw) = rows(50, 77, torch.bfloat16, gpu), weights(16, 77, gpu, lead=(3,))
    q, sx = int8_quantize(x)
    y = int8_grouped_linear(x, w, sw, torch.tensor([0, 10, 30, 50], device=gpu))
    check_grouped(y, q, sx, w, sw, [0, 10, 30, 50], torch.bfloat16)
    assert torch.equal(y, int8_grouped_linear(q, w, sw, torch.tensor([0, 10, 30, 50], device=gpu), x_scale=sx))


def test_workspace_without_slices(gpu):
    """Room for the codes alone, and for the slices of k too: the same bits; what is behind the workspace stays."""
    m, n, k = 200, 72, 4096
    x, (w, sw) = rows(m, k, torch.bfloat16, gpu), weights(n, k, gpu)
    want = int8_linear(x, w, sw)
    need = int(N.library().kq_int8_linear_workspace_size(N.DT_BF16, m, n, k))
    codes = m * k + (4 * m + 15) // 16 * 16
    assert need > codes
    for size in (codes, need - 4, need):
        ws = torch.full((need + 4096,), 77, dtype=torch.uint8, device=gpu)
        y = torch.full((m + 1, n), 7.0, dtype=torch.bfloat16, device=gpu)
        N.call("kq_int8_linear", N.DT_BF16, N.ptr(x), k, None, N.ptr(w), N.ptr(sw), m, n, k, 0, None, 0, None, n, N.DT_BF16,
               N.ptr(y), n, N.ptr(ws), size, N.stream(x.device))
        assert torch.equal(y[:m], want) and (y[m] == 7).all()
        assert (ws[max(size, codes):] == 77).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m", [3, 40, 100, 300])
def test_rows_are_independent(gpu, m, dtype):
    """A row's bits depend neither on the path that its batch takes nor on the alignment of what it is written to."""
    x, (w, sw) = rows(m, 272, dtype, gpu, m), weights(264, 272, gpu)
    g = torch.Generator(device=gpu).manual_seed(4)
    bias, residual = torch.randn(264, generator=g, device=gpu), torch.randn(m, 264, generator=g, device=gpu).to(dtype)
    for keywords in ({}, {"bias": bias}, {"residual": residual}, *({"bias": bias, "activation": kind, "residual": residual}
                                                                  for kind in KINDS)):
        y = int8_linear(x, w, sw, **keywords)
        one = dict(keywords)
        for r in (0, m - 1):
            if "residual" in one:
                one["residual"] = residual[r:r + 1]
            assert torch.equal(int8_linear(x[r:r + 1], w, sw, **one), y[r:r + 1])
        cut = dict(keywords)
        for name in ("bias", "residual"):
            if name in cut:
                cut[name] = cut[name][..., 1:]
        assert torch.equal(int8_linear(x, w[1:], sw[1:], **cut), y[:, 1:])  # 263 columns: no whole 16-byte pieces


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_signs_of_zeros(gpu, dtype):
    """Rows of zeros with negative channel scales: -0 without a bias or residual, whatever the batch."""
    w, sw = weights(264, 256, gpu)
    for m in (1, 40, 100, 300):
        y = int8_linear(torch.zeros(m, 256, device=gpu, dtype=dtype), w, -sw)
        assert not y.any() and torch.signbit(y).all(), m
        z = int8_linear(torch.zeros(m, 256, device=gpu, dtype=dtype), w, -sw, residual=torch.zeros_like(y))
        assert not z.any() and not torch.signbit(z).any(), m


def test_empty_results(gpu):
    w, sw = weights(0, 256, gpu)
    x = torch.ones(2, 3, 256, device=gpu, dtype=torch.bfloat16)
    y = int8_linear(x, w, sw, residual=torch.zeros(2, 3, 0, device=gpu, dtype=torch.bfloat16))
    assert y.shape == (2, 3, 0)
    w, sw = weights(24, 256, gpu)
    assert int8_linear(x[:, :0], w, sw, activation="relu").shape == (2, 0, 24)
