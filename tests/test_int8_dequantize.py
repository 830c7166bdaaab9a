"""Dequantized 8-bit integers: one rounding of the exact product of a code (8
bits) and a scale (24 bits), which float64 holds exactly.  Nearest values of 16
bits are found by search among all of them, not by a conversion."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from kquant_amd import _native as N
from kquant_amd.int8 import int8_dequantize

CODES = torch.arange(-128, 128).to(torch.int8)


def scales():
    """Of every size, beside borders of 8 and 11 bits, subnormal products and overflows among them."""
    g = torch.Generator().manual_seed(11)
    some = torch.exp(4 * torch.randn(2000, generator=g))
    # scales whose product with 3, 7, 127 lies just beside (m + 1/2) 2^e of bf16 and fp16
    near = []
    for bits in (8, 11):
        m = torch.arange(1 << (bits - 1), 1 << bits, dtype=torch.float64) + 0.5
        for q in (3, 5, 7, 11, 85, 127):
            near.append((m / q).float())
    edges = torch.tensor([0.0, 2.0 ** -149, 2.0 ** -133, 2.0 ** -126, 1.5 * 2.0 ** -126, 2.0 ** -24 / 7, 2.0 ** -14 / 127, 516.0,
                          2.0 ** 9 * (1 + 2.0 ** -23), 2.6e36, 2.0 ** 121, 3.4e38])
    return torch.cat([some, *near, edges, some * 1e-6, some * 2.0 ** -130])


def nearest16(exact: np.ndarray, dtype) -> np.ndarray:
    """The nearest of all 16-bit values to each |exact|, ties to the even pattern; past the last border infinity."""
    grid = torch.arange(0, 0x7f80 if dtype == torch.bfloat16 else 0x7c00).to(torch.int16).view(dtype).double().numpy()
    grid = np.append(grid, 2 * grid[-1] - grid[-2])  # where infinity stands
    a = np.abs(exact)
    hi = np.clip(np.searchsorted(grid, a), 1, len(grid) - 1)
    lo = hi - 1
    down, up = a - grid[lo], grid[hi] - a  # exact: few bits apart
    pick = np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    value = np.append(grid[:-1], np.inf)[pick]
    return np.copysign(value, exact)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_sixteen_bits_are_rounded_once(dtype):
    s = scales()
    q = CODES.expand(s.numel(), 256)
    got = int8_dequantize(q, s, dtype=dtype)
    assert got.dtype == dtype
    exact = q.double().numpy() * s.double().numpy()[:, None]
    assert np.array_equal(got.double().numpy(), nearest16(exact, dtype))


def test_wider_results():
    s = scales()
    q = CODES.expand(s.numel(), 256)
    exact = q.double() * s.double()[:, None]
    assert torch.equal(int8_dequantize(q, s), exact.float())
    assert torch.equal(int8_dequantize(q, s, dtype=torch.float64), exact)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_special_scales_and_shapes(dtype):
    s = torch.tensor([[float("nan"), float("inf")], [1.0, -0.7]])
    q = torch.tensor([-3, 0, 5], dtype=torch.int8).expand(2, 2, 3)
    y = int8_dequantize(q, s, dtype=dtype)
    assert torch.isnan(y[0, 0]).all() and torch.isnan(y[0, 1, 1]) and torch.isinf(y[0, 1, ::2]).all()
    assert torch.equal(y[1], (q[1].double() * s[1].double()[:, None]).to(dtype))
    assert int8_dequantize(q[:0], s[:0], dtype=dtype).shape == (0, 2, 3)
    assert torch.equal(int8_dequantize(q.transpose(0, 1), s.T, dtype=dtype)[:, 1], y[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_derivatives_and_batches(dtype):
    """The sum of code times upstream value, in both modes."""
    q, s = torch.tensor([[3, -7, 127]], dtype=torch.int8), torch.tensor([0.3], requires_grad=True)
    up = torch.tensor([[1.0, 2.0, -0.5]])
    (int8_dequantize(q, s, dtype=dtype).float() * up).sum().backward()
    assert s.grad.item() == 3 - 14 - 63.5
    _, tangent = torch.func.jvp(lambda v: int8_dequantize(q, v, dtype=dtype), (s.detach(),), (torch.ones(1),))
    assert torch.equal(tangent.float(), q.float())
    q, s = CODES.reshape(2, 128), torch.tensor([0.3, 7.0])
    each = torch.func.vmap(lambda a, b: int8_dequantize(a, b, dtype=dtype))(q, s)
    assert torch.equal(each, int8_dequantize(q, s, dtype=dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float64], ids=str)
def test_on_the_gpu(gpu, dtype):
    s = scales()
    q = CODES.expand(s.numel(), 256)
    got = int8_dequantize(q.to(gpu), s.to(gpu), dtype=dtype)
    assert torch.equal(got.cpu(), int8_dequantize(q, s, dtype=dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("k", [1, 7, 8, 33, 2048, 2049, 7168, 5003])
def test_rows_strides_and_shapes(gpu, dtype, k):
    g = torch.Generator(device=gpu).manual_seed(k)
    base = torch.randint(-128, 128, (11, k + 24), generator=g, device=gpu, dtype=torch.int8)
    s = torch.exp(3 * torch.randn(11, generator=g, device=gpu))
    for q, scale in ((base[:, :k], s), (base[:, 3:k + 3], s), (base[:, 16:k + 16], s), (base[::2, :k], s[::2]),
                     (base[:1, :k].expand(5, k), s[:5]), (base[4, :k], s[4]), (base[:0, :k], s[:0]), (base.T[:11], s),
                     (base[:10, :k].reshape(2, 5, k), s[:10].reshape(5, 2).T)):
        want = int8_dequantize(q.cpu(), scale.cpu(), dtype=dtype)
        assert torch.equal(int8_dequantize(q, scale, dtype=dtype).cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_derivatives_on_the_gpu(gpu, dtype):
    q, s = CODES.reshape(2, 128).to(gpu), torch.tensor([0.3, 7.0], device=gpu, requires_grad=True)
    y = int8_dequantize(q, s, dtype=dtype)
    assert torch.equal(y.detach(), int8_dequantize(q, s.detach(), dtype=dtype))
    (grad,) = torch.autograd.grad(y.float().sum(), s)
    assert torch.equal(grad, q.float().sum(1))
    each = torch.func.vmap(lambda a, b: int8_dequantize(a, b, dtype=dtype))(q, s.detach())
    assert torch.equal(each, y.detach())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("pad", [3, 8])
def test_surroundings(gpu, dtype, pad):
    for m, k in ((5, 264), (3, 2100)):
        q = torch.randint(-128, 128, (m, k), device=gpu, dtype=torch.int8)
        s = torch.rand(m, device=gpu)
        y = torch.full((m + 2, k + pad), 7.0, dtype=dtype, device=gpu)
        N.call("kq_int8_dequantize", N.ptr(q), k, N.ptr(s), m, k, N.DTYPE_CODES[dtype], N.ptr(y[1:]), k + pad, N.stream(gpu))
        assert torch.equal(y[1:m + 1, :k], int8_dequantize(q, s, dtype=dtype))
        assert (y[0] == 7).all() and (y[m + 1] == 7).all() and (y[1:, k:] == 7).all()


@pytest.mark.gpu
def test_more_rows_than_a_launch(gpu):
    m = (1 << 23) + 5
    q = torch.randint(-128, 128, (m, 2), device=gpu, dtype=torch.int8)
    s = torch.rand(m, device=gpu)
    assert torch.equal(int8_dequantize(q, s), q.float() * s[:, None])


def test_c_entry_refusals():
    p, odd = ctypes.c_void_p(256), ctypes.c_void_p(257)  # never read: validation fails first
    ok = [p, 64, p, 10, 64, N.DT_BF16, p, 64, None]
    for at, value, status, text in ((1, 63, N.KQ_ERR_INVALID, b"row strides"), (3, -1, N.KQ_ERR_INVALID, b"rows >= 0"),
                                    (4, 0, N.KQ_ERR_INVALID, b"k >= 1"), (5, N.DT_I8, N.KQ_ERR_INVALID, b"dtype"),
                                    (7, 63, N.KQ_ERR_INVALID, b"row strides"), (0, None, N.KQ_ERR_INVALID, b"null"),
                                    (2, None, N.KQ_ERR_INVALID, b"null"), (6, None, N.KQ_ERR_INVALID, b"null"),
                                    (2, ctypes.c_void_p(258), N.KQ_ERR_INVALID, b"aligned"), (6, odd, N.KQ_ERR_INVALID, b"aligned")):
        args = list(ok)
        args[at] = value
        assert N.library().kq_int8_dequantize(*args) == status and text in N.library().kq_last_error(), (at, value)
