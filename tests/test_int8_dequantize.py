"""Dequantized 8-bit integers: one rounding of the exact product of a code (8
bits) and a scale (24 bits), which float64 holds exactly.  Nearest values of 16
bits are found by search among all of them, not by a conversion."""

from __future__ import annotations

import numpy as np
import pytest
import torch

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
def test_gradient_of_the_scale(dtype):
    """The sum of code times upstream value, in both modes."""
    q, s = torch.tensor([[3, -7, 127]], dtype=torch.int8), torch.tensor([0.3], requires_grad=True)
    up = torch.tensor([[1.0, 2.0, -0.5]])
    (int8_dequantize(q, s, dtype=dtype).float() * up).sum().backward()
    assert s.grad.item() == 3 - 14 - 63.5
    _, tangent = torch.func.jvp(lambda v: int8_dequantize(q, v, dtype=dtype), (s.detach(),), (torch.ones(1),))
    assert torch.equal(tangent.float(), q.float())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float64], ids=str)
def test_on_the_gpu(gpu, dtype):
    s = scales()
    q = CODES.expand(s.numel(), 256)
    got = int8_dequantize(q.to(gpu), s.to(gpu), dtype=dtype)
    assert torch.equal(got.cpu(), int8_dequantize(q, s, dtype=dtype))
