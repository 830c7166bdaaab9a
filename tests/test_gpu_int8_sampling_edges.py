"""Calls at the edges of what the int8 products and the sampling allow: smallest
temperatures and logits with both cuts, rows of NaN through every epilogue, and
results that end a batch."""

from __future__ import annotations

import math

import pytest
import torch

from kquant_amd.int8 import int8_quantize
from kquant_amd.linear import int8_linear

from .test_gpu_int8 import DTYPES, check, rows, weights
from .test_gpu_linear_epilogue import KINDS
from .test_gpu_sampling import check as check_sample
from .test_gpu_sampling import rows as logits

pytestmark = pytest.mark.gpu
CUTS = [{"top_k": 30, "top_p": 0.9}, {"top_k": 6000, "top_p": 0.99}, {"top_p": 0.5}, {"top_k": 7, "min_p": 0.2}, {"top_k": 1},
        {"top_k": 5, "top_p": 1e-30}]


@pytest.mark.parametrize("vocab", [900, 9001])
@pytest.mark.parametrize("settings", CUTS, ids=str)
def test_smallest_temperatures(gpu, vocab, settings):
    """Subnormal ones, as numbers and as rows' own: the largest logits alone have weight, equal ones share it."""
    z, u = logits(6, vocab, torch.float32, gpu, 17)
    z[1] = torch.round(z[1])
    z[2] = 1.5
    z[3, ::2] = -math.inf
    z[4] *= 2.0 ** -140
    for t in (5e-324, 1e-300, 1e-45, 1e-38):
        check_sample(z, u, temperature=t, **settings)
    check_sample(z, u, temperature=torch.tensor([1e-45, 1e-40, 3e-39, 1e-38, 1e-42, 1e-37], device=gpu), **settings)


@pytest.mark.parametrize("vocab", [900, 9001])
@pytest.mark.parametrize("settings", [{}, *CUTS], ids=str)
def test_subnormal_logits(gpu, vocab, settings):
    z, u = logits(4, vocab, torch.float32, gpu, 19)
    for scale in (2.0 ** -130, 2.0 ** -146):
        check_sample(z * scale, u, **settings)
        check_sample(z * scale, u, temperature=scale, **settings)


@pytest.mark.parametrize("m,n", [(3, 264), (30, 264), (100, 264), (300, 777), (1030, 4104)])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_rows_of_nan_through_the_epilogue(gpu, m, n, dtype):
    """A row with an infinity or a NaN stays NaN under every activation, and the rows beside it stay as they were."""
    k = 272
    x, (w, sw) = rows(m, k, dtype, gpu, m), weights(n, k, gpu, n)
    bias, residual = torch.randn(n, device=gpu), torch.randn(m, n, device=gpu).to(dtype)
    bad = x.clone()
    bad[0, k - 1], bad[m - 1, 0] = -math.inf, math.nan
    q, sx = int8_quantize(x)
    for kind in KINDS:
        for given in ({"bias": bias}, {"residual": residual}, {"bias": bias, "residual": residual}):
            clean, y = (int8_linear(v, w, sw, activation=kind, **given) for v in (x, bad))
            check(clean, q, sx, w, sw, given.get("bias"), kind, given.get("residual"), dtype)
            assert torch.isnan(y[0]).all() and torch.isnan(y[m - 1]).all() and torch.equal(y[1:m - 1], clean[1:m - 1])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_far_arguments_of_activations(gpu, kind, dtype):
    """Products of magnitudes at which exponentials overflow or end."""
    g = torch.Generator(device=gpu).manual_seed(5)
    for m in (3, 300):
        q = torch.randint(-127, 128, (m, 64), generator=g, device=gpu, dtype=torch.int8)
        w, sw = weights(72, 64, gpu, 3)
        sx = torch.exp2(torch.randint(-20, 100, (m,), generator=g, device=gpu).float())
        y = int8_linear(q, w, sw, source_scale=sx, activation=kind, out_dtype=dtype)
        assert torch.isfinite(y).all()
        check(y, q, sx, w, sw, None, kind, None, dtype)
