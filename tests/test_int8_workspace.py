"""The int8 linear's workspace, as the public header states it."""

from __future__ import annotations

import ctypes

import pytest
import torch

from kquant_amd import _native as N

P = ctypes.c_void_p(256)  # never read: validation fails first


def up16(v):
    return (v + 15) // 16 * 16


def size(dtype, m, n, k):
    return int(N.library().kq_int8_linear_workspace_size(dtype, m, n, k))


def codes_room(dtype, m, n, k):
    inside = m <= 4 and k <= 8192 and m * n * k <= 3.5e8
    return 0 if dtype == N.DT_I8 or inside else up16(m * k) + up16(4 * m)


FEW = [(1, 24, 64), (4, 24, 8192), (4, 24, 8208), (1, 24, 16384), (5, 24, 64), (16, 24, 64), (4, 12288, 7168), (1, 48816, 7168),
       (1, 48832, 7168), (3, 16, 16)]


@pytest.mark.parametrize("shape", FEW, ids=str)
@pytest.mark.parametrize("dtype", [N.DT_BF16, N.DT_F16, N.DT_F32, N.DT_I8])
def test_room_of_few_rows(dtype, shape):
    """Up to 16 rows take no slices: exactly the codes' room; a call of rows to be quantized is refused without it."""
    need = codes_room(dtype, *shape)
    assert size(dtype, *shape) == need
    m, n, k = shape
    if need:
        args = [dtype, P, k, None, P, P, m, n, k, 0, None, 0, None, n, N.DT_BF16, P, n]
        for ws, room in ((None, 0), (None, need), (P, need - 1)):
            assert N.library().kq_int8_linear(*args, ws, room, None) == N.KQ_ERR_INVALID
            assert b"workspace needs %d bytes" % need in N.library().kq_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(200, 72, 4096), (83, 70, 4096), (300, 384, 7168)])
def test_slices_are_optional(gpu, m, n, k):
    """Codes may use room for slices too, and need none; rows need their codes' alone."""
    g = torch.Generator(device=gpu).manual_seed(2)
    x = torch.randn(m, k, generator=g, device=gpu).to(torch.bfloat16)
    q = torch.randint(-127, 128, (m, k), generator=g, device=gpu, dtype=torch.int8)
    w = torch.randint(-127, 128, (n, k), generator=g, device=gpu, dtype=torch.int8)
    sx, sw = torch.rand(m, generator=g, device=gpu), torch.rand(n, generator=g, device=gpu)
    for dtype, a, scale in ((N.DT_I8, q, sx), (N.DT_BF16, x, None)):
        need, codes = size(dtype, m, n, k), codes_room(dtype, m, n, k)
        assert need > codes and (need - codes) % (4 * m * n) == 0
        got = []
        for room in (codes, need):
            ws = torch.zeros(max(room, 16), dtype=torch.uint8, device=gpu)
            y = torch.empty(m, n, dtype=torch.float32, device=gpu)
            N.call("kq_int8_linear", dtype, N.ptr(a), k, N.ptr(scale), N.ptr(w), N.ptr(sw), m, n, k, 0, None, 0, None, n,
                   N.DT_F32, N.ptr(y), n, N.ptr(ws) if room else None, room, N.stream(gpu))
            got.append(y)
        assert torch.equal(got[0], got[1])
