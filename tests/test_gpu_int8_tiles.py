"""The int8 products on every kernel that a shape can take: dense tiles of each
height with the epilogue, grouped tiles whose weights stream and whose number
passes the workers', and the few-row grouped kernel with more than one block of
rows in a group.

Results are compared with their definition in float64 within the tolerances of
tests/test_gpu_int8.py, and a row's bits with those of the row alone."""

from __future__ import annotations

import math

import pytest
import torch

from kquant_amd import _native as N
from kquant_amd.grouped import int8_grouped_linear
from kquant_amd.int8 import int8_quantize
from kquant_amd.linear import int8_linear

from .test_gpu_int8 import DTYPES, check, check_grouped, rows, weights
from .test_gpu_linear_epilogue import KINDS

pytestmark = pytest.mark.gpu


# ------------------------------------------------------- dense tiles' heights --

def cut(m, n, k, cus, split=True):
    """The rule by which the library cuts an m x n product over k: (rows of a tile, slices of k)."""
    best, least = None, 0.0
    ntiles, steps = -(-n // 256), -(-k // 128)
    for tm in (32, 64, 96, 128, 256):
        tiles = -(-m // tm) * ntiles
        for slices in (1, 2, 3, 4, 6, 8, 12, 16):
            if slices > 1 and (not split or tiles * slices > cus or steps < 2 * slices):
                break
            each = -(-steps // slices)
            used = -(-steps // each)
            cost = float(-(-tiles * used // cus)) * (88 + tm) * 0.0042 * each
            if used > 1:
                cost += 4.0 + float(m) * n * (4.0 * used + 4.0) / 4e6
            if least == 0.0 or cost <= least:
                least, best = cost, (tm, used)
    return best


def workers(gpu):
    cus = torch.cuda.get_device_properties(gpu).multi_processor_count
    return max(cus // 8 * 8, 8)


def test_the_rule_is_the_librarys(gpu):
    """Its slices show in the workspace of codes."""
    size = N.library().kq_int8_linear_workspace_size
    sliced = 0
    for m in (65, 83, 100, 200, 300, 520, 777, 1187, 2000):
        for n in (24, 74, 264, 777, 2000, 5000):
            for k in (144, 512, 1040, 4096, 7168, 16432):
                _, slices = cut(m, n, k, workers(gpu))
                sliced += slices > 1
                assert int(size(N.DT_I8, m, n, k)) == (4 * slices * m * n if slices > 1 else 0), (m, n, k)
    assert 0 < sliced < 9 * 6 * 6


# (rows, columns, k): a tile's rows, its workers' rounds
DENSE = [((90, 8200, 144), 32, 1), ((250, 12288, 1040), 64, 1), ((898, 8200, 144), 64, 2), ((777, 5000, 7168), 96, 1),
         ((1927, 8200, 144), 96, 3), ((520, 12296, 144), 128, 1), ((1794, 8200, 144), 128, 2), ((1030, 12296, 144), 256, 1),
         ((4100, 8200, 144), 256, 3), ((4099, 12301, 144), 256, 4)]


@pytest.mark.parametrize("shape,height,rounds", DENSE, ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_dense_tiles(gpu, shape, height, rounds, dtype):
    """Bias, every activation and a residual on whole and partial tiles, a worker's first and later ones; rows alone;
    and results that are no whole 16-byte pieces."""
    m, n, k = shape
    assert cut(m, n, k, workers(gpu)) == (height, 1)
    assert workers(gpu) != 256 or -(-(-(-m // height) * -(-n // 256)) // 256) == rounds
    x, (w, sw) = rows(m, k, dtype, gpu, m), weights(n, k, gpu, n)
    g = torch.Generator(device=gpu).manual_seed(6)
    bias, residual = torch.randn(n, generator=g, device=gpu), torch.randn(m, n, generator=g, device=gpu).to(dtype)
    q, sx = int8_quantize(x)
    y = int8_linear(x, w, sw)
    check(y, q, sx, w, sw, None, None, None, dtype)
    for kind in KINDS:
        y = int8_linear(x, w, sw, bias=bias, activation=kind, residual=residual)
        check(y, q, sx, w, sw, bias, kind, residual, dtype)
        for r in (0, m // 2, m - 1):
            alone = int8_linear(x[r:r + 1], w, sw, bias=bias, activation=kind, residual=residual[r:r + 1])
            assert torch.equal(alone, y[r:r + 1])
        less = int8_linear(q, w[1:], sw[1:], source_scale=sx, bias=bias[1:], activation=kind, residual=residual[:, 1:],
                           out_dtype=dtype)
        assert torch.equal(less, y[:, 1:])
    assert torch.equal(int8_linear(x, w, sw, residual=residual)[m - 1:], int8_linear(x[m - 1:], w, sw, residual=residual[m - 1:]))


# ---------------------------------------------------------------- few rows --

@pytest.mark.parametrize("n,k", [(264, 272), (40, 1024), (4104, 144)])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_grouped_few_rows_in_one_group(gpu, dtype, n, k):
    """At most four rows a group on average, and groups of more than the 16 rows of a block: the same bits as on tiles."""
    sizes = [0, 17, 1, 0, 33, 0, 0, 2, 0, 0, 0, 0, 0, 5, 0, 0]
    starts = [2, *(2 + torch.tensor(sizes).cumsum(0)).tolist()]
    m = starts[-1] + 3
    assert max(sizes) > 32 and m <= 4 * len(sizes)
    x, (w, sw) = rows(m, k, dtype, gpu, 3), weights(n, k, gpu, 4, (len(sizes),))
    q, sx = int8_quantize(x)
    offsets = torch.tensor(starts, device=gpu)
    y = int8_grouped_linear(x, w, sw, offsets)
    check_grouped(y, q, sx, w, sw, starts, dtype)
    more = int8_grouped_linear(torch.cat([x, x.new_zeros(4 * len(sizes), k)]), w, sw, offsets)
    assert torch.equal(more[:m], y) and not more[m:].any()
    # all rows in one group
    one = torch.tensor([0] * 8 + [m] * 9, device=gpu)
    check_grouped(int8_grouped_linear(x, w, sw, one), q, sx, w, sw, one.tolist(), dtype)


# ----------------------------------------------------------- grouped tiles --

def starts_of(sizes, before):
    at = [before]
    for v in sizes:
        at.append(at[-1] + v)
    return at


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_grouped_weights_that_stream(gpu, dtype):
    """More weights than the last-level cache holds, groups of every tile height, several tiles a worker."""
    sizes = [0, 1, 40, 70, 90, 96, 97, 120, 130, 600, 32, 33, 64, 65, 128, 129, 256, 257, 0, 300, 5, 513, 17, 80] * 2
    n, k, starts = 2048, 3584, starts_of(sizes, 7)
    assert len(sizes) * n * k > 256 << 20 and sum(-(-v // 256) for v in sizes) * (n // 256) > workers(gpu)
    m = starts[-1] + 11
    x, (w, sw) = rows(m, k, dtype, gpu, 8), weights(n, k, gpu, 9, (len(sizes),))
    q, sx = int8_quantize(x)
    y = int8_grouped_linear(x, w, sw, torch.tensor(starts, device=gpu))
    check_grouped(y, q, sx, w, sw, starts, dtype)
    assert torch.equal(int8_grouped_linear(q, w, sw, torch.tensor(starts, device=gpu), x_scale=sx, out_dtype=dtype), y)
    for e in (1, 3, 9, 17, 47):  # a row has the bits of the linear's
        r = starts[e + 1] - 1
        assert torch.equal(int8_linear(q[r:r + 1], w[e], sw[e], source_scale=sx[r:r + 1], out_dtype=dtype), y[r:r + 1])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_grouped_more_tiles_than_workers(gpu, dtype):
    sizes = [1300, 90, 0, 70, 2600, 256, 900]
    n, k, starts = 4104, 144, starts_of(sizes, 5)
    assert sum(-(-v // 256) for v in sizes) * -(-n // 256) > workers(gpu)
    m = starts[-1]
    x, (w, sw) = rows(m, k, dtype, gpu, 8), weights(n, k, gpu, 9, (len(sizes),))
    q, sx = int8_quantize(x)
    y = int8_grouped_linear(x, w, sw, torch.tensor(starts, device=gpu))
    check_grouped(y, q, sx, w, sw, starts, dtype)


@pytest.mark.parametrize("m", [4_400_001, 17_000_001])
def test_grouped_long_tables(gpu, m):
    """More tiles a worker than one entry of its table has, and than the table has for one worker a CU."""
    starts = [0, 5, m // 3, m // 3, m // 2 + 1, m - 300, m - 2]
    assert m // 256 > 64 * workers(gpu)
    (w, sw), g = weights(8, 16, gpu, 9, (6,)), torch.Generator(device=gpu).manual_seed(5)
    q = torch.randint(-127, 128, (m, 16), generator=g, device=gpu, dtype=torch.int8)
    sx = torch.rand(m, generator=g, device=gpu)
    y = int8_grouped_linear(q, w, sw, torch.tensor(starts, device=gpu), x_scale=sx)
    check_grouped(y, q, sx, w, sw, starts, torch.bfloat16)


# ------------------------------------------------------------------ scales --

@pytest.mark.parametrize("exponent", [-60, 0, 7, 100])
def test_scales_beside_a_127th(gpu, exponent):
    """The scale is one fp32 product with the fp32 number below 1 / 127, (1 - 2^-28) / 127: every mantissa's is within
    1/2 + 1/16 of a step of a 127th of the row's largest magnitude (the nearest number: within 1/2)."""
    bits = (127 + exponent << 23) + torch.arange(1 << 23, device=gpu, dtype=torch.int32)
    x = bits.view(torch.float32)[:, None]
    _, scale = int8_quantize(x)
    s = scale.double()
    step = torch.exp2(torch.floor(torch.log2(s)) - 23)
    off = (127 * s - x[:, 0].double()).abs() / 127  # 127 s has 31 bits
    assert math.isfinite(float(s.sum())) and bool((off <= (0.5 + 0.0625) * step * (1 + 2.0 ** -40)).all())
