"""Sampling against its definition, row by row in 64 bits (80 for the sums).

Tokens are compared for equality.  That holds where no border between two tokens
lies nearer to the number drawn than the weights' unit lets it move: each token's
weight is off by at most 2^-46 of the largest, so a border by V 2^-46 of a total
of at least 1, and the numbers are multiples of 2^-24, of which a test's rows draw
a few hundred: that one of them falls into a border's reach has a chance below
1e-5 for the largest vocabulary.  Where borders are hit exactly (equal logits,
numbers that are multiples of 1 / V), weights are all 1 and sums exact on both sides.

Log probabilities: the kernel's are fp64 values rounded once to fp32 (2^-24), of
a total that V units of 2^-46 move: 2^-24 |logprob| + V 2^-46 + 1e-12."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from kquant_amd.sampling import sample_tokens

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def draw(z, u, t, k, p, m):
    """(token, logprob, kept tokens) of one row z of float64 logits."""
    if np.isnan(z).any() or not (z > -np.inf).any():
        return -1, math.nan, 0
    order = np.lexsort((np.arange(z.size), -z))
    if not t > 0:
        return int(order[0]), 0.0, 1
    top = z[order[0]]
    with np.errstate(invalid="ignore"):
        d = np.where(z == top, 0.0, (z - top) / t).astype(np.longdouble)
    w = np.exp(d)
    w[w < 2.0 ** -46] = 0  # the documented floor
    keep = z.size if k <= 0 else min(k, z.size)
    if p < 1:
        upto = np.cumsum(w[order[:keep]])
        before = np.concatenate([[np.longdouble(0)], upto[:-1]])
        keep = max(1, int(np.count_nonzero(before < np.longdouble(p) * upto[-1])))
    kept = order[:keep]
    kept = kept[(w[kept] >= m) | (np.arange(keep) == 0)]
    kept = np.sort(kept)
    upto = np.cumsum(w[kept])
    hit = np.nonzero(upto > np.longdouble(u) * upto[-1])[0] if u < 1 else []
    at = hit[0] if len(hit) else np.nonzero(w[kept])[0][-1]
    return int(kept[at]), float(np.log(w[kept[at]] / upto[-1])), kept.size


def each(value, rows, default):
    return [default if value is None else value] * rows if not isinstance(value, torch.Tensor) else value.tolist()


def check(z, u, **settings):
    tokens, logprobs = sample_tokens(z, u, return_logprobs=True, **settings)
    assert tokens.dtype == torch.int64 and logprobs.dtype == torch.float32
    assert tokens.shape == logprobs.shape == z.shape[:-1]
    assert torch.equal(sample_tokens(z, u, **settings), tokens)
    rows, vocab = z.shape
    host, us = z.double().cpu().numpy(), u.double().tolist()
    t, k = each(settings.get("temperature"), rows, 1.0), each(settings.get("top_k"), rows, 0)
    p, m = each(settings.get("top_p"), rows, 1.0), each(settings.get("min_p"), rows, 0.0)
    kept = []
    for r in range(rows):
        token, logprob, n = draw(host[r], us[r], t[r], k[r], p[r], m[r])
        assert int(tokens[r]) == token, (r, int(tokens[r]), token, us[r])
        got = float(logprobs[r])
        assert math.isnan(got) == math.isnan(logprob)
        if token >= 0:
            assert abs(got - logprob) <= 2.0 ** -24 * abs(logprob) + vocab * 2.0 ** -46 + 1e-12, (r, got, logprob)
        kept.append(n)
    return tokens, kept


def rows(m, vocab, dtype, gpu, seed=0, spread=3.0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    z = torch.randn(m, vocab, generator=g, device=gpu) * spread
    return z.to(dtype), torch.rand(m, generator=g, device=gpu)


SETTINGS = [{}, {"temperature": 0.7}, {"top_k": 20}, {"top_p": 0.9}, {"min_p": 0.05}, {"top_k": 50, "top_p": 0.95},
            {"temperature": 1.5, "top_k": 200, "top_p": 0.5, "min_p": 0.01}, {"temperature": 0.0}]


@pytest.mark.parametrize("vocab", [1, 2, 5, 63, 64, 65, 511, 512, 513, 1000, 2049, 8192, 50257])
@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_settings(gpu, vocab, settings, dtype):
    z, u = rows(3, vocab, dtype, gpu, vocab)
    check(z, u, **settings)


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("vocab,dtype", [(129280, torch.float32), (262144, torch.bfloat16)], ids=str)
def test_wide(gpu, vocab, dtype, settings):
    z, u = rows(2, vocab, dtype, gpu, 1)
    check(z, u, **settings)


@pytest.mark.parametrize("m", [1, 2, 9, 33, 150, 300])
def test_own_settings(gpu, m):
    """Each row its own settings, greedy and unfiltered rows among them."""
    z, u = rows(m, 3001, torch.float32, gpu, m)
    g = torch.Generator(device=gpu).manual_seed(m)
    pick = lambda v: torch.tensor(v, device=gpu)[torch.randint(0, len(v), (m,), generator=g, device=gpu)]  # noqa: E731
    settings = {"temperature": pick([0.0, 0.5, 1.0, 2.0, -1.0]), "top_k": pick([0, 1, 7, 300, 3001, 5000, -3]),
                "top_p": pick([1.0, 0.9, 0.3, 2.0]), "min_p": pick([0.0, 0.02, 0.5])}
    tokens, _ = check(z, u, **settings)
    settings["top_k"] = settings["top_k"].int()
    assert torch.equal(sample_tokens(z, u, **settings), tokens)
    # a row's token does not depend on the batch
    for r in range(0, m, 7):
        own = {name: v[r:r + 1] for name, v in settings.items()}
        assert int(sample_tokens(z[r:r + 1], u[r:r + 1], **own)) == int(tokens[r])


def test_every_token_has_its_share(gpu):
    """A grid of numbers over a small vocabulary: the tokens' shares, in order of index."""
    z = torch.tensor([[0.5, -1.0, 2.0, 2.0, 0.0]], device=gpu).expand(1000, 5)
    u = torch.arange(1000, device=gpu).float() / 1000
    for settings in SETTINGS[:7]:
        tokens, _ = check(z, u, **settings)
        assert (tokens[1:] >= tokens[:-1]).all()


@pytest.mark.parametrize("vocab", [7, 512, 1000, 20000])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_ties(gpu, vocab, dtype):
    """Equal logits: the order is the index's, and each has the same share."""
    z = torch.zeros(64, vocab, dtype=dtype, device=gpu)
    z[:, ::2] = -0.0
    u = torch.arange(64, device=gpu).float() / 64
    for settings in ({}, {"top_k": 3}, {"top_p": 0.5}, {"top_k": vocab // 2, "top_p": 0.25}, {"min_p": 1.0}):
        check(z, u, **settings)
    tokens, kept = check(z, u, top_k=5)
    assert max(kept) == min(5, vocab) and int(tokens.max()) == min(5, vocab) - 1


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
def test_few_values(gpu, settings):
    """Rows of a few values, many of them equal: cuts fall among ties."""
    g = torch.Generator(device=gpu).manual_seed(2)
    z = torch.randint(-4, 4, (12, 30000), generator=g, device=gpu).float() / 2
    z[6:] = z[6:] * 1e-4
    u = torch.rand(12, generator=g, device=gpu)
    check(z, u, **settings)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("settings", SETTINGS, ids=str)
def test_masks(gpu, dtype, settings):
    """Masked logits at -inf and at the type's lowest value, infinities, NaN, and rows with nothing left."""
    z, u = rows(12, 5000, dtype, gpu, 4)
    low = torch.finfo(dtype).min
    z[0, 1:] = -math.inf
    z[1] = -math.inf
    z[2, 17] = math.nan
    z[3] = low
    z[4, :4999] = low
    z[5, 100], z[5, 4000] = math.inf, math.inf
    z[6, ::2] = -math.inf
    z[7], z[7, 3] = -math.inf, math.nan
    z[8, 4999] = math.inf
    z[9, :] = -math.inf
    z[9, 4321] = low
    z[10, 0] = torch.finfo(dtype).max
    tokens, _ = check(z, u, **settings)
    assert tokens[1] == -1 and tokens[2] == -1 and tokens[7] == -1 and tokens[9] == 4321 and tokens[8] == 4999


def test_numbers_outside(gpu):
    z, _ = rows(6, 100, torch.float32, gpu)
    u = torch.tensor([0.0, 1.0, 2.0, -1.0, math.nan, 1 - 2.0 ** -24], device=gpu)
    tokens = sample_tokens(z, u, top_k=10)
    kept = z.topk(10, dim=1).indices
    assert tokens.tolist() == [int(kept[0].min()), int(kept[1].max()), int(kept[2].max()), int(kept[3].min()),
                               int(kept[4].max()), int(kept[5].max())]


@pytest.mark.parametrize("temperature", [1e-30, 1e-6, 0.01, 50.0, 1e6, 1e30])
def test_temperatures(gpu, temperature):
    for dtype in DTYPES:
        z, u = rows(4, 3000, dtype, gpu, 6)
        for settings in ({}, {"top_k": 100}, {"top_p": 0.7}, {"min_p": 0.3}):
            check(z, u, temperature=temperature, **settings)


@pytest.mark.parametrize("scale", [1e-6, 1e-3, 30.0, 1e4, 1e37])
def test_spreads(gpu, scale):
    z, u = rows(4, 9001, torch.float32, gpu, 8, spread=1.0)
    z = (z * scale).clamp(-3e38, 3e38)
    for settings in SETTINGS:
        check(z, u, **settings)


def test_strides_and_shapes(gpu):
    base, u = rows(8, 4100, torch.float32, gpu, 3)
    for z in (base[:, :4000], base[:, 1:4001], base[:, 8:], base[:, ::2], base[::2].repeat_interleave(2, 0), base[:1].expand(8, 4100)):
        assert torch.equal(sample_tokens(z, u, top_p=0.8), sample_tokens(z.contiguous().clone(), u, top_p=0.8))
    z = base.reshape(2, 4, 4100)
    assert torch.equal(sample_tokens(z, u.reshape(2, 4), top_k=9), sample_tokens(base, u, top_k=9).reshape(2, 4))
    assert sample_tokens(base[0], u[0]).shape == ()
    assert sample_tokens(base[:0], u[:0]).shape == (0,)
    assert torch.equal(sample_tokens(base.cpu(), u.cpu(), top_k=9), sample_tokens(base, u, top_k=9).cpu())


@pytest.mark.parametrize("m", [1, 3, 70, 1100])
@pytest.mark.parametrize("vocab", [4097, 5003, 8192])
def test_many_slices(gpu, m, vocab):
    """One slice a row and many; chunks and pieces that end inside the row."""
    for dtype in DTYPES[:2]:
        z, u = rows(m, vocab, dtype, gpu, m)
        for settings in ({"top_k": 40, "top_p": 0.9}, {"temperature": 0.8, "min_p": 0.001}):
            check(z[:70], u[:70], **settings)
            all_rows = sample_tokens(z, u, **settings)
            assert torch.equal(all_rows[-70:], sample_tokens(z[-70:], u[-70:], **settings))


@pytest.mark.parametrize("settings", [{"top_k": 5000}, {"top_p": 0.5}, {"top_k": 20000, "top_p": 0.7}, {"top_k": 9000, "min_p": 0.1}],
                         ids=str)
def test_long_lists(gpu, settings):
    """More equal logits at a cut than a list holds."""
    g = torch.Generator(device=gpu).manual_seed(11)
    z = torch.zeros(6, 40001, device=gpu)
    z[1, ::2] = -1.0
    z[2] = torch.randint(-1, 2, (40001,), generator=g, device=gpu).float()
    z[3, :8000] = -1e-7
    z[4] = -torch.arange(40001, device=gpu) // 4096
    z[5, 30000:] = 9.0
    check(z, torch.rand(6, generator=g, device=gpu), **settings)


def test_cuts_at_every_place(gpu):
    """Every top_k around a list's and a bin's ends, and a row of shares for top_p."""
    z, _ = rows(1, 6000, torch.bfloat16, gpu, 13)
    k = torch.cat([torch.arange(1, 300, device=gpu), torch.arange(5900, 6002, device=gpu)])
    u = torch.rand(k.numel(), generator=torch.Generator(device=gpu).manual_seed(1), device=gpu)
    check(z.expand(k.numel(), 6000), u, top_k=k)
    p = torch.linspace(0.0005, 0.9995, 301, device=gpu)
    check(z.expand(301, 6000), u[:301], top_p=p)
    check(z.expand(301, 6000), u[:301], top_p=p, top_k=k[:301] * 3)


@pytest.mark.parametrize("vocab", [1000, 20000])
@pytest.mark.parametrize("settings", [{}, {"top_k": 50}, {"top_p": 0.9}, {"top_k": 50, "top_p": 0.9}, {"min_p": 0.5}], ids=str)
def test_infinite_temperatures(gpu, vocab, settings):
    """A row's own temperature may be infinite: its finite logits share the draw, or its infinite ones where there are."""
    m = 24
    z, u = rows(m, vocab, torch.float32, gpu, 21)
    z[:, ::3] = -math.inf
    z[::2, 7] = z[::2, vocab - 2 - (vocab - 2) % 3 + 1] = math.inf
    t = torch.full((m,), math.inf, device=gpu)
    tokens, logprobs = sample_tokens(z, u, temperature=t, return_logprobs=True, **settings)
    picked = z.gather(1, tokens[:, None])[:, 0]
    assert torch.equal(picked == math.inf, torch.arange(m, device=gpu) % 2 == 0) and not (picked == -math.inf).any()
    if "top_p" not in settings:  # logarithms of whole numbers, in fp64 rounded once
        odd = min(settings.get("top_k", vocab), int((z[1] > -math.inf).sum()))
        for r in range(m):
            assert abs(logprobs[r].item() + math.log(odd if r % 2 else 2)) <= 2.0 ** -24 * 12 + 1e-12


@pytest.mark.parametrize("settings", [{}, {"top_k": 20, "top_p": 0.9, "min_p": 0.01}], ids=str)
def test_more_rows_than_a_set_of_launches(gpu, settings):
    m, vocab = 8192 + 300, 4100
    z, u = rows(m, vocab, torch.bfloat16, gpu, 31)
    own = {name: torch.full((m,), value, device=gpu, dtype=torch.int32 if name == "top_k" else torch.float32)
           for name, value in (settings | {"temperature": 0.9}).items()}
    own["temperature"][1::2] = 1.3
    tokens, logprobs = sample_tokens(z, u, return_logprobs=True, **own)
    for a, b in ((0, 700), (8000, 8400), (8192, m)):
        part = sample_tokens(z[a:b], u[a:b], return_logprobs=True, **{name: v[a:b] for name, v in own.items()})
        assert torch.equal(part[0], tokens[a:b]) and torch.equal(part[1], logprobs[a:b])
    check(z[8190:8195], u[8190:8195], **{name: v[8190:8195] for name, v in own.items()})
