"""The int8 products and the sampling as they are used one after another: a layer
of routed experts in 8-bit integers, the dense layer behind it, the vocabulary
head, and the token.  And as a server calls them: captured and replayed, on
several streams, into buffers whose surroundings stay.

Each stage is compared with its definition on what it was given, within its own
tolerance (tests/test_gpu_int8.py, tests/test_gpu_sampling.py)."""

from __future__ import annotations

import math

import pytest
import torch

from kquant_amd import _native as N
from kquant_amd.grouped import int8_grouped_linear
from kquant_amd.int8 import int8_dequantize, int8_quantize
from kquant_amd.linear import int8_linear
from kquant_amd.sampling import sample_tokens
from kquant_amd.tp_simulator import kimi_topk, swiglu

from .test_gpu_int8 import check as check_linear
from .test_gpu_int8 import check_codes, check_grouped
from .test_gpu_sampling import check as check_sample

pytestmark = pytest.mark.gpu
HIDDEN, INTER, EXPERTS, TOPK, VOCAB = 320, 208, 6, 2, 5003


def model(gpu):
    g = torch.Generator(device=gpu).manual_seed(3)

    def weight(*shape):
        return int8_quantize(torch.randn(*shape, generator=g, device=gpu) / math.sqrt(shape[-1]))

    return {"router": torch.randn(EXPERTS, HIDDEN, generator=g, device=gpu), "w1": weight(EXPERTS, INTER, HIDDEN),
            "w3": weight(EXPERTS, INTER, HIDDEN), "w2": weight(EXPERTS, HIDDEN, INTER), "dense": weight(HIDDEN, HIDDEN),
            "bias": torch.randn(HIDDEN, generator=g, device=gpu), "head": weight(VOCAB, HIDDEN)}


def route(h, w):
    """Gates, tokens and offsets of the (token, expert) pairs in expert order."""
    tokens = h.shape[0]
    gates, ids = kimi_topk(h.float() @ w["router"].T, torch.zeros(EXPERTS, device=h.device), TOPK)
    need = max(int(N.library().kq_route_sort_workspace_size(tokens, TOPK, EXPERTS)), 256)
    ws = torch.empty(need, dtype=torch.uint8, device=h.device)
    offsets = torch.empty(EXPERTS + 1, dtype=torch.int64, device=h.device)
    rows = torch.empty(tokens * TOPK, dtype=torch.int32, device=h.device)
    sorted_gates = torch.empty(tokens * TOPK, dtype=torch.float32, device=h.device)
    N.call("kq_route_sort", N.ptr(ids), tokens, TOPK, EXPERTS, N.ptr(gates), N.ptr(offsets), N.ptr(rows), None,
           N.ptr(sorted_gates), N.ptr(ws), need, N.stream(h.device))
    return sorted_gates, rows.long(), offsets


def step(h, u, w, **settings):
    """One token for each state, and what each stage took and gave."""
    gates, rows, offsets = route(h, w)
    q, s = int8_quantize(h)  # once for both products of the experts
    x, xs = q[rows], s[rows]
    gate = int8_grouped_linear(x, *w["w1"], offsets, x_scale=xs)
    up = int8_grouped_linear(x, *w["w3"], offsets, x_scale=xs)
    act = swiglu(gate, up)
    down = int8_grouped_linear(act, *w["w2"], offsets)
    order = torch.argsort(rows, stable=True)  # (index_add's atomics would add a token's experts in any order)
    parts = (gates[:, None] * down.float())[order].reshape(-1, TOPK, HIDDEN)
    out = (h.float() + parts.sum(1)).to(torch.bfloat16)
    top = int8_linear(out, *w["dense"], bias=w["bias"], activation="silu", residual=out)
    logits = int8_linear(top, *w["head"], out_dtype=torch.float32)
    tokens, logprobs = sample_tokens(logits, u, return_logprobs=True, **settings)
    return locals()


@pytest.mark.parametrize("tokens", [1, 5, 70, 301])
def test_decode_step(gpu, tokens):
    w = model(gpu)
    g = torch.Generator(device=gpu).manual_seed(tokens)
    h = torch.randn(tokens, HIDDEN, generator=g, device=gpu).to(torch.bfloat16)
    u = torch.rand(tokens, generator=g, device=gpu)
    t = step(h, u, w, temperature=0.9, top_k=200, top_p=0.97)
    check_codes(t["q"], t["s"], h)
    starts = t["offsets"].tolist()
    for y, name in ((t["gate"], "w1"), (t["up"], "w3")):
        check_grouped(y, t["x"], t["xs"], *w[name], starts, torch.bfloat16)
    aq, as_ = int8_quantize(t["act"])
    check_codes(aq, as_, t["act"])
    check_grouped(t["down"], aq, as_, *w["w2"], starts, torch.bfloat16)
    oq, os_ = int8_quantize(t["out"])
    check_linear(t["top"], oq, os_, *w["dense"], w["bias"], "silu", t["out"], torch.bfloat16)
    tq, ts = int8_quantize(t["top"])
    check_linear(t["logits"], tq, ts, *w["head"], None, None, None, torch.float32)
    tokens_, _ = check_sample(t["logits"], u, temperature=0.9, top_k=200, top_p=0.97)
    assert torch.equal(tokens_, t["tokens"])
    # a row's result does not depend on the rows beside it, where they take the same route through the kernels' sizes or not
    alone = step(h[:1], u[:1], w, temperature=0.9, top_k=200, top_p=0.97)
    assert torch.equal(alone["logits"], t["logits"][:1]) and torch.equal(alone["tokens"], t["tokens"][:1])


def test_codes_stand_for_their_values(gpu):
    """A product of codes is the product of the values they stand for."""
    w = model(gpu)
    h = torch.randn(40, HIDDEN, device=gpu)
    q, s = int8_quantize(h)
    values, weight = int8_dequantize(q, s).double(), int8_dequantize(*w["dense"]).double()
    want = values @ weight.T
    # both sides: each value rounded once (2^-24), the product's scaling 3 2^-24
    tol = 6 * 2.0 ** -24 * (values.abs() @ weight.abs().T)
    assert ((int8_linear(q, *w["dense"], source_scale=s, out_dtype=torch.float32).double() - want).abs() <= tol).all()


@pytest.mark.parametrize("tokens", [3, 90])
def test_captured_and_replayed(gpu, tokens):
    w = model(gpu)
    g = torch.Generator(device=gpu).manual_seed(1)
    fresh = lambda: (torch.randn(tokens, HIDDEN, generator=g, device=gpu).to(torch.bfloat16),  # noqa: E731
                     torch.rand(tokens, generator=g, device=gpu))
    h, u = fresh()
    t = torch.full((tokens,), 0.8, device=gpu)

    def run():
        logits = int8_linear(int8_linear(h, *w["dense"], bias=w["bias"], activation="gelu", residual=h), *w["head"],
                             out_dtype=torch.float32)
        rows = int8_grouped_linear(h, *w["w1"], offsets)
        return logits, rows, *sample_tokens(logits, u, temperature=t, top_k=50, top_p=0.9, min_p=0.01, return_logprobs=True)

    offsets = torch.linspace(0, tokens, EXPERTS + 1, device=gpu).long()
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = run()
    for i in range(4):
        h2, u2 = fresh()
        h.copy_(h2)
        u.copy_(u2)
        t.fill_(0.5 + 0.3 * i)
        offsets.copy_(torch.sort(torch.randint(0, tokens + 1, (EXPERTS + 1,), generator=g, device=gpu)).values)
        graph.replay()
        got = [v.clone() for v in kept]
        torch.cuda.synchronize()
        for a, b in zip(got, run()):  # the program's own work between the replays
            assert torch.equal(a, b)


def test_two_graphs_and_streams(gpu):
    """Two captured calls, replayed on two streams at once beside eager ones on a third, share no workspace."""
    g = torch.Generator(device=gpu).manual_seed(2)
    weight, scale = int8_quantize(torch.randn(72, 4096, generator=g, device=gpu))
    z = [torch.randn(9, 30011, generator=g, device=gpu) * 3 for _ in range(3)]
    x = [torch.randn(200, 4096, generator=g, device=gpu).to(torch.bfloat16) for _ in range(3)]
    u = torch.rand(9, generator=g, device=gpu)
    call = lambda i: (int8_linear(x[i], weight, scale), sample_tokens(z[i], u, top_k=100, top_p=0.9))  # noqa: E731
    want = [tuple(v.clone() for v in call(i)) for i in range(3)]
    torch.cuda.synchronize()
    graphs, kept = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            kept.append(call(i))
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        with torch.cuda.stream(streams[2]):
            eager = call(2)
        torch.cuda.synchronize()
        for got, right in zip([*kept, eager], want):
            assert all(torch.equal(a, b) for a, b in zip(got, right))


def test_repeated(gpu):
    """Bitwise the same from call to call."""
    w = model(gpu)
    h = torch.randn(130, HIDDEN, device=gpu).to(torch.bfloat16)
    u = torch.rand(130, device=gpu)
    first = step(h, u, w, top_p=0.9)
    for _ in range(5):
        again = step(h, u, w, top_p=0.9)
        for name in ("q", "gate", "down", "top", "logits", "tokens", "logprobs"):
            assert torch.equal(first[name], again[name])


@pytest.mark.parametrize("m,n", [(1, 264), (30, 72), (100, 264), (100, 777), (300, 1032)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_surroundings_of_results(gpu, m, n, dtype):
    """Results in a wider buffer: what lies between the rows, before and behind stays."""
    k = 272
    q = torch.randint(-128, 128, (m, k), device=gpu, dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k), device=gpu, dtype=torch.int8)
    sx, sw = torch.rand(m, device=gpu), torch.rand(n, device=gpu) * 0.01
    want = int8_linear(q, w, sw, source_scale=sx, out_dtype=dtype)
    for pad in (8, 3):
        y = torch.full((m + 2, n + pad), 7.0, dtype=dtype, device=gpu)
        need = int(N.library().kq_int8_linear_workspace_size(N.DT_I8, m, n, k))
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=gpu)
        N.call("kq_int8_linear", N.DT_I8, N.ptr(q), k, N.ptr(sx), N.ptr(w), N.ptr(sw), m, n, k, 0, None, 0, None, n,
               N.DTYPE_CODES[dtype], N.ptr(y[1:]), n + pad, N.ptr(ws), need, N.stream(q.device))
        assert torch.equal(y[1:m + 1, :n], want)
        assert (y[0] == 7).all() and (y[m + 1] == 7).all() and (y[1:m + 1, n:] == 7).all()
        codes = torch.full((m + 2, k + pad), 7, dtype=torch.int8, device=gpu)
        scale = torch.full((m + 2,), 7.0, device=gpu)
        x = torch.randn(m, k, device=gpu).to(dtype)
        N.call("kq_int8_quantize", N.DTYPE_CODES[dtype], N.ptr(x), k, m, k, N.ptr(codes[1:]), k + pad, N.ptr(scale[1:]),
               N.stream(x.device))
        a, b = int8_quantize(x)
        assert torch.equal(codes[1:m + 1, :k], a) and torch.equal(scale[1:m + 1], b)
        assert (codes[0] == 7).all() and (codes[m + 1] == 7).all() and (codes[1:m + 1, k:] == 7).all()
        assert scale[0] == 7 and scale[m + 1] == 7


@pytest.mark.parametrize("rows", [6, 200])
def test_surroundings_of_grouped_results(gpu, rows):
    q = torch.randint(-128, 128, (rows, 64), device=gpu, dtype=torch.int8)
    w = torch.randint(-128, 128, (3, 40, 64), device=gpu, dtype=torch.int8)
    sx, sw = torch.rand(rows, device=gpu), torch.rand(3, 40, device=gpu)
    offsets = torch.tensor([1, rows // 2, rows // 2, rows - 2], device=gpu)
    want = int8_grouped_linear(q, w, sw, offsets, x_scale=sx)
    y = torch.full((rows + 2, 48), 7.0, dtype=torch.bfloat16, device=gpu)
    N.call("kq_int8_grouped_linear", N.ptr(q), 64, N.ptr(sx), rows, N.ptr(offsets), 3, N.ptr(w), N.ptr(sw), 40, 64, N.DT_BF16,
           N.ptr(y[1:]), 48, N.stream(q.device))
    assert torch.equal(y[1:rows + 1, :40], want)
    assert (y[0] == 7).all() and (y[rows + 1] == 7).all() and (y[1:rows + 1, 40:] == 7).all()
    assert not want[0].any() and not want[rows - 2:].any()


def test_surroundings_of_samples(gpu):
    """Logits inside a wider buffer whose other values would win or spoil a row; nothing but the results is written."""
    for vocab, dtype in ((700, torch.float32), (5003, torch.float32), (5004, torch.bfloat16), (70000, torch.float16)):
        wide = torch.full((6, vocab + 24), math.nan, dtype=dtype, device=gpu)
        for first in (0, 3, 8):
            z = wide[1:5, first:first + vocab]
            z.copy_(torch.randn(4, vocab, device=gpu))
            before = wide.clone()
            u = torch.rand(4, device=gpu)
            for settings in ({}, {"top_k": 30, "top_p": 0.9}, {"top_p": 0.5}):
                assert torch.equal(sample_tokens(z, u, **settings), sample_tokens(z.clone(), u, **settings))
            assert torch.equal(torch.isnan(wide), torch.isnan(before)) and torch.equal(wide.nan_to_num(), before.nan_to_num())
            wide.fill_(math.nan)


def test_long_offsets(gpu):
    """Rows and weights past 2^31 bytes."""
    m, n, k = 40, 17000, 131056
    w = torch.randint(-128, 128, (n, k), device=gpu, dtype=torch.int8)  # 2.2 GB
    q = torch.randint(-128, 128, (m, k), device=gpu, dtype=torch.int8)
    one = torch.ones(m, device=gpu)
    last = w[-300:].contiguous()
    for rows in (2, 20, 40):
        y = int8_linear(q[:rows], w, torch.ones(n, device=gpu), source_scale=one[:rows], out_dtype=torch.float32)
        want = (q[:rows].double() @ last.double().T).float()
        assert torch.equal(y[:, -300:], want)
    y = int8_linear(q.repeat(4, 1), w, torch.ones(n, device=gpu), source_scale=one.repeat(4), out_dtype=torch.float32)
    assert torch.equal(y[:m, -300:], (q.double() @ last.double().T).float()) and torch.equal(y[:m], y[-m:])
    del w
    z = torch.randn(20000, 60000, device=gpu, dtype=torch.bfloat16)  # 2.4 GB
    u = torch.rand(20000, device=gpu)
    tokens = sample_tokens(z, u, top_k=40)
    assert torch.equal(tokens[-8:], sample_tokens(z[-8:].clone(), u[-8:], top_k=40))
    q, s = int8_quantize(z)
    check_codes(q[-5:], s[-5:], z[-5:])
