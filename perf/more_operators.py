"""Operator cases: the token path of a model held in 8-bit integers.

Four families, each through the public Python entry points:

  quantize  rows to int8 codes with one fp32 scale a row (``int8.int8_quantize``)
  linear    the dense int8 linear with scales of each token and channel, bias,
            activation and residual (``linear.int8_linear``), from rows in 16 or
            32 bits or from rows that are quantized already
  grouped   the same product grouped by expert (``grouped.int8_grouped_linear``)
  sample    one token for each row of logits from given uniform numbers, with
            temperature, top-k, top-p and min-p (``sampling.sample_tokens``)

``listed()`` gives the fixed cases, ``draw(rng)`` further ones of the same
ranges.  A case is a dict of plain values; ``prepare`` builds the inputs from a
seed, ``run`` makes one pass, in plain torch operations or, where ``own`` is
true, through the library.  ``exact`` states each result in float64.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZEOF = {"bf16": 2, "f16": 2, "f32": 4, "int8": 1}
DEVICE = "cuda"


# ------------------------------------------------------------------ cases --

def listed() -> list[dict]:
    return [
        # a prefill batch's rows, quantized once for the layers that read them
        {"name": "quantize_prefill", "family": "quantize", "dtype": "bf16", "m": 8192, "k": 7168},
        # a small odd batch in fp32
        {"name": "quantize_odd", "family": "quantize", "dtype": "f32", "m": 333, "k": 1033},
        # one decoded token through an ungated MLP layer: latency and weight bytes
        {"name": "linear_decode", "family": "linear", "dtype": "bf16", "out": "bf16", "m": 1, "n": 12288, "k": 7168,
         "bias": True, "activation": "silu", "residual": True},
        # a decode batch's rows, quantized before for two layers, to logits in fp32 under a wide head
        {"name": "linear_head", "family": "linear", "dtype": "int8", "out": "f32", "m": 16, "n": 129280, "k": 7168,
         "bias": False, "activation": "none", "residual": False},
        # a ragged chunk of a prompt in fp16
        {"name": "linear_ragged", "family": "linear", "dtype": "f16", "out": "f16", "m": 777, "n": 5000, "k": 7168,
         "bias": True, "activation": "gelu", "residual": True},
        # a full prefill chunk
        {"name": "linear_prefill", "family": "linear", "dtype": "bf16", "out": "bf16", "m": 4096, "n": 12288, "k": 7168,
         "bias": True, "activation": "gelu_tanh", "residual": True},
        # one decode batch (8 tokens x top-8) through a GPU's share of the experts
        {"name": "grouped_decode", "family": "grouped", "dtype": "bf16", "rows": 64, "pad": 0, "groups": 48, "n": 4096,
         "k": 7168, "skew": "uniform"},
        # a prefill batch's gate/up product on that share, popular and rare experts, the row buffer padded
        {"name": "grouped_prefill", "family": "grouped", "dtype": "bf16", "rows": 8192, "pad": 333, "groups": 48,
         "n": 4096, "k": 7168, "skew": "zipf"},
        # one user's token: latency
        {"name": "sample_one", "family": "sample", "dtype": "f32", "rows": 1, "vocab": 129280, "spread": 3.0,
         "masked": 0.0, "settings": "top_k+top_p"},
        # a serving batch whose users chose different settings
        {"name": "sample_batch", "family": "sample", "dtype": "f32", "rows": 64, "vocab": 129280, "spread": 3.0,
         "masked": 0.0, "settings": "mixed"},
        # answers drawn for training, from the whole distribution
        {"name": "sample_rollout", "family": "sample", "dtype": "bf16", "rows": 256, "vocab": 65536, "spread": 3.0,
         "masked": 0.0, "settings": "temperature"},
        # answers held to a grammar that leaves a tenth of an odd vocabulary
        {"name": "sample_masked", "family": "sample", "dtype": "f32", "rows": 7, "vocab": 50257, "spread": 2.0,
         "masked": 0.9, "settings": "min_p"},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    family = rng.choice(["quantize", "linear", "linear", "grouped", "sample", "sample"])
    if family == "quantize":
        return {"family": family, "dtype": rng.choice(["bf16", "f16", "f32"]), "m": _log_int(rng, 1, 8192),
                "k": _log_int(rng, 64, 7168)}
    if family == "linear":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32", "int8"])
        return {"family": family, "dtype": dtype, "out": rng.choice(["bf16", "f32"]) if dtype == "int8" else dtype,
                "m": _log_int(rng, 1, 4096), "n": _log_int(rng, 64, 12288), "k": 16 * rng.randint(8, 448),
                "bias": rng.choice([False, True]),
                "activation": rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]),
                "residual": rng.choice([False, True])}
    if family == "grouped":
        return {"family": family, "dtype": rng.choice(["bf16", "bf16", "f16"]), "rows": _log_int(rng, 1, 8192),
                "pad": rng.choice([0, rng.randint(1, 500)]), "groups": _log_int(rng, 1, 48),
                "n": 8 * _log_int(rng, 8, 512), "k": 16 * _log_int(rng, 8, 448),
                "skew": rng.choice(["zipf", "uniform", "half"])}
    return {"family": family, "dtype": rng.choice(["f32", "f32", "bf16", "f16"]), "rows": _log_int(rng, 1, 256),
            "vocab": _log_int(rng, 100, 65536), "spread": rng.choice([1.0, 2.0, 3.0]),
            "masked": rng.choice([0.0, 0.0, 0.9]),
            "settings": rng.choice(["temperature", "top_k", "top_p", "top_k+top_p", "min_p", "mixed"])}


# ----------------------------------------------------------------- inputs --

def _activations(rows: int, k: int, dtype: torch.dtype, g: torch.Generator) -> torch.Tensor:
    channel = torch.exp(0.5 * torch.randn(k, generator=g, device=DEVICE))
    return (torch.randn(rows, k, generator=g, device=DEVICE) * channel).to(dtype)


def _weight(shape, g: torch.Generator) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes of normally distributed rows under a scale of each row that spreads by a few times."""
    codes = torch.empty(shape, dtype=torch.int8, device=DEVICE)
    flat = codes.reshape(-1)
    for i in range(0, flat.numel(), 1 << 28):
        part = flat[i:i + (1 << 28)]
        part.copy_((torch.randn(part.numel(), generator=g, device=DEVICE) * 32).round_().clamp_(-127, 127))
    return codes, torch.exp(0.5 * torch.randn(shape[:-1], generator=g, device=DEVICE)) * (0.02 / 32)


def _counts(case: dict, seed: int) -> list[int]:
    """Rows of each expert: uniform or Zipf(1.1) popularity, or only every other expert taken."""
    g = torch.Generator().manual_seed(seed)
    groups = case["groups"]
    p = torch.ones(groups)
    if case["skew"] == "zipf":
        p = torch.arange(1, groups + 1).float().pow(-1.1)[torch.randperm(groups, generator=g)]
    elif case["skew"] == "half":
        p[1::2] = 0.0
    picks = torch.multinomial(p, case["rows"], replacement=True, generator=g)
    return torch.bincount(picks, minlength=groups).tolist()


def _settings(case: dict, g: torch.Generator) -> dict:
    """Keywords of ``sample_tokens``: one value for all rows, or (mixed) each row its own, some rows greedy."""
    kind, rows, vocab = case["settings"], case["rows"], case["vocab"]
    if kind == "mixed":
        pick = lambda values: torch.tensor(values, device=DEVICE)[  # noqa: E731
            torch.randint(0, len(values), (rows,), generator=g, device=DEVICE)]
        return {"temperature": pick([0.0, 0.6, 0.8, 1.0, 1.3]), "top_k": pick([0, 20, 50, 1000, vocab]).to(torch.int32),
                "top_p": pick([1.0, 0.95, 0.9, 0.5]), "min_p": pick([0.0, 0.0, 0.05])}
    s: dict = {"temperature": 1.0 if kind == "temperature" else 0.8}
    if "top_k" in kind:
        s["top_k"] = 50
    if "top_p" in kind:
        s["top_p"] = 0.95
    if kind == "min_p":
        s["min_p"] = 0.05
    return s


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    s: dict = {"case": case}
    if case["family"] == "quantize":
        s["x"] = _activations(case["m"], case["k"], DTYPES[case["dtype"]], g)
        return s
    if case["family"] == "grouped":
        starts = [0]
        for c in _counts(case, seed):
            starts.append(starts[-1] + c)
        s["starts"] = starts
        s["offsets"] = torch.tensor(starts, dtype=torch.int64, device=DEVICE)
        s["x"] = _activations(case["rows"] + case["pad"], case["k"], DTYPES[case["dtype"]], g)
        s["w"], s["scale"] = _weight((case["groups"], case["n"], case["k"]), g)
        return s
    if case["family"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        z = torch.randn(rows, vocab, generator=g, device=DEVICE) * case["spread"]
        # a few tokens that the model finds likely
        z.scatter_add_(1, torch.randint(0, vocab, (rows, 8), generator=g, device=DEVICE),
                       4 * case["spread"] * torch.rand(rows, 8, generator=g, device=DEVICE))
        if case["masked"]:
            z[torch.rand(rows, vocab, generator=g, device=DEVICE) < case["masked"]] = -math.inf
            z[:, vocab - 1] = 0.0
        s["logits"] = z.to(DTYPES[case["dtype"]])
        s["uniform"] = torch.rand(rows, generator=g, device=DEVICE)
        s["settings"] = _settings(case, g)
        return s
    m, n, k = case["m"], case["n"], case["k"]
    if case["dtype"] == "int8":
        x = _activations(m, k, torch.float32, g)
        s["x_scale"] = x.abs().amax(1) / 127
        s["x"] = (x / s["x_scale"][:, None]).round().to(torch.int8)
    else:
        s["x"], s["x_scale"] = _activations(m, k, DTYPES[case["dtype"]], g), None
    s["w"], s["scale"] = _weight((n, k), g)
    out = DTYPES[case["out"]]
    s["bias"] = (torch.randn(n, generator=g, device=DEVICE) * 0.5).to(torch.bfloat16) if case["bias"] else None
    s["residual"] = torch.randn(m, n, generator=g, device=DEVICE).to(out) if case["residual"] else None
    return s


# ------------------------------------------------------------ plain forms --

def _plain_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    scale = (x.float().abs().amax(dim=1) / 127).clamp(min=2.0 ** -126)
    # in 64 bits: a quotient beside a border between two codes
    return (x.double() / scale.double()[:, None]).round().to(torch.int8), scale


def _plain_linear(s: dict) -> torch.Tensor:
    case = s["case"]
    q, scale = (s["x"], s["x_scale"]) if case["dtype"] == "int8" else _plain_quantize(s["x"])
    z = (q.float() @ s["w"].float().T) * scale[:, None] * s["scale"]
    if case["bias"]:
        z = z + s["bias"].float()
    kind = case["activation"]
    if kind == "relu":
        z = z.clamp(min=0)
    elif kind == "silu":
        z = z / (1 + torch.exp(-z))
    elif kind == "gelu":
        z = 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    elif kind == "gelu_tanh":
        z = 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if case["residual"]:
        z = z + s["residual"].float()
    return z.to(DTYPES[case["out"]])


def _plain_grouped(s: dict) -> torch.Tensor:
    x, w, starts = s["x"], s["w"], s["starts"]
    q, scale = _plain_quantize(x)
    y = torch.zeros(x.shape[0], s["case"]["n"], dtype=x.dtype, device=x.device)
    for e, (a, b) in enumerate(zip(starts, starts[1:])):
        if a < b:
            y[a:b] = ((q[a:b].float() @ w[e].float().T) * scale[a:b, None] * s["scale"][e]).to(x.dtype)
    return y


def _plain_sample(s: dict) -> tuple[torch.Tensor, torch.Tensor]:
    z, chosen = s["logits"], s["settings"]
    rows, vocab = z.shape

    def column(name: str, default: float) -> torch.Tensor:
        v = chosen.get(name, default)
        return v.double()[:, None] if isinstance(v, torch.Tensor) else torch.full((rows, 1), float(v), dtype=torch.float64,
                                                                                 device=z.device)

    t, top_p, min_p = column("temperature", 1.0), column("top_p", 1.0), column("min_p", 0.0)
    top_k = column("top_k", 0.0)
    ordered, index = torch.sort(z, dim=1, descending=True, stable=True)  # ties: the lowest index first
    d = (ordered.double() - ordered[:, :1].double()) / torch.where(t > 0, t, 1.0)
    w = torch.exp(d)
    place = torch.arange(vocab, device=z.device)
    w = torch.where((place < top_k) | (top_k <= 0), w, 0.0)
    upto = torch.cumsum(w, dim=1)
    w = torch.where((upto - w < top_p * upto[:, -1:]) | (top_p >= 1), w, 0.0)
    w = torch.where((torch.exp(d) >= min_p) | (place == 0), w, 0.0)
    w = torch.where((t > 0) | (place == 0), w, 0.0)
    kept = torch.zeros_like(w).scatter_(1, index, w)
    upto = torch.cumsum(kept, dim=1)
    token = (upto > s["uniform"].double()[:, None] * upto[:, -1:]).int().argmax(dim=1)
    return token, torch.log(kept.gather(1, token[:, None])[:, 0] / upto[:, -1]).float()


# ------------------------------------------------------------------- pass --

def _own_linear(s: dict) -> torch.Tensor:
    from kquant_amd.linear import int8_linear

    case = s["case"]
    kind = None if case["activation"] == "none" else case["activation"]
    return int8_linear(s["x"], s["w"], s["scale"], source_scale=s["x_scale"], bias=s["bias"], activation=kind,
                       residual=s["residual"], out_dtype=DTYPES[case["out"]])


def run(state: dict):
    family = state["case"]["family"]
    if family == "quantize":
        if own:
            from kquant_amd.int8 import int8_quantize

            return int8_quantize(state["x"])
        return _plain_quantize(state["x"])
    if family == "linear":
        return _own_linear(state) if own else _plain_linear(state)
    if family == "grouped":
        if own:
            from kquant_amd.grouped import int8_grouped_linear

            return int8_grouped_linear(state["x"], state["w"], state["scale"], state["offsets"])
        return _plain_grouped(state)
    if own:
        from kquant_amd.sampling import sample_tokens

        return sample_tokens(state["logits"], state["uniform"], **state["settings"], return_logprobs=True)
    return _plain_sample(state)


# ------------------------------------------------------------------- work --

def work(case: dict) -> dict:
    """Each input read once and each output written once."""
    if case["family"] == "quantize":
        m, k = case["m"], case["k"]
        return {"bytes": float(m * k * (SIZEOF[case["dtype"]] + 1) + 4 * m), "flops": 3.0 * m * k}
    if case["family"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        return {"bytes": float(rows * vocab * SIZEOF[case["dtype"]] + 16 * rows), "flops": 4.0 * rows * vocab}
    if case["family"] == "grouped":
        size, rows, n, k = SIZEOF[case["dtype"]], case["rows"], case["n"], case["k"]
        held = sum(c > 0 for c in _counts(case, 0))
        return {"bytes": float(size * (rows * k + (rows + case["pad"]) * n) + held * n * (k + 4)),
                "flops": 2.0 * rows * n * k}
    m, n, k, out = case["m"], case["n"], case["k"], SIZEOF[case["out"]]
    extra = (2 * n if case["bias"] else 0) + (out * m * n if case["residual"] else 0)
    return {"bytes": float(SIZEOF[case["dtype"]] * m * k + n * (k + 4) + out * m * n + extra), "flops": 2.0 * m * n * k}


# ------------------------------------------------------------------ exact --

def _codes64(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The scale is the fp32 number nearest to a 127th of the largest magnitude; a code the whole number nearest to
    the quotient, the even one of two."""
    largest = x.double().abs().max(dim=1).values
    scale = (largest / 127.0).float().double().clamp(min=2.0 ** -126)
    quotient = x.double() / scale.unsqueeze(1)
    below = torch.floor(quotient)
    part = quotient - below
    up = (part > 0.5) | ((part == 0.5) & (below.remainder(2.0) == 1.0))
    return below + up.double(), scale


def _activate64(z: torch.Tensor, kind: str) -> torch.Tensor:
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if kind == "silu":
        return z * torch.sigmoid(z)
    if kind == "gelu":
        return z * torch.special.ndtr(z)
    if kind == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z


def _draw64(z: np.ndarray, u: float, t: float, top_k: int, top_p: float, min_p: float) -> tuple[int, float]:
    """One row in extended precision: the order, the three cuts as lengths of it, and the draw by index."""
    order = np.lexsort((np.arange(z.size), -z))
    if t <= 0:
        return int(order[0]), 0.0
    w = np.exp((z.astype(np.longdouble) - np.longdouble(z[order[0]])) / np.longdouble(t))
    sorted_w = w[order]
    length = z.size if top_k <= 0 else min(top_k, z.size)
    if top_p < 1:
        before = np.concatenate([[np.longdouble(0)], np.cumsum(sorted_w[:length])])
        length = max(1, int(np.searchsorted(before[:-1], np.longdouble(top_p) * before[-1], side="left")))
    length = max(1, min(length, int(np.count_nonzero(sorted_w >= np.longdouble(min_p)))))
    kept = np.sort(order[:length])
    upto = np.cumsum(w[kept])
    at = min(int(np.searchsorted(upto, np.longdouble(u) * upto[-1], side="right")), length - 1)
    return int(kept[at]), float(np.log(w[kept[at]] / upto[-1]))


def exact(case: dict, seed: int):
    with torch.no_grad():
        s = prepare(case, seed)
        if case["family"] == "sample":
            z, u = s["logits"].double().cpu().numpy(), s["uniform"].double().cpu().numpy()
            given = {}
            for name, default in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)):
                v = s["settings"].get(name, default)
                given[name] = v.cpu().tolist() if isinstance(v, torch.Tensor) else [v] * case["rows"]
            drawn = [_draw64(z[r], u[r], given["temperature"][r], given["top_k"][r], given["top_p"][r], given["min_p"][r])
                     for r in range(case["rows"])]
            return (torch.tensor([d[0] for d in drawn], device=DEVICE),
                    torch.tensor([d[1] for d in drawn], dtype=torch.float64, device=DEVICE))
        if case["family"] == "linear" and case["dtype"] == "int8":
            q, scale = s["x"].double(), s["x_scale"].double()
        else:
            q, scale = _codes64(s["x"])
        if case["family"] == "quantize":
            return q.to(torch.int8), scale
        if case["family"] == "grouped":
            ends, out = s["offsets"].tolist(), []
            for e in range(case["groups"]):
                rows = slice(ends[e], ends[e + 1])
                out.append(torch.matmul(q[rows] * scale[rows].unsqueeze(1),
                                        (s["w"][e].double() * s["scale"][e].double().unsqueeze(1)).transpose(0, 1)))
            return torch.cat(out + [torch.zeros(case["pad"], case["n"], dtype=torch.float64, device=DEVICE)])
        z = torch.matmul(q, s["w"].double().transpose(0, 1)) * torch.outer(scale, s["scale"].double())
        if s["bias"] is not None:
            z += s["bias"].double()
        z = _activate64(z, case["activation"])
        return z if s["residual"] is None else z + s["residual"].double()
