"""Operator cases: the products a model runs around its quantized experts.

Three families, each through the public Python entry points:

  grouped   matrix products grouped by expert over dense bf16 / fp16 weights
            (``grouped.grouped_linear``): the forward pass, and a training
            step with the gradients of the rows and of the weights
  loss      softmax cross entropy of a vocabulary head without keeping the
            logits (``loss.linear_cross_entropy``): per-token losses, and a
            training step with the gradients of the rows and of the head;
            the head dense bf16, or frozen MXFP8 / MXFP4
  linear    the dense MXFP8 / MXFP4 linear with bias, activation and residual
            in its epilogue (``linear.mxfp8_linear`` / ``mxfp4_linear``)

``listed()`` gives the fixed cases, ``draw(rng)`` further ones of the same
ranges.  A case is a dict of plain values; ``prepare`` builds the inputs from a
seed, ``run`` makes one pass, in plain torch operations or, where ``own`` is
true, through the library.  ``exact`` states each result in float64.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZEOF = {"bf16": 2, "f16": 2, "f32": 4}
DEVICE = "cuda"
IGNORE = -100


# ------------------------------------------------------------------ cases --

def listed() -> list[dict]:
    return [
        # one decode batch (8 tokens x top-8) through a GPU's share of the experts: latency and weight bytes
        {"name": "grouped_decode", "family": "grouped", "train": False, "dtype": "bf16", "rows": 64, "pad": 0,
         "groups": 48, "n": 4096, "k": 7168, "skew": "uniform"},
        # a prefill batch's gate/up product on that share, popular and rare experts
        {"name": "grouped_prefill", "family": "grouped", "train": False, "dtype": "bf16", "rows": 8192, "pad": 0,
         "groups": 48, "n": 4096, "k": 7168, "skew": "zipf"},
        # a training step of that share's down product, the row buffer padded past the routed rows
        {"name": "grouped_train", "family": "grouped", "train": True, "dtype": "bf16", "rows": 8192, "pad": 333,
         "groups": 48, "n": 7168, "k": 2048, "skew": "zipf"},
        # a small odd training batch in fp16
        {"name": "grouped_train_small", "family": "grouped", "train": True, "dtype": "f16", "rows": 333, "pad": 7,
         "groups": 12, "n": 1416, "k": 1032, "skew": "zipf"},
        # scoring a few sampled tokens against a wide MXFP8 head: latency and head bytes
        {"name": "loss_score_few", "family": "loss", "train": False, "head": "mxfp8", "tokens": 5, "vocab": 129280,
         "k": 7168, "ignored": 0.0},
        # perplexity of an odd chunk of text under the dense head
        {"name": "loss_eval", "family": "loss", "train": False, "head": "bf16", "tokens": 777, "vocab": 129280,
         "k": 7168, "ignored": 0.0},
        # a training step's loss with the head's gradient, a tenth of the tokens not counted
        {"name": "loss_train", "family": "loss", "train": True, "head": "bf16", "tokens": 4096, "vocab": 65536,
         "k": 4096, "ignored": 0.1},
        # recovery of a quantized model: the gradient through a frozen MXFP4 head of an odd vocabulary
        {"name": "loss_train_frozen", "family": "loss", "train": True, "head": "mxfp4", "tokens": 2048,
         "vocab": 50257, "k": 2048, "ignored": 0.3},
        # one decoded token through an ungated MLP layer of an MXFP8 model
        {"name": "linear_decode", "family": "linear", "fmt": "mxfp8", "dtype": "bf16", "m": 1, "n": 12288, "k": 7168,
         "bias": True, "activation": "silu", "residual": True},
        # a ragged chunk of a prompt, MXFP4 weights
        {"name": "linear_ragged", "family": "linear", "fmt": "mxfp4", "dtype": "bf16", "m": 777, "n": 5000, "k": 7168,
         "bias": True, "activation": "gelu", "residual": True},
        # a full prefill chunk
        {"name": "linear_prefill", "family": "linear", "fmt": "mxfp8", "dtype": "bf16", "m": 4096, "n": 12288,
         "k": 7168, "bias": True, "activation": "gelu_tanh", "residual": True},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    family = rng.choice(["grouped", "loss", "linear"])
    if family == "grouped":
        train = rng.choice([False, True])
        return {"family": family, "train": train, "dtype": rng.choice(["bf16", "bf16", "f16"]),
                "rows": _log_int(rng, 1, 8192), "pad": rng.choice([0, rng.randint(1, 500)]),
                "groups": _log_int(rng, 1, 48), "n": 8 * _log_int(rng, 8, 512), "k": 8 * _log_int(rng, 8, 448),
                "skew": rng.choice(["zipf", "uniform", "half"])}
    if family == "loss":
        train = rng.choice([False, True])
        head = rng.choice(["bf16", "bf16", "mxfp8", "mxfp4"])
        tokens = _log_int(rng, 1, 2048)
        return {"family": family, "train": train, "head": head, "tokens": tokens,
                "vocab": _log_int(rng, 100, 65536),
                "k": 8 * _log_int(rng, 8, 512) if head == "bf16" else 64 * _log_int(rng, 4, 64),
                "ignored": rng.choice([0.0, 0.1, 0.5])}
    dtype = rng.choice(["bf16", "bf16", "f32"])
    return {"family": family, "fmt": rng.choice(["mxfp8", "mxfp4"]), "dtype": dtype,
            "m": _log_int(rng, 1, 1024 if dtype == "f32" else 4096), "n": _log_int(rng, 64, 12288),
            "k": 64 * rng.randint(4, 112), "bias": rng.choice([False, True]),
            "activation": rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]),
            "residual": rng.choice([False, True])}


# ----------------------------------------------------------------- inputs --

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _mx_rows(w: torch.Tensor, fmt: str) -> tuple[torch.Tensor, torch.Tensor]:
    """Block-scaled codes of fp32 rows: E4M3 bytes (or packed E2M1) and E8M0 bytes."""
    b = w.reshape(w.shape[0], -1, 32)
    qmax = 448.0 if fmt == "mxfp8" else 6.0
    e = torch.log2(b.abs().amax(-1).clamp(min=1e-30) / qmax).ceil().clamp(-127, 127)
    y = (b / torch.exp2(e)[..., None]).reshape(w.shape)
    scale = (e + 127).to(torch.uint8)
    if fmt == "mxfp8":
        return y.clamp(-448, 448).to(torch.float8_e4m3fn), scale
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=w.device)
    codes = torch.bucketize(y.abs(), edges).to(torch.uint8) | (torch.signbit(y).to(torch.uint8) << 3)
    return codes[:, 0::2] | (codes[:, 1::2] << 4), scale


def _mx_weight(rows: int, k: int, fmt: str, std: float, g: torch.Generator):
    parts = [_mx_rows(torch.randn(min(8192, rows - r), k, generator=g, device=DEVICE) * std, fmt)
             for r in range(0, rows, 8192)]
    return torch.cat([p[0].view(torch.uint8) for p in parts]).view(parts[0][0].dtype), torch.cat([p[1] for p in parts])


def _dense(shape, std: float, dtype: torch.dtype, g: torch.Generator) -> torch.Tensor:
    out = torch.empty(shape, dtype=dtype, device=DEVICE)
    flat = out.reshape(-1)
    for i in range(0, flat.numel(), 1 << 28):
        part = flat[i:i + (1 << 28)]
        part.copy_(torch.randn(part.numel(), generator=g, device=DEVICE) * std)
    return out


def _activations(rows: int, k: int, dtype: torch.dtype, g: torch.Generator) -> torch.Tensor:
    channel = torch.exp(0.5 * torch.randn(k, generator=g, device=DEVICE))
    return (torch.randn(rows, k, generator=g, device=DEVICE) * channel).to(dtype)


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


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    s: dict = {"case": case}
    if case["family"] == "grouped":
        dtype = DTYPES[case["dtype"]]
        rows, n, k, groups = case["rows"] + case["pad"], case["n"], case["k"], case["groups"]
        starts = [0]
        for c in _counts(case, seed):
            starts.append(starts[-1] + c)
        s["starts"] = starts
        s["offsets"] = torch.tensor(starts, dtype=torch.int64, device=DEVICE)
        s["x"] = _activations(rows, k, dtype, g)
        s["w"] = _dense((groups, n, k), 0.02, dtype, g)
        if case["train"]:
            s["dy"] = _dense((rows, n), 0.05, dtype, g)
            s["x"].requires_grad_(own)
            s["w"].requires_grad_(own)
        return s
    if case["family"] == "loss":
        tokens, vocab, k = case["tokens"], case["vocab"], case["k"]
        # a normed last state under a head whose logits spread over a few units
        s["h"] = _dense((tokens, k), 1.0, torch.bfloat16, g)
        std = 2.0 / math.sqrt(k)
        if case["head"] == "bf16":
            s["w"], s["scale"] = _dense((vocab, k), std, torch.bfloat16, g), None
        else:
            s["w"], s["scale"] = _mx_weight(vocab, k, case["head"], std, g)
        target = torch.randint(0, vocab, (tokens,), generator=g, device=DEVICE)
        target[torch.rand(tokens, generator=g, device=DEVICE) < case["ignored"]] = IGNORE
        target[0] = vocab - 1  # the last column, and one counted token at least
        s["target"] = target
        if case["train"]:
            s["h"].requires_grad_(own)
            if case["head"] == "bf16":
                s["w"].requires_grad_(own)
        return s
    dtype = DTYPES[case["dtype"]]
    s["x"] = _activations(case["m"], case["k"], dtype, g)
    s["w"], s["scale"] = _mx_weight(case["n"], case["k"], case["fmt"], 0.015, g)
    s["bias"] = _dense((case["n"],), 0.5, dtype, g) if case["bias"] else None
    s["residual"] = _dense((case["m"], case["n"]), 1.0, dtype, g) if case["residual"] else None
    return s


# ------------------------------------------------------------ plain forms --

def _values(q: torch.Tensor, scale: torch.Tensor | None) -> torch.Tensor:
    """fp32 weight of dense, MXFP8 or packed MXFP4 rows."""
    if scale is None:
        return q.float()
    if q.dtype == torch.float8_e4m3fn:
        v = q.float()
    else:
        lut = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=q.device)
        v = lut[torch.stack([q & 15, q >> 4], dim=-1).reshape(q.shape[0], -1).int()]
    factor = torch.exp2(scale.float() - 127.0)
    return (v.reshape(v.shape[0], -1, 32) * factor[..., None]).reshape(v.shape)


def _plain_grouped(s: dict):
    case, x, w, starts = s["case"], s["x"], s["w"], s["starts"]
    y = torch.zeros(x.shape[0], case["n"], dtype=x.dtype, device=x.device)
    dx, dw = (torch.zeros_like(x), torch.zeros_like(w)) if case["train"] else (None, None)
    for e, (a, b) in enumerate(zip(starts, starts[1:])):
        if a == b:
            continue
        xe, we = x[a:b].float(), w[e].float()
        y[a:b] = (xe @ we.T).to(x.dtype)
        if case["train"]:
            dy = s["dy"][a:b].float()
            dx[a:b] = (dy @ we).to(x.dtype)
            dw[e] = (dy.T @ xe).to(x.dtype)
    return (y, dx, dw) if case["train"] else y


def _plain_loss(s: dict):
    case, target = s["case"], s["target"]
    h, w = s["h"].float(), _values(s["w"], s["scale"])
    z = h @ w.T
    top = z.amax(dim=1, keepdim=True)
    p = torch.exp(z - top)
    total = p.sum(dim=1, keepdim=True)
    counted = target != IGNORE
    column = target.clamp(min=0)[:, None]
    losses = (top + torch.log(total) - z.gather(1, column)).squeeze(1)
    losses = torch.where(counted, losses, torch.zeros_like(losses))
    if not case["train"]:
        return losses
    count = counted.sum()
    d = p / total
    d.scatter_add_(1, column, -torch.ones_like(column, dtype=d.dtype))
    d = d * (counted[:, None] / count)
    loss = losses.sum() / count
    dh = (d @ w).to(torch.bfloat16)
    if case["head"] != "bf16":
        return loss, dh
    return loss, dh, (d.T @ h).to(torch.bfloat16)


def _plain_linear(s: dict):
    case = s["case"]
    z = s["x"].float() @ _values(s["w"], s["scale"]).T
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
    return z.to(s["x"].dtype)


# ------------------------------------------------------------------- pass --

def _own_grouped(s: dict):
    from kquant_amd.grouped import grouped_linear

    y = grouped_linear(s["x"], s["w"], s["offsets"])
    if not s["case"]["train"]:
        return y
    dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
    return y.detach(), dx, dw


def _own_loss(s: dict):
    from kquant_amd.loss import linear_cross_entropy

    case = s["case"]
    if not case["train"]:
        return linear_cross_entropy(s["h"], s["w"], s["target"], s["scale"], ignore_index=IGNORE, reduction="none")
    loss = linear_cross_entropy(s["h"], s["w"], s["target"], s["scale"], ignore_index=IGNORE)
    leaves = (s["h"], s["w"]) if case["head"] == "bf16" else (s["h"],)
    return (loss.detach(), *torch.autograd.grad(loss, leaves))


def _own_linear(s: dict):
    from kquant_amd import linear

    case = s["case"]
    f = linear.mxfp8_linear if case["fmt"] == "mxfp8" else linear.mxfp4_linear
    kind = None if case["activation"] == "none" else case["activation"]
    return f(s["x"], s["w"], s["scale"], bias=s["bias"], activation=kind, residual=s["residual"])


def run(state: dict):
    family = state["case"]["family"]
    if own:
        return {"grouped": _own_grouped, "loss": _own_loss, "linear": _own_linear}[family](state)
    return {"grouped": _plain_grouped, "loss": _plain_loss, "linear": _plain_linear}[family](state)


# ------------------------------------------------------------------- work --

def work(case: dict) -> dict:
    """Each input read once and each output written once; a training step's
    products are three (the gradients' two and the forward's)."""
    if case["family"] == "grouped":
        size, rows, n, k = SIZEOF[case["dtype"]], case["rows"], case["n"], case["k"]
        held = sum(c > 0 for c in _counts(case, 0))
        out = (rows + case["pad"]) * n
        nbytes = size * (rows * k + held * n * k + out)
        flops = 2.0 * rows * n * k
        if case["train"]:  # and dy read, dx and every expert's dw written
            nbytes += size * (rows * n + (rows + case["pad"]) * k + case["groups"] * n * k)
            flops *= 3
        return {"bytes": float(nbytes), "flops": flops}
    if case["family"] == "loss":
        t, v, k = case["tokens"], case["vocab"], case["k"]
        head = v * k * {"bf16": 2.0, "mxfp8": 33 / 32, "mxfp4": 17 / 32}[case["head"]]
        if not case["train"]:
            return {"bytes": head + 2.0 * t * k + 12.0 * t, "flops": 2.0 * t * v * k}
        counted = t * (1 - case["ignored"])
        products = 3 if case["head"] == "bf16" else 2
        grads = 2.0 * t * k + (head if case["head"] == "bf16" else 0.0)
        return {"bytes": head + 2.0 * t * k + 8.0 * t + grads, "flops": products * 2.0 * counted * v * k}
    m, n, k, size = case["m"], case["n"], case["k"], SIZEOF[case["dtype"]]
    weight = n * k * (33 / 32 if case["fmt"] == "mxfp8" else 17 / 32)
    extra = size * ((n if case["bias"] else 0) + (m * n if case["residual"] else 0))
    return {"bytes": size * (m * k + m * n) + weight + extra, "flops": 2.0 * m * n * k}


# ------------------------------------------------------------------ exact --

def _weight64(q: torch.Tensor, scale: torch.Tensor | None) -> torch.Tensor:
    if scale is None:
        return q.double()
    if q.dtype == torch.uint8:
        lo, hi = (q % 16).long(), (q // 16).long()
        code = torch.empty(q.shape[0], 2 * q.shape[1], dtype=torch.long, device=q.device)
        code[:, 0::2], code[:, 1::2] = lo, hi
        exponent, fraction = (code // 2) % 4, (code % 2).double()
        size = torch.where(exponent == 0, fraction / 2, (1 + fraction / 2) * 2.0 ** (exponent - 1).double())
        v = torch.where(code >= 8, -size, size)
    else:
        v = q.double()
    return v * torch.pow(2.0, scale.double() - 127).repeat_interleave(32, dim=1)


def exact(case: dict, seed: int):
    with torch.no_grad():
        s = prepare(case, seed)
        for name in ("x", "w", "h"):
            if name in s:
                s[name] = s[name].detach()
        if case["family"] == "grouped":
            ends = s["offsets"].tolist()
            ys, dxs, dws = [], [], []
            for e in range(case["groups"]):
                xe, we = s["x"][ends[e]:ends[e + 1]].double(), s["w"][e].double()
                ys.append(torch.matmul(xe, we.transpose(0, 1)))
                if case["train"]:
                    de = s["dy"][ends[e]:ends[e + 1]].double()
                    dxs.append(torch.matmul(de, we))
                    dws.append(torch.matmul(de.transpose(0, 1), xe))
            pad = lambda width: [torch.zeros(case["pad"], width, dtype=torch.float64, device=DEVICE)]  # noqa: E731
            y = torch.cat(ys + pad(case["n"]))
            return (y, torch.cat(dxs + pad(case["k"])), torch.stack(dws)) if case["train"] else y
        if case["family"] == "loss":
            h, target = s["h"].double(), s["target"]
            keep = (target != IGNORE).nonzero().squeeze(1)
            hk, tk = h[keep], target[keep]
            cuts = list(range(0, case["vocab"], 16384))
            piece = lambda c: _weight64(s["w"][c:c + 16384], None if s["scale"] is None  # noqa: E731
                                        else s["scale"][c:c + 16384])
            lse = torch.full((keep.numel(),), -math.inf, dtype=torch.float64, device=DEVICE)
            hit = torch.zeros_like(lse)
            for c in cuts:
                z = torch.matmul(hk, piece(c).transpose(0, 1))
                lse = torch.logaddexp(lse, torch.logsumexp(z, dim=1))
                here = ((tk >= c) & (tk < c + z.shape[1])).nonzero().squeeze(1)
                hit[here] = z[here, tk[here] - c]
            losses = torch.zeros(h.shape[0], dtype=torch.float64, device=DEVICE)
            losses[keep] = lse - hit
            if not case["train"]:
                return losses
            dh = torch.zeros_like(h)
            dw = torch.empty(case["vocab"], case["k"], dtype=torch.float64, device=DEVICE) if case["head"] == "bf16" else None
            for c in cuts:
                wc = piece(c)
                d = torch.exp(torch.matmul(hk, wc.transpose(0, 1)) - lse[:, None])
                here = ((tk >= c) & (tk < c + wc.shape[0])).nonzero().squeeze(1)
                d[here, tk[here] - c] -= 1
                d /= keep.numel()
                dh[keep] += torch.matmul(d, wc)
                if dw is not None:
                    dw[c:c + wc.shape[0]] = torch.matmul(d.transpose(0, 1), hk)
            loss = losses.sum() / keep.numel()
            return (loss, dh) if dw is None else (loss, dh, dw)
        out = torch.matmul(s["x"].double(), _weight64(s["w"], s["scale"]).transpose(0, 1))
        if s["bias"] is not None:
            out += s["bias"].double()
        kind = case["activation"]
        if kind == "relu":
            out = torch.where(out > 0, out, torch.zeros_like(out))
        elif kind == "silu":
            out = out * torch.sigmoid(out)
        elif kind == "gelu":
            out = out * torch.special.ndtr(out)
        elif kind == "gelu_tanh":
            inner = out + 0.044715 * out ** 3
            out = out * torch.sigmoid(2 * math.sqrt(2 / math.pi) * inner)
        if s["residual"] is not None:
            out += s["residual"].double()
        return out
