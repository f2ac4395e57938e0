"""What a training step does between its token ids and its losses, as
measurable cases.

A case is a dict of plain values; "op" says which operator it takes:

* ``embedding``: rows of a vocabulary's matrix looked up by token id and scaled;
  forward, or forward and the matrix's gradient;
* ``layer_norm``: layer norm over the last dimension; forward, or forward and
  the gradients of the input, the weight and the bias;
* ``experts``: tokens brought into their experts' order (the order itself, then
  the rows) and the experts' rows brought back, weighted and summed; forward, or
  forward and the gradients of the tokens, the experts' rows and the weights.

``listed`` gives the cases, ``draw`` one more of the same ranges, ``prepare``
what a program holds before the call, ``run`` one pass (in plain torch
operations in 32 bits, or, with ``own``, through the library), ``work`` the
bytes and operations a pass cannot do without, and ``exact`` the results in
64 bits.
"""

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5
# Token ids follow a Zipf-Mandelbrot law, low ids first, as a byte-pair
# vocabulary's do: the chance of rank r is proportional to about 1 / (r + 2.7).
ZIPF = 2.7

# Most elements of a drawn case: the largest listed one's of its operator.
MAX_EMBEDDING = 65536 * 4096 + 32000 * 4096
MAX_NORM = 65536 * 4096
MAX_EXPERTS = 131072 * 8 * 512


def listed():
    return [
        # One step of a small batch's decoding: eight rows of a large matrix.
        {"name": "embedding_decode_bf16", "op": "embedding", "dtype": "bf16", "train": False, "tokens": 8, "dim": 2048,
         "vocab": 128256, "scale": 1.0, "padded": 0.0},
        # A small model's step in fp16 at odd sizes, its padding without gradient.
        {"name": "embedding_small_f16", "op": "embedding", "dtype": "f16", "train": True, "tokens": 129, "dim": 200,
         "vocab": 1031, "scale": 1.0, "padded": 0.1},
        # Pretraining in fp32 over an odd vocabulary, rows scaled by the root of
        # their length.
        {"name": "embedding_train_f32", "op": "embedding", "dtype": "f32", "train": True, "tokens": 8191, "dim": 768,
         "vocab": 50257, "scale": 768 ** 0.5, "padded": 0.0},
        # Fine-tuning over a large vocabulary, most rows of which no token takes.
        {"name": "embedding_train_bf16", "op": "embedding", "dtype": "bf16", "train": True, "tokens": 4096,
         "dim": 2048, "vocab": 128256, "scale": 1.0, "padded": 0.3},
        # A large batch over a smaller vocabulary: frequent tokens come
        # thousands of times.
        {"name": "embedding_large_bf16", "op": "embedding", "dtype": "bf16", "train": True, "tokens": 65536,
         "dim": 4096, "vocab": 32000, "scale": 1.0, "padded": 0.0},
        # The norm before the head for one step of a small batch's decoding.
        {"name": "norm_decode_f16", "op": "layer_norm", "dtype": "f16", "train": False, "rows": 8, "dim": 2048,
         "affine": "both", "params": "same"},
        # A small model's norm in fp32, an odd number of tokens.
        {"name": "norm_train_f32", "op": "layer_norm", "dtype": "f32", "train": True, "rows": 2047, "dim": 768,
         "affine": "both", "params": "same"},
        # A large batch in bf16, the norm's own parameters kept in fp32.
        {"name": "norm_large_bf16", "op": "layer_norm", "dtype": "bf16", "train": True, "rows": 65536, "dim": 4096,
         "affine": "both", "params": "f32"},
        # One step of a small batch's decoding through 256 experts.
        {"name": "experts_decode_bf16", "op": "experts", "dtype": "bf16", "train": False, "tokens": 8, "dim": 2048,
         "experts": 256, "top": 8, "masked": 0.0, "weights": "f32"},
        # A small batch over few experts in fp32.
        {"name": "experts_small_f32", "op": "experts", "dtype": "f32", "train": True, "tokens": 512, "dim": 768,
         "experts": 8, "top": 2, "masked": 0.0, "weights": "same"},
        # A training step with padding tokens, an odd number of tokens.
        {"name": "experts_train_bf16", "op": "experts", "dtype": "bf16", "train": True, "tokens": 16383, "dim": 2048,
         "experts": 64, "top": 6, "masked": 0.25, "weights": "same"},
        # A large batch over many small experts.
        {"name": "experts_large_bf16", "op": "experts", "dtype": "bf16", "train": True, "tokens": 131072, "dim": 512,
         "experts": 256, "top": 8, "masked": 0.0, "weights": "f32"},
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _dim(rng, lo, hi):
    dim = _log_int(rng, lo, hi)
    return min(hi, -(-dim // 64) * 64) if rng.random() < 0.6 else dim


def draw(rng):
    op = rng.choice(["embedding", "layer_norm", "experts"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    train = rng.random() < 0.7
    if op == "embedding":
        most = MAX_EMBEDDING // 2 if dtype == "f32" else MAX_EMBEDDING
        vocab = _log_int(rng, 100, 131072)
        dim = _dim(rng, 32, 4096)
        tokens = _log_int(rng, 1, max(1, min(65536, most // dim - vocab)))
        return {"op": op, "dtype": dtype, "train": train, "tokens": tokens, "dim": dim, "vocab": vocab,
                "scale": rng.choice([1.0, math.sqrt(dim)]), "padded": rng.choice([0.0, 0.0, 0.3])}
    if op == "layer_norm":
        most = MAX_NORM // 2 if dtype == "f32" else MAX_NORM
        dim = _dim(rng, 16, 16384)
        return {"op": op, "dtype": dtype, "train": train, "rows": _log_int(rng, 1, min(65536, most // dim)),
                "dim": dim, "affine": rng.choice(["both", "both", "weight", "none"]),
                "params": rng.choice(["same", "f32"])}
    most = MAX_EXPERTS // 2 if dtype == "f32" else MAX_EXPERTS
    experts = rng.choice([8, 16, 60, 64, 128, 160, 256, 384])
    top = rng.randint(1, 8)
    dim = _dim(rng, 32, 4096)
    return {"op": op, "dtype": dtype, "train": train, "tokens": _log_int(rng, 1, min(131072, most // (dim * top))),
            "dim": dim, "experts": experts, "top": top, "masked": rng.choice([0.0, 0.25]),
            "weights": rng.choice(["f32", "same"])}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _randn(gen, *shape):
    return torch.randn(*shape, device=DEVICE, generator=gen)


def _embedding_state(case, gen):
    n, d, v, dtype = case["tokens"], case["dim"], case["vocab"], DTYPES[case["dtype"]]
    u = torch.rand(n, device=DEVICE, generator=gen, dtype=torch.float64)
    index = (ZIPF * ((v / ZIPF + 1) ** u - 1)).long().clamp_(max=v - 1)
    # padding behind a text, its token the vocabulary's last
    padding = v - 1 if case["padded"] else None
    if case["padded"]:
        index[n - int(n * case["padded"]):] = padding
    state = {"index": index, "weight": (_randn(gen, v, d) * (1.0 / math.sqrt(d))).to(dtype), "padding": padding}
    if case["train"]:
        state["weight"].requires_grad_(True)
        state["upstream"] = _randn(gen, n, d).to(dtype)
    return state


def _norm_state(case, gen):
    n, d, dtype = case["rows"], case["dim"], DTYPES[case["dtype"]]
    params = dtype if case["params"] == "same" else torch.float32
    # a residual stream: columns of their own size and offset, a few of them large
    size = torch.exp(_randn(gen, d) * 0.5)
    x = _randn(gen, n, d).mul_(size).add_(_randn(gen, d) * 0.5)
    x[:, torch.randint(0, d, (1 + d // 512,), device=DEVICE, generator=gen)] *= 10
    state = {"x": x.to(dtype), "weight": None, "bias": None}
    if case["affine"] != "none":
        state["weight"] = (_randn(gen, d) * 0.2 + 1).to(params)
    if case["affine"] == "both":
        state["bias"] = (_randn(gen, d) * 0.2).to(params)
    if case["train"]:
        state["upstream"] = _randn(gen, n, d).to(dtype)
        state["leaves"] = [state[k].requires_grad_(True) for k in ("x", "weight", "bias") if state[k] is not None]
    return state


def _experts_state(case, gen):
    t, d, e, k, dtype = case["tokens"], case["dim"], case["experts"], case["top"], DTYPES[case["dtype"]]
    logits = _randn(gen, t, e) * 1.5 + _randn(gen, e)
    top = logits.topk(k, -1)
    weights = torch.softmax(top.values, -1).to(dtype if case["weights"] == "same" else torch.float32)
    mask = torch.rand(t, device=DEVICE, generator=gen) >= case["masked"] if case["masked"] else None
    state = {"x": _randn(gen, t, d).to(dtype), "index": top.indices, "weights": weights, "mask": mask,
             # what the experts made of their rows
             "rows": _randn(gen, t * k, d).to(dtype)}
    if case["train"]:
        state["leaves"] = [state[name].requires_grad_(True) for name in ("x", "rows", "weights")]
        state["upstream"] = [_randn(gen, t * k, d).to(dtype), _randn(gen, t, d).to(dtype)]
    return state


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    make = {"embedding": _embedding_state, "layer_norm": _norm_state, "experts": _experts_state}[case["op"]]
    return {"case": case, **make(case, gen)}


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def _embedding_plain(s):
    case, index, weight = s["case"], s["index"], s["weight"].detach()
    out = weight[index].float().mul_(case["scale"]).to(weight.dtype)
    if not case["train"]:
        return [out]
    g = s["upstream"].float()
    if s["padding"] is not None:
        g = g * (index != s["padding"])[:, None]
    grad = torch.zeros(weight.shape, device=DEVICE).index_add_(0, index, g).mul_(case["scale"])
    return [out, grad.to(weight.dtype)]


def _norm_plain(s):
    x = s["x"].detach().float()
    w = s["weight"].detach().float() if s["weight"] is not None else None
    mean = x.mean(-1, keepdim=True)
    x = x - mean
    rstd = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    xhat = x.mul_(rstd)
    y = xhat * w if w is not None else xhat
    if s["bias"] is not None:
        y = y + s["bias"].detach().float()
    out = [y.to(s["x"].dtype)]
    if not s["case"]["train"]:
        return out
    g = s["upstream"].float()
    gw = g * w if w is not None else g
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - xhat * (gw * xhat).mean(-1, keepdim=True))
    out.append(dx.to(s["x"].dtype))
    if w is not None:
        out.append((g * xhat).sum(0).to(s["weight"].dtype))
    if s["bias"] is not None:
        out.append(g.sum(0).to(s["bias"].dtype))
    return out


def _experts_plain(s):
    case, index = s["case"], s["index"]
    t, k = index.shape
    e, dtype = case["experts"], s["x"].dtype
    live = (index >= 0) & (index < e)
    if s["mask"] is not None:
        live = live & s["mask"][:, None]
    # entries in their experts' order, those that are dropped behind all others
    key = torch.where(live, index, e).reshape(-1)
    source = key.sort(stable=True).indices
    row = torch.empty_like(source)
    row[source] = torch.arange(t * k, device=DEVICE)
    row = row.view(t, k)
    counts = torch.zeros(e + 1, dtype=torch.int64, device=DEVICE).scatter_add_(0, key, torch.ones_like(key))[:e]
    position = torch.where(live, row, -1 - row).int()
    on = live.reshape(-1)[source][:, None]
    x = s["x"].detach().float()
    rows = x[torch.div(source, k, rounding_mode="floor")].mul_(on).to(dtype)
    made = s["rows"].detach().float()[row] * live[..., None]
    w = torch.where(live, s["weights"].detach().float(), 0.0)
    y = (made * w[..., None]).sum(1).to(dtype)
    out = [position, counts, rows, y]
    if not case["train"]:
        return out
    d_rows, d_y = s["upstream"]
    dx = d_rows.float()[row].mul_(live[..., None]).sum(1).to(dtype)
    g = d_y.float()
    d_weights = (made * g[:, None]).sum(-1).to(s["weights"].dtype)
    d_made = torch.empty_like(made.view(t * k, -1))
    d_made[row.reshape(-1)] = (g[:, None] * w[..., None]).view(t * k, -1)
    return out + [dx, d_made.to(dtype), d_weights]


def _embedding_own(s):
    import fuselse_amd

    out = fuselse_amd.embedding(s["index"], s["weight"], scale=s["case"]["scale"], padding_idx=s["padding"])
    if not s["case"]["train"]:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, s["weight"], s["upstream"])]


def _norm_own(s):
    import fuselse_amd

    out = fuselse_amd.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS)
    if not s["case"]["train"]:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, s["leaves"], s["upstream"])]


def _experts_own(s):
    import fuselse_amd

    order = fuselse_amd.expert_order(s["index"], s["case"]["experts"], mask=s["mask"])
    rows = fuselse_amd.expert_dispatch(s["x"], order)
    y = fuselse_amd.expert_combine(s["rows"], s["weights"], order)
    out = [order.position, order.counts, rows.detach(), y.detach()]
    if not s["case"]["train"]:
        return out
    return out + list(torch.autograd.grad((rows, y), s["leaves"], s["upstream"]))


def run(state):
    op = state["case"]["op"]
    if own:
        return {"embedding": _embedding_own, "layer_norm": _norm_own, "experts": _experts_own}[op](state)
    return {"embedding": _embedding_plain, "layer_norm": _norm_plain, "experts": _experts_plain}[op](state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def _distinct(tokens, vocab):
    """How many different ids that many tokens take, on average."""
    edges = np.log(np.arange(vocab + 1) / ZIPF + 1) / math.log(vocab / ZIPF + 1)
    return float((1 - (1 - np.diff(edges)) ** tokens).sum())


def work(case):
    size, d = SIZES[case["dtype"]], case["dim"]
    if case["op"] == "embedding":
        n, v = case["tokens"], case["vocab"]
        text = n - int(n * case["padded"])
        nbytes = 8 * n + size * d * (_distinct(text, v) + n)
        flops = n * d
        if case["train"]:
            nbytes += size * d * (text + v)
            flops += text * d
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "layer_norm":
        n = case["rows"]
        arrays = {"both": 2, "weight": 1, "none": 0}[case["affine"]]
        params = d * arrays * (size if case["params"] == "same" else 4)
        nbytes = 2 * size * n * d + params
        flops = 7 * n * d
        if case["train"]:
            nbytes += 2 * size * n * d + params
            flops += 14 * n * d
        return {"bytes": nbytes, "flops": flops}
    t, k = case["tokens"], case["top"]
    live = 1 - case["masked"]
    weights = t * k * (size if case["weights"] == "same" else 4)
    # ids and positions; tokens in, rows out; rows in, tokens out
    nbytes = 12 * t * k + (t if case["masked"] else 0) + 8 * case["experts"] + weights
    nbytes += size * d * (t * live + t * k) + size * d * (t * k * live + t)
    flops = 2 * t * k * d * live
    if case["train"]:
        nbytes += size * d * (t * k * live + t) + size * d * (t * live + t * k) + weights
        flops *= 4
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------
# The results in 64 bits: torch's own lookup and norm, and autograd in float64
# ---------------------------------------------------------------------------
def _embedding_exact(s):
    case = s["case"]
    weight = s["weight"].detach().double().requires_grad_(case["train"])
    out = torch.nn.functional.embedding(s["index"], weight, padding_idx=s["padding"]) * case["scale"]
    if not case["train"]:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, weight, s["upstream"].double())]


def _norm_exact(s):
    w, b = (s[k].detach().double() if s[k] is not None else None for k in ("weight", "bias"))
    x = s["x"].detach().double()
    if not s["case"]["train"]:
        return [torch.nn.functional.layer_norm(x, x.shape[-1:], w, b, EPS)]
    leaves = [v.requires_grad_(True) for v in (x, w, b) if v is not None]
    out = torch.nn.functional.layer_norm(x, x.shape[-1:], w, b, EPS)
    return [out.detach(), *torch.autograd.grad(out, leaves, s["upstream"].double())]


def _experts_exact(s):
    case, index = s["case"], s["index"]
    t, k = index.shape
    d = case["dim"]
    drop = torch.zeros_like(index, dtype=torch.bool) if s["mask"] is None else (~s["mask"])[:, None].expand_as(index)
    # a number of its own for each entry, in the order of expert, token and choice
    entry = torch.arange(t * k, device=DEVICE).view(t, k)
    rank = (index.masked_fill(drop, case["experts"]) * (t * k) + entry).reshape(-1).argsort().argsort().view(t, k)
    counts = torch.bincount(index[~drop], minlength=case["experts"])
    x, made, w = (s[name].detach().double().requires_grad_(case["train"]) for name in ("x", "rows", "weights"))
    keep = (~drop).reshape(-1).nonzero()[:, 0]
    at = rank.reshape(-1)[keep]
    token = keep // k
    rows = torch.zeros(t * k, d, dtype=torch.float64, device=DEVICE).index_copy(0, at, x[token])
    y = torch.zeros(t, d, dtype=torch.float64, device=DEVICE)
    y = y.index_add(0, token, made[at] * w.reshape(-1)[keep][:, None])
    out = [torch.where(drop, -1 - rank, rank).int(), counts, rows.detach(), y.detach()]
    if not case["train"]:
        return out
    return out + list(torch.autograd.grad((rows, y), (x, made, w), [g.double() for g in s["upstream"]]))


def exact(case, seed):
    state = prepare(case, seed)
    return {"embedding": _embedding_exact, "layer_norm": _norm_exact, "experts": _experts_exact}[case["op"]](state)
