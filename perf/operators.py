"""The losses of a language model's training as measurable cases.

A case is a dict of plain values; "op" says which operator it takes:

* ``linear_ce``: softmax cross entropy of hidden states against a vocabulary
  projection, without the logits being kept; forward, or forward and backward
  to the hidden states and the projection;
* ``distill``: distillation from a teacher's top-K logits, over logits in
  fp32 / fp16 / bf16 that are a shifted view of a batch of sequences;
* ``router``: the balance loss, the z loss and the per-expert counts of a
  mixture-of-experts router.

``listed`` gives the cases, ``draw`` one more of the same ranges, ``prepare``
what a program holds before the call, ``run`` one pass (in plain torch
operations in 32 bits, or, with ``own``, through the library), ``work`` the
bytes and operations a pass cannot do without, and ``exact`` the results in
64 bits.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
IGNORE = -100
# What a gradient scaler multiplies a mean loss's gradient with in fp16, so
# that it stays above the type's smallest values.
SCALES = {"f32": 1.0, "f16": 8192.0, "bf16": 1.0}

# Most work of a drawn case: the largest listed one of its operator.
MAX_LINEAR = 4096 * 128256 * 2048
MAX_DISTILL = 4 * 1024 * 128256
MAX_ROUTER = 131072 * 256


def listed():
    return [
        # Scoring a handful of tokens (the last step of a small batch): the
        # projection is read once for few rows.
        {"name": "linear_score_bf16", "op": "linear_ce", "dtype": "bf16", "train": False, "rows": 8, "dim": 2048,
         "vocab": 128256, "ignored": 0.0, "reduction": "none", "z_loss": 0.0},
        # A small model's training step in fp32 at odd sizes: launches count.
        {"name": "linear_small_f32", "op": "linear_ce", "dtype": "f32", "train": True, "rows": 129, "dim": 200,
         "vocab": 1031, "ignored": 0.1, "reduction": "mean", "z_loss": 0.0},
        # Evaluation of a text: the loss of every token, no gradients.
        {"name": "linear_eval_bf16", "op": "linear_ce", "dtype": "bf16", "train": False, "rows": 4096, "dim": 4096,
         "vocab": 32000, "ignored": 0.0, "reduction": "none", "z_loss": 0.0},
        # Fine-tuning over a large vocabulary: prompts are ignored, the
        # normaliser is kept small by the z term.
        {"name": "linear_train_bf16", "op": "linear_ce", "dtype": "bf16", "train": True, "rows": 4096, "dim": 2048,
         "vocab": 128256, "ignored": 0.3, "reduction": "mean", "z_loss": 1e-4},
        # Policy gradients in fp16 over an odd vocabulary and an odd number of
        # tokens, each loss weighted by an advantage of its own.
        {"name": "linear_policy_f16", "op": "linear_ce", "dtype": "f16", "train": True, "rows": 2047, "dim": 768,
         "vocab": 50257, "ignored": 0.0, "reduction": "none", "z_loss": 0.0},
        # Pretraining in fp32.
        {"name": "linear_train_f32", "op": "linear_ce", "dtype": "f32", "train": True, "rows": 2048, "dim": 1024,
         "vocab": 32000, "ignored": 0.0, "reduction": "sum", "z_loss": 0.0},
        # Distillation step of a large vocabulary in bf16, 64 teacher logits a
        # token.
        {"name": "distill_train_bf16", "op": "distill", "dtype": "bf16", "train": True, "batch": 4, "seq": 1024,
         "vocab": 128256, "top": 64, "temperature": 1.0, "unused": 0.2},
        # The same in fp32 over an odd vocabulary with a softened teacher.
        {"name": "distill_train_f32", "op": "distill", "dtype": "f32", "train": True, "batch": 3, "seq": 512,
         "vocab": 50257, "top": 20, "temperature": 2.0, "unused": 0.0},
        # A few tokens of a validation batch in fp16.
        {"name": "distill_eval_f16", "op": "distill", "dtype": "f16", "train": False, "batch": 2, "seq": 17,
         "vocab": 32000, "top": 8, "temperature": 1.0, "unused": 0.0},
        # The router of a small batch over few experts.
        {"name": "router_small_f32", "op": "router", "dtype": "f32", "tokens": 512, "experts": 8, "top": 2,
         "masked": 0.0},
        # A training step's router with padding tokens.
        {"name": "router_train_bf16", "op": "router", "dtype": "bf16", "tokens": 16383, "experts": 64, "top": 6,
         "masked": 0.25},
        # The routers of a large batch over many experts.
        {"name": "router_large_f32", "op": "router", "dtype": "f32", "tokens": 131072, "experts": 256, "top": 8,
         "masked": 0.0},
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear_ce", "linear_ce", "distill", "router"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if op == "linear_ce":
        most = MAX_LINEAR // 8 if dtype == "f32" else MAX_LINEAR
        vocab = _log_int(rng, 100, 131072)
        dim = _log_int(rng, 32, 4096)
        if rng.random() < 0.6:
            dim = -(-dim // 64) * 64
        rows = _log_int(rng, 1, min(4096, most // (vocab * dim)))
        return {"op": op, "dtype": dtype, "train": rng.random() < 0.7, "rows": rows, "dim": dim, "vocab": vocab,
                "ignored": rng.choice([0.0, 0.0, 0.1, 0.5]), "reduction": rng.choice(["mean", "sum", "none"]),
                "z_loss": rng.choice([0.0, 1e-4])}
    if op == "distill":
        batch = rng.randint(1, 8)
        vocab = _log_int(rng, 300, 131072)
        most = MAX_DISTILL // 2 if dtype == "f32" else MAX_DISTILL
        return {"op": op, "dtype": dtype, "train": rng.random() < 0.7, "batch": batch,
                "seq": _log_int(rng, 2, max(2, min(2048, most // (batch * vocab)))), "vocab": vocab,
                "top": _log_int(rng, 1, 256), "temperature": rng.choice([1.0, 2.0, 0.7]),
                "unused": rng.choice([0.0, 0.2])}
    experts = rng.choice([8, 16, 60, 64, 128, 160, 256, 384])
    return {"op": op, "dtype": dtype, "tokens": _log_int(rng, 1, MAX_ROUTER // experts), "experts": experts,
            "top": rng.randint(1, 8), "masked": rng.choice([0.0, 0.25])}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _linear_state(case, gen):
    n, d, v, dtype = case["rows"], case["dim"], case["vocab"], DTYPES[case["dtype"]]
    # rows of the projection of norm 2, so that a normalised hidden state has
    # logits of standard deviation 2
    weight = torch.randn(v, d, device=DEVICE, generator=gen).mul_(2.0 / math.sqrt(d))
    target = torch.randint(0, v, (n,), device=DEVICE, generator=gen)
    x = torch.randn(n, d, device=DEVICE, generator=gen)
    # a trained model gives most targets a high logit: 3 from the noise's 2
    # per row up to about log(vocab) + 2
    known = (torch.rand(n, 1, device=DEVICE, generator=gen) < 0.7).float()
    x += known * weight[target] * ((math.log(v) + 1.0) / 4.0)
    # prompts and padding, in one run as they come at the front of a batch
    hidden = int(n * case["ignored"])
    target[:hidden] = IGNORE
    state = {"x": x.to(dtype), "weight": weight.to(dtype), "target": target}
    if case["reduction"] == "none":
        state["upstream"] = torch.randn(n, device=DEVICE, generator=gen)
    else:
        scale = SCALES[case["dtype"]] if case["reduction"] == "mean" else 1.0
        state["upstream"] = torch.full((), scale, device=DEVICE)
    if case["train"]:
        state["x"].requires_grad_(True)
        state["weight"].requires_grad_(True)
    return state


def _distill_state(case, gen):
    b, s, v, k, dtype = case["batch"], case["seq"], case["vocab"], case["top"], DTYPES[case["dtype"]]
    logits = torch.randn(b, s, v, device=DEVICE, generator=gen).mul_(2.0)
    # distinct tokens for each position: a random first one and a random odd
    # multiple of steps from it
    step = max(1, v // k)
    first = torch.randint(0, v, (b, s, 1), device=DEVICE, generator=gen)
    order = torch.rand(b, s, k, device=DEVICE, generator=gen).argsort(-1)
    index = (first + order * step) % v
    teacher = torch.randn(b, s, k, device=DEVICE, generator=gen).mul_(2.0).add_(6.0)
    teacher, by = teacher.sort(-1, descending=True)
    index = index.gather(-1, by)
    # the student agrees with the teacher up to noise
    near = teacher + torch.randn(b, s, k, device=DEVICE, generator=gen)
    logits.scatter_(-1, index, near)
    if case["unused"]:
        # a teacher cut to its nucleus leaves places of its top-K unused, and
        # some tokens (prompts) have no teacher at all
        keep = torch.randint(1, k + 1, (b, s, 1), device=DEVICE, generator=gen)
        teacher = teacher.masked_fill(torch.arange(k, device=DEVICE) >= keep, -math.inf)
        none = torch.rand(b, s, 1, device=DEVICE, generator=gen) < case["unused"]
        teacher = teacher.masked_fill(none, -math.inf)
    # the logits of positions 0 .. s-2 predict tokens 1 .. s-1
    view = logits.to(dtype)[:, :-1].detach()
    state = {"logits": view, "teacher": teacher[:, :-1].to(dtype).contiguous(), "index": index[:, :-1].contiguous(),
             "upstream": torch.full((), SCALES[case["dtype"]], device=DEVICE)}
    if case["train"]:
        view.requires_grad_(True)
    return state


def _router_state(case, gen):
    t, e, dtype = case["tokens"], case["experts"], DTYPES[case["dtype"]]
    bias = torch.randn(e, device=DEVICE, generator=gen)
    logits = (torch.randn(t, e, device=DEVICE, generator=gen) * 1.5 + bias).to(dtype)
    index = logits.float().topk(case["top"], -1).indices
    mask = None
    if case["masked"]:
        mask = torch.rand(t, device=DEVICE, generator=gen) >= case["masked"]
    return {"logits": logits.requires_grad_(True), "index": index, "mask": mask,
            "balance_weight": torch.full((), 0.01 * SCALES[case["dtype"]], device=DEVICE),
            "z_weight": torch.full((), 0.001 * SCALES[case["dtype"]], device=DEVICE)}


def prepare(case, seed):
    gen = _generator(seed)
    make = {"linear_ce": _linear_state, "distill": _distill_state, "router": _router_state}[case["op"]]
    return {"case": case, **make(case, gen)}


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def _linear_plain(s):
    case = s["case"]
    z, target = case["z_loss"], s["target"]
    x, w = s["x"].detach().float(), s["weight"].detach().float()
    live = target != IGNORE
    t = target.clamp(min=0)[:, None]
    logits = x @ w.t()
    at_target = logits.gather(1, t)[:, 0]
    top = logits.amax(1, keepdim=True)
    e = logits.sub_(top).exp_()
    total = e.sum(1, keepdim=True)
    lse = (total.log() + top)[:, 0]
    loss = torch.where(live, lse - at_target + z * lse * lse, 0.0)
    scale = live.float()
    if case["reduction"] == "mean":
        count = live.sum().clamp(min=1)
        loss = loss.sum() / count
        scale = scale / count
    elif case["reduction"] == "sum":
        loss = loss.sum()
    if not case["train"]:
        return [loss]
    g = s["upstream"] * scale
    grad = e.mul_((g * (1 + 2 * z * lse))[:, None] / total)
    grad.scatter_add_(1, t, -g[:, None])
    return [loss, (grad @ w).to(s["x"].dtype), (grad.t() @ x).to(s["weight"].dtype)]


def _distill_plain(s):
    case = s["case"]
    temp = case["temperature"]
    x = s["logits"].detach().float() / temp
    t = s["teacher"].float() / temp
    top = t.amax(-1, keepdim=True)
    live = top > -math.inf
    p = torch.where(live, (t - torch.where(live, top, 0.0)).exp(), 0.0)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    peak = x.amax(-1, keepdim=True)
    e = (x - peak).exp_()
    total = e.sum(-1, keepdim=True)
    logq = x.gather(-1, s["index"]) - peak - total.log()
    logp = torch.where(p > 0, p, 1.0).log()
    rows = (temp * temp) * torch.where(p > 0, p * (logp - logq), 0.0).sum(-1)
    if not case["train"]:
        return [rows]
    count = live.sum().clamp(min=1)
    loss = rows.sum() / count
    g = torch.where(live, s["upstream"] * temp / count, 0.0)
    grad = e.mul_(g / total)
    grad.scatter_add_(-1, s["index"], -g * p)
    return [loss, grad.to(s["logits"].dtype)]


def _router_plain(s):
    x = s["logits"].detach().float()
    tokens, experts = x.shape
    index = s["index"]
    live = s["mask"] if s["mask"] is not None else torch.ones(tokens, dtype=torch.bool, device=x.device)
    n = live.sum().clamp(min=1)
    picked = live[:, None].expand_as(index).to(torch.int64)
    counts = torch.zeros(experts, dtype=torch.int64, device=x.device)
    counts.scatter_add_(0, index.reshape(-1), picked.reshape(-1))
    top = x.amax(1, keepdim=True)
    e = (x - top).exp()
    total = e.sum(1, keepdim=True)
    lse = total.log() + top
    p = torch.where(live[:, None], e / total, 0.0)
    share = counts.float() / (n * index.shape[1])
    balance = experts * (share * (p.sum(0) / n)).sum()
    z = torch.where(live[:, None], lse * lse, 0.0).sum() / n
    mean_share = (p * share).sum(1, keepdim=True)
    grad = p * (s["balance_weight"] * experts / n * (share - mean_share) + s["z_weight"] * 2 / n * lse)
    return [balance, z, counts, grad.to(s["logits"].dtype)]


def _linear_own(s):
    import fuselse_amd

    case = s["case"]
    loss = fuselse_amd.linear_cross_entropy(s["x"], s["weight"], s["target"], ignore_index=IGNORE,
                                            reduction=case["reduction"], z_loss=case["z_loss"])
    if not case["train"]:
        return [loss]
    dx, dw = torch.autograd.grad(loss, (s["x"], s["weight"]), s["upstream"])
    return [loss.detach(), dx, dw]


def _distill_own(s):
    import fuselse_amd

    case = s["case"]
    loss = fuselse_amd.topk_distillation(s["logits"], s["teacher"], s["index"], temperature=case["temperature"],
                                         reduction="mean" if case["train"] else "none")
    if not case["train"]:
        return [loss]
    (grad,) = torch.autograd.grad(loss, s["logits"], s["upstream"])
    return [loss.detach(), grad]


def _router_own(s):
    import fuselse_amd

    out = fuselse_amd.router_balance(s["logits"], s["index"], mask=s["mask"])
    (grad,) = torch.autograd.grad((out.balance_loss, out.z_loss), s["logits"], (s["balance_weight"], s["z_weight"]))
    return [out.balance_loss.detach(), out.z_loss.detach(), out.counts, grad]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear_ce": _linear_own, "distill": _distill_own, "router": _router_own}[op](state)
    return {"linear_ce": _linear_plain, "distill": _distill_plain, "router": _router_plain}[op](state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "linear_ce":
        n, d, v = case["rows"], case["dim"], case["vocab"]
        live = n - int(n * case["ignored"])
        losses = 4 * n if case["reduction"] == "none" else 4
        nbytes = size * (live * d + v * d) + 8 * n + losses
        flops = 2 * live * d * v
        if case["train"]:
            nbytes += size * (n * d + v * d)
            flops *= 3
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "distill":
        rows = case["batch"] * (case["seq"] - 1)
        teacher = rows * case["top"] * (size + 8)
        passes = 2 if case["train"] else 1
        return {"bytes": size * rows * case["vocab"] * passes + teacher + (4 if case["train"] else 4 * rows), "flops": 3 * rows * case["vocab"] * passes}
    t, e, k = case["tokens"], case["experts"], case["top"]
    return {"bytes": 2 * size * t * e + 8 * t * k + (t if case["masked"] else 0) + 8 * e + 8, "flops": 8 * t * e}


# ---------------------------------------------------------------------------
# The results in 64 bits: torch's own log-sum-exp and autograd in float64
# ---------------------------------------------------------------------------
def _linear_exact(s):
    case = s["case"]
    x = s["x"].detach().double().requires_grad_(case["train"])
    w = s["weight"].detach().double().requires_grad_(case["train"])
    keep = (s["target"] != IGNORE).nonzero()[:, 0]
    logits = x[keep] @ w.t()
    lse = torch.logsumexp(logits, 1)
    rows = lse - logits[torch.arange(len(keep), device=DEVICE), s["target"][keep]] + case["z_loss"] * lse ** 2
    if case["reduction"] == "none":
        loss = torch.zeros(case["rows"], dtype=torch.float64, device=DEVICE).index_copy(0, keep, rows)
    else:
        loss = rows.sum() / (max(1, len(keep)) if case["reduction"] == "mean" else 1)
    if not case["train"]:
        return [loss]
    return [loss.detach(), *torch.autograd.grad(loss, (x, w), s["upstream"].double())]


def _distill_exact(s):
    case = s["case"]
    temp = case["temperature"]
    x = s["logits"].detach().double().requires_grad_(case["train"])
    t = s["teacher"].double() / temp
    taught = torch.isfinite(t).any(-1)
    logq = torch.log_softmax(x[taught] / temp, -1).gather(-1, s["index"][taught])
    logp = torch.log_softmax(t[taught], -1)
    p = logp.exp()
    terms = torch.where(p > 0, p * (logp.clamp(min=-1e6) - logq), 0.0)
    if not case["train"]:
        rows = torch.zeros(taught.shape, dtype=torch.float64, device=DEVICE)
        rows[taught] = temp ** 2 * terms.sum(-1)
        return [rows]
    loss = temp ** 2 * terms.sum() / max(1, int(taught.sum()))
    return [loss.detach(), *torch.autograd.grad(loss, x, s["upstream"].double())]


def _router_exact(s):
    x = s["logits"].detach().double().requires_grad_(True)
    live = s["mask"] if s["mask"] is not None else torch.ones(len(x), dtype=torch.bool, device=DEVICE)
    chosen = s["index"][live]
    counts = torch.bincount(chosen.reshape(-1), minlength=x.shape[1])
    n = max(1, len(chosen))
    probs = torch.softmax(x[live], 1)
    balance = x.shape[1] * (counts.double() / (n * chosen.shape[1]) * probs.sum(0) / n).sum()
    z = (torch.logsumexp(x[live], 1) ** 2).sum() / n
    (grad,) = torch.autograd.grad((balance, z), x, (s["balance_weight"].double(), s["z_weight"].double()))
    return [balance.detach(), z.detach(), counts, grad]


def exact(case, seed):
    state = prepare(case, seed)
    return {"linear_ce": _linear_exact, "distill": _distill_exact, "router": _router_exact}[case["op"]](state)
