"""The distillation and the router balance on logits with a large value in
common: neither depends on it, and neither may lose digits to it.

A difference from the maximum is exact where logits of a few units lie next to
a multiple of 2^-11 in fp32; what is left is half a step an operation."""

import math

import pytest
import torch

import fuselse_amd
from fuselse_amd import ext
from test_gpu_losses import E23, u, tiny, within

pytestmark = pytest.mark.gpu


def spread(cuda, shape, offset, seed, scale=2.0):
    """Multiples of 2^-11 of standard deviation `scale` around offset: exact in
    fp32 up to 2^12."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    return (torch.randn(*shape, device=cuda, generator=g) * scale * 2 ** 11).round() / 2 ** 11 + offset


def distill_exact(s, t, i, temp, up):
    """(losses, ds, bounds) in 64 bits of rows that all have a teacher."""
    sd, td = s.detach().double(), t.double()
    sd, td = sd - sd.amax(-1, keepdim=True), td - td.amax(-1, keepdim=True)
    lq, lp = torch.log_softmax(sd / temp, -1), torch.log_softmax(td / temp, -1)
    q, p = lq.exp(), lp.exp()
    v, k = s.shape[-1], t.shape[-1]
    terms = p * (lp - lq.gather(-1, i))
    loss = temp ** 2 * terms.sum(-1)
    # an exponent d / T is off by three roundings of its size, log2 e's and 1 / T's
    # among them: sums by the mean of that, and by their additions (v / 256 a
    # thread one after another, 64 for the merges); the log of a sum, its storing
    # and its subtraction by half a step of its size each
    step = 2.0 ** -22
    log_sum = lambda x: torch.logsumexp(x / temp, -1) * 2.0 ** -21
    dq = (q * sd.abs() / temp).sum(-1) * step + (v / 256 + 64) * E23 + log_sum(sd)
    dp = (p * td.abs() / temp).sum(-1) * step + (k / 64 + 64) * E23 + log_sum(td)
    size = (p * (lp.abs() + lq.gather(-1, i).abs())).sum(-1)
    # a probability's error counts with the size of its term
    err = (p * ((td.abs() / temp * step + dp[..., None]) * (1 + (lp - lq.gather(-1, i)).abs()))).sum(-1)
    loss_b = temp ** 2 * (dq + dp + err + size * (k / 64 + 16) * E23)
    g = up.double()[..., None] * temp
    ps = torch.zeros_like(q).scatter_add_(-1, i, p)
    ds = g * (q - ps)
    pe = torch.zeros_like(q).scatter_add_(-1, i, p * (td.abs() / temp * step + dp[..., None] + 2.0 ** -21))
    ds_b = g.abs() * (q * (sd.abs() / temp * step + dq[..., None] + 2.0 ** -21) + pe + (q + ps) * 2.0 ** -22) \
        + u(s.dtype) * ds.abs() + 2.0 ** -126 * (1 + g.abs())
    return loss, ds, loss_b, ds_b


OFFSETS = [0.0, 100.0, -1000.0, 2000.0]


@pytest.mark.parametrize("offset", OFFSETS)
@pytest.mark.parametrize("rows,v,k,temp", [(5, 4096, 16, 1.0), (3, 50257, 200, 1.0), (33, 1001, 5, 2.0),
                                           (2000, 300, 8, 0.7), (4, 40000, 64, 3.0)])
def test_distillation_of_shifted_logits_loss(cuda, rows, v, k, temp, offset):
    print(f"case distill offset loss {rows} {v} {k} {temp} {offset}", flush=True)
    s, t = spread(cuda, (rows, v), offset, v), spread(cuda, (rows, k), -offset, k)
    i = torch.rand(rows, v, device=cuda).argsort(-1)[:, :k].contiguous()
    up = torch.ones(rows, device=cuda)
    want, _, b, _ = distill_exact(s, t, i, temp, up)
    within(fuselse_amd.topk_distillation(s, t, i, temperature=temp, reduction="none"), want, b, "loss")


@pytest.mark.parametrize("offset", OFFSETS)
@pytest.mark.parametrize("rows,v,k,temp", [(5, 4096, 16, 1.0), (3, 50257, 200, 1.0), (33, 1001, 5, 2.0),
                                           (2000, 300, 8, 0.7), (4, 40000, 64, 3.0)])
def test_distillation_of_shifted_logits_gradient(cuda, rows, v, k, temp, offset):
    print(f"case distill offset gradient {rows} {v} {k} {temp} {offset}", flush=True)
    s, t = spread(cuda, (rows, v), offset, v), spread(cuda, (rows, k), -offset, k)
    i = torch.rand(rows, v, device=cuda).argsort(-1)[:, :k].contiguous()
    up = torch.randn(rows, device=cuda, generator=torch.Generator(device=cuda).manual_seed(3))
    _, want, _, b = distill_exact(s, t, i, temp, up)
    s.requires_grad_(True)
    loss = fuselse_amd.topk_distillation(s, t, i, temperature=temp, reduction="none")
    within(torch.autograd.grad(loss, s, up)[0], want, b, "ds")


def test_distillation_gradient_without_pairs(cuda):
    """The checked calls with and without pairs: the same loss, the gradient
    off by the log-sum-exps' rounding alone."""
    print("case distill pairs", flush=True)
    rows, v, k = 6, 3001, 12
    s, t = spread(cuda, (rows, v), 0.0, 1), spread(cuda, (rows, k), 0.0, 2)
    i = torch.rand(rows, v, device=cuda).argsort(-1)[:, :k].contiguous()
    up = torch.ones(rows, device=cuda)
    loss, lse, tlse, norm = ext.topk_distillation(s, t, i, 2.0, "none")
    loss2, _, _, _, pairs = ext.topk_distillation(s, t, i, 2.0, "none", with_pairs=True)
    assert torch.equal(loss, loss2) and pairs.shape == (rows, 4)
    a = ext.topk_distillation_backward(up, s, t, i, lse, tlse, norm, 2.0)
    b = ext.topk_distillation_backward(up, s, t, i, lse, tlse, norm, 2.0, pairs=pairs)
    _, want, _, bound = distill_exact(s, t, i, 2.0, up)
    within(b, want, bound, "with pairs")
    # exponents, and with them an element's parts, off by a step of 16 at most
    within(a, want, bound + 2.0 ** -18 * want.abs().amax(1, keepdim=True), "without")
    with pytest.raises(RuntimeError, match="pairs must be"):
        ext.topk_distillation_backward(up, s, t, i, lse, tlse, norm, 2.0, pairs=pairs[:3])


@pytest.mark.parametrize("offset", [0.0, 100.0, -1000.0, 2000.0])
@pytest.mark.parametrize("tokens,e,k", [(300, 8, 2), (1000, 60, 4), (700, 256, 8), (5000, 384, 6), (400, 1000, 2)])
def test_router_balance_of_shifted_logits(cuda, tokens, e, k, offset):
    print(f"case router offset {tokens} {e} {k} {offset}", flush=True)
    x = spread(cuda, (tokens, e), offset, e)
    index = x.topk(k, 1).indices
    x.requires_grad_(True)
    out = fuselse_amd.router_balance(x, index)
    (gx,) = torch.autograd.grad(out.balance_loss, x)
    xd = x.detach().double()
    xd = xd - xd.amax(1, keepdim=True)
    p = torch.softmax(xd, 1)
    f = torch.bincount(index.reshape(-1), minlength=e).double() / (tokens * k)
    balance = e * (f * p.mean(0)).sum()
    dot = (p * f).sum(1, keepdim=True)
    want = p * (e / tokens * (f - dot))
    # an exponent is off by three roundings of its size, a sum by the mean of that
    # and by its additions: 16 a lane, and 64 for the merges
    rel = xd.abs() * 2.0 ** -22
    rel = rel + (p * rel).sum(1, keepdim=True) + (e / 64 + 80) * E23
    # a lane adds its tokens' probabilities one after another
    bal_b = e * (f * (p * rel).mean(0)).sum() + balance * (tokens / 256 + 64) * E23
    within(out.balance_loss, balance, bal_b, "balance")
    size = p * (e / tokens * (f + dot))
    bound = size * (rel + 2.0 ** -21) + p * (e / tokens) * (p * f * (rel + (e / 64 + 16) * E23)).sum(1, keepdim=True) \
        + 2.0 ** -126
    within(gx, want, bound + u(torch.float32) * want.abs(), "dlogits")
