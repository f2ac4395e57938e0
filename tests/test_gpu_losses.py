"""The training losses (linear cross entropy, distillation from top logits,
router balance) against plain implementations in 64 bits, forward and
backward, at the sizes and masks where the kernels change path.

Tolerances.  A rounding to type t is off by at most half a step, eps_t / 2
relative (u(t) below).  An fp32 sum of n terms is off by at most n 2^-23 of the
sum of their magnitudes (2^-23 a step covers an accumulator that truncates).
fp32 operands' products are 2^-21 off (three of four partial products of two
fp16 parts, six of nine of three bf16 parts)."""

import math

import pytest
import torch

import fuselse_amd
from fuselse_amd import ext

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
E23 = 2.0 ** -23


def u(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the smallest step of the type: what an underflow loses."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def product_loss(dtype):
    return 2.0 ** -21 if dtype == torch.float32 else 0.0


def within(got, want, bound, what):
    got, want = got.detach().double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), (what, "NaN in other places")
    off = (got - want).abs()
    off = torch.where(got.isnan() | (got == want), torch.zeros_like(off), off)
    bad = ~(off <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((off / (bound + 1e-300)).max()))


# ---------------------------------------------------------------------------
# Linear cross entropy
# ---------------------------------------------------------------------------
def linear_inputs(cuda, n, d, v, dtype, ignored=0.0, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    w = (torch.randn(v, d, device=cuda, generator=g) * (2.0 / math.sqrt(d))).to(dtype)
    t = torch.randint(0, v, (n,), device=cuda, generator=g)
    x = torch.randn(n, d, device=cuda, generator=g)
    known = (torch.rand(n, 1, device=cuda, generator=g) < 0.7).float()
    x = (x + known * w[t].float() * ((math.log(v) + 1) / 4)).to(dtype)
    if ignored:
        t[torch.rand(n, device=cuda, generator=g) < ignored] = -100
    return x, w, t


def linear_reference(x, w, t, ignore, reduction, z, upstream):
    """(loss, dx, dw, bounds of the three) in 64 bits; t holds no bad target."""
    dtype = x.dtype
    xd, wd = x.detach().double(), w.detach().double()
    n, d = xd.shape
    live = t != ignore
    xd = torch.where(live[:, None], xd, 0.0)
    ts = torch.where(live, t, 0)
    logits = xd @ wd.t()
    lse = torch.logsumexp(logits, 1)
    rows = torch.where(live, lse - logits.gather(1, ts[:, None])[:, 0] + z * lse ** 2, 0.0)
    count = max(1, int(live.sum()))
    by = 1.0 / count if reduction == "mean" else 1.0
    loss = rows if reduction == "none" else rows.sum() * by
    g = torch.where(live, upstream.double() * by, 0.0)
    a, b = g * (1 + 2 * z * lse), -g
    p = (logits - lse[:, None]).exp()
    onehot = torch.zeros_like(p).scatter_(1, ts[:, None], 1.0)
    G = a[:, None] * p + b[:, None] * onehot
    dx, dw = G @ wd, G.t() @ xd
    # a logit's error, the same for all of a row
    size = (xd.abs() @ wd.abs().t()).amax(1)
    dl = size * (d * E23 + product_loss(dtype)) + 2.0 ** -22 * lse.abs()
    # the log of a sum: at most 256 additions one after another, and the exponentials
    dlse = dl + 2.0 ** -15
    rows_b = (dl + dlse) * (1 + 2 * z * lse.abs()) + 2.0 ** -22 * (rows.abs() + lse.abs())
    rows_b = torch.where(live, rows_b, 0.0)
    loss_b = rows_b if reduction == "none" else rows_b.sum() * by + 2.0 ** -22 * loss.abs()
    g_abs = a.abs()[:, None] * p + b.abs()[:, None] * onehot
    rel = (dl + dlse)[:, None] + u(dtype) + product_loss(dtype) + 2.0 ** -20
    top = float(torch.maximum(a.abs(), b.abs()).max()) if n else 0.0
    under = tiny(dtype) * top / 2 ** 9 if dtype == torch.float16 else 0.0
    # an fp32 exponential below 2^-126 is 0, and so is a bf16 part of G, which
    # is taken at least 2^9 / top times larger: 2^-126 top (1 + 3 2^-9) at most
    under += 2.0 ** -125 * top
    v = wd.shape[0]
    err = g_abs * rel + under
    dx_b = err @ wd.abs() + (g_abs @ wd.abs()) * (v * E23) + u(dtype) * dx.abs() + tiny(dtype)
    dw_b = err.t() @ xd.abs() + (g_abs.t() @ xd.abs()) * (n * E23) + u(dtype) * dw.abs() + tiny(dtype)
    # what is not live is exactly zero
    dx_b = torch.where(live[:, None], dx_b, 0.0)
    return loss, dx, dw, loss_b, dx_b, dw_b


def linear_upstream(cuda, n, reduction, seed=1):
    g = torch.Generator(device=cuda).manual_seed(seed)
    if reduction == "none":
        return torch.randn(n, device=cuda, generator=g)
    return torch.full((), 1.5, device=cuda)


def check_linear(x, w, t, reduction, z=0.0, ignore=-100):
    up = linear_upstream(x.device, x.shape[0], reduction)
    x.requires_grad_(True)
    w.requires_grad_(True)
    loss = fuselse_amd.linear_cross_entropy(x, w, t, ignore_index=ignore, reduction=reduction, z_loss=z)
    assert loss.dtype == torch.float32
    dx, dw = torch.autograd.grad(loss, (x, w), up)
    assert dx.dtype == x.dtype and dw.dtype == w.dtype and dx.shape == x.shape and dw.shape == w.shape
    want, rx, rw, b, bx, bw = linear_reference(x, w, t, ignore, reduction, z, up)
    within(loss, want, b, "loss")
    within(dx, rx, bx, "dx")
    within(dw, rw, bw, "dw")
    # without gradients few rows take another path
    plain = fuselse_amd.linear_cross_entropy(x.detach(), w.detach(), t, ignore_index=ignore, reduction=reduction,
                                             z_loss=z)
    within(plain, want, b, "loss without gradients")


LINEAR_SHAPES = [(1, 1, 1), (1, 64, 100), (2, 33, 7), (5, 130, 1000), (17, 64, 65), (64, 31, 129), (65, 128, 300),
                 (129, 200, 1031), (300, 72, 515), (257, 320, 257), (40, 1000, 2049), (513, 64, 97)]


@pytest.mark.parametrize("n,d,v", LINEAR_SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_shapes(cuda, n, d, v, dtype):
    print(f"case linear {n} {d} {v} {dtype}", flush=True)
    x, w, t = linear_inputs(cuda, n, d, v, dtype, ignored=0.2)
    check_linear(x, w, t, "mean", z=1e-2)


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("ignored", [0.0, 0.6, 1.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_reductions_and_ignored_rows(cuda, reduction, ignored, dtype):
    print(f"case linear {reduction} {ignored} {dtype}", flush=True)
    x, w, t = linear_inputs(cuda, 150, 96, 333, dtype, ignored=ignored, seed=3)
    if ignored == 1.0:
        t.fill_(-100)
    check_linear(x, w, t, reduction, z=1e-3 if reduction != "sum" else 0.0)


@pytest.mark.parametrize("n,d,v", [(70, 40, 16500), (300, 64, 40000), (8, 128, 50257), (1, 200, 32003)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_several_pieces(cuda, n, d, v, dtype):
    print(f"case linear pieces {n} {d} {v} {dtype}", flush=True)
    x, w, t = linear_inputs(cuda, n, d, v, dtype, ignored=0.1, seed=4)
    t[0] = v - 1
    check_linear(x, w, t, "sum")


@pytest.mark.parametrize("n", [1, 3, 16, 17, 33, 64, 65])
@pytest.mark.parametrize("d,v", [(64, 1), (68, 33), (192, 4097), (320, 70001), (1088, 32003)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_few_rows(cuda, n, d, v, dtype):
    """Rows that one pass over the projection serves, K ending inside a stage,
    vocabularies of less and more than a row group a wave."""
    print(f"case linear few {n} {d} {v} {dtype}", flush=True)
    x, w, t = linear_inputs(cuda, n, d, v, dtype, ignored=0.3, seed=n)
    t[-1] = v - 1
    check_linear(x, w, t, "none", z=1e-3)


@pytest.mark.parametrize("n,d,v", [(700, 130, 5000), (1500, 320, 9000), (130, 500, 20000), (1100, 64, 300),
                                   (260, 2048, 520), (3000, 200, 70), (2000, 66, 3)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_tile_sizes(cuda, n, d, v, dtype):
    """Sizes whose products take the large and the middle tiles, with several
    tiles a block and several splits."""
    print(f"case linear tiles {n} {d} {v} {dtype}", flush=True)
    x, w, t = linear_inputs(cuda, n, d, v, dtype, ignored=0.25, seed=v)
    check_linear(x, w, t, "sum", z=1e-4)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_ignored_rows_may_hold_anything(cuda, dtype):
    print(f"case linear garbage {dtype}", flush=True)
    x, w, t = linear_inputs(cuda, 200, 64, 300, dtype, ignored=0.5, seed=5)
    bad = t == -100
    clean = fuselse_amd.linear_cross_entropy(x, w, t)
    x[bad] = float("nan")
    x[bad.nonzero()[0, 0]] = float("inf")
    x.requires_grad_(True)
    w.requires_grad_(True)
    loss = fuselse_amd.linear_cross_entropy(x, w, t)
    dx, dw = torch.autograd.grad(loss, (x, w))
    assert torch.equal(loss.detach(), clean)
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all() and (dx[bad] == 0).all()


def test_linear_bad_target_is_nan(cuda):
    print("case linear bad target", flush=True)
    x, w, t = linear_inputs(cuda, 70, 64, 300, torch.bfloat16, seed=6)
    want = fuselse_amd.linear_cross_entropy(x, w, t, reduction="none")
    t2 = t.clone()
    t2[3], t2[40] = 300, -1
    x.requires_grad_(True)
    loss = fuselse_amd.linear_cross_entropy(x, w, t2, reduction="none")
    bad = torch.zeros(70, dtype=torch.bool, device=cuda)
    bad[[3, 40]] = True
    assert loss[bad].isnan().all() and torch.equal(loss[~bad].detach(), want[~bad])
    (dx,) = torch.autograd.grad(loss, x, torch.ones_like(loss))
    assert dx[bad].isnan().all() and torch.isfinite(dx[~bad]).all()
    assert fuselse_amd.linear_cross_entropy(x.detach(), w, t2).isnan()


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_strides_dims_and_integer_types(cuda, dtype):
    print(f"case linear strides {dtype}", flush=True)
    x, w, t = linear_inputs(cuda, 60, 130, 257, dtype, ignored=0.2, seed=7)
    want = fuselse_amd.linear_cross_entropy(x, w, t, reduction="none")
    wide = torch.full((60, 143), 7.0, dtype=dtype, device=cuda)
    wide[:, 5:135] = x
    wwide = torch.full((257, 131), -3.0, dtype=dtype, device=cuda)
    wwide[:, 1:] = w
    got = fuselse_amd.linear_cross_entropy(wide[:, 5:135], wwide[:, 1:], t.to(torch.int32), reduction="none")
    assert torch.equal(got, want)
    got = fuselse_amd.linear_cross_entropy(x.view(3, 4, 5, 130), w, t.view(3, 4, 5), reduction="none")
    assert got.shape == (3, 4, 5) and torch.equal(got.reshape(-1), want)
    # a head kept as (D, V), and hidden states of a shifted batch
    xs = torch.zeros(3, 21, 130, dtype=dtype, device=cuda)
    xs[:, :-1] = x.view(3, 20, 130)
    xs.requires_grad_(True)
    wt = w.t().contiguous().requires_grad_(True)
    loss = fuselse_amd.linear_cross_entropy(xs[:, :-1], wt.t(), t.view(3, 20), reduction="none")
    assert torch.equal(loss.detach().reshape(-1), want)
    up = linear_upstream(cuda, 60, "none").view(3, 20)
    gx, gw = torch.autograd.grad(loss, (xs, wt), up)
    x.requires_grad_(True)
    w.requires_grad_(True)
    rx, rw = torch.autograd.grad(fuselse_amd.linear_cross_entropy(x, w, t, reduction="none"), (x, w), up.reshape(-1))
    assert torch.equal(gx[:, :-1].reshape(60, 130), rx) and (gx[:, -1] == 0).all() and torch.equal(gw.t(), rw)


def test_linear_one_gradient_only_and_expanded_upstream(cuda):
    print("case linear one gradient", flush=True)
    x, w, t = linear_inputs(cuda, 90, 64, 200, torch.float16, seed=8)
    xg, wg = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    both = torch.autograd.grad(fuselse_amd.linear_cross_entropy(xg, wg, t, reduction="none").sum(), (xg, wg))
    (dx,) = torch.autograd.grad(fuselse_amd.linear_cross_entropy(xg, w, t, reduction="none").sum(), xg)
    (dw,) = torch.autograd.grad(fuselse_amd.linear_cross_entropy(x, wg, t, reduction="none").sum(), wg)
    assert torch.equal(dx, both[0]) and torch.equal(dw, both[1])


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_linear_no_rows(cuda, reduction):
    print(f"case linear no rows {reduction}", flush=True)
    x = torch.zeros(0, 64, device=cuda, requires_grad=True)
    w = torch.ones(10, 64, device=cuda, requires_grad=True)
    loss = fuselse_amd.linear_cross_entropy(x, w, torch.zeros(0, dtype=torch.int64, device=cuda), reduction=reduction)
    assert loss.shape == ((0,) if reduction == "none" else ()) and (loss == 0).all()
    dx, dw = torch.autograd.grad(loss, (x, w), torch.ones_like(loss))
    assert dx.shape == (0, 64) and (dw == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_large_logits(cuda, dtype):
    """Logits of some thousands, whose exponentials overflow without the
    running maximum."""
    print(f"case linear large {dtype}", flush=True)
    x, w, t = linear_inputs(cuda, 50, 64, 400, dtype, seed=9)
    check_linear((x * 30).to(dtype), (w * 30).to(dtype), t, "none")


def test_linear_fp16_small_upstream(cuda):
    """Small upstream gradients keep their digits inside the products: the
    results differ by the results' own underflow alone."""
    print("case linear small upstream", flush=True)
    x, w, t = linear_inputs(cuda, 128, 64, 300, torch.float16, seed=10)
    x.requires_grad_(True)
    small = fuselse_amd.linear_cross_entropy(x, w, t, reduction="none")
    up = torch.full((128,), 2.0 ** -8, device=cuda)
    (a,) = torch.autograd.grad(small, x, up)
    x2 = x.detach().clone().requires_grad_(True)
    (b,) = torch.autograd.grad(fuselse_amd.linear_cross_entropy(x2, w, t, reduction="none"), x2, up * 2.0 ** 8)
    # powers of two: the same digits up to the results' own underflow
    assert ((a.double() * 2.0 ** 8 - b.double()).abs() <= tiny(torch.float16) * 2.0 ** 8).all()


@pytest.mark.parametrize("large", ["weight", "input"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_gradients_near_the_types_largest(cuda, dtype, large):
    """Gradients of the size of weight (of input) while it is 2^116 times
    larger and its partner as much smaller: sums on the way stay finite."""
    print(f"case linear near the largest {dtype} {large}", flush=True)
    x, w, t = linear_inputs(cuda, 20, 64, 300, dtype, ignored=0.2, seed=12)
    # no element of the small side is below the type's smallest normal
    x, w = (torch.where(v.abs() < 2.0 ** -6, 2.0 ** -6, v) for v in (x, w))
    e = 2.0 ** (116 if large == "weight" else -116)
    x, w = (x * (1 / e)).requires_grad_(True), (w * e).requires_grad_(True)
    up = linear_upstream(cuda, 20, "none")
    loss = fuselse_amd.linear_cross_entropy(x, w, t, reduction="none")
    want, rx, rw, b, bx, bw = linear_reference(x, w, t, -100, "none", 0.0, up)
    within(loss, want, b, "loss")
    dx, dw = torch.autograd.grad(loss, (x, w), up)
    if large == "weight":
        within(dx, rx, bx, "dx")
    else:
        within(dw, rw, bw, "dw")


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_few_rows_at_any_alignment(cuda, dtype):
    """Rows of x that begin at odd elements, where one pass serves them."""
    print(f"case linear few unaligned {dtype}", flush=True)
    x, w, t = linear_inputs(cuda, 7, 192, 4000, dtype, seed=13)
    for off, stride in ((1, 193), (3, 201), (0, 192)):
        room = torch.full((7 * stride + off,), float("nan"), device=cuda, dtype=dtype)
        there = room[off:].as_strided((7, 192), (stride, 1))
        there.copy_(x)
        got = fuselse_amd.linear_cross_entropy(there, w, t, reduction="none")
        assert torch.equal(got, fuselse_amd.linear_cross_entropy(x, w, t, reduction="none")), (off, stride)


def test_linear_gradient_against_differences(cuda):
    print("case linear differences", flush=True)
    x, w, t = linear_inputs(cuda, 6, 16, 40, torch.float32, seed=11)
    x.requires_grad_(True)
    w.requires_grad_(True)
    dx, dw = torch.autograd.grad(fuselse_amd.linear_cross_entropy(x, w, t, reduction="sum", z_loss=0.01), (x, w))
    g = torch.Generator(device=cuda).manual_seed(2)
    for leaf, grad in ((x, dx), (w, dw)):
        d = torch.randn(leaf.shape, device=cuda, generator=g)
        d = d / d.norm()
        h = 2.0 ** -6
        with torch.no_grad():
            a = leaf.detach() + h * d
            b = leaf.detach() - h * d
            la = fuselse_amd.linear_cross_entropy(*((a, w) if leaf is x else (x, a)), t, reduction="none", z_loss=0.01)
            lb = fuselse_amd.linear_cross_entropy(*((b, w) if leaf is x else (x, b)), t, reduction="none", z_loss=0.01)
        num = float((la.double() - lb.double()).sum()) / (2 * h)
        want = float((grad.double() * d.double()).sum())
        # third derivatives of at most 8 |logit change|^3 a row: 6 h^2 8 (|w| = 2)^3 / 6; rounding 6 rows x 40 x 2^-22 / h
        assert abs(num - want) <= 64 * h * h + 6 * 40 * 2.0 ** -22 / h, (num, want)


def test_linear_twice_differentiable_is_refused(cuda):
    print("case linear double backward", flush=True)
    x, w, t = linear_inputs(cuda, 6, 16, 40, torch.float32)
    x.requires_grad_(True)
    (g,) = torch.autograd.grad(fuselse_amd.linear_cross_entropy(x, w, t), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# ---------------------------------------------------------------------------
# Distillation
# ---------------------------------------------------------------------------
def distill_inputs(cuda, lead, v, k, dtype, tdtype, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    s = (torch.randn(*lead, v, device=cuda, generator=g) * 3).to(dtype)
    t = (torch.randn(*lead, k, device=cuda, generator=g) * 2).to(tdtype)
    i = torch.rand(*lead, v, device=cuda, generator=g).argsort(-1)[..., :k].contiguous() if k <= v else \
        torch.randint(0, v, (*lead, k), device=cuda, generator=g)
    return s, t, i


def distill_reference(s, t, i, temp, reduction, up):
    """(loss, ds, bounds) in 64 bits; indices of unused entries may be anything."""
    dtype = s.dtype
    v = s.shape[-1]
    sd, td = s.detach().double() / temp, t.double() / temp
    used = td > -math.inf
    live = used.any(-1)
    td = torch.where(live[..., None], td, 0.0)
    p = torch.softmax(td, -1) * live[..., None] if t.shape[-1] else torch.zeros_like(td)
    ii = torch.where(used, i, 0)
    lse = torch.logsumexp(sd, -1, keepdim=True)
    terms = torch.where(p > 0, p * ((p + (p == 0)).log() - (sd.gather(-1, ii) - lse)), 0.0)
    rows = temp ** 2 * terms.sum(-1)
    by = 1.0 / max(1, int(live.sum())) if reduction == "mean" else 1.0
    loss = rows if reduction == "none" else rows.sum() * by
    g = (up.double() * by).expand(live.shape) * live * temp
    q = (sd - lse).exp()
    ps = torch.zeros_like(q).scatter_add_(-1, ii, p)
    ds = g[..., None] * (q - ps)
    # exponents are rounded: 2^-22 of their magnitude, and of the two log-sum-exps'
    big = torch.where(sd.isfinite(), sd.abs(), 0.0).amax(-1) + lse[..., 0].abs() + 1
    if t.shape[-1]:
        big = big + torch.where(td.isfinite(), td.abs(), 0.0).amax(-1)
    # a lane folds v / 256 values one after another at most, with the merges
    rel = big * 2.0 ** -21 + (v / 256 + 64) * E23
    rows_b = temp ** 2 * (rel + (t.shape[-1] / 64 + 8) * E23 * terms.abs().sum(-1) + rel * terms.abs().sum(-1)) * live
    loss_b = rows_b if reduction == "none" else rows_b.sum() * by + 2.0 ** -22 * loss.abs()
    ds_b = g.abs()[..., None] * (rel[..., None] + 2.0 ** -20 + t.shape[-1] * E23) * (q + ps) + u(dtype) * ds.abs() \
        + tiny(dtype) + g.abs()[..., None] * 2.0 ** -126
    return loss, ds, loss_b, ds_b


def check_distill(s, t, i, temp, reduction):
    rows = s.shape[:-1]
    gen = torch.Generator(device=s.device).manual_seed(5)
    up = torch.randn(rows, device=s.device, generator=gen) if reduction == "none" else \
        torch.full((), 0.75, device=s.device)
    s = s.detach().requires_grad_(True)
    loss = fuselse_amd.topk_distillation(s, t, i, temperature=temp, reduction=reduction)
    (ds,) = torch.autograd.grad(loss, s, up)
    assert loss.dtype == torch.float32 and ds.dtype == s.dtype
    want, rs, b, bs = distill_reference(s, t, i, temp, reduction, up)
    within(loss, want, b, "loss")
    within(ds, rs, bs, "ds")
    assert torch.equal(fuselse_amd.topk_distillation(s.detach(), t, i, temperature=temp, reduction=reduction),
                       loss.detach())
    return ds


DISTILL_SHAPES = [((1,), 1, 1), ((3,), 5, 2), ((2,), 64, 64), ((7,), 1000, 10), ((33,), 4099, 65), ((5,), 32000, 200),
                  ((2,), 128256, 1024), ((300,), 513, 3), ((2000,), 77, 5), ((3,), 20, 30)]


@pytest.mark.parametrize("lead,v,k", DISTILL_SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_distill_shapes(cuda, lead, v, k, dtype):
    print(f"case distill {lead} {v} {k} {dtype}", flush=True)
    s, t, i = distill_inputs(cuda, lead, v, k, dtype, dtype, seed=v)
    check_distill(s, t, i, 1.0, "mean")


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("temp", [0.5, 3.0])
@pytest.mark.parametrize("tdtype", DTYPES)
def test_distill_reductions_temperatures_and_teacher_types(cuda, reduction, temp, tdtype):
    print(f"case distill {reduction} {temp} {tdtype}", flush=True)
    s, t, i = distill_inputs(cuda, (4, 9), 2050, 16, torch.bfloat16, tdtype, seed=2)
    t[0, 3] = -math.inf
    t[1, :, 5:] = -math.inf
    i[1, :, 5:] = -7                      # unused places may hold any index
    i[0, 3, 0] = 10 ** 12
    check_distill(s, t, i, temp, reduction)


@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_distill_no_teacher(cuda, reduction):
    print(f"case distill no teacher {reduction}", flush=True)
    s, t, i = distill_inputs(cuda, (6,), 300, 4, torch.float32, torch.float32)
    t.fill_(-math.inf)
    s[2] = float("nan")                   # a row without a teacher may hold anything
    ds = s.requires_grad_(True)
    loss = fuselse_amd.topk_distillation(s, t, i, reduction=reduction)
    (ds,) = torch.autograd.grad(loss.sum(), s)
    assert (loss == 0).all() and (ds == 0).all()
    loss = fuselse_amd.topk_distillation(s.detach(), t[:, :0], i[:, :0], reduction=reduction)
    assert (loss == 0).all()


def test_distill_repeated_index_takes_the_sum(cuda):
    print("case distill repeated", flush=True)
    for dtype in DTYPES:
        s, t, i = distill_inputs(cuda, (5,), 9001, 12, dtype, torch.float32, seed=4)
        i[:, 3] = i[:, 0]
        i[:, 7] = i[:, 0]
        i[:, 11] = i[:, 10]
        first = check_distill(s, t, i, 2.0, "sum")
        assert torch.equal(first, check_distill(s, t, i, 2.0, "sum"))


@pytest.mark.parametrize("v", [8193, 8195, 8197, 8199, 16385, 16393, 16399, 32777])
@pytest.mark.parametrize("dtype", DTYPES)
def test_distill_teacher_at_a_rows_end(cuda, v, dtype):
    """Rows a little longer than whole chunks of the backward, at every phase
    of their first line, with the teacher's entries in the last columns."""
    print(f"case distill end {v} {dtype}", flush=True)
    s, t, i = distill_inputs(cuda, (64,), v, 12, dtype, dtype, seed=v)
    i[:] = v - 1 - torch.arange(12, device=cuda)
    check_distill(s, t, i, 1.0, "none")


@pytest.mark.parametrize("k", [3, 4, 5, 63, 255, 256, 257, 1021, 1022, 1023, 1024])
def test_distill_many_entries_in_one_chunk(cuda, k):
    """All of a row's entries in one chunk of the backward, most of them several
    times, unused ones between them."""
    print(f"case distill many {k}", flush=True)
    for dtype in DTYPES:
        s, t, i = distill_inputs(cuda, (9,), 300, k, dtype, torch.float32, seed=k)
        i %= 150
        t[:, 1::7] = -math.inf
        check_distill(s, t, i, 1.0, "none")


def test_distill_masked_student_and_special_values(cuda):
    print("case distill special", flush=True)
    for dtype in DTYPES:
        s, t, i = distill_inputs(cuda, (8,), 5000, 6, dtype, torch.float32, seed=6)
        low = torch.finfo(dtype).min
        for r in range(8):
            free = torch.ones(5000, dtype=torch.bool, device=cuda)
            free[i[r]] = False
            s[r, free & (torch.arange(5000, device=cuda) % 3 == 0)] = -math.inf if r % 2 else low
        check_distill(s, t, i, 1.0, "none")
        # a used entry the student masks: infinite loss, gradient -p there
        s[0, i[0, 0]] = -math.inf
        x = s.clone().requires_grad_(True)
        loss = fuselse_amd.topk_distillation(x, t, i, reduction="none")
        (ds,) = torch.autograd.grad(loss, x, torch.ones_like(loss))
        assert loss[0] == math.inf and torch.isfinite(loss[1:]).all() and torch.isfinite(ds).all()
        want = -torch.softmax(t[0].double(), 0)[0]
        assert abs(float(ds[0, i[0, 0]]) - float(want)) <= float(abs(want)) * (u(dtype) + 2.0 ** -18)
        # a bad used index, a NaN: the row alone
        i2 = i.clone()
        i2[4, 2] = 5000
        x2 = s.clone()
        x2[6, 17] = float("nan")
        x2.requires_grad_(True)
        l2 = fuselse_amd.topk_distillation(x2, t, i2, reduction="none")
        (d2,) = torch.autograd.grad(l2, x2, torch.ones_like(l2))
        rows = [0, 1, 2, 3, 5, 7]
        assert l2[[4, 6]].isnan().all() and d2[[4, 6]].isnan().all()
        assert torch.equal(l2[rows].detach(), loss[rows].detach()) and torch.equal(d2[rows], ds[rows])


@pytest.mark.parametrize("v", [1000, 1001, 50257])
@pytest.mark.parametrize("dtype", DTYPES)
def test_distill_shifted_batch_is_read_in_place(cuda, v, dtype):
    print(f"case distill shifted {v} {dtype}", flush=True)
    s, t, i = distill_inputs(cuda, (3, 7), v, 9, dtype, dtype, seed=8)
    ds = check_distill(s[:, :-1], t[:, :-1].contiguous(), i[:, :-1].contiguous(), 1.0, "sum")
    flat = check_distill(s[:, :-1].contiguous(), t[:, :-1], i[:, :-1].to(torch.int32), 1.0, "sum")
    assert torch.equal(ds, flat)
    # through the batch, and rows one after the other in other strides
    x = s.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(fuselse_amd.topk_distillation(x[:, :-1], t[:, :-1], i[:, :-1], reduction="sum"), x,
                               torch.full((), 0.75, device=cuda))
    assert torch.equal(g[:, :-1], ds) and (g[:, -1] == 0).all()
    odd = torch.zeros(3, 6, v + 3, dtype=dtype, device=cuda)
    odd[..., 1:v + 1] = s[:, :-1]
    assert torch.equal(check_distill(odd[..., 1:v + 1], t[:, :-1], i[:, :-1], 1.0, "sum"), ds)
    tr = s[:, :-1].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(check_distill(tr, t[:, :-1], i[:, :-1], 1.0, "sum"), ds)


def test_distill_one_row_and_four_dimensions(cuda):
    print("case distill dims", flush=True)
    s, t, i = distill_inputs(cuda, (2, 2, 3), 200, 4, torch.float32, torch.float32)
    want = fuselse_amd.topk_distillation(s.view(12, 200), t.view(12, 4), i.view(12, 4), reduction="none")
    got = fuselse_amd.topk_distillation(s, t, i, reduction="none")
    assert got.shape == (2, 2, 3) and torch.equal(got.reshape(-1), want)
    one = fuselse_amd.topk_distillation(s[0, 0, 0], t[0, 0, 0], i[0, 0, 0], reduction="none")
    assert one.shape == () and one == want[0]
    none = fuselse_amd.topk_distillation(s[:0], t[:0], i[:0])
    assert none == 0


# ---------------------------------------------------------------------------
# Router balance
# ---------------------------------------------------------------------------
def router_reference(x, index, mask, gb, gz):
    dtype = x.dtype
    xd = x.detach().double()
    T, E = xd.shape
    k = index.shape[1]
    live = mask if mask is not None else torch.ones(T, dtype=torch.bool, device=x.device)
    n = int(live.sum())
    xd = torch.where(live[:, None], xd, 0.0)
    chosen = index[live].reshape(-1)
    counts = torch.bincount(chosen[(chosen >= 0) & (chosen < E)], minlength=E)
    m = max(1, n)
    p = torch.softmax(xd, 1) * live[:, None]
    lse = torch.logsumexp(xd, 1) * live
    f = counts.double() / (m * max(1, k))
    bal = E * (f * p.sum(0) / m).sum()
    z = (lse ** 2).sum() / m
    dot = (p * f).sum(1, keepdim=True)
    gx = p * (gb * E / m * (f - dot) + gz * 2 * lse[:, None] / m)
    big = torch.where(xd.isfinite(), xd.abs(), 0.0).amax(1, keepdim=True) + lse.abs()[:, None] + 1
    rel = big * 2.0 ** -21 + (E / 4 + 64) * E23
    # a lane adds up its tokens' probabilities one after another
    worst = float(rel.max()) + (T / 256 + 256) * E23
    gx_b = rel * gx.abs() + p * (abs(gb) * E / m * (rel * (f + dot) + E * E23 * dot) + abs(gz) * 2 / m * rel * big) \
        + 2.0 ** -20 * p * (abs(gb) * E / m * (f + dot) + abs(gz) * 2 * lse.abs()[:, None] / m) \
        + u(dtype) * gx.abs() + tiny(dtype) + 2.0 ** -126
    z_b = float((2 * lse.abs() * big[:, 0] * 2.0 ** -21 + 2 * lse.abs() * (E / 4 + 64) * E23).sum()) / m + 2.0 ** -22 * float(z)
    return bal, z, counts, gx, bal * worst + 2.0 ** -22, z_b + 1e-30, gx_b


def check_router(x, index, mask=None, gb=0.7, gz=-0.3):
    x = x.detach().requires_grad_(True)
    out = fuselse_amd.router_balance(x, index, mask=mask)
    ups = torch.tensor(gb, device=x.device), torch.tensor(gz, device=x.device)
    (gx,) = torch.autograd.grad((out.balance_loss, out.z_loss), x, ups)
    i2 = index.reshape(x.shape[:-1].numel(), index.shape[-1]).long()
    bal, z, counts, rx, bb, zb, bx = router_reference(x.reshape(-1, x.shape[-1]), i2,
                                                      mask.reshape(-1) if mask is not None else None,
                                                      float(ups[0]), float(ups[1]))
    assert out.counts.dtype == torch.int64 and torch.equal(out.counts, counts)
    within(out.balance_loss, bal, bb, "balance")
    within(out.z_loss, z, zb, "z")
    within(gx.reshape(rx.shape), rx, bx, "dlogits")
    plain = fuselse_amd.router_balance(x.detach(), index, mask=mask)
    assert torch.equal(plain.balance_loss, out.balance_loss.detach()) and torch.equal(plain.z_loss, out.z_loss.detach())
    return gx


def router_inputs(cuda, t, e, k, dtype, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = (torch.randn(t, e, device=cuda, generator=g) * 2 + torch.randn(e, device=cuda, generator=g)).to(dtype)
    return x, x.float().topk(min(k, e), 1).indices


@pytest.mark.parametrize("e", [1, 2, 3, 8, 17, 60, 64, 100, 128, 160, 256, 257, 384, 512, 1000, 1024])
@pytest.mark.parametrize("dtype", DTYPES)
def test_router_experts(cuda, e, dtype):
    print(f"case router {e} {dtype}", flush=True)
    x, i = router_inputs(cuda, 777, e, 4, dtype, seed=e)
    check_router(x, i)


@pytest.mark.parametrize("t", [1, 2, 63, 129, 5000, 70001])
@pytest.mark.parametrize("e,k", [(8, 2), (64, 6), (384, 8)])
def test_router_tokens_and_masks(cuda, t, e, k):
    print(f"case router {t} {e} {k}", flush=True)
    x, i = router_inputs(cuda, t, e, k, torch.bfloat16, seed=t)
    g = torch.Generator(device=cuda).manual_seed(1)
    mask = torch.rand(t, device=cuda, generator=g) < 0.7
    x[~mask] = float("nan")               # masked tokens may hold anything
    gx = check_router(x, i, mask)
    assert (gx[~mask] == 0).all()
    gx = check_router(x, i, torch.zeros_like(mask))
    assert (gx == 0).all()


def test_router_choices_strides_and_special_values(cuda):
    print("case router special", flush=True)
    x, i = router_inputs(cuda, 300, 60, 4, torch.float32)
    check_router(x, i[:, :0])
    i2 = i.clone()
    i2[5, 1], i2[7, 0] = -1, 60            # dropped choices
    i2[9, 2] = i2[9, 3]                    # the same expert twice
    check_router(x, i2.to(torch.int32))
    wide = torch.zeros(300, 75, device=cuda)
    wide[:, 3:63] = x
    assert torch.equal(check_router(wide[:, 3:63], i), check_router(x, i))
    check_router(x.view(3, 100, 60), i.view(3, 100, 4), torch.arange(300, device=cuda).view(3, 100) % 3 != 0)
    # experts a router masks
    x[:, ::7] = -math.inf
    x[:, 1] = torch.finfo(torch.float32).min
    check_router(x, i)
    out = fuselse_amd.router_balance(x[:0], i[:0])
    assert out.balance_loss == 0 and out.z_loss == 0 and (out.counts == 0).all()
    # one loss of the two
    xg = x.clone().requires_grad_(True)
    o = fuselse_amd.router_balance(xg, i)
    (a,) = torch.autograd.grad(o.balance_loss, xg, retain_graph=True)
    (b,) = torch.autograd.grad(o.z_loss, xg, retain_graph=True)
    (c,) = torch.autograd.grad((o.balance_loss, o.z_loss), xg)
    # each is rounded on its own: a part of 2^-22 of either's magnitude
    assert ((a + b - c).abs() <= 2.0 ** -22 * (a.abs() + b.abs()) + 2.0 ** -126).all()
    assert not o.counts.requires_grad


# ---------------------------------------------------------------------------
# All together, on streams and in graphs
# ---------------------------------------------------------------------------
def _moe_step(s):
    """One training step's losses and gradients of a small distilled
    mixture-of-experts model: router, hidden states, head."""
    route = fuselse_amd.router_balance(s["router"], s["choices"], mask=s["mask"])
    ce = fuselse_amd.linear_cross_entropy(s["hidden"], s["head"], s["target"], z_loss=1e-4)
    logits = s["hidden"][:32] @ s["head"].t()
    kd = fuselse_amd.topk_distillation(logits, s["teacher"], s["top"], temperature=2.0)
    total = ce + 0.5 * kd + 0.01 * route.balance_loss + 0.001 * route.z_loss
    grads = torch.autograd.grad(total, (s["router"], s["hidden"], s["head"]))
    return [total.detach(), ce.detach(), kd.detach(), route.counts, *grads]


def _moe_state(cuda, seed=0):
    x, w, t = linear_inputs(cuda, 100, 64, 500, torch.bfloat16, ignored=0.3, seed=seed)
    r, choices = router_inputs(cuda, 100, 16, 2, torch.float32, seed=seed)
    _, teacher, top = distill_inputs(cuda, (32,), 500, 10, torch.bfloat16, torch.bfloat16, seed=seed)
    return {"router": r.requires_grad_(True), "choices": choices, "mask": t != -100, "hidden": x.requires_grad_(True),
            "head": w.requires_grad_(True), "target": t, "teacher": teacher, "top": top}


def _moe_reference(s):
    xd = s["hidden"].detach().double().requires_grad_(True)
    wd = s["head"].detach().double().requires_grad_(True)
    rd = s["router"].detach().double().requires_grad_(True)
    live = s["target"] != -100
    logits = xd @ wd.t()
    lse = torch.logsumexp(logits, 1)
    ce = (lse - logits.gather(1, s["target"].clamp(min=0)[:, None])[:, 0] + 1e-4 * lse ** 2)[live].mean()
    logp = torch.log_softmax(logits[:32] / 2, 1).gather(1, s["top"])
    tp = torch.softmax(s["teacher"].double() / 2, 1)
    kd = 4 * (tp * (tp.log() - logp)).sum(1).mean()
    counts = torch.bincount(s["choices"][live].reshape(-1), minlength=16)
    n = int(live.sum())
    bal = 16 * (counts.double() / (2 * n) * torch.softmax(rd[live], 1).mean(0)).sum()
    z = (torch.logsumexp(rd[live], 1) ** 2).mean()
    total = ce + 0.5 * kd + 0.01 * bal + 0.001 * z
    return [total.detach(), ce.detach(), kd.detach(), counts, *torch.autograd.grad(total, (rd, xd, wd))]


def test_losses_together(cuda):
    print("case together", flush=True)
    s = _moe_state(cuda)
    got, want = _moe_step(s), _moe_reference(s)
    assert torch.equal(got[3], want[3])
    for k in (0, 1, 2):
        # the distilled logits are rounded to bf16: at most 2^-8 of 16 each
        assert abs(float(got[k]) - float(want[k])) <= 2.0 ** -8 * 16 * (1 if k != 1 else 2.0 ** -6), k
    for a, b in zip(got[4:], want[4:]):
        # roundings to bf16 on the way: of a logit, of a probability, of the results
        assert float((a.double() - b).norm()) <= 0.05 * float(b.norm())


def test_losses_in_a_hip_graph(cuda):
    print("case graph", flush=True)
    s = _moe_state(cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _moe_step(s)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = _moe_step(s)
    for seed in range(1, 5):
        other = _moe_state(cuda, seed)
        with torch.no_grad():
            for k in s:
                s[k].copy_(other[k])
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want = _moe_step(other)
        torch.cuda.synchronize()
        for k, (a, b) in enumerate(zip(outs, want)):
            assert torch.equal(a, b), (seed, k)


def test_losses_on_two_streams(cuda):
    print("case streams", flush=True)
    states = [_moe_state(cuda, k) for k in (0, 1)]
    want = [_moe_step(s) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    for _ in range(3):
        got = []
        for st, s in zip(streams, states):
            with torch.cuda.stream(st):
                got.append(_moe_step(s))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_backward_twice_and_saved_hooks(cuda):
    print("case hooks", flush=True)
    s = _moe_state(cuda, 3)
    ce = fuselse_amd.linear_cross_entropy(s["hidden"], s["head"], s["target"])
    a = torch.autograd.grad(ce, (s["hidden"], s["head"]), retain_graph=True)
    b = torch.autograd.grad(ce, (s["hidden"], s["head"]))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    with torch.autograd.graph.save_on_cpu():
        ce = fuselse_amd.linear_cross_entropy(s["hidden"], s["head"], s["target"])
        rt = fuselse_amd.router_balance(s["router"], s["choices"], mask=s["mask"])
    c = torch.autograd.grad(ce, (s["hidden"], s["head"]))
    assert all(torch.equal(x, y) for x, y in zip(a, c))
    torch.autograd.grad(rt.balance_loss, s["router"])


# ---------------------------------------------------------------------------
# Tensors of more than 2^32 bytes, and elements past 2^31
# ---------------------------------------------------------------------------
def test_linear_offsets_past_32_bits(cuda):
    print("case linear large offsets", flush=True)
    n, d, v, dtype = 40, 2048, 1_100_000, torch.bfloat16
    g = torch.Generator(device=cuda).manual_seed(20)
    w = torch.empty(v, d, device=cuda, dtype=dtype).normal_(0.0, 2.0 / math.sqrt(d), generator=g)
    t = torch.randint(v - 1000, v, (n,), device=cuda, generator=g)
    t[0], t[1] = 0, -100
    x = (torch.randn(n, d, device=cuda, generator=g) + 2 * w[t].float()).to(dtype)
    up = linear_upstream(cuda, n, "none")
    x.requires_grad_(True)
    w.requires_grad_(True)
    loss = fuselse_amd.linear_cross_entropy(x, w, t, reduction="none")
    dx, dw = torch.autograd.grad(loss, (x, w), up)
    plain = fuselse_amd.linear_cross_entropy(x.detach()[:12], w.detach(), t[:12], reduction="none")
    want, rx, rw, b, bx, bw = linear_reference(x, w, t, -100, "none", 0.0, up)
    within(loss, want, b, "loss")
    within(plain, want[:12], b[:12], "loss of few rows")
    within(dx, rx, bx, "dx")
    for part in (slice(0, 1000), slice(v - 1000, v)):
        within(dw[part], rw[part], bw[part], "dw")


def test_distill_offsets_past_32_bits(cuda):
    print("case distill large offsets", flush=True)
    rows, v, k = 17000, 128256, 8
    g = torch.Generator(device=cuda).manual_seed(21)
    s = torch.empty(rows, v, device=cuda, dtype=torch.bfloat16).normal_(0.0, 3.0, generator=g).requires_grad_(True)
    t = torch.randn(rows, k, device=cuda, generator=g)
    i = torch.arange(k, device=cuda) * 7919 + torch.arange(rows, device=cuda)[:, None]
    up = torch.randn(rows, device=cuda, generator=g)
    loss = fuselse_amd.topk_distillation(s, t, i, reduction="none")
    (ds,) = torch.autograd.grad(loss, s, up)
    for part in (slice(0, 20), slice(rows - 20, rows)):
        want, rs, b, bs = distill_reference(s[part], t[part], i[part], 1.0, "none", up[part])
        within(loss[part], want, b, "loss")
        within(ds[part], rs, bs, "ds")


def test_router_offsets_past_32_bits(cuda):
    """A batch repeated: the losses of one copy, its counts times the copies,
    and its gradient over the copies in each."""
    print("case router large offsets", flush=True)
    tokens, e, k, copies = 4096, 1024, 2, 520
    g = torch.Generator(device=cuda).manual_seed(22)
    base = (torch.randn(tokens, e, device=cuda, generator=g)).to(torch.float16)
    index = torch.randint(0, e, (tokens, k), device=cuda, generator=g)
    x = base.repeat(copies, 1).requires_grad_(True)
    out = fuselse_amd.router_balance(x, index.repeat(copies, 1))
    xd = base.double()
    p = torch.softmax(xd, 1)
    counts = torch.bincount(index.flatten(), minlength=e)
    f = counts.double() / (tokens * k)
    balance, z = e * (f * p.mean(0)).sum(), (torch.logsumexp(xd, 1) ** 2).mean()
    assert torch.equal(out.counts, counts * copies)
    # a lane adds at most tokens copies / (256 blocks 16 groups) probabilities
    # one after another, of exponents that are rounded by 2^-21 each
    rel = tokens * copies / (256 * 16) * E23 + 2.0 ** -20
    assert abs(float(out.balance_loss) - float(balance)) <= rel * float(balance)
    assert abs(float(out.z_loss) - float(z)) <= 2.0 ** -18 * float(z)
    # upstream gradients that bring an element's to the size of p: within fp16
    scale = float(tokens * copies)
    (dx,) = torch.autograd.grad(out.balance_loss, x, torch.full((), scale, device=cuda))
    want = p * (e * f - (p * (e * f)).sum(1, keepdim=True))
    bound = (2.0 ** -18 * p * (e * f + (p * (e * f)).sum(1, keepdim=True)) + u(torch.float16) * want.abs()
             + tiny(torch.float16))
    for c in (0, copies - 1):
        within(dx[c * tokens:(c + 1) * tokens], want, bound, f"dx of copy {c}")
