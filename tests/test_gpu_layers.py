"""The layers around the training losses (embedding lookup, layer norm, the
experts' order) against plain implementations in 64 bits, forward and backward,
at the sizes and masks where the kernels change path.

Tolerances.  A rounding to type t is off by at most half a step, eps_t / 2
relative (u(t)).  An fp32 sum of n terms is off by at most n 2^-23 of the sum of
their magnitudes, in whatever order."""

import math

import pytest
import torch

import fuselse_amd
from fuselse_amd import ext
from test_gpu_losses import DTYPES, E23, tiny, u, within

pytestmark = pytest.mark.gpu


def randn(cuda, *shape, seed=0):
    return torch.randn(*shape, device=cuda, generator=torch.Generator(device=cuda).manual_seed(seed))


def randint(cuda, high, *shape, seed=0):
    return torch.randint(0, high, shape, device=cuda, generator=torch.Generator(device=cuda).manual_seed(seed))


# ---------------------------------------------------------------------------
# Embedding
# ---------------------------------------------------------------------------
def check_embedding(index, w, scale=1.0, padding=None, grad=None, seed=0):
    cuda, dtype = w.device, w.dtype
    V, D = w.shape
    w.requires_grad_(True)
    out = fuselse_amd.embedding(index, w, scale=scale, padding_idx=padding)
    assert out.shape == (*index.shape, D) and out.dtype == dtype
    g = randn(cuda, *out.shape, seed=seed + 1).to(dtype) if grad is None else grad(out)
    (dw,) = torch.autograd.grad(out, w, g)
    assert dw.shape == w.shape and dw.dtype == dtype
    flat = index.reshape(-1).long()
    inside = (flat >= 0) & (flat < V)
    rows = out.detach().reshape(-1, D)
    want = w.detach().double()[flat[inside]] * scale
    if scale == 1.0:
        assert torch.equal(rows[inside], w.detach()[flat[inside]])
    assert rows[~inside].isnan().all()
    # the scale's rounding, the product's, and the one to the type
    within(rows[inside], want, (u(dtype) + 2.0 ** -22) * want.abs() + tiny(dtype), "out")
    keep = inside
    if padding is not None:
        keep = keep & (flat != padding % V)
    gd = g.reshape(-1, D).double()[keep]
    total = torch.zeros(V, D, dtype=torch.float64, device=cuda).index_add_(0, flat[keep], gd)
    size = torch.zeros(V, D, dtype=torch.float64, device=cuda).index_add_(0, flat[keep], gd.abs())
    count = torch.bincount(flat[keep], minlength=V)[:, None].double()
    bound = size * abs(scale) * (count * E23 + 2.0 ** -22) + u(dtype) * abs(scale) * total.abs() + tiny(dtype)
    bound = torch.where(count > 0, bound, 0.0)
    within(dw, total * scale, bound, "dw")
    # the same bits again, and without autograd
    assert torch.equal(ext.embedding_backward(g.reshape(-1, D).contiguous(), flat.contiguous(), V, scale,
                                              -1 if padding is None else padding % V), dw)
    with torch.no_grad():
        again = fuselse_amd.embedding(index, w, scale=scale, padding_idx=padding)
    assert torch.equal(again.nan_to_num(nan=3.0), out.detach().nan_to_num(nan=3.0))
    return dw


EMBEDDING = [(1, 1, 1), (3, 5, 7), (2, 3, 2), (31, 4, 8), (33, 4, 9), (129, 1031, 200), (1000, 1023, 64),
             (1000, 1024, 24), (4095, 50257, 65), (4096, 50257, 64), (4097, 1000, 40), (8191, 50257, 24),
             (8192, 300, 513), (20000, 37, 33), (5000, (1 << 20) - 1, 4), (5000, 1 << 20, 4), (300, (1 << 20) + 5, 3),
             (9000, (1 << 20) + 5, 3), (9000, 1 << 20, 2), (8193, 5, 7)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,d", EMBEDDING)
def test_embedding(cuda, n, v, d, dtype):
    print(f"case embedding {n} {v} {d} {dtype}", flush=True)
    w = randn(cuda, v, d).to(dtype)
    # low ids come often, as in a text
    index = (randint(cuda, 1 << 20, n, seed=2).double() / (1 << 20)).pow(3).mul(v).long().clamp(max=v - 1)
    check_embedding(index, w)
    check_embedding(index, w.detach(), scale=math.sqrt(d) if d > 1 else 0.3, padding=-1)


@pytest.mark.parametrize("n", [2, 32, 33, 64, 65, 1025, 5000, 40000])
@pytest.mark.parametrize("d", [5, 64, 520])
def test_embedding_one_token_many_times(cuda, n, d):
    print(f"case embedding one token {n} {d}", flush=True)
    w = randn(cuda, 77, d).bfloat16()
    check_embedding(torch.full((n,), 41, device=cuda), w)
    # runs that end at and around the borders of 32 entries
    index = torch.arange(n, device=cuda) // 31
    check_embedding(index % 77, w.detach())
    check_embedding((torch.arange(n, device=cuda) // 32) % 77, w.detach())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,d", [(131071, 3000, 8), (131072, 3000, 3), (131073, 5, 65), (200001, 70000, 24),
                                   (65536, 4000, 520)])
def test_embedding_many_tokens_of_short_rows(cuda, n, v, d, dtype):
    print(f"case embedding many tokens {n} {v} {d} {dtype}", flush=True)
    w = randn(cuda, v, d).to(dtype)
    check_embedding(randint(cuda, v, n, seed=3), w)
    # runs that end at and around the borders of 64 entries
    for run in (63, 64, 65):
        check_embedding((torch.arange(n, device=cuda) // run) % v, w.detach(), padding=0)


@pytest.mark.parametrize("n", [0, 1, 40, 5000])
def test_embedding_indexes_outside_and_padding(cuda, n):
    print(f"case embedding outside {n}", flush=True)
    w = randn(cuda, 50, 12)
    index = randint(cuda, 70, n) - 10
    if n > 2:
        index[:3] = torch.tensor([2 ** 62, -2 ** 63, 50], device=cuda)
    check_embedding(index, w, padding=0)
    check_embedding(torch.full((n,), 7, device=cuda), w.detach(), padding=7)
    check_embedding(torch.full((n,), 50, device=cuda), w.detach())
    assert not check_embedding(torch.full((n,), -1, device=cuda), w.detach()).any()


@pytest.mark.parametrize("itype", [torch.int32, torch.int64, torch.uint8, torch.int16])
def test_embedding_views(cuda, itype):
    print(f"case embedding views {itype}", flush=True)
    # rows apart, and a start that is no multiple of 16 bytes
    for view in (lambda b: b[:, 3:43], lambda b: b[:, :40], lambda b: b.t()[:40].t()):
        base = randn(cuda, 90, 45).half()
        w = view(base).detach()
        index = randint(cuda, 90, 4, 2, 9).to(itype)
        check_embedding(index, w)
        check_embedding(index[:, :, ::2], w.detach())
        check_embedding(index[1, 1, 4], w.detach())  # a single token
    # gradients that are expanded, transposed or rows apart
    w = randn(cuda, 90, 40)
    index = randint(cuda, 90, 33)
    check_embedding(index, w, grad=lambda o: torch.ones((), device=cuda).expand_as(o))
    check_embedding(index, w.detach(), grad=lambda o: randn(cuda, 40, 33).t())
    check_embedding(index, w.detach(), grad=lambda o: randn(cuda, 33, 50)[:, 3:43])


def test_embedding_refusals(cuda):
    w, i = randn(cuda, 5, 4), torch.zeros(2, dtype=torch.int64, device=cuda)
    for bad in (5, -6):
        with pytest.raises(RuntimeError, match="padding_idx"):
            fuselse_amd.embedding(i, w, padding_idx=bad)
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        fuselse_amd.embedding(i, w.double())
    with pytest.raises(RuntimeError, match="2D"):
        fuselse_amd.embedding(i, w[0])
    with pytest.raises(RuntimeError, match="not be empty"):
        fuselse_amd.embedding(i, w[:0])
    with pytest.raises(RuntimeError, match="at least one column"):
        fuselse_amd.embedding(i, w[:, :0])
    with pytest.raises(RuntimeError, match="index must be CUDA"):
        fuselse_amd.embedding(i.cpu(), w)
    with pytest.raises(RuntimeError, match="contiguous rows"):
        ext.embedding(w.t(), i)


# ---------------------------------------------------------------------------
# Layer norm
# ---------------------------------------------------------------------------
def check_norm(x, w, b, eps=1e-5, grad=None, seed=0):
    cuda, dtype = x.device, x.dtype
    D = x.shape[-1]
    leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
    y = fuselse_amd.layer_norm(x, w, b, eps=eps)
    assert y.shape == x.shape and y.dtype == dtype
    g = randn(cuda, *y.shape, seed=seed + 5).to(dtype) if grad is None else grad(y)
    got = list(torch.autograd.grad(y, leaves, g))

    xd = x.detach().double().reshape(-1, D)
    gd = g.double().reshape(-1, D)
    wd = w.detach().double() if w is not None else torch.ones(D, dtype=torch.float64, device=cuda)
    bd = b.detach().double() if b is not None else torch.zeros(D, dtype=torch.float64, device=cuda)
    N = xd.shape[0]
    mean = xd.mean(1, keepdim=True)
    c = xd - mean
    var = c.square().mean(1, keepdim=True)
    rstd = 1 / (var + eps).sqrt()
    h = c * rstd
    # steps of a sum over a row: at most D
    nE = D * E23
    # the first mean's error, which the differences then carry
    e0 = nE * xd.abs().mean(1, keepdim=True) + E23 * mean.abs()
    d_abs, d_sq = (c.abs() + e0), var + e0 ** 2
    c_err = E23 * (d_abs + c.abs()) + (nE + 2 * E23) * d_abs.mean(1, keepdim=True)
    rel = 0.5 * (nE + 4 * E23) * d_sq / (var + eps) + 4 * E23
    h_err = rstd * c_err + h.abs() * rel
    y_err = wd.abs() * h_err + 2 * E23 * ((wd * h).abs() + bd.abs())
    want = h * wd + bd
    within(y.reshape(-1, D), want, y_err + u(dtype) * want.abs() + tiny(dtype), "y")

    a = gd * wd
    m0, m1 = a.mean(1, keepdim=True), (a * h).mean(1, keepdim=True)
    dx = rstd * (a - m0 - h * m1)
    size = a.abs() + m0.abs() + (h * m1).abs()
    m0_err = (nE + 2 * E23) * a.abs().mean(1, keepdim=True)
    m1_err = (nE + 3 * E23) * (a * h).abs().mean(1, keepdim=True) + (a.abs() * h_err).mean(1, keepdim=True)
    dx_err = rstd * (m0_err + h.abs() * m1_err + m1.abs() * h_err + 4 * E23 * size + h_err * m1_err)
    dx_err = dx_err + rel * rstd * size
    within(got[0].reshape(-1, D), dx, dx_err + u(dtype) * dx.abs() + tiny(dtype), "dx")
    rest = got[1:]
    if w is not None:
        dw = (gd * h).sum(0)
        err = (gd.abs() * h_err).sum(0) + (N + 1) * E23 * (gd * h).abs().sum(0)
        within(rest.pop(0), dw, err + u(w.dtype) * dw.abs() + tiny(w.dtype), "dw")
    if b is not None:
        db = gd.sum(0)
        within(rest.pop(0), db, N * E23 * gd.abs().sum(0) + u(b.dtype) * db.abs() + tiny(b.dtype), "db")
    # the same bits again, and without autograd
    assert all(torch.equal(p, q) for p, q in zip(
        got, torch.autograd.grad(fuselse_amd.layer_norm(x, w, b, eps=eps), leaves, g)))
    with torch.no_grad():
        assert torch.equal(fuselse_amd.layer_norm(x, w, b, eps=eps), y.detach())


def norm_inputs(cuda, n, d, dtype, pdtype, seed=0):
    x = (randn(cuda, n, d, seed=seed) * torch.exp(0.5 * randn(cuda, d, seed=seed + 1)) + randn(cuda, d, seed=seed + 2))
    return (x.to(dtype), (1 + 0.3 * randn(cuda, d, seed=seed + 3)).to(pdtype),
            randn(cuda, d, seed=seed + 4).to(pdtype))


NORM_D = [1, 2, 3, 8, 63, 64, 65, 127, 128, 129, 200, 256, 500, 512, 1000, 1024, 1028, 2047, 2048, 2056, 4096, 4104,
          8192, 8200, 16384, 16392, 20001, 32768, 32776]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", NORM_D)
def test_layer_norm(cuda, d, dtype):
    print(f"case norm {d} {dtype}", flush=True)
    for n in (1, 5, 37):
        x, w, b = norm_inputs(cuda, n, d, dtype, dtype)
        check_norm(x, w, b)


@pytest.mark.parametrize("n", [2, 63, 64, 65, 511, 512, 513, 2047, 9000])
@pytest.mark.parametrize("d", [40, 768, 2051])
def test_layer_norm_many_rows(cuda, n, d):
    print(f"case norm rows {n} {d}", flush=True)
    x, w, b = norm_inputs(cuda, n, d, torch.bfloat16, torch.float32)
    check_norm(x, w, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", range(1, 10))
def test_layer_norm_short_rows(cuda, d, dtype):
    print(f"case norm short {d} {dtype}", flush=True)
    for n, pdtype in ((255, torch.float32), (257, dtype), (200001, torch.float32)):
        x, w, b = norm_inputs(cuda, n, d, dtype, pdtype)
        check_norm(x, w, b)
    check_norm(x.detach()[:1000], None, None)
    check_norm(randn(cuda, 300, d + 3).to(dtype)[:, 2:2 + d], w.detach(), None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("has", ["w", "b", ""])
def test_layer_norm_parameters(cuda, dtype, has):
    print(f"case norm parameters {has} {dtype}", flush=True)
    for pdtype in DTYPES:
        x, w, b = norm_inputs(cuda, 21, 136, dtype, pdtype)
        check_norm(x, w if "w" in has else None, b if "b" in has else None)
        check_norm(x.detach(), w.detach(), b.detach().float())  # of different types


def test_layer_norm_one_gradient_alone(cuda):
    x, w, b = norm_inputs(cuda, 100, 96, torch.float32, torch.float32)
    g = randn(cuda, 100, 96, seed=9)
    for t in (x, w, b):
        t.requires_grad_(True)
    all_three = torch.autograd.grad(fuselse_amd.layer_norm(x, w, b), (x, w, b), g)
    for i, leaf in enumerate((x, w, b)):
        others = [t if t is leaf else t.detach() for t in (x, w, b)]
        (one,) = torch.autograd.grad(fuselse_amd.layer_norm(*others), leaf, g)
        assert torch.equal(one, all_three[i])


@pytest.mark.parametrize("d", [96, 2048, 5000, 40000])
def test_layer_norm_common_value_and_constant_rows(cuda, d):
    """A value that a row's elements have in common takes no digits from the
    result; a constant row has variance 0."""
    print(f"case norm common {d}", flush=True)
    x = (randn(cuda, 6, d) + torch.tensor([0.0, 1e3, -3e4, 1e5, 7.0, 123.456], device=cuda)[:, None])
    x[4] = 7.0
    x[5] = 123.456
    check_norm(x, *norm_inputs(cuda, 1, d, torch.float32, torch.float32)[1:])
    xd = x.detach()[3].double()
    want = (xd - xd.mean()) / (xd.var(correction=0) + 1e-5).sqrt()
    off = (fuselse_amd.layer_norm(x.detach())[3].double() - want).abs().max()
    # one mean in fp32 would be off by half a step of 1e5, 2^-8
    assert off < 1e-4, off
    assert fuselse_amd.layer_norm(x.detach())[4:].abs().max() < 1e-3
    assert fuselse_amd.layer_norm(torch.zeros_like(x.detach()), eps=0.0).isnan().all()


def test_layer_norm_rows_that_are_not_finite(cuda):
    """They leave the other rows as they are."""
    for d in (96, 1100, 9000, 40000):
        x, w, b = norm_inputs(cuda, 9, d, torch.float32, torch.float32)
        y = fuselse_amd.layer_norm(x, w, b)
        stray = x.clone()
        stray[2, 3], stray[5, d - 1], stray[7] = math.inf, math.nan, -math.inf
        z = fuselse_amd.layer_norm(stray, w, b)
        live = torch.ones(9, dtype=torch.bool, device=cuda)
        live[[2, 5, 7]] = False
        assert torch.equal(z[live], y[live]) and z[~live].isnan().all()


def test_layer_norm_views_and_empty(cuda):
    print("case norm views", flush=True)
    _, w, b = norm_inputs(cuda, 1, 72, torch.float16, torch.float16)
    check_norm(randn(cuda, 4, 5, 80).half()[:, :, 3:75], w, b)
    check_norm(randn(cuda, 4, 5, 72).half()[:, :-1], w.detach(), b.detach())
    check_norm(randn(cuda, 72, 11).half().t(), w.detach(), b.detach())
    check_norm(randn(cuda, 72).half(), w.detach(), b.detach())
    check_norm(randn(cuda, 1, 72).half().expand(7, 72), w.detach(), b.detach())
    check_norm(randn(cuda, 9, 72).half(), w.detach(), b.detach(), grad=lambda y: torch.ones((), device=cuda).half().expand_as(y))
    check_norm(randn(cuda, 9, 72).half(), randn(cuda, 144).half()[::2], None)
    x = torch.zeros(0, 72, device=cuda, dtype=torch.float16, requires_grad=True)
    got = torch.autograd.grad(fuselse_amd.layer_norm(x, w, b), (x, w, b), torch.zeros_like(x))
    assert got[0].shape == (0, 72) and not got[1].any() and not got[2].any()


def test_layer_norm_refusals(cuda):
    x, w, b = norm_inputs(cuda, 3, 8, torch.float32, torch.float32)
    for args in ((x.double(),), (x, w[:7], None), (x, w[None], None), (x, w.double(), None), (x, w.cpu(), None)):
        with pytest.raises(RuntimeError):
            fuselse_amd.layer_norm(*args)
    for eps in (-1.0, math.nan):
        with pytest.raises(RuntimeError, match="eps"):
            fuselse_amd.layer_norm(x, eps=eps)
    with pytest.raises(RuntimeError, match="one type"):
        ext.layer_norm(x.half(), w.half(), b)


# ---------------------------------------------------------------------------
# The experts' order
# ---------------------------------------------------------------------------
def plain_order(index, experts, mask=None):
    flat = index.reshape(-1, index.shape[-1]).long()
    live = (flat >= 0) & (flat < experts)
    if mask is not None:
        live &= mask.reshape(-1)[:, None]
    key = torch.where(live, flat, experts).reshape(-1).cpu()
    place = torch.empty_like(key)
    place[key.sort(stable=True).indices] = torch.arange(key.numel())
    counts = torch.bincount(key, minlength=experts + 1)[:experts]
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])
    place = place.to(index.device).reshape(flat.shape)
    return (torch.where(live, place, -1 - place).reshape(index.shape).int(), counts.to(index.device),
            offsets.int().to(index.device))


def check_order(index, experts, mask=None):
    got = fuselse_amd.expert_order(index, experts, mask=mask)
    for a, b, what in zip(got, plain_order(index, experts, mask), ("position", "counts", "offsets")):
        assert a.dtype == b.dtype and torch.equal(a, b), what
    return got


ORDERS = [(1, 1, 1), (1, 8, 256), (8, 8, 256), (5, 3, 4), (64, 1, 2), (63, 2, 7), (512, 2, 8), (1024, 4, 1024),
          (4096, 1, 60), (4097, 1, 60), (2731, 3, 64), (16383, 6, 64), (70001, 2, 1023), (9000, 17, 1024),
          (300000, 1, 3), (20, 1024, 8)]


@pytest.mark.parametrize("t,k,e", ORDERS)
def test_expert_order(cuda, t, k, e):
    print(f"case order {t} {k} {e}", flush=True)
    # experts of different load
    index = (randint(cuda, 1 << 20, t, k).double() / (1 << 20)).pow(2).mul(e).long()
    check_order(index, e)
    check_order(index.int(), e, mask=randint(cuda, 4, t, seed=3) > 0)
    check_order(index + randint(cuda, 5, t, k, seed=4) - 2, e)  # some outside
    check_order(torch.full_like(index, e - 1), e)
    check_order(index, e, mask=torch.zeros(t, dtype=torch.bool, device=cuda))


def test_expert_order_views_and_refusals(cuda):
    index = randint(cuda, 9, 3, 5, 4)
    got = check_order(index, 9, mask=randint(cuda, 2, 3, 5).bool())
    assert got.position.shape == (3, 5, 4)
    check_order(index[:, ::2, 1:], 9, mask=randint(cuda, 2, 3, 6).bool()[:, ::2])
    check_order(index[0, 0], 9)
    check_order(index[:0], 9)
    check_order(torch.tensor([[2 ** 62, -2 ** 63, 4]], device=cuda), 9)
    for args in ((index, 0), (index, 1025), (index[..., :0], 9), (index.float(), 9)):
        with pytest.raises(RuntimeError):
            fuselse_amd.expert_order(*args)
    with pytest.raises(RuntimeError, match="bool"):
        fuselse_amd.expert_order(index, 9, mask=torch.ones(3, 5, device=cuda))


def check_rows(t, k, e, d, dtype, wdtype, mask=None, index=None, view=lambda a: a, seed=0):
    cuda = torch.device("cuda:0")
    index = randint(cuda, e, t, k, seed=seed) if index is None else index
    order = fuselse_amd.expert_order(index, e, mask=mask)
    live = order.position >= 0
    place = torch.where(live, order.position, -1 - order.position).long()
    x = view(randn(cuda, t, d, seed=seed + 1).to(dtype)).detach()
    made = view(randn(cuda, t * k, d, seed=seed + 2).to(dtype)).detach()
    w = randn(cuda, t, k, seed=seed + 3).to(wdtype)
    # what is dropped may hold anything
    made[place[~live]] = math.nan
    w[~live] = math.inf
    if mask is not None:
        x[~mask] = math.nan
    for leaf in (x, made, w):
        leaf.requires_grad_(True)
    rows = fuselse_amd.expert_dispatch(x, order)
    y = fuselse_amd.expert_combine(made, w, order)
    assert rows.shape == (t * k, d) and y.shape == (t, d) and rows.dtype == y.dtype == dtype
    g_rows, g_y = randn(cuda, t * k, d, seed=seed + 4).to(dtype), randn(cuda, t, d, seed=seed + 5).to(dtype)
    g_rows[place[~live]] = math.nan
    got = torch.autograd.grad((rows, y), (x, made, w), (g_rows, g_y))

    on = live[..., None]
    token = torch.arange(t, device=cuda)[:, None].expand(t, k)
    want = torch.zeros_like(rows)
    want[place[live]] = x.detach()[token[live]]
    assert torch.equal(rows, want)
    md = torch.where(on, made.detach().double()[place], 0.0)
    wd = torch.where(live, w.detach().double(), 0.0)[..., None]
    gy = g_y.double()[:, None]
    gr = torch.where(on, g_rows.double()[place], 0.0)

    def held(got, want, size, steps, what):
        # a dropped entry's is exactly 0
        bound = steps * E23 * size + u(got.dtype) * want.abs() + torch.where(size > 0, tiny(got.dtype), 0.0)
        within(got, want, bound, what)

    held(y, (wd * md).sum(1), (wd * md).abs().sum(1), k, "y")
    held(got[0], gr.sum(1), gr.abs().sum(1), k, "dx")
    held(got[1][place], wd * gy, (wd * gy).abs(), 1, "d_rows")
    dots = torch.where(on, gy * md, 0.0)
    held(got[2], dots.sum(-1), dots.abs().sum(-1), d, "d_weights")
    again = torch.autograd.grad((fuselse_amd.expert_dispatch(x, order), fuselse_amd.expert_combine(made, w, order)),
                                (x, made, w), (g_rows, g_y))
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    # one gradient without the other
    assert torch.equal(torch.autograd.grad(fuselse_amd.expert_combine(made, w.detach(), order), made, g_y)[0], got[1])
    assert torch.equal(torch.autograd.grad(fuselse_amd.expert_combine(made.detach(), w, order), w, g_y)[0], got[2])
    with torch.no_grad():
        assert torch.equal(fuselse_amd.expert_dispatch(x, order), rows)
        assert torch.equal(fuselse_amd.expert_combine(made, w, order), y)


ROWS = [(1, 1, 1, 1), (1, 8, 256, 2048), (3, 2, 4, 3), (7, 3, 5, 7), (5, 2, 3, 8), (33, 6, 8, 9), (8, 9, 16, 65),
        (100, 8, 64, 128), (64, 17, 24, 136), (20, 2, 8, 511), (20, 2, 8, 512), (31, 4, 8, 513), (9, 8, 16, 1100),
        (512, 2, 8, 768), (3, 40, 64, 4104), (1000, 6, 60, 200), (600, 1, 4, 1030), (700, 2, 8, 1041), (520, 5, 8, 1544), (30, 1, 4, 3001), (30, 2, 4, 1900), (30, 2, 4, 700), (30, 1, 4, 600),
        (9, 1, 4, 5000), (9, 2, 4, 5001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,k,e,d", ROWS)
def test_expert_rows(cuda, t, k, e, d, dtype):
    print(f"case rows {t} {k} {e} {d} {dtype}", flush=True)
    check_rows(t, k, e, d, dtype, torch.float32)
    check_rows(t, k, e, d, dtype, dtype, mask=randint(cuda, 3, t, seed=8) > 0)
    check_rows(t, k, e, d, dtype, torch.float32, index=randint(cuda, e + 2, t, k, seed=9) - 1)


def test_expert_rows_masks_and_views(cuda):
    print("case rows masks", flush=True)
    none = torch.zeros(40, dtype=torch.bool, device=cuda)
    check_rows(40, 3, 8, 96, torch.bfloat16, torch.float32, mask=none)
    check_rows(40, 3, 8, 600, torch.float32, torch.float32, mask=none)
    # a token that chooses one expert several times
    check_rows(40, 3, 8, 96, torch.float16, torch.float16, index=torch.full((40, 3), 5, device=cuda))

    def apart(a):
        b = torch.zeros(a.shape[0], a.shape[1] + 5, dtype=a.dtype, device=a.device)
        b[:, 3:3 + a.shape[1]] = a
        return b[:, 3:3 + a.shape[1]]

    for d in (40, 43, 700):
        check_rows(50, 4, 8, d, torch.bfloat16, torch.float32, view=apart)
        check_rows(50, 4, 8, d, torch.float32, torch.float32, view=lambda a: a.t().contiguous().t())


def test_expert_leading_shapes_types_and_empty(cuda):
    index = randint(cuda, 6, 2, 5, 3)
    order = fuselse_amd.expert_order(index, 6)
    x, made = randn(cuda, 2, 5, 24).bfloat16(), randn(cuda, 30, 24, seed=1).bfloat16()
    w = torch.softmax(randn(cuda, 2, 5, 3, seed=2), -1)
    flat = fuselse_amd.ExpertOrder(order.position.reshape(10, 3), *order[1:])
    assert torch.equal(fuselse_amd.expert_dispatch(x, order), fuselse_amd.expert_dispatch(x.reshape(10, 24), flat))
    y = fuselse_amd.expert_combine(made, w, order)
    assert y.shape == (2, 5, 24) and torch.equal(y.reshape(10, 24), fuselse_amd.expert_combine(made, w.reshape(10, 3), flat))
    # weights of another 16-bit type are taken in fp32
    h = w.half()
    assert torch.equal(fuselse_amd.expert_combine(made, h, order), fuselse_amd.expert_combine(made, h.float(), order))
    empty = fuselse_amd.expert_order(index[:0], 6)
    assert not empty.counts.any() and not empty.offsets.any()
    x0 = torch.zeros(0, 5, 24, device=cuda, requires_grad=True)
    r0 = torch.zeros(0, 24, device=cuda, requires_grad=True)
    rows, y = fuselse_amd.expert_dispatch(x0, empty), fuselse_amd.expert_combine(r0, w[:0], empty)
    assert rows.shape == (0, 24) and y.shape == (0, 5, 24)
    assert torch.autograd.grad(rows.sum() + y.sum(), x0)[0].shape == x0.shape


def test_expert_refusals(cuda):
    order = fuselse_amd.expert_order(randint(cuda, 4, 6, 2), 4)
    x, w = randn(cuda, 6, 8), randn(cuda, 6, 2)
    with pytest.raises(RuntimeError, match="tokens of order"):
        fuselse_amd.expert_dispatch(x[:5], order)
    with pytest.raises(RuntimeError, match=r"\(tokens \* top, D\)"):
        fuselse_amd.expert_combine(x, w, order)
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        fuselse_amd.expert_dispatch(x.double(), order)
    with pytest.raises(RuntimeError, match="weights must be"):
        fuselse_amd.expert_combine(randn(cuda, 12, 8), w.double(), order)
    with pytest.raises(RuntimeError, match="position must be"):
        fuselse_amd.expert_dispatch(x, order._replace(position=order.position.long()))


@pytest.mark.parametrize("t,k,d", [(1, 1, 520), (1023, 1, 512), (1024, 1, 512), (127, 8, 516), (128, 9, 2048),
                                   (250, 3, 2052), (256, 3, 2050), (60, 16, 8200)])
def test_expert_rows_around_the_fewest_waves(cuda, t, k, d):
    print(f"case rows of few waves {t} {k} {d}", flush=True)
    check_rows(t, k, 32, d, torch.bfloat16, torch.bfloat16, index=randint(cuda, 33, t, k, seed=9))
    check_rows(t, k, 32, d, torch.float32, torch.float32, mask=randint(cuda, 2, t, seed=8) > 0)


@pytest.mark.parametrize("t,k,d", [(3, 1024, 40), (5, 100, 520), (2, 1000, 2100), (70, 25, 9), (11, 16, 1024)])
def test_expert_rows_of_many_choices(cuda, t, k, d):
    print(f"case rows of many choices {t} {k} {d}", flush=True)
    check_rows(t, k, 64, d, torch.bfloat16, torch.float32)
    check_rows(t, k, 64, d, torch.float32, torch.float32, mask=randint(cuda, 2, t, seed=8) > 0)
    check_rows(t, k, 64, d, torch.float16, torch.float16, index=randint(cuda, 70, t, k, seed=9) - 3)


def test_places_outside_the_rows_are_dropped(cuda):
    """Places that no order gives are bounds-checked by the kernels."""
    pos = torch.tensor([[0, 4], [2 ** 31 - 1, -2 ** 31], [-9, 1]], dtype=torch.int32, device=cuda)
    for d in (8, 11, 600):
        x, rows, w = randn(cuda, 3, d), randn(cuda, 6, d, seed=1), randn(cuda, 3, 2, seed=2)
        out = ext.expert_dispatch(x, pos)
        assert torch.equal(out[[0, 4, 1]], x[[0, 0, 2]])
        y = ext.expert_combine(rows, None, pos)
        want = torch.stack([rows[0] + rows[4], torch.zeros(d, device=cuda), rows[1]])
        assert torch.equal(y, want)
        d_rows, d_w = ext.expert_combine_backward(x, rows, w, pos)
        assert torch.equal(d_rows[[0, 4, 1]], x[[0, 0, 2]] * w[[0, 0, 2], [0, 1, 1]][:, None])
        assert not d_w[1].any() and d_w[2, 0] == 0
