"""The linear cross entropy where its rows differ in size, its vocabulary takes
several pieces and its digits are claimed, against plain implementations in 64
bits.

Tolerances are those of the other tests of the training losses: half a step of
the type a rounding, 2^-23 of the sum of magnitudes an addition.  A product's
sum over K takes 32 additions inside a matrix instruction and one more for
every 32 of K, and the splits' sums are joined one after another (64 at most)."""

import math

import pytest
import torch

import fuselse_amd
from fuselse_amd import _lib
from test_gpu_losses import DTYPES, E23, linear_inputs, tiny, u, within

pytestmark = pytest.mark.gpu


def live_reference(x, w, t, up, dl, z=0.0):
    """(losses, dx, dw, their bounds, G, a p) in 64 bits of rows that are all
    live, reduction "none"; dl: a logit's error.  G's rounding to a 16-bit type
    counts for every entry but the target's."""
    dtype = x.dtype
    xd, wd, g = x.detach().double(), w.detach().double(), up.double()
    n, v = len(xd), len(wd)
    logits = xd @ wd.t()
    lse = torch.logsumexp(logits, 1)
    loss = lse - logits.gather(1, t[:, None])[:, 0] + z * lse ** 2
    a, b = (g * (1 + 2 * z * lse))[:, None], -g[:, None]
    ap = a * (logits - lse[:, None]).exp()
    onehot = torch.zeros_like(ap).scatter_(1, t[:, None], 1.0)
    G = ap + b * onehot
    dx, dw = G @ wd, G.t() @ xd
    # the log of a sum: at most 256 additions one after another, and the exponentials
    dlse = dl + 2.0 ** -15 + 2.0 ** -22 * lse.abs()
    loss_b = (dl + dlse) * (1 + 2 * abs(z) * lse.abs()) + 2.0 ** -22 * (loss.abs() + lse.abs())
    # an exponential's argument and result, a product and a sum in fp32
    rel = (dl + dlse)[:, None] + 2.0 ** -20
    rounding = u(dtype) if dtype != torch.float32 else 0.0
    err = ap.abs() * (rel + rounding * (1 - onehot)) + (ap.abs() + b.abs()) * onehot * 2.0 ** -22
    top = float(torch.maximum(a.abs(), b.abs()).max())
    under = 2.0 ** -125 * top + (tiny(dtype) * top / 2 ** 9 if dtype == torch.float16 else 0.0)
    err = err + under
    # fp32 operands go in as parts whose left-out products are below 2^-21
    parts = 2.0 ** -21 if dtype == torch.float32 else 0.0
    dx_b = err @ wd.abs() + (G.abs() @ wd.abs()) * ((v / 32 + 96) * E23 + parts) + u(dtype) * dx.abs() + tiny(dtype)
    dw_b = err.t() @ xd.abs() + (G.abs().t() @ xd.abs()) * ((n / 32 + 96) * E23 + parts) + u(dtype) * dw.abs() \
        + tiny(dtype)
    return loss, dx, dw, loss_b, dx_b, dw_b, G


def logit_error(x, w):
    """One a row: the largest sum of magnitudes times the sum's and the parts' errors."""
    d = x.shape[1]
    size = (x.detach().double().abs() @ w.detach().double().abs().t()).amax(1)
    return size * ((d / 32 + 96) * E23 + (2.0 ** -21 if x.dtype == torch.float32 else 0.0))


def own(x, w, t, up, z=0.0):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = fuselse_amd.linear_cross_entropy(x, w, t, reduction="none", z_loss=z)
    return loss, *torch.autograd.grad(loss, (x, w), up)


def upstream(cuda, n, seed=1):
    return torch.randn(n, device=cuda, generator=torch.Generator(device=cuda).manual_seed(seed))


# ---------------------------------------------------------------------------
# Rows of very different magnitudes
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("e", [20, 30, 60])
@pytest.mark.parametrize("n,d,v", [(80, 64, 300), (140, 200, 1031), (700, 130, 5000)])
def test_one_large_row_leaves_the_others_their_digits(cuda, n, d, v, e):
    """fp32: a row of x and a row of w 2^e times the others'.  The large row of
    w has logits that underflow in every softmax, so that the other rows'
    losses and gradients are those without either."""
    print(f"case linear large row {n} {d} {v} {e}", flush=True)
    x, w, t = linear_inputs(cuda, n, d, v, torch.float32, seed=e)
    x = x.abs() + 0.25
    t[t == 5] = 6
    big_x, big_w = x.clone(), w.clone()
    big_x[3] *= 2.0 ** e
    big_w[5] = -(w[5].abs() + 0.25) * 2.0 ** e
    up = upstream(cuda, n)
    loss, dx, dw = own(big_x, big_w, t, up)
    rows = torch.arange(n, device=cuda) != 3
    others = torch.arange(v, device=cuda) != 5
    ts = torch.where(t > 5, t - 1, t)
    want, rx, _, b, bx, _, _ = live_reference(x[rows], w[others], ts[rows], up[rows], logit_error(x[rows], w[others]))
    within(loss[rows], want, b, "loss")
    within(dx[rows], rx, bx, "dx")
    plain = fuselse_amd.linear_cross_entropy(big_x, big_w, t, reduction="none")
    within(plain[rows], want, b, "loss without gradients")
    # dw without the large row's part: its upstream gradient is 0
    up[3] = 0.0
    _, _, dw = own(big_x, big_w, t, up)
    _, _, rw, _, _, bw, _ = live_reference(x[rows], w[others], ts[rows], up[rows], logit_error(x[rows], w[others]))
    within(dw[others], rw, bw, "dw")


# ---------------------------------------------------------------------------
# Several pieces of the vocabulary
# ---------------------------------------------------------------------------
def assert_several_pieces(n, d, v, dtype, w):
    """G of a piece, in the gradients' parts, lies in the backward's workspace:
    where G of the whole vocabulary would not fit there, there are several."""
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    parts = 3 if dtype == torch.float32 else 1
    nbytes = _lib.load().fl_linear_ce_workspace_bytes(n, v, d, code, 2, w.data_ptr(), d)
    assert 2 * parts * (-(-n // 64) * 64) * v > nbytes > 0


PIECES = [(torch.float32, 2048, 64, 45000, 0.1), (torch.float32, 22016, 68, 16389, 0.93),
          (torch.bfloat16, 4096, 130, 70000, 0.2), (torch.bfloat16, 4096, 192, 70000, 0.5),
          (torch.float16, 65536, 64, 16389, 0.96), (torch.bfloat16, 65536, 100, 16389, 0.97)]


@pytest.mark.parametrize("dtype,n,d,v,ignored", PIECES)
def test_vocabularies_of_several_pieces(cuda, dtype, n, d, v, ignored):
    """Targets on both sides of every multiple of 256, where pieces end, last
    pieces of 5 entries (9 pieces of 2048), packed and unpacked projections."""
    print(f"case linear several pieces {dtype} {n} {d} {v}", flush=True)
    x, w, t = linear_inputs(cuda, n, d, v, dtype, ignored=ignored, seed=v)
    assert_several_pieces(n, d, v, dtype, w)
    edges = torch.arange(256, v, 256, device=cuda)
    edges = torch.cat([edges - 1, edges, torch.tensor([0, v - 1], device=cuda)])
    at = (t != -100).nonzero()[:, 0]
    assert len(at) > len(edges)
    t[at[:: len(at) // len(edges)][:len(edges)]] = edges
    live = t != -100
    up = upstream(cuda, n)
    loss, dx, dw = own(x, w, t, up, z=1e-3)
    want, rx, rw, b, bx, bw, _ = live_reference(x[live], w, t[live], up[live], logit_error(x[live], w), z=1e-3)
    assert (loss[~live] == 0).all() and (dx[~live] == 0).all()
    within(loss[live], want, b, "loss")
    within(dx[live], rx, bx, "dx")
    within(dw, rw, bw, "dw")


# ---------------------------------------------------------------------------
# The rounding of the targets' entries, and of the logits
# ---------------------------------------------------------------------------
def dominated_inputs(cuda, n, d, v, dtype, targets, seed=0):
    """Targets' entries dominate both gradients: all probabilities are about
    1 / v, only targets' rows of w are large, and logits are exact (x whole
    multiples of 2^-12 below 2^-4, w quarters from 1 to 1.75, the others +-2^-6)."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    sign = lambda *s: torch.randint(0, 2, s, device=cuda, generator=g) * 2.0 - 1.0
    x = torch.randint(128, 256, (n, d), device=cuda, generator=g) * sign(n, d) * 2.0 ** -12
    w = sign(v, d) * 2.0 ** -6
    large = targets.unique()
    w[large] *= 2.0 ** 6 + 2.0 ** 4 * torch.randint(0, 4, (len(large), d), device=cuda, generator=g)
    return x.to(dtype), w.to(dtype)


def rounded(G, dtype):
    """G as the products would take it with every entry rounded to dtype."""
    scale = 2.0 ** (13 - math.frexp(float(G.abs().max()))[1])
    return (G * scale).to(dtype).double() / scale


@pytest.mark.parametrize("n,d,v,kind", [
    (300, 64, 20000, "few"),        # several rows a target, several targets a group of 64
    (300, 130, 20000, "one"),       # one target of every row; rows that are no whole vectors
    (513, 64, 9000, "each"),        # a target of its own for nearly every row
    (2469, 64, 125, "weighted"),    # many rows a group: its targets in several waves
    (65536, 64, 16389, "ignored"),  # several pieces
    (1500, 320, 40000, "few"),      # dw in whole sums, tiles of 256
])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_the_rounding_of_a_targets_entry_is_given_back(cuda, n, d, v, kind, dtype):
    print(f"case linear target rounding {n} {d} {v} {kind} {dtype}", flush=True)
    g = torch.Generator(device=cuda).manual_seed(n + d)
    if kind == "few":
        t = torch.tensor([64, 65, 66, 127, 700, v - 1], device=cuda)[torch.randint(0, 6, (n,), device=cuda, generator=g)]
    elif kind == "one":
        t = torch.full((n,), v - 3, device=cuda)
    else:
        t = torch.randint(0, 20 if kind == "weighted" else v, (n,), device=cuda, generator=g) * (5 if kind == "weighted" else 1)
    if kind == "ignored":
        t[torch.rand(n, device=cuda, generator=g) < 0.99] = -100
    x, w = dominated_inputs(cuda, n, d, v, dtype, t[t != -100], seed=v)
    up = upstream(cuda, n)
    if kind == "ignored":
        assert_several_pieces(n, d, v, dtype, w)
    if kind == "weighted":  # few rows carry the gradients
        up = torch.where(torch.arange(n, device=cuda) % 157 == 0, up, 2.0 ** -14)
    live = t != -100
    xl, tl, ul = x[live], t[live], up[live]
    loss, dx, dw = own(x, w, t, up)
    want, rx, rw, b, bx, bw, G = live_reference(xl, w, tl, ul, 0.0)
    # the bounds tell: without the rounding given back each gradient breaks them
    wrong = rounded(G, dtype)
    for name, bad, right, bound in (("dx", (wrong @ w.double()).to(dtype), rx, bx),
                                    ("dw", (wrong.t() @ xl.double()).to(dtype), rw, bw)):
        assert ((bad.double() - right).abs() > bound).any(), f"{name}: the bound does not tell"
    within(loss[live], want, b, "loss")
    within(dx[live], rx, bx, "dx")
    within(dw, rw, bw, "dw")


@pytest.mark.parametrize("n,d,v", [(300, 2048, 1000), (129, 4096, 300)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_exact_logits_of_many_columns(cuda, n, d, v, dtype):
    """x and w of -1, 0 and 1 times powers of two: logits have no error, and
    the results that of the exponentials, G's rounding and the sums alone."""
    print(f"case linear exact logits {n} {d} {v} {dtype}", flush=True)
    g = torch.Generator(device=cuda).manual_seed(d)
    x = (torch.randint(-1, 2, (n, d), device=cuda, generator=g) * 2.0 ** -2).to(dtype)
    w = (torch.randint(-1, 2, (v, d), device=cuda, generator=g) * 2.0 ** -2).to(dtype)
    t = torch.randint(0, v, (n,), device=cuda, generator=g)
    up = upstream(cuda, n)
    loss, dx, dw = own(x, w, t, up, z=1e-3)
    want, rx, rw, b, bx, bw, _ = live_reference(x, w, t, up, 0.0, z=1e-3)
    within(loss, want, b, "loss")
    within(dx, rx, bx, "dx")
    within(dw, rw, bw, "dw")


# ---------------------------------------------------------------------------
# Rows that are not finite
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_row_that_is_not_finite_stays_alone(cuda, value, dtype):
    print(f"case linear not finite {value} {dtype}", flush=True)
    x, w, t = linear_inputs(cuda, 90, 64, 300, dtype, seed=31)
    up = upstream(cuda, 90)
    bad_x = x.clone()
    bad_x[11, 5] = value
    loss, dx, dw = own(bad_x, w, t, up)
    rows = torch.arange(90, device=cuda) != 11
    want, rx, _, b, bx, _, _ = live_reference(x[rows], w, t[rows], up[rows], logit_error(x[rows], w))
    within(loss[rows], want, b, "loss")
    within(dx[rows], rx, bx, "dx")
    assert not torch.isfinite(loss[11]) and dx[11].isnan().all() and not torch.isfinite(dw[:, 5]).any()


# ---------------------------------------------------------------------------
# Forwards whose rows' pairs are joined piece by piece
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,n,d,v", [(torch.bfloat16, 65539, 64, 70001), (torch.float16, 65539, 72, 140003),
                                         (torch.float32, 65539, 64, 70001), (torch.bfloat16, 100, 32, 44_000_003)])
def test_pairs_joined_piece_by_piece(cuda, dtype, n, d, v):
    print(f"case linear join {dtype} {n} {d} {v}", flush=True)
    x, w, t = linear_inputs(cuda, n, d, v, dtype, ignored=0.1, seed=41)
    t[0], t[n - 1] = v - 1, 0
    loss = fuselse_amd.linear_cross_entropy(x, w, t, reduction="none")
    some = torch.arange(0, n, max(1, n // 99), device=cuda)
    some[-1] = n - 1
    xs, ts = x[some].double(), t[some]
    lse, size = torch.full((len(some),), -math.inf, dtype=torch.float64, device=cuda), 0.0
    for v0 in range(0, v, 1 << 20):
        part = w[v0:v0 + (1 << 20)].double()
        lse = torch.logaddexp(lse, torch.logsumexp(xs @ part.t(), 1))
        size = torch.maximum((xs.abs() @ part.abs().t()).amax(1), torch.as_tensor(size, device=cuda))
    live = ts != -100
    want = torch.where(live, lse - (xs * w[torch.where(live, ts, 0)].double()).sum(1), 0.0)
    dl = size * ((d / 32 + 96) * E23 + (2.0 ** -21 if dtype == torch.float32 else 0.0))
    bound = torch.where(live, 2 * dl + 2.0 ** -15 + 2.0 ** -21 * lse.abs(), 0.0)
    within(loss[some], want, bound, "loss")
    # a row's loss does not depend on the rows beside it, nor on the pieces
    few = fuselse_amd.linear_cross_entropy(x[some], w, t[some], reduction="none")
    within(few, want, bound, "loss of some rows")


# ---------------------------------------------------------------------------
# More elements of x than one launch has threads
# ---------------------------------------------------------------------------
def test_more_rows_than_one_packing_launch_covers(cuda):
    """2^23 rows of 4096 columns are 2^32 threads of 8 elements; all but a few
    are ignored, and hold whatever the memory held."""
    print("case linear long", flush=True)
    n, d, v = 1 << 23, 4096, 300
    torch.cuda.empty_cache()
    g = torch.Generator(device=cuda).manual_seed(51)
    x = torch.empty(n, d, dtype=torch.bfloat16, device=cuda)
    w = (torch.randn(v, d, device=cuda, generator=g) / 32).to(torch.bfloat16)
    at = torch.tensor([0, 1, 4097, n // 2, n - 3, n - 1], device=cuda)
    t = torch.full((n,), -100, device=cuda)
    t[at] = torch.randint(0, v, (len(at),), device=cuda, generator=g)
    x[at] = torch.randn(len(at), d, device=cuda, generator=g).to(torch.bfloat16)
    loss = fuselse_amd.linear_cross_entropy(x, w, t, reduction="none")
    xs = x[at].clone()
    del x
    torch.cuda.empty_cache()
    want, _, _, b, _, _, _ = live_reference(xs, w, t[at], torch.ones(len(at), device=cuda), logit_error(xs, w))
    within(loss[at], want, b, "loss")
    assert int((loss != 0).sum()) == len(at)
