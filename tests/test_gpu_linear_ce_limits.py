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
