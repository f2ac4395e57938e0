"""Layer norm of rows whose sums, or whose squares' sums, leave fp32 though the
elements do not, and of rows of equal or all but equal elements, in every kind of
kernel (rows of a thread, of lanes, of a block, of 1024 threads, read again).

Tolerances.  Steps of a sum over a row are at most D, each of 2^-23 relative (nE).
Once the mean is known to a rounding of itself (E23 |mean|) and the differences to it
are summed, what is left of the mean's error is nE of their mean magnitude."""

import math

import pytest
import torch

import fuselse_amd
from test_gpu_layers import randn
from test_gpu_losses import E23, tiny, u, within

pytestmark = pytest.mark.gpu

D = [3, 4, 7, 8, 40, 129, 768, 1028, 4096, 5000, 8200, 20001, 32768, 40000]


def check(x, w, b, eps=1e-5):
    cuda, dtype, d = x.device, x.dtype, x.shape[-1]
    x = x.detach().requires_grad_(True)
    y = fuselse_amd.layer_norm(x, w, b, eps=eps)
    g = randn(cuda, *y.shape, seed=7).to(dtype)
    dx, dw = torch.autograd.grad(y, (x, w), g)
    xd, gd, wd, bd = x.detach().double(), g.double(), w.detach().double(), b.detach().double()
    mean = xd.mean(1, keepdim=True)
    c = xd - mean
    var = c.square().mean(1, keepdim=True)
    rstd = 1 / (var + eps).sqrt()
    h = c * rstd
    nE = d * E23
    e0 = E23 * mean.abs() + 2 * nE * c.abs().mean(1, keepdim=True)
    d_abs = c.abs() + e0
    c_err = E23 * (d_abs + c.abs()) + (nE + 2 * E23) * d_abs.mean(1, keepdim=True)
    rel = 0.5 * (nE + 4 * E23) * (var + e0 ** 2) / (var + eps) + 4 * E23
    h_err = rstd * c_err + h.abs() * rel
    want = h * wd + bd
    within(y, want, wd.abs() * h_err + 2 * E23 * ((wd * h).abs() + bd.abs()) + u(dtype) * want.abs() + tiny(dtype), "y")
    a = gd * wd
    m0, m1 = a.mean(1, keepdim=True), (a * h).mean(1, keepdim=True)
    want = rstd * (a - m0 - h * m1)
    size = a.abs() + m0.abs() + (h * m1).abs()
    m0_err = (nE + 2 * E23) * a.abs().mean(1, keepdim=True)
    m1_err = (nE + 3 * E23) * (a * h).abs().mean(1, keepdim=True) + (a.abs() * h_err).mean(1, keepdim=True)
    err = rstd * (m0_err + h.abs() * m1_err + m1.abs() * h_err + 4 * E23 * size + h_err * m1_err) + rel * rstd * size
    # products with a subnormal reciprocal of the spread: three steps of 2^-149 and the elements' factors
    err = err + 2.0 ** -149 * (4 + size)
    within(dx, want, err + u(dtype) * want.abs() + tiny(dtype), "dx")
    want = (gd * h).sum(0)
    within(dw, want, (gd.abs() * h_err).sum(0) + (x.shape[0] + 1) * E23 * (gd * h).abs().sum(0) + u(w.dtype) * want.abs(),
           "dw")
    return y.detach()


def params(cuda, d):
    return (1 + 0.3 * randn(cuda, d, seed=3)).requires_grad_(True), randn(cuda, d, seed=4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", D)
def test_rows_whose_sums_leave_fp32(cuda, d, dtype):
    print(f"case norm range {d} {dtype}", flush=True)
    w, b = params(cuda, d)
    r = randn(cuda, 9, d)
    r[1] = torch.where(torch.arange(d, device=cuda) % 2 == 0, 1.0, -1.0)
    r[6] = 0
    r[6, d // 2] = 1
    r[8] = r[8].abs() + 1
    power = torch.tensor([0, 58, 62, 63, 64, 100, 126, -20, 122], device=cuda)
    check((r.double() * 2.0 ** power.double()[:, None]).to(dtype), w, b)
    # the usual rows among them are as by themselves
    ordinary = r[[0, 7]].to(dtype)
    y = fuselse_amd.layer_norm(ordinary, w, b).detach()
    mixed = torch.cat([ordinary[:1], torch.full((1, d), 2.0 ** 120, device=cuda, dtype=dtype), ordinary[1:]])
    assert torch.equal(fuselse_amd.layer_norm(mixed, w, b).detach()[[0, 2]], y)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", D)
def test_rows_of_equal_elements(cuda, d, dtype):
    """The variance is 0 and y the bias, exactly, whatever the value.

    The first mean is off by at most 50 + D / 1024 roundings of 2^-24, the mean of the
    differences, all equal, by as many of itself: together far less than half a step of
    the value, so that the mean moves to the value and all differences are 0."""
    print(f"case norm equal {d} {dtype}", flush=True)
    w, b = params(cuda, d)
    values = [0.0, 1.0, 123.456, -7e4, 65504.0, 1.2345e-7]
    if dtype != torch.float16:
        values += [1.1e10, 3.3e15, -1.7e18, 1e36, 1.6e38, -1.1e-38]
    x = torch.tensor(values, device=cuda).to(dtype).clamp(-65504 if dtype == torch.float16 else -math.inf)
    x = x[:, None].repeat(1, d).requires_grad_(True)
    for eps in (1e-5, 1e-12):
        y = fuselse_amd.layer_norm(x, w, b, eps=eps)
        assert torch.equal(y, b.to(dtype).expand_as(y))
        (dw,) = torch.autograd.grad(y, w, torch.ones_like(y))
        assert not dw.any()


@pytest.mark.parametrize("d", D)
def test_rows_of_all_but_equal_elements(cuda, d):
    """Differences of a few steps of fp32 to a large common value."""
    print(f"case norm all but equal {d}", flush=True)
    w, b = params(cuda, d)
    k = torch.randint(-4, 5, (6, d), device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)).double()
    k[3] = 0
    k[3, 0] = 1
    power = torch.tensor([10, 40, 63, 100, 120, 126], device=cuda).double()[:, None]
    check((1.2 * 2.0 ** power * (1 + k * 2.0 ** -22)).float(), w, b)


def test_rows_that_no_scale_holds(cuda):
    """Elements that are farther from the mean than fp32's largest make a row NaN, and
    leave the others as they are."""
    for d in (4, 40, 1028, 9000, 40000):
        w, b = params(cuda, d)
        x = randn(cuda, 3, d)
        y = fuselse_amd.layer_norm(x, w, b)
        x[1] = -3.4e38
        x[1, 0] = 3.4e38
        z = fuselse_amd.layer_norm(x, w, b)
        assert torch.equal(z[[0, 2]], y[[0, 2]]) and z[1].isnan().all()
