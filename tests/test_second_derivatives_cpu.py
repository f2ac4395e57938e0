"""A gradient that depends on a saved tensor that requires a gradient is no
constant, whatever its upstream gradient: a gradient penalty on it has to raise,
not to lose its share.  The launches are stubbed, so this runs without a GPU; the
compiled calls have the same test on it."""

import pytest
import torch

from fuselse_amd import ext, layers, losses


def grads(y, leaves):
    return torch.autograd.grad(y, leaves, torch.ones_like(y), create_graph=True)


def refused(g):
    with pytest.raises(RuntimeError, match="once"):
        g.pow(2).sum().backward()


@pytest.fixture
def norm(monkeypatch):
    monkeypatch.setattr(ext, "_norm_fwd", lambda x, w, b, eps, stats: (x * 2, x.new_zeros(x.shape[0], 4)))
    monkeypatch.setattr(ext, "_norm_bwd", lambda g, x, w, dt, st, *need: tuple(
        t if n else None for t, n in zip((g * 3, g.sum(0), g.sum(0)), need)))
    return lambda x, w, b: layers._LayerNorm.apply(x, w, b, 1e-5)


def test_layer_norm(norm):
    x, w, b = torch.randn(3, 4), torch.randn(4), torch.randn(4)

    def leaves(*names):
        return [t.clone().requires_grad_(n in names) for n, t in zip("xwb", (x, w, b))]

    X, W, B = leaves("x", "w", "b")
    dx, dw, db = grads(norm(X, W, B), (X, W, B))
    refused(dx)
    refused(dw)
    assert not db.requires_grad  # sums of the upstream gradient
    X, W, B = leaves("w", "b")
    dw, db = grads(norm(X, W, B), (W, B))
    assert not dw.requires_grad and not db.requires_grad
    X, W, B = leaves("x")
    refused(grads(norm(X, W, B), (X,))[0])
    # an upstream gradient that requires one, and no second derivative at all
    X, W, B = leaves("b")
    y = norm(X, W, B)
    up = torch.ones_like(y).requires_grad_()
    refused(torch.autograd.grad(y, B, up, create_graph=True)[0])
    y = norm(X, W, B)
    assert not torch.autograd.grad(y, B, up)[0].requires_grad


def test_experts(monkeypatch):
    monkeypatch.setattr(ext, "_dispatch", lambda x, p: x.repeat(2, 1))
    monkeypatch.setattr(ext, "_combine", lambda r, w, p: r[:2] * 1)
    monkeypatch.setattr(ext, "_combine_bwd", lambda g, r, w, p, need_r, need_w: (
        g.repeat(2, 1) if need_r else None, torch.ones_like(w) if need_w else None))
    p = torch.zeros(2, 2, dtype=torch.int32)
    x = torch.randn(2, 3, requires_grad=True)
    (dx,) = grads(layers._Dispatch.apply(x, p), (x,))
    assert not dx.requires_grad  # linear: a constant
    r, w = torch.randn(4, 3, requires_grad=True), torch.randn(2, 2, requires_grad=True)
    dr, dw = grads(layers._Combine.apply(r, w, p), (r, w))
    refused(dr)
    refused(dw)
    assert not grads(layers._Combine.apply(r, w.detach(), p), (r,))[0].requires_grad
    assert not grads(layers._Combine.apply(r.detach(), w, p), (w,))[0].requires_grad


def test_losses(monkeypatch):
    loss = torch.zeros(())
    monkeypatch.setattr(ext, "_linear_fwd", lambda x, w, *a: (loss.clone(), loss))
    monkeypatch.setattr(ext, "_linear_bwd", lambda g, x, w, *a: (x * 2, w * 2))
    x, w, i = torch.randn(2, 3, requires_grad=True), torch.randn(5, 3, requires_grad=True), torch.zeros(2, dtype=torch.int64)
    for t in torch.autograd.grad(losses._LinearCrossEntropy.apply(x, w, i, -100, 2, 0.0), (x, w), create_graph=True):
        refused(t)
    monkeypatch.setattr(ext, "_distill_fwd", lambda x, *a: (loss.clone(), None, None, loss, loss))
    monkeypatch.setattr(ext, "_distill_bwd", lambda g, x, *a: x * 2)
    (g,) = torch.autograd.grad(losses._TopkDistillation.apply(x, x.detach(), i, 1.0, 2), x, create_graph=True)
    refused(g)
    monkeypatch.setattr(ext, "_router_fwd", lambda x, i, m: (loss.clone(), loss.clone(), i, loss, loss))
    monkeypatch.setattr(ext, "_router_bwd", lambda gb, gz, x, *a: x * 2)
    b, z, _ = losses._RouterBalance.apply(x, i, None)
    (g,) = torch.autograd.grad(b + z, x, create_graph=True)
    refused(g)
