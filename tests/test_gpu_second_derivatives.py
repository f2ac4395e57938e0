"""Gradient penalties on the layers and losses: a gradient that depends on a saved
tensor that requires a gradient raises where it is differentiated again, also
under a constant upstream gradient; one that does not is a constant."""

import pytest
import torch

import fuselse_amd
from fuselse_amd import layers
from test_gpu_followed_calls import _None
from test_gpu_layers_calls import inputs

pytestmark = pytest.mark.gpu


def state(cuda, *names):
    """inputs with these as the only leaves that require a gradient."""
    s = inputs(cuda, torch.float32)
    s["x"] = s["g"].clone()
    for k in ("x", "table", "w", "b", "gates", "made"):
        s[k] = s[k].detach().clone().requires_grad_(k in names)
    s["order"] = fuselse_amd.expert_order(s["index"], s["experts"])
    return s


CALLS = {
    "embedding": lambda s: fuselse_amd.embedding(s["ids"], s["table"]),
    "norm": lambda s: fuselse_amd.layer_norm(s["x"], s["w"], s["b"]),
    "dispatch": lambda s: fuselse_amd.expert_dispatch(s["x"], s["order"]),
    "combine": lambda s: fuselse_amd.expert_combine(s["made"], s["gates"], s["order"]),
    "linear": lambda s: fuselse_amd.linear_cross_entropy(s["x"], s["table"], s["ids"]),
    "distillation": lambda s: fuselse_amd.topk_distillation(s["x"], s["b"].expand(150, 72)[:, :2],
                                                            (s["ids"] % 72)[:, None].expand(-1, 2)),
    "router": lambda s: fuselse_amd.router_balance(s["x"], (s["ids"] % 72)[:, None]).z_loss,
}
# the call, what requires a gradient, and which of the gradients depend on it
CASES = [("embedding", ["table"], []), ("norm", ["x", "w", "b"], ["x", "w"]), ("norm", ["x"], ["x"]),
         ("norm", ["w", "b"], []), ("norm", ["x", "b"], ["x"]), ("norm", ["b"], []), ("dispatch", ["x"], []),
         ("combine", ["made", "gates"], ["made", "gates"]), ("combine", ["made"], []), ("combine", ["gates"], []),
         ("linear", ["x", "table"], ["x", "table"]), ("linear", ["x"], ["x"]), ("distillation", ["x"], ["x"]),
         ("router", ["x"], ["x"])]


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("name,leaves,depend", CASES)
def test_gradient_penalty(cuda, monkeypatch, name, leaves, depend, python):
    if python:
        monkeypatch.setattr(layers, "_common", _None())
    print(f"case second {name} {leaves} {python}", flush=True)
    s = state(cuda, *leaves)
    at = [s[k] for k in leaves]
    y = CALLS[name](s)
    plain = torch.autograd.grad(y, at, torch.ones_like(y), retain_graph=True)
    got = torch.autograd.grad(y, at, torch.ones_like(y), create_graph=True)
    for k, g, p in zip(leaves, got, plain):
        assert torch.equal(g.detach(), p) and not p.requires_grad
        assert g.requires_grad == (k in depend), k
        if k in depend:
            with pytest.raises(RuntimeError, match="once"):
                (g.pow(2).sum() + at[0].sum()).backward()
    # under an upstream gradient that requires one, all of them
    up = torch.ones_like(y).requires_grad_()
    for g in torch.autograd.grad(CALLS[name](s), at, up, create_graph=True):
        with pytest.raises(RuntimeError, match="once"):
            g.sum().backward()
