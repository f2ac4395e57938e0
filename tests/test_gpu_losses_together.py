"""A training step of the three losses against the same losses one by one."""

import pytest
import torch

import fuselse_amd
from test_gpu_losses import _moe_state, _moe_step, u

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", [0, 1, 2])
def test_a_steps_gradients_are_the_sums_of_each_losss(cuda, seed):
    """Each leaf's gradient in the step is the sum of what the losses alone give,
    rounded to the leaf's type: half a step of the sum where two gradients of a
    type are added, 2^-22 of both magnitudes where the router's backward takes
    both of its losses at once."""
    print(f"case together {seed}", flush=True)
    s = _moe_state(cuda, seed)
    got = dict(zip(("router", "hidden", "head"), _moe_step(s)[4:]))

    def ce():
        return fuselse_amd.linear_cross_entropy(s["hidden"], s["head"], s["target"], z_loss=1e-4)

    def kd():
        logits = s["hidden"][:32] @ s["head"].t()
        return 0.5 * fuselse_amd.topk_distillation(logits, s["teacher"], s["top"], temperature=2.0)

    def route():
        return fuselse_amd.router_balance(s["router"], s["choices"], mask=s["mask"])

    for leaf in ("hidden", "head"):
        a, b = (torch.autograd.grad(f(), s[leaf])[0].double() for f in (ce, kd))
        assert ((got[leaf].double() - (a + b)).abs() <= u(torch.bfloat16) * (a + b).abs()).all(), leaf
        assert float(a.norm()) > 0 and float(b.norm()) > 0
    a, b = (torch.autograd.grad(f, s["router"])[0].double()
            for f in (0.01 * route().balance_loss, 0.001 * route().z_loss))
    assert ((got["router"].double() - (a + b)).abs() <= 2.0 ** -22 * (a.abs() + b.abs()) + 2.0 ** -126).all()
