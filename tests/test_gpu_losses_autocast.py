"""The training losses under torch.autocast, as mixed-precision training calls
them: hidden states of the region's type beside a head kept in fp32."""

import pytest
import torch

import fuselse_amd
from test_gpu_losses import distill_inputs, linear_inputs, router_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("region", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("types", [(None, torch.float32), (torch.float32, None), (torch.float16, torch.bfloat16)])
@pytest.mark.parametrize("n", [7, 150])
def test_operands_of_two_types_take_the_regions(cuda, region, types, n):
    """The same bits as with both cast by hand, gradients in the operands' own
    types; None stands for the region's type."""
    print(f"case autocast {region} {types} {n}", flush=True)
    tx, tw = (t or region for t in types)
    x, w, t = linear_inputs(cuda, n, 96, 333, torch.float32, ignored=0.2, seed=n)
    x, w = x.to(tx).requires_grad_(True), w.to(tw).requires_grad_(True)
    up = torch.full((), 1.5, device=cuda)
    want = fuselse_amd.linear_cross_entropy(x.to(region), w.to(region), t, z_loss=1e-3)
    rx, rw = torch.autograd.grad(want, (x, w), up)
    with torch.autocast("cuda", dtype=region):
        loss = fuselse_amd.linear_cross_entropy(x, w, t, z_loss=1e-3)
        dx, dw = torch.autograd.grad(loss, (x, w), up, retain_graph=True)
        with torch.no_grad():
            plain = fuselse_amd.linear_cross_entropy(x, w, t, z_loss=1e-3)
            assert torch.equal(plain, fuselse_amd.linear_cross_entropy(x.to(region), w.to(region), t, z_loss=1e-3))
    assert loss.dtype == torch.float32 and dx.dtype == tx and dw.dtype == tw
    assert torch.equal(loss, want) and torch.equal(dx, rx) and torch.equal(dw, rw)
    # a backward outside the region
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, (x, w), up), (rx, rw)))


def test_a_head_behind_a_layer_in_a_region(cuda):
    print("case autocast head", flush=True)
    x, w, t = linear_inputs(cuda, 64, 96, 333, torch.float32, seed=2)
    body = torch.nn.Linear(96, 96, device=cuda)
    head = torch.nn.Linear(96, 333, bias=False, device=cuda)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        hidden = body(x)
        assert hidden.dtype == torch.bfloat16
        fuselse_amd.linear_cross_entropy(hidden, head.weight, t).backward()
    assert head.weight.grad.dtype == torch.float32 and torch.isfinite(head.weight.grad).all()
    assert body.weight.grad.dtype == torch.float32 and float(body.weight.grad.abs().max()) > 0


def test_equal_types_and_the_other_losses_are_as_outside(cuda):
    print("case autocast equal", flush=True)
    x, w, t = linear_inputs(cuda, 90, 96, 333, torch.float32, seed=3)
    s, teacher, i = distill_inputs(cuda, (20,), 333, 6, torch.float32, torch.bfloat16)
    r, chosen = router_inputs(cuda, 90, 16, 2, torch.float32)

    def all_three():
        b = fuselse_amd.router_balance(r, chosen)
        return [fuselse_amd.linear_cross_entropy(x, w, t), fuselse_amd.topk_distillation(s, teacher, i), b.balance_loss,
                b.z_loss]

    want = all_three()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert all(torch.equal(a, b) for a, b in zip(all_three(), want))


def test_operands_of_two_types_outside_a_region_are_refused(cuda):
    x, w, t = linear_inputs(cuda, 9, 64, 33, torch.float32)
    with pytest.raises(RuntimeError, match="weight must have x's dtype"):
        fuselse_amd.linear_cross_entropy(x.bfloat16(), w, t)
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=False):
        with pytest.raises(RuntimeError, match="weight must have x's dtype"):
            fuselse_amd.linear_cross_entropy(x.bfloat16(), w, t)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        with pytest.raises(RuntimeError, match="x must be float32"):
            fuselse_amd.linear_cross_entropy(x.double(), w, t)
