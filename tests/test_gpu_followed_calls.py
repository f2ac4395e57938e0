"""Calls that torch follows by more than a backward, on the GPU: forward-mode
derivatives and tracers are refused by the compiled calls too (the drop-ins leave
the first to torch); modes that only watch, and torch.compile's way around calls
it cannot see into, change no result."""

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

import fuselse_amd
from fuselse_amd import layers
from test_gpu_layers import randint, randn
from test_gpu_layers_calls import chain, inputs, same

pytestmark = pytest.mark.gpu


class _None:
    """Stands in for the compiled calls and leaves every call to Python."""

    def __getattr__(self, name):
        return lambda *args: None


def calls(cuda):
    """A call of one tensor each, and the tensor."""
    s = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in inputs(cuda, torch.float32).items()}
    order = fuselse_amd.expert_order(s["index"], s["experts"])
    target = s["ids"] % 72
    return {
        "embedding": (lambda t: fuselse_amd.embedding(s["ids"], t), s["table"]),
        "norm input": (lambda t: fuselse_amd.layer_norm(t, s["w"], s["b"]), s["g"]),
        "norm weight": (lambda t: fuselse_amd.layer_norm(s["g"], t, s["b"]), s["w"]),
        "norm bias": (lambda t: fuselse_amd.layer_norm(s["g"], s["w"], t), s["b"]),
        "dispatch": (lambda t: fuselse_amd.expert_dispatch(t, order), s["g"]),
        "combine rows": (lambda t: fuselse_amd.expert_combine(t, s["gates"], order), s["made"]),
        "combine weights": (lambda t: fuselse_amd.expert_combine(s["made"], t, order), s["gates"]),
        "linear": (lambda t: fuselse_amd.linear_cross_entropy(t, s["table"], s["ids"]), s["g"]),
        "distillation": (lambda t: fuselse_amd.topk_distillation(t, s["g"][:, :2], target[:, None].expand(-1, 2)), s["g"]),
        "router": (lambda t: fuselse_amd.router_balance(t, target[:, None]).balance_loss, s["g"]),
    }


@pytest.mark.parametrize("python", [False, True])
def test_forward_mode_and_tracers_are_refused(cuda, monkeypatch, python):
    if python:
        monkeypatch.setattr(layers, "_common", _None())
    for name, (f, x) in calls(cuda).items():
        print(f"case followed {name}", flush=True)
        want = f(x)
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                f(forward_ad.make_dual(x, torch.ones_like(x)))
            assert torch.equal(f(x), want)
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(f)(x)
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(f, (x,))
        # functorch's wrappers have no memory that a kernel could read
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (x,), (x,))
        with pytest.raises(RuntimeError):
            torch.func.vmap(f)(x[None].clone())
        assert torch.equal(f(x), want)
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(lambda i: fuselse_amd.expert_order(i, 4).position)(randint(cuda, 4, 5, 2))


def test_drop_ins_leave_forward_mode_to_torch(cuda):
    x, v = randn(cuda, 5, 33), randn(cuda, 5, 33, seed=1)
    i = randint(cuda, 33, 5)
    p = torch.softmax(x.double(), -1)
    lse = (p * v).sum(-1)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, v)
        torch.testing.assert_close(forward_ad.unpack_dual(fuselse_amd.logsumexp(d)).tangent.double(), lse,
                                   rtol=1e-5, atol=1e-5)
        torch.testing.assert_close(forward_ad.unpack_dual(fuselse_amd.selective_log_softmax(d, i)).tangent.double(),
                                   v.double()[range(5), i] - lse, rtol=1e-5, atol=1e-5)


def test_modes_that_watch_change_nothing(cuda):
    from torch.utils.flop_counter import FlopCounterMode

    s = inputs(cuda)
    want = chain(s)
    with FlopCounterMode(display=False):
        assert same(chain(s), want)


def test_torch_compile_goes_around_the_calls(cuda):
    s = inputs(cuda)

    def step(ids, table, w, b, index, gates):
        x = fuselse_amd.layer_norm(fuselse_amd.embedding(ids, table) * 2, w, b)
        order = fuselse_amd.expert_order(index, 6)
        return fuselse_amd.expert_combine(fuselse_amd.expert_dispatch(x, order) + 1, gates, order) * 3

    args = [s[k] for k in ("ids", "table", "w", "b", "index", "gates")]
    want = step(*args)
    got = torch.compile(step, backend="eager")(*args)
    assert torch.equal(got, want)
    leaves = [s[k] for k in ("table", "w", "b", "gates")]
    assert same(torch.autograd.grad(got, leaves, s["g"]), torch.autograd.grad(want, leaves, s["g"]))
