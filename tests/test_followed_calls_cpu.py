"""Calls that torch would have to follow by more than a backward: of tensors
with a forward-mode derivative, and under tracers.  What the kernels write is
no torch operation, so either would get a wrong result without an error: the
layers and losses refuse, the drop-ins leave such calls to torch.  The refusals
come before all other checks, so CPU tensors show them."""

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

import fuselse_amd
from fuselse_amd import ExpertOrder
from fuselse_amd.autograd import make_fuselse_logsumexp
from fuselse_amd.selective import make_selective_log_softmax

IDS = torch.zeros(2, dtype=torch.int64)
CHOICES = torch.zeros(2, 2, dtype=torch.int64)
ORDER = ExpertOrder(torch.zeros(2, 2, dtype=torch.int32), torch.zeros(4, dtype=torch.int64),
                    torch.zeros(5, dtype=torch.int32))

# a call of one tensor each
CALLS = {
    "embedding": (lambda t: fuselse_amd.embedding(IDS, t), (5, 4)),
    "norm input": (lambda t: fuselse_amd.layer_norm(t), (2, 4)),
    "norm weight": (lambda t: fuselse_amd.layer_norm(torch.zeros(2, 4), t), (4,)),
    "norm bias": (lambda t: fuselse_amd.layer_norm(torch.zeros(2, 4), None, t), (4,)),
    "dispatch": (lambda t: fuselse_amd.expert_dispatch(t, ORDER), (2, 4)),
    "combine rows": (lambda t: fuselse_amd.expert_combine(t, torch.zeros(2, 2), ORDER), (4, 4)),
    "combine weights": (lambda t: fuselse_amd.expert_combine(torch.zeros(4, 4), t, ORDER), (2, 2)),
    "linear input": (lambda t: fuselse_amd.linear_cross_entropy(t, torch.zeros(5, 4), IDS), (2, 4)),
    "linear weight": (lambda t: fuselse_amd.linear_cross_entropy(torch.zeros(2, 4), t, IDS), (5, 4)),
    "distillation": (lambda t: fuselse_amd.topk_distillation(t, torch.zeros(2, 2), CHOICES), (2, 4)),
    "teacher": (lambda t: fuselse_amd.topk_distillation(torch.zeros(2, 4), t, CHOICES), (2, 2)),
    "router": (lambda t: fuselse_amd.router_balance(t, CHOICES).balance_loss, (2, 4)),
}


@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_is_refused(name):
    call, shape = CALLS[name]
    x = torch.ones(shape)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(forward_ad.make_dual(x, x))
        # a level alone changes nothing
        with pytest.raises(RuntimeError, match="must be"):
            call(x)


@pytest.mark.parametrize("name", CALLS)
def test_tracers_are_refused(name):
    call, shape = CALLS[name]
    x = torch.ones(shape)
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(call)(x)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(call, (x,))


def test_an_order_is_not_traced():
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(lambda i: fuselse_amd.expert_order(i, 4).position)(CHOICES)


class FakeCuda(torch.Tensor):
    @property
    def is_cuda(self):
        return True


class NoKernels:
    def __getattr__(self, name):
        def call(*args, **kwargs):
            raise AssertionError(f"{name} was called")

        return call


@pytest.mark.parametrize("half", [False, True])
def test_logsumexp_leaves_forward_mode_to_torch(half):
    x = torch.randn(3, 7).to(torch.bfloat16 if half else torch.float32).as_subclass(FakeCuda)
    v = torch.randn(3, 7).to(x.dtype)
    f = make_fuselse_logsumexp(NoKernels(), half_inputs=half)
    with pytest.raises(AssertionError):
        f(x)
    with forward_ad.dual_level():
        got = forward_ad.unpack_dual(f(forward_ad.make_dual(x, v)))
        want = forward_ad.unpack_dual(torch.logsumexp(forward_ad.make_dual(x.as_subclass(torch.Tensor), v), -1))
        assert torch.equal(got.primal.as_subclass(torch.Tensor), want.primal)
        assert torch.equal(got.tangent.as_subclass(torch.Tensor), want.tangent)


def test_selective_log_softmax_leaves_forward_mode_to_torch():
    x, v = torch.randn(3, 7).as_subclass(FakeCuda), torch.randn(3, 7)
    i = torch.tensor([1, 6, 0])
    f = make_selective_log_softmax(NoKernels(), original=lambda a, b: a.log_softmax(-1)[range(3), b])
    with pytest.raises(AssertionError):
        f(x, i)
    with forward_ad.dual_level():
        got = forward_ad.unpack_dual(f(forward_ad.make_dual(x, v), i)).tangent
        want = v[range(3), i] - (torch.softmax(x.as_subclass(torch.Tensor), -1) * v).sum(-1)
        torch.testing.assert_close(got.as_subclass(torch.Tensor), want)
