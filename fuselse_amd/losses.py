"""Losses of a language model's training on the log-sum-exp kernels, with
autograd: the cross entropy of a vocabulary projection without its logits, the
distillation from a teacher's top logits, and the balance loss of a
mixture-of-experts router.  No counterpart in the reference.

All take CUDA tensors only and raise RuntimeError for anything the kernels do
not take; there is no CPU fallback.  They are differentiable once, backward,
and cannot be traced into a graph (torch.jit.trace, make_fx).  A call holds no
state: its workspace comes from torch's allocator on the current stream, so
calls may run on several streams and be captured into graphs.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import ext


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A 2-D view of t with contiguous rows (a copy where there is none)."""
    if t.dim() != 2:
        t = t.reshape(t.shape[:-1].numel(), t.shape[-1])
    if (t.stride(1) != 1 and t.shape[1] != 1) or (t.stride(0) < t.shape[1] and t.shape[0] > 1):
        t = t.contiguous()
    return t


def _integers(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dtype == torch.int64:
        return t
    ext._check(not (t.is_floating_point() or t.is_complex() or t.dtype == torch.bool),
               f"{name} must be an integer tensor")
    return t.to(torch.int64)


def _one_type(a: torch.Tensor, b: torch.Tensor):
    """In an autocast region two tensors of different types brought to the
    region's, as its matrix products take them; else the tensors themselves."""
    if a.dtype != b.dtype and torch.is_autocast_enabled("cuda"):
        to = torch.get_autocast_dtype("cuda")
        a, b = (t.to(to) if t.dtype in ext._DTYPE_CODE else t for t in (a, b))
    return a, b


def _once(backward):
    """A backward whose results are constants: with create_graph, those that
    depend on what requires a gradient (the upstream one, or, where ctx.saved
    says so, saved tensors) are an error where they are differentiated again."""

    def run(ctx, *grads):
        if not torch.is_grad_enabled():
            return backward(ctx, *grads)
        with torch.no_grad():
            out = backward(ctx, *grads)
        out = out if isinstance(out, tuple) else (out,)
        saved = (True,) * len(out) if any(g is not None and g.requires_grad for g in grads) else ctx.saved
        return tuple(_constant(t) if t is not None and s else t for t, s in zip(out, saved))

    return staticmethod(run)


def _constant(t: torch.Tensor) -> torch.Tensor:
    error = torch._C._functions.DelayedError(
        b"trying to differentiate twice a function that is differentiable once", 1)
    return error(t.detach().requires_grad_())


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target, ignore_index, reduction, z_loss):
        loss, lse = ext._linear_fwd(x, weight, target, ignore_index, reduction, z_loss, True)
        ctx.save_for_backward(x, weight, target, lse)
        ctx.args = (ignore_index, reduction, z_loss)
        ctx.saved = (True, True, False, False, False, False)
        return loss

    @_once
    def backward(ctx, grad):
        x, weight, target, lse = ctx.saved_tensors
        need = ctx.needs_input_grad
        # in rows again, which a saved-tensor hook may have changed
        dx, dw = ext._linear_bwd(grad.contiguous(), _rows(x), _rows(weight), target, lse, *ctx.args, need[0], need[1])
        return dx, dw, None, None, None, None


def linear_cross_entropy(input: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: int = -100,
                         reduction: str = "mean", z_loss: float = 0.0) -> torch.Tensor:
    """Cross entropy of the logits input @ weight.T, which are never stored.

    input (..., D) and weight (V, D) in fp32, fp16 or bf16, target (...)
    integers.  With l the logits of a token and lse their log-sum-exp, its
    loss is lse - l[target] + z_loss * lse^2, in fp32.  Tokens whose target is
    ignore_index have loss 0 and gradient 0 and cost nothing: their input is
    not read.  Another target outside [0, V) makes the loss NaN, and with it
    the gradients.  reduction: "none" (a loss per token, target's shape), "sum",
    or "mean" over the tokens that are not ignored (0 where all are).

    input and weight are of one type; in a torch.autocast region they may differ
    and are then both cast to the region's.

    Gradients reach input and weight.  The backward makes the logits again in
    pieces of the vocabulary; its workspace, and the forward's, grow with
    N * D and with N and D times one piece, not with N * V.

    Sums are fp32, and fp32 products good to 2^-21; an fp32 element's digits
    below 2^-39 of the largest magnitude in its row do not enter the logits,
    and magnitudes above 2^116 may overflow in the gradients.  In fp16 and bf16
    the gradient of the logits is rounded to the type before its products; in
    fp16 what lies below 2^-39 of the largest row's is lost.  At most 2^23
    tokens, 2^28 vocabulary entries and 2^20 columns.
    """
    ext._check_eager(input, weight)
    ext._check(input.dim() >= 1 and tuple(input.shape[:-1]) == tuple(target.shape),
               "target must have input's shape without its last dimension")
    input, weight = _one_type(input, weight)
    x, w = _rows(input), _rows(weight) if weight.dim() == 2 else weight
    t = _integers(target, "target").reshape(-1).contiguous()
    ext._check_linear(x, w, t)
    red = ext._reduction(reduction)
    if torch.is_grad_enabled() and (input.requires_grad or weight.requires_grad):
        loss = _LinearCrossEntropy.apply(x, w, t, ignore_index, red, z_loss)
    else:
        loss, _ = ext._linear_fwd(x, w, t, ignore_index, red, z_loss, False)
    return loss.reshape(target.shape) if reduction == "none" and target.dim() != 1 else loss


class _TopkDistillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher, index, temperature, reduction):
        loss, _, _, norm, pairs = ext._distill_fwd(logits, teacher, index, temperature, reduction, True)
        ctx.save_for_backward(logits, teacher, index, norm, pairs)
        ctx.temperature = temperature
        ctx.saved = (True, False, False, False, False)
        return loss

    @_once
    def backward(ctx, grad):
        logits, teacher, index, norm, pairs = ctx.saved_tensors
        if logits.stride(-1) != 1 and logits.shape[-1] != 1:  # as a saved-tensor hook may give it back
            logits = logits.contiguous()
        g = ext._distill_bwd(grad.contiguous(), logits, teacher, index, None, None, norm, ctx.temperature, pairs)
        return g, None, None, None, None


def topk_distillation(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_index: torch.Tensor,
                      temperature: float = 1.0, reduction: str = "mean") -> torch.Tensor:
    """Distillation of a student from a teacher's top-K logits.

    logits (..., V), teacher_logits (..., K) in fp32, fp16 or bf16,
    teacher_index (..., K) integers, the columns of the teacher's entries.  A
    row's loss is temperature^2 * KL(p || q) in fp32, p the softmax of its
    teacher_logits / temperature over the K entries, q the softmax of logits /
    temperature over all columns.  Teacher entries of -inf are unused, whatever
    their index; a row without any other has loss and gradient 0.  A used index
    outside [0, V) makes the row's loss and gradient NaN; an index that comes
    several times takes the sum of its probabilities.  reduction: "none",
    "sum", or "mean" over the rows that have a teacher (0 where none has).

    At most 2^22 rows of 2^28 columns and 1024 teacher entries a row; the
    temperature's square and its inverse have to be normal fp32 numbers.

    The gradient reaches logits, in their type; the teacher gets none.  3-D
    logits whose last dimension is contiguous are read where they are
    (logits[:, :-1] of a batch of sequences is not copied).
    """
    ext._check_eager(logits, teacher_logits)
    ext._check(logits.dim() >= 1 and tuple(logits.shape[:-1]) == tuple(teacher_logits.shape[:-1])
               and teacher_logits.shape == teacher_index.shape,
               "teacher_logits and teacher_index must be (..., K) with the rows of logits")
    lead = logits.shape[:-1]
    x, t, i = logits, teacher_logits.detach(), _integers(teacher_index, "teacher_index")
    if x.dim() not in (2, 3):
        x, t, i = (u.reshape(lead.numel(), u.shape[-1]) for u in (x, t, i))
    if x.stride(-1) != 1 and x.shape[-1] != 1:
        x = x.contiguous()
    t, i = t.contiguous(), i.contiguous()
    ext._check_distill(x, t, i)
    red = ext._reduction(reduction)
    if torch.is_grad_enabled() and logits.requires_grad:
        loss = _TopkDistillation.apply(x, t, i, temperature, red)
    else:
        loss = ext._distill_fwd(x, t, i, temperature, red, False)[0]
    return loss.reshape(lead) if reduction == "none" else loss


class RouterBalance(NamedTuple):
    """What router_balance returns."""

    balance_loss: torch.Tensor
    z_loss: torch.Tensor
    counts: torch.Tensor


class _RouterBalance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, index, mask):
        balance, z, counts, lse, coef = ext._router_fwd(logits, index, mask)
        ctx.save_for_backward(logits, mask, lse, coef)
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)
        ctx.saved = (True, False, False)
        return balance, z, counts

    @_once
    def backward(ctx, grad_balance, grad_z, _):
        if grad_balance is None and grad_z is None:
            return None, None, None
        logits, mask, lse, coef = ctx.saved_tensors
        return ext._router_bwd(grad_balance, grad_z, _rows(logits), mask, lse, coef), None, None


def router_balance(logits: torch.Tensor, index: torch.Tensor, mask: Optional[torch.Tensor] = None) -> RouterBalance:
    """Balance loss, z loss and per-expert counts of a mixture-of-experts
    router.

    logits (..., experts) in fp32, fp16 or bf16, index (..., top) integers, the
    experts each token chose, mask (...) bool, the tokens that take part (None:
    all; the others may hold anything).  Over the n tokens that do:
    counts[e] = how many of their choices are e (int64), balance_loss =
    experts * sum_e counts[e] / (n * top) * mean of softmax(logits)[e], z_loss =
    mean of logsumexp(logits)^2, both fp32 and 0 where n is 0.  Choices outside
    [0, experts) count for no expert.  Gradients of both losses reach logits;
    the counts are constants.  At most 1024 experts, 1024 choices a token and
    2^31 - 1 choices.
    """
    ext._check_eager(logits)
    ext._check(logits.dim() >= 1 and tuple(logits.shape[:-1]) == tuple(index.shape[:-1]) and index.dim() >= 1,
               "index must be (..., top) with the tokens of logits")
    ext._check(mask is None or tuple(mask.shape) == tuple(logits.shape[:-1]),
               "mask must have the shape of logits' tokens")
    x = _rows(logits)
    i = _integers(index, "index")
    i = i.reshape(x.shape[0], i.shape[-1]).contiguous() if i.dim() != 2 else i.contiguous()
    m = mask.reshape(-1).contiguous() if mask is not None else None
    ext._check_router(x, i, m)
    if torch.is_grad_enabled() and logits.requires_grad:
        return RouterBalance(*_RouterBalance.apply(x, i, m))
    return RouterBalance(*ext._router_fwd(x, i, m)[:3])
