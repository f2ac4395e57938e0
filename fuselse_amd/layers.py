"""Layers of a language model's training step around its losses, with
autograd: the embedding lookup, layer norm, and tokens brought into their
experts' order and back.  No counterpart in the reference.

All take CUDA tensors only and raise RuntimeError for anything the kernels do
not take; there is no CPU fallback.  They are differentiable once, backward,
and cannot be traced into a graph (torch.jit.trace, make_fx).  A call holds no
state: its workspace comes from torch's allocator on the current stream, so
calls may run on several streams and be captured into graphs.  Sums are fp32
and results are rounded once, to the input's type, in autocast regions too.

A call on contiguous tensors of the current device that need no conversion is
made by compiled code (``_layers.so``), autograd and all, since the host's part
is most of a small call; what follows here is every other call, and what refuses.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib, ext
from .losses import _integers, _once, _rows

_common = None


def _bind():
    """The compiled calls, which need the library and torch loaded first."""
    global _common
    _lib.load()
    try:
        from . import _layers
    except ImportError as e:
        raise _lib.NativeLibraryMissing(
            f"fuselse_amd: cannot load fuselse_amd/_layers.so ({e}); run "
            "`python -c 'import __graft_entry__ as g; g.build()'`") from e
    _common = _layers
    return _layers


def _flat(t: torch.Tensor) -> torch.Tensor:
    """t in rows, as the kernels take them."""
    t = t.resolve_neg()
    return t if t.dim() == 2 and t.is_contiguous() else _rows(t)


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, index, scale, padding):
        ctx.save_for_backward(index)
        ctx.args = (weight.shape[0], scale, padding)
        ctx.saved = (False,) * 4
        return ext._embedding_fwd(weight, index, scale)

    @_once
    def backward(ctx, grad):
        (index,) = ctx.saved_tensors
        return ext._embedding_bwd(_flat(grad), index.contiguous(), *ctx.args), None, None, None


def embedding(index: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
              padding_idx: Optional[int] = None) -> torch.Tensor:
    """scale * weight[index], as torch.nn.functional.embedding takes them.

    index (...) integers, weight (V, D) in fp32, fp16 or bf16; the result is
    (..., D) of weight's type, exact copies of its rows where scale is 1.  An
    index outside [0, V) gives a row of NaN and no gradient.

    The gradient reaches weight, dense: each row the sum of its tokens'
    gradients, in an order that index alone decides, times scale; tokens of
    padding_idx (negative: from the end) give none.  At most 2^30 tokens and vocabulary entries and
    2^20 columns.
    """
    padding = -1
    if padding_idx is not None:
        V = weight.shape[0] if weight.dim() else 0
        ext._check(-V <= padding_idx < V, "padding_idx must be within the rows of weight")
        padding = padding_idx % V
    out = (_common or _bind()).embedding(index, weight, scale, padding)
    if out is not None:
        return out
    ext._check_eager(weight)
    i = _integers(index, "index").reshape(-1).contiguous()
    w = _flat(weight) if weight.dim() == 2 else weight
    ext._check_embedding(w, i)
    if weight.requires_grad and torch.is_grad_enabled():
        out = _Embedding.apply(w, i, scale, padding)
    else:
        out = ext._embedding_fwd(w, i, scale)
    return out if index.dim() == 1 else out.reshape(*index.shape, w.shape[1])


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = ext._norm_fwd(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        of = weight if weight is not None else bias
        ctx.params_dtype = of.dtype if of is not None else None
        of_x, of_weight = ctx.needs_input_grad[:2]
        ctx.saved = (of_x or of_weight, of_x, False, False)
        return y

    @_once
    def backward(ctx, grad):
        x, weight, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        # as they were saved, which a saved-tensor hook may have changed
        weight = weight.contiguous() if weight is not None else None
        dx, dw, db = ext._norm_bwd(_flat(grad), _flat(x), weight, ctx.params_dtype, stats.contiguous(), *need[:3])
        return dx, dw, db, None


def layer_norm(input: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the last dimension.

    input (..., D) in fp32, fp16 or bf16; weight and bias (D,), each may be
    None; they may be of any of these types and are taken in fp32 where they
    are not of input's.  y = (x - mean) / sqrt(variance + eps) * weight + bias
    in input's type, the variance over D; a value that a row's elements have in
    common costs no digits, and equal elements give the bias exactly (eps 0:
    NaN).  Elements may be of any size: only a row in which one differs from
    the mean by more than fp32 holds is NaN.  Gradients reach all three.  At
    most 2^31 - 1 rows and 2^24 columns.
    """
    out = (_common or _bind()).layer_norm(input, weight, bias, eps)
    if out is not None:
        return out
    ext._check_eager(input, weight, bias)
    ext._check(input.dim() >= 1, "input must have a last dimension")
    x = _flat(input)
    needs = input.requires_grad
    if weight is not None or bias is not None:
        needs = needs or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)
        if any(t is not None and t.dtype != x.dtype for t in (weight, bias)):
            weight, bias = (t.float() if t is not None and t.dtype in ext._DTYPE_CODE else t for t in (weight, bias))
        weight, bias = (t.resolve_neg().contiguous() if t is not None else None for t in (weight, bias))
    ext._check_norm(x, weight, bias)
    if needs and torch.is_grad_enabled():
        y = _LayerNorm.apply(x, weight, bias, eps)
    else:
        y = ext._norm_fwd(x, weight, bias, eps, False)[0]
    return y if input.dim() == 2 else y.reshape(input.shape)


class ExpertOrder(NamedTuple):
    """What expert_order returns."""

    position: torch.Tensor
    counts: torch.Tensor
    offsets: torch.Tensor


def expert_order(index: torch.Tensor, num_experts: int, mask: Optional[torch.Tensor] = None) -> ExpertOrder:
    """The order that brings tokens to their experts.

    index (..., top) integers, the experts each token chose, mask (...) bool,
    the tokens that take part (None: all), both as router_balance takes them.
    The entries of index are put in the order of their experts, and in their own
    within one; entries of the other tokens, and of no expert of [0,
    num_experts), are dropped and come last.  position (index's shape, int32):
    an entry's place p, or -1 - p where it is dropped; counts (num_experts,
    int64); offsets (num_experts + 1, int32): expert e has the places
    [offsets[e], offsets[e + 1]), offsets[1:] are the ends a grouped product
    takes.  At most 1024 experts, 1024 choices a token, 2^30 tokens and 2^31 - 1
    choices.
    """
    out = (_common or _bind()).expert_order(index, num_experts, mask)
    if out is not None:
        return ExpertOrder._make(out)
    ext._check_eager()
    ext._check(index.dim() >= 1, "index must be (..., top)")
    i, m = _integers(index, "index"), mask
    i = i.reshape(i.shape[:-1].numel(), i.shape[-1]).contiguous()
    if m is not None:
        ext._check(m.shape == index.shape[:-1], "mask must have the shape of index's tokens")
        m = m.reshape(-1).contiguous()
    ext._check_order(i, num_experts, m)
    position, counts, offsets = ext._order(i, num_experts, m)
    return ExpertOrder(position if index.dim() == 2 else position.reshape(index.shape), counts, offsets)


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, position):
        ctx.save_for_backward(position)
        ctx.saved = (False, False)
        return ext._dispatch(x, position)

    @_once
    def backward(ctx, grad):
        (position,) = ctx.saved_tensors
        return ext._combine(_flat(grad), None, position.contiguous()), None


def expert_dispatch(input: torch.Tensor, order: ExpertOrder) -> torch.Tensor:
    """The tokens' rows in their experts' order: (entries, D), row p of input
    the row of the token whose entry has place p, zeros at the places of dropped
    entries.

    input (..., D) in fp32, fp16 or bf16 with the tokens of the index that
    order was made of.  The gradient reaches input: a token's is the sum of its
    rows', in the order of its choices.  At most 2^24 columns.
    """
    out = (_common or _bind()).expert_dispatch(input, order.position)
    if out is not None:
        return out
    ext._check_eager(input)
    ext._check(input.dim() >= 1 and input.shape[:-1] == order.position.shape[:-1],
               "input must be (..., D) with the tokens of order")
    x, position = _flat(input), _flat(order.position)
    ext._check_dispatch(x, position)
    if input.requires_grad and torch.is_grad_enabled():
        return _Dispatch.apply(x, position)
    return ext._dispatch(x, position)


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, position):
        ctx.save_for_backward(rows, weights, position)
        ctx.saved = (ctx.needs_input_grad[1], ctx.needs_input_grad[0], False)
        return ext._combine(rows, weights, position)

    @_once
    def backward(ctx, grad):
        rows, weights, position = ctx.saved_tensors
        need = ctx.needs_input_grad
        d_rows, d_weights = ext._combine_bwd(_flat(grad), _flat(rows), weights.contiguous(), position.contiguous(),
                                             need[0], need[1])
        return d_rows, d_weights, None


def expert_combine(rows: torch.Tensor, weights: torch.Tensor, order: ExpertOrder) -> torch.Tensor:
    """The experts' rows back at their tokens: (..., D), each token's sum of its
    entries' rows times their weights, in the order of its choices.

    rows (entries, D) in fp32, fp16 or bf16, in the order that expert_dispatch
    gives; weights (..., top), order's index's shape, taken in fp32 where they
    are not of rows' type.  Dropped entries give nothing: their rows and weights
    may hold anything, and their gradients are 0.  Gradients
    reach rows and weights.  At most 2^24 columns.
    """
    out = (_common or _bind()).expert_combine(rows, weights, order.position)
    if out is not None:
        return out
    ext._check_eager(rows, weights)
    ext._check(weights.shape == order.position.shape, "weights must have the shape of order's index")
    needs = rows.requires_grad or weights.requires_grad
    w = weights
    if w.dtype != rows.dtype and w.dtype in ext._DTYPE_CODE:
        w = w.float()
    r, w, position = _flat(rows) if rows.dim() == 2 else rows, _flat(w).contiguous(), _flat(order.position)
    ext._check_combine(r, w, position)
    if needs and torch.is_grad_enabled():
        out = _Combine.apply(r, w, position)
    else:
        out = ext._combine(r, w, position)
    return out if weights.dim() == 2 else out.reshape(*weights.shape[:-1], r.shape[1])
