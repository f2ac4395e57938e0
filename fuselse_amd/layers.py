"""Layers of a language model's training step around its losses, with
autograd: the embedding lookup, layer norm, and tokens brought into their
experts' order and back.  No counterpart in the reference.

All take CUDA tensors only and raise RuntimeError for anything the kernels do
not take; there is no CPU fallback.  They are differentiable once.  A call
holds no state: its workspace comes from torch's allocator on the current
stream, so calls may run on several streams and be captured into graphs.
Sums are fp32 and results are rounded once, to the input's type, in autocast
regions too.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import ext
from .losses import _integers, _rows


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, index, scale, padding):
        ctx.save_for_backward(index)
        ctx.args = (weight.shape[0], scale, padding)
        return ext._embedding_fwd(weight, index, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (index,) = ctx.saved_tensors
        return ext._embedding_bwd(_rows(grad), index, *ctx.args), None, None, None


def embedding(index: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
              padding_idx: Optional[int] = None) -> torch.Tensor:
    """scale * weight[index], as torch.nn.functional.embedding takes them.

    index (...) integers, weight (V, D) in fp32, fp16 or bf16; the result is
    (..., D) of weight's type, exact copies of its rows where scale is 1.  An
    index outside [0, V) gives a row of NaN and no gradient.

    The gradient reaches weight, dense: each row the sum of its tokens'
    gradients in their order, times scale; tokens of padding_idx (negative:
    from the end) give none.  At most 2^30 tokens and vocabulary entries and
    2^20 columns.
    """
    w = _rows(weight) if weight.dim() == 2 else weight
    i = _integers(index, "index").reshape(-1).contiguous()
    ext._check_embedding(w, i)
    V, D = w.shape
    padding = -1
    if padding_idx is not None:
        ext._check(-V <= padding_idx < V, "padding_idx must be within the rows of weight")
        padding = padding_idx % V
    if torch.is_grad_enabled() and weight.requires_grad:
        out = _Embedding.apply(w, i, scale, padding)
    else:
        out = ext._embedding_fwd(w, i, scale)
    return out if index.dim() == 1 else out.reshape(*index.shape, D)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = ext._norm_fwd(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, bias, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, bias, stats = ctx.saved_tensors
        # in rows again, which a saved-tensor hook may have changed
        return *ext._norm_bwd(_rows(grad), _rows(x), weight, bias, stats, *ctx.needs_input_grad[:3]), None


def layer_norm(input: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the last dimension.

    input (..., D) in fp32, fp16 or bf16; weight and bias (D,), each may be
    None; they may be of any of these types and are taken in fp32 where they
    are not of input's.  y = (x - mean) / sqrt(variance + eps) * weight + bias
    in input's type, the variance over D; a value that a row's elements have in
    common costs no digits.  Rows that spread over more than about 2^63
    overflow.  Gradients reach all three.  At most 2^31 - 1 rows and 2^24
    columns.
    """
    ext._check(input.dim() >= 1, "input must have a last dimension")
    x = _rows(input)
    params = [t for t in (weight, bias) if t is not None]
    if params and not all(t.dtype == x.dtype for t in params):
        weight, bias = (t.float() if t is not None and t.dtype in ext._DTYPE_CODE else t for t in (weight, bias))
    weight, bias = (t.contiguous() if t is not None else None for t in (weight, bias))
    ext._check_norm(x, weight, bias)
    if torch.is_grad_enabled() and (input.requires_grad or any(t.requires_grad for t in params)):
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
    ext._check(index.dim() >= 1, "index must be (..., top)")
    ext._check(mask is None or tuple(mask.shape) == tuple(index.shape[:-1]),
               "mask must have the shape of index's tokens")
    i = _integers(index, "index")
    i = i.reshape(i.shape[:-1].numel(), i.shape[-1]) if i.dim() != 2 else i
    i = i.contiguous()
    m = mask.reshape(-1).contiguous() if mask is not None else None
    ext._check_order(i, num_experts, m)
    position, counts, offsets = ext._order(i, num_experts, m)
    return ExpertOrder(position if index.dim() == 2 else position.reshape(index.shape), counts, offsets)


def _position(order: ExpertOrder) -> torch.Tensor:
    p = order.position
    if p.dim() != 2:
        p = p.reshape(p.shape[:-1].numel(), p.shape[-1])
    return p.contiguous()


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, position):
        ctx.save_for_backward(position)
        return ext._dispatch(x, position)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (position,) = ctx.saved_tensors
        return ext._combine(_rows(grad), None, position), None


def expert_dispatch(input: torch.Tensor, order: ExpertOrder) -> torch.Tensor:
    """The tokens' rows in their experts' order: (entries, D), row p of input
    the row of the token whose entry has place p, zeros at the places of dropped
    entries.

    input (..., D) in fp32, fp16 or bf16 with the tokens of the index that
    order was made of.  The gradient reaches input: a token's is the sum of its
    rows', in the order of its choices.  At most 2^24 columns.
    """
    ext._check(input.dim() >= 1 and tuple(input.shape[:-1]) == tuple(order.position.shape[:-1]),
               "input must be (..., D) with the tokens of order")
    x, position = _rows(input), _position(order)
    ext._check_dispatch(x, position)
    if torch.is_grad_enabled() and input.requires_grad:
        return _Dispatch.apply(x, position)
    return ext._dispatch(x, position)


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, position):
        ctx.save_for_backward(rows, weights, position)
        return ext._combine(rows, weights, position)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        rows, weights, position = ctx.saved_tensors
        return *ext._combine_bwd(_rows(grad), _rows(rows), weights, position, *ctx.needs_input_grad[:2]), None


def expert_combine(rows: torch.Tensor, weights: torch.Tensor, order: ExpertOrder) -> torch.Tensor:
    """The experts' rows back at their tokens: (..., D), each token's sum of its
    entries' rows times their weights, in the order of its choices.

    rows (entries, D) in fp32, fp16 or bf16, in the order that expert_dispatch
    gives; weights (..., top), order's index's shape, taken in fp32 where they
    are not of rows' type.  Dropped entries give nothing: their rows and weights
    are not read and may hold anything, and their gradients are 0.  Gradients
    reach rows and weights.  At most 2^24 columns.
    """
    ext._check(weights.shape == order.position.shape, "weights must have the shape of order's index")
    if weights.dtype != rows.dtype and weights.dtype in ext._DTYPE_CODE:
        weights = weights.float()
    r, position = _rows(rows) if rows.dim() == 2 else rows, _position(order)
    w = weights.reshape(position.shape).contiguous()
    ext._check_combine(r, w, position)
    if torch.is_grad_enabled() and (rows.requires_grad or weights.requires_grad):
        out = _Combine.apply(r, w, position)
    else:
        out = ext._combine(r, w, position)
    return out if weights.dim() == 2 else out.reshape(*weights.shape[:-1], rows.shape[1])
