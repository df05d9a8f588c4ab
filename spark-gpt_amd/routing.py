"""Routing of tokens to experts, on gfx950 kernels: what a mixture-of-experts
layer does around its experts.

* ``route_tokens(logits, top_k, ...)``      the experts of each token and their weights
* ``expert_order(selected, num_experts)``   the rows' order by expert: what
  ``_FP8Experts`` (and ``ops.moe_plan``) take, spark-gpt's bookkeeping of
  train.py:2268-2290
* ``combine_experts(rows, weights, ...)``   the weighted sum of each token's rows
* ``fp8_routed_experts(x, logits, experts, top_k, ...)``  the layer: the three
  around ``_FP8Experts``

Weights are fp32, indices int64, as in the reference.  Nothing here
synchronises the device: a padded batch keeps its shape, its padding tokens
are masked, and their slots (-1) come last in the expert order, where no kernel
reads them.  ``route_tokens`` and ``combine_experts`` are differentiable once,
in the logits and in the rows and weights.  There is no CPU fallback.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ops
from . import torch_ops  # the sparkfp8:: operators and their implementations
from .moe import _FP8Experts


class _RouteTokens(torch.autograd.Function):
    """(weights, selected) of ``route_tokens`` in a compiled graph (an eager call
    makes the same node in C++); the selection has no gradient."""

    @staticmethod
    def forward(ctx, logits, bias, mask, score, groups, top_groups, group_best, top_k, renormalize, scale):
        weights, selected, picked = torch_ops.op("route_fwd")(logits, bias, mask, score, groups, top_groups, group_best,
                                                              top_k, renormalize, scale)
        # the logits' values are read again for the plain softmax alone; else only their shape and type are
        ctx.save_for_backward(logits, selected, picked)
        ctx.route = (score, renormalize, scale)
        ctx.mark_non_differentiable(selected)
        ctx.set_materialize_grads(False)
        return weights, selected

    @staticmethod
    @once_differentiable
    def backward(ctx, dweights, _dselected):
        if dweights is None:
            return (None,) * 10
        logits, selected, picked = ctx.saved_tensors
        return (torch_ops.op("route_bwd")(dweights, selected, picked, logits, *ctx.route),) + (None,) * 9


def route_tokens(logits: torch.Tensor, top_k: int, *, score: str = "softmax", bias: torch.Tensor | None = None,
                 mask: torch.Tensor | None = None, groups: int = 1, top_groups: int | None = None,
                 group_best: int = 1, renormalize: bool = True, scale: float = 1.0):
    """The ``top_k`` experts of each token and their weights:
    ``(weights fp32 [T, top_k], selected int64 [T, top_k])`` in descending order.

    ``logits`` [T, E] fp32, bf16 or fp16 (any row stride), E <= 1024, top_k <= 64.

    * ``score``: ``"softmax"`` over the experts or ``"sigmoid"`` of each logit.
    * ``bias`` (fp32 [E]): added to the scores for the order alone, neither to
      the weights nor to the gradient (balance without a loss).  Without it the
      experts are ordered by their logits.
    * ``groups``, ``top_groups``, ``group_best``: the experts are ``groups``
      groups of E / groups in a row, and only the ``top_groups`` best take
      part (default: all).  A group's value is the best order value in it
      (``group_best=1``) or the sum of its two best scores, biases included (2);
      two sums that 64 bits do not tell apart may come either way.
    * ``renormalize``: weights are scores over the sum of the chosen ones;
      ``scale`` multiplies the weights.
    * ``mask`` (bool [T]): tokens that are False are not routed.

    Equal order values go to the lowest index; an expert whose logit (or order
    value) is -inf is never taken, and NaN ranks first.  Slots that no expert
    is left for, and those of masked tokens, get index -1 and weight 0."""
    compiling = torch.compiler.is_compiling()
    apply = _RouteTokens.apply if compiling else ops.route_tokens
    if compiling and bias is not None:
        bias = bias.detach()  # as in the eager call: weights require a gradient where the logits do
    return apply(logits, bias, mask, score, groups, groups if top_groups is None else top_groups, group_best, top_k,
                 renormalize, float(scale))


def expert_order(selected: torch.Tensor, num_experts: int):
    """``(token_index int64 [T * k], inverse_permutation int64 [T * k], offsets
    int32 [E])`` of ``selected`` [T, k]: the slots in stable order by expert.
    Row r of the order belongs to token ``token_index[r]``; slot s's row is
    ``inverse_permutation[s]``; expert e owns rows ``offsets[e - 1] ..
    offsets[e] - 1``.  Slots that name no expert (-1, or anything outside
    [0, E)) come last, in order, and have -1 in ``inverse_permutation``."""
    return torch_ops.op("expert_order")(selected, num_experts)


class _CombineExperts(torch.autograd.Function):
    """The weighted top-k sum of ``combine_experts`` in a compiled graph."""

    @staticmethod
    def forward(ctx, rows, weights, inverse_permutation, offsets):
        ctx.save_for_backward(rows, weights, inverse_permutation, offsets)
        return torch_ops.op("combine_fwd")(rows, weights, inverse_permutation)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        rows, weights, inverse_permutation, offsets = ctx.saved_tensors
        drows, dweights = torch_ops.op("combine_bwd")(dout, rows, weights, inverse_permutation, offsets)
        return drows, dweights, None, None


def combine_experts(rows: torch.Tensor, weights: torch.Tensor, inverse_permutation: torch.Tensor,
                    offsets: torch.Tensor) -> torch.Tensor:
    """``out[t] = sum over j of weights[t, j] * rows[inverse_permutation[t * k + j]]``
    [T, D]: rows [R, D] bf16, fp16 or fp32 in expert order, weights [T, k]
    (k <= 64), ``inverse_permutation`` and ``offsets`` of ``expert_order`` (the
    latter is not read: the slots say which rows there are).  The
    sum is taken in 32 bits in slot order and rounded once; slots without a row
    (-1, or anything outside [0, R)) add nothing.  In the backward pass a row that
    no slot names gets zeros and one that several name the sum of theirs, in 32
    bits and slot order; the latter costs a pass over the slots for each such row."""
    if torch.compiler.is_compiling():
        return _CombineExperts.apply(rows, weights.float(), inverse_permutation, offsets)
    return ops.combine_experts(rows, weights, inverse_permutation, offsets)


def fp8_routed_experts(x: torch.Tensor, logits: torch.Tensor, experts, top_k: int, **route):
    """The FP8 mixture-of-experts layer after its router's product: ``(out [T, D]
    bf16, selected [T, top_k])``.  ``x`` [T, D] bf16, ``logits`` [T, E]; ``experts``
    has the reference's packed ``gate_up_proj`` [E, 2I, D], ``down_proj`` [E, D, I],
    ``fp8_scale`` and ``fp8_amax`` (train.py:2252-2260); ``route`` are the keyword
    arguments of ``route_tokens``."""
    if logits.dim() != 2 or logits.shape != (x.shape[0], experts.gate_up_proj.shape[0]):
        raise ValueError(f"logits must be [{x.shape[0]}, {experts.gate_up_proj.shape[0]}], one row for each token and one "
                         f"column for each expert, got {tuple(logits.shape)}")
    weights, selected = route_tokens(logits, top_k, **route)
    token_index, inverse_permutation, offsets = expert_order(selected, logits.shape[1])
    rows = _FP8Experts.apply(x, experts.gate_up_proj, experts.down_proj, token_index, inverse_permutation, offsets,
                             top_k, experts.fp8_scale, experts.fp8_amax)
    return combine_experts(rows, weights, inverse_permutation, offsets), selected
