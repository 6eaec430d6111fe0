"""Routing of tokens to experts: ``weights, indices = route(logits, top_k, ...)``.

Scores are ``s = softmax(logits)`` or ``sigmoid(logits)``.  Experts are chosen by
``s + bias`` (a balance bias that gets no gradient and does not enter the weights), if
asked within the ``topk_groups`` best of ``num_groups`` groups of experts (a group's score
is the sum of its two largest), ties going to the lowest index.  The weights are the
chosen experts' scores, divided by their sum if ``renormalize``, times ``scale``.

The selection is the one exact arithmetic would make: it does not depend on how the scores
round.  A logit of -inf masks an expert: it is chosen only when nothing else is left, with
weight 0.  The reference has no mixture of experts; this feeds ``FusedSwiGLUExperts``.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _launch


def _forward(logits, bias, top_k, score, renormalize, scale, num_groups, topk_groups):
    assert logits.ndim >= 2, "Expected logits of shape (..., num_experts)"
    assert score in ("softmax", "sigmoid"), f"Expected score 'softmax' or 'sigmoid', got {score!r}"
    E = logits.shape[-1]
    if bias is not None:
        assert bias.shape == (E,), f"Expected a bias of shape ({E},), got {tuple(bias.shape)}"
    z = logits.reshape(-1, E) if logits.ndim != 2 else logits
    if z.stride(1) != 1 or (z.shape[0] > 1 and z.stride(0) < E):
        z = z.contiguous()
    return (z, *_launch.route(z, bias, int(top_k), score, bool(renormalize), float(scale), int(num_groups), int(topk_groups)))


class FusedRouter(Function):
    """``FusedRouter.apply(logits, bias, top_k, score, renormalize, scale, num_groups,
    topk_groups)``; see :func:`route`."""

    @staticmethod
    def forward(ctx, logits, bias, top_k, score, renormalize, scale, num_groups, topk_groups):
        z, weights, indices = _forward(logits, bias, top_k, score, renormalize, scale, num_groups, topk_groups)
        ctx.save_for_backward(z, indices)
        ctx.set_materialize_grads(False)  # no zeros for the indices' gradient
        ctx.args = (score, bool(renormalize), float(scale))
        ctx.in_shape = logits.shape
        if logits.ndim != 2:
            shape = logits.shape[:-1] + (int(top_k),)
            weights, indices = weights.view(shape), indices.view(shape)
        ctx.mark_non_differentiable(indices)
        return weights, indices

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_weights, _grad_indices):
        dz = None
        if ctx.needs_input_grad[0] and grad_weights is not None:
            z, indices = ctx.saved_tensors
            score, renormalize, scale = ctx.args
            dw = grad_weights.reshape(indices.shape).contiguous()
            dz = _launch.route_backward(z, indices, dw, score, renormalize, scale)
            if len(ctx.in_shape) != 2:
                dz = dz.view(ctx.in_shape)
        return dz, None, None, None, None, None, None, None


def route(logits: torch.Tensor, top_k: int, *, bias: Optional[torch.Tensor] = None, score: str = "softmax",
          renormalize: bool = True, scale: float = 1.0, num_groups: int = 1,
          topk_groups: int = 1) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(weights, indices)`` of the ``top_k`` experts of each token, best first: fp32 and
    int32, shape (..., top_k), for logits (..., num_experts) in bf16, fp16 or fp32.

    At most 1024 experts, 32 of them per token, 32 groups of equal size.  ``bias``: one
    value per expert, added to the scores for the selection only."""
    if logits.requires_grad and torch.is_grad_enabled():
        return FusedRouter.apply(logits, bias, top_k, score, renormalize, scale, num_groups, topk_groups)
    # nothing to differentiate: autograd's bookkeeping costs more than the kernel
    _, weights, indices = _forward(logits, bias, top_k, score, renormalize, scale, num_groups, topk_groups)
    if logits.ndim != 2:
        shape = logits.shape[:-1] + (int(top_k),)
        weights, indices = weights.view(shape), indices.view(shape)
    return weights, indices
