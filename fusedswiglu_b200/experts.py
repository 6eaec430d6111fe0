"""Routed SwiGLU experts (mixture of experts).

``y[t] = sum_j weights[t, j] * (silu(x[t] @ w_gate[e]) * (x[t] @ w_up[e])) @ w_down[e]``
with ``e = indices[t, j]``, for bf16 or fp16 tensors with fp32 accumulation.  All experts'
products are one launch each of the library's tcgen05 kernel over rows sorted by expert;
the number of tokens per expert stays on the device.

Shapes: x (..., d_model); weights, indices (..., top_k), as ``route`` returns them;
w_gate, w_up (num_experts, d_model, d_intermediate); w_down (num_experts, d_intermediate,
d_out); y (..., d_out).  ``weights`` is fp32 or of x's type.  A pair whose index is outside
[0, num_experts) contributes nothing (an expert on another rank, a padded token).
"""
from __future__ import annotations

import math

import torch
from torch import nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _launch
from .router import route


def check_args(x, weights, indices, w_gate, w_up, w_down):
    assert x.ndim >= 2 and w_gate.ndim == 3 and w_down.ndim == 3, "Incorrect number of dimensions"
    assert w_gate.shape == w_up.shape, "Expected both weight matrices to have same shape"
    assert x.shape[-1] == w_gate.shape[1] and w_gate.shape[2] == w_down.shape[1] and w_gate.shape[0] == w_down.shape[0], "Dimension mismatch"
    assert x.dtype == w_gate.dtype == w_up.dtype == w_down.dtype, "Expected tensors of one dtype"
    check_routing(x, weights, indices)


def check_routing(x, weights, indices):
    assert weights.shape == indices.shape and weights.shape[:-1] == x.shape[:-1], (
        f"Expected weights and indices of shape {tuple(x.shape[:-1])} + (top_k,), got {tuple(weights.shape)} and {tuple(indices.shape)}")
    assert indices.dtype in (torch.int32, torch.int64), f"Expected int32 or int64 indices, got {indices.dtype}"
    assert weights.dtype in (torch.float32, x.dtype), f"Expected weights in float32 or {x.dtype}, got {weights.dtype}"


def _forward(x, weights, indices, w_gate, w_up, w_down, save):
    """(y, saved, weights, w_gate, w_up, w_down), the last four contiguous."""
    check_args(x, weights, indices, w_gate, w_up, w_down)
    x2d = (x if x.ndim == 2 else x.reshape(-1, x.shape[-1])).contiguous()
    r = (weights if weights.ndim == 2 else weights.reshape(-1, weights.shape[-1])).contiguous()
    wg, wu, wd = w_gate.contiguous(), w_up.contiguous(), w_down.contiguous()
    y, saved = _launch.experts_forward(x2d, r, _launch.expert_indices(indices, wg.shape[0]), wg, wu, wd, save=save)
    return (y if x.ndim == 2 else y.view(x.shape[:-1] + (wd.shape[2],)), saved, r, wg, wu, wd)


class FusedSwiGLUExperts(Function):
    """``FusedSwiGLUExperts.apply(x, weights, indices, w_gate, w_up, w_down)``."""

    @classmethod
    def apply(cls, x, weights, indices, w_gate, w_up, w_down):
        if torch.is_grad_enabled() and any(t.requires_grad for t in (x, weights, w_gate, w_up, w_down)):
            return super().apply(x, weights, indices, w_gate, w_up, w_down)
        # nothing to differentiate: nothing is saved, and autograd's bookkeeping is left out
        return _forward(x, weights, indices, w_gate, w_up, w_down, False)[0]

    @staticmethod
    def forward(ctx, x, weights, indices, w_gate, w_up, w_down):
        need = any(ctx.needs_input_grad)
        y, saved, *kept = _forward(x, weights, indices, w_gate, w_up, w_down, need)
        if need:
            ctx.save_for_backward(*kept, saved)
        ctx.in_shape, ctx.weights_shape = x.shape, weights.shape
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        r, wg, wu, wd, saved = ctx.saved_tensors
        need_x, need_r, _, need_g, need_u, need_d = ctx.needs_input_grad
        dy = grad_y.reshape(-1, wd.shape[2]).contiguous()
        dx, dr, dwg, dwu, dwd = _launch.experts_backward(dy, r, wg, wu, wd, saved, need_x=need_x, need_weights=need_r,
                                                         need_gate_up=need_g or need_u, need_down=need_d)
        return (dx.view(ctx.in_shape) if need_x else None, dr.view(ctx.weights_shape) if need_r else None, None,
                dwg if need_g else None, dwu if need_u else None, dwd if need_d else None)


class SwiGLUMoE(nn.Module):
    """Mixture-of-experts block: router, routed SwiGLU experts, weighted sum.

    Parameters: ``w_router`` (d_model, num_experts) and the experts' weights, all of
    ``dtype``; the buffer ``balance_bias`` (num_experts) steers the selection of experts
    (to even out their load, from outside autograd) when ``use_balance_bias`` is set."""

    def __init__(self, d_model: int, d_intermediate: int, num_experts: int, top_k: int, *, score: str = "softmax",
                 renormalize: bool = True, scale: float = 1.0, num_groups: int = 1, topk_groups: int = 1,
                 use_balance_bias: bool = False, dtype: torch.dtype = torch.bfloat16, device=None):
        super().__init__()
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("SwiGLUMoE supports torch.bfloat16 and torch.float16 parameters")
        if d_model % 8 or d_intermediate % 8 or num_experts % 8:
            raise ValueError("feature sizes and the number of experts must be multiples of 8")
        self.top_k = top_k
        self.routing = dict(score=score, renormalize=renormalize, scale=scale, num_groups=num_groups,
                            topk_groups=topk_groups)

        def init(*shape):
            w = torch.randn(*shape, device=device, dtype=torch.float32).mul_(1.0 / math.sqrt(shape[-2]))
            return nn.Parameter(w.to(dtype))

        self.w_router = init(d_model, num_experts)
        self.w_gate, self.w_up = init(num_experts, d_model, d_intermediate), init(num_experts, d_model, d_intermediate)
        self.w_down = init(num_experts, d_intermediate, d_model)
        bias = torch.zeros(num_experts, device=device, dtype=torch.float32) if use_balance_bias else None
        self.register_buffer("balance_bias", bias)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        logits = RouterLogits.apply(x, self.w_router)
        weights, indices = route(logits, self.top_k, bias=self.balance_bias, **self.routing)
        return FusedSwiGLUExperts.apply(x, weights, indices, self.w_gate, self.w_up, self.w_down)


class RouterLogits(Function):
    """``x @ w_router`` and its gradients on the library's GEMM."""

    @staticmethod
    def forward(ctx, x, w_router):
        assert x.dtype == w_router.dtype, "Expected tensors of one dtype"
        x2d, w = x.reshape(-1, x.shape[-1]).contiguous(), w_router.contiguous()
        ctx.save_for_backward(x2d, w)
        ctx.in_shape = x.shape
        return _launch.gemm(x2d, w).view(x.shape[:-1] + (w.shape[1],))

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x2d, w = ctx.saved_tensors
        dz = grad.reshape(-1, w.shape[1]).contiguous()
        dx = _launch.gemm(dz, w, trans_b=True).view(ctx.in_shape) if ctx.needs_input_grad[0] else None
        dw = None
        if ctx.needs_input_grad[1]:
            T = x2d.shape[0]
            if T == 0:
                return dx, torch.zeros_like(w)
            if T % 8:  # the GEMM wants the transposed operand's rows in multiples of 8: rows of zeros add nothing
                pad = 8 - T % 8
                x2d = torch.cat([x2d, x2d.new_zeros(pad, x2d.shape[1])])
                dz = torch.cat([dz, dz.new_zeros(pad, dz.shape[1])])
            dw = _launch.gemm(x2d, dz, trans_a=True)
        return dx, dw
