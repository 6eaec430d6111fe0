"""Serving in 8-bit floating point (e4m3) with a scale for each block of 128.

A quantised weight is ``(q, scale)``: q (d_out, d_in) ``torch.float8_e4m3fn`` and scale
(ceil(d_out / 128), ceil(d_in / 128)) fp32, any positive numbers, so 8-bit checkpoints of
that form are used as they are; ``fp8_quantize_weight`` makes one from a 16-bit weight in this package's
(d_in, d_out) layout.  Activations are quantised inside the calls, each row in blocks of
128 columns with a power-of-two scale.  Products accumulate in fp32.

The calls are for inference: no gradients (they refuse inputs that ask for one).  d_in is a
multiple of 16, d_out of 8.
"""
from __future__ import annotations

from typing import Tuple

import torch
from torch import nn

from . import _launch
from .experts import RouterLogits, SwiGLUMoE, check_routing
from .mlp import SwiGLUMLP
from .router import route


def _no_grad(*tensors) -> None:
    assert not (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)), (
        "Expected inputs without gradients: the 8-bit products are for inference")


def _check_weight(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor, ndim: int = 2) -> None:
    assert x.ndim >= 2 and q.ndim == ndim, "Incorrect number of dimensions"
    assert q.dtype == torch.float8_e4m3fn, f"Expected a float8_e4m3fn weight, got {q.dtype}"
    *outer, n, d = q.shape
    want = (*outer, -(-n // 128), -(-d // 128))
    assert scale.dtype == torch.float32 and scale.shape == want, (
        f"Expected float32 scales of shape {want}, got {scale.dtype} {tuple(scale.shape)}")
    assert x.shape[-1] == q.shape[-1], f"Dimension mismatch. Expected x.shape[-1] ({x.shape[-1]}) to be equal to the weight's inner size ({q.shape[-1]})"


def _check_mlp(x, w_gate, s_gate, w_up, s_up, w_down, s_down, ndim):
    _no_grad(x)
    _check_weight(x, w_gate, s_gate, ndim)
    _check_weight(x, w_up, s_up, ndim)
    assert w_gate.shape == w_up.shape, "Expected both weight matrices to have same shape"
    assert w_down.ndim == ndim and w_down.shape[-1] == w_gate.shape[-2] and w_down.shape[:-2] == w_gate.shape[:-2], "Dimension mismatch"
    _check_weight(x.new_empty(0, w_down.shape[-1], device="meta"), w_down, s_down, ndim)


def fp8_quantize(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, scale) of the rows of x (T, d), bf16 or fp16: q (T, d) e4m3, scale
    (T, ceil(d / 128)) fp32 (stored block by block), with q * scale ~ x.  The scale is the
    smallest power of two under which the block's largest magnitude is at most 448; 1 for a
    block of zeros, NaN for one that holds inf or NaN."""
    assert x.ndim == 2, "Incorrect number of dimensions"
    _no_grad(x)
    return _launch.fp8_quantize_rows(x.contiguous())


def fp8_quantize_weight(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, scale) of a weight (d_in, d_out), or of a stack (E, d_in, d_out), in bf16 or fp16."""
    assert w.ndim in (2, 3), "Incorrect number of dimensions"
    q, s = _launch.fp8_quantize_weight(w.detach().contiguous().view((-1,) + w.shape[-2:]))
    return (q, s) if w.ndim == 3 else (q[0], s[0])


def fp8_matmul(xq: torch.Tensor, x_scale: torch.Tensor, q: torch.Tensor, scale: torch.Tensor,
               dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """y (T, d_out) in ``dtype`` from quantised rows (T, d_in) and a quantised weight."""
    _check_weight(xq, q, scale)
    assert xq.ndim == 2 and xq.dtype == torch.float8_e4m3fn, "Expected float8_e4m3fn rows of shape (T, d_in)"
    assert x_scale.dtype == torch.float32 and x_scale.shape == (xq.shape[0], -(-xq.shape[1] // 128)), (
        f"Expected float32 row scales of shape {(xq.shape[0], -(-xq.shape[1] // 128))}, got {x_scale.dtype} {tuple(x_scale.shape)}")
    return _launch.fp8_gemm(xq.contiguous(), x_scale, q.contiguous(), scale.contiguous(), dtype)


def fp8_linear(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """y (..., d_out) in x's type: x (..., d_in), bf16 or fp16, times a quantised weight."""
    _no_grad(x)
    _check_weight(x, q, scale)
    if x.ndim == 2:
        return _launch.fp8_linear(x.contiguous(), q.contiguous(), scale.contiguous())
    x2d = x.reshape(-1, x.shape[-1]).contiguous()
    return _launch.fp8_linear(x2d, q.contiguous(), scale.contiguous()).view(x.shape[:-1] + (q.shape[0],))


def fp8_swiglu_mlp(x, w_gate, s_gate, w_up, s_up, w_down, s_down) -> torch.Tensor:
    """``(silu(x @ w_gate) * (x @ w_up)) @ w_down`` on quantised weights: gate and up
    (d_intermediate, d_in), down (d_out, d_intermediate)."""
    _check_mlp(x, w_gate, s_gate, w_up, s_up, w_down, s_down, 2)
    x2d = x.reshape(-1, x.shape[-1]).contiguous()
    y = _launch.fp8_mlp(x2d, *(t.contiguous() for t in (w_gate, s_gate, w_up, s_up, w_down, s_down)))
    return y.view(x.shape[:-1] + (w_down.shape[0],))


def fp8_swiglu_experts(x, weights, indices, w_gate, s_gate, w_up, s_up, w_down, s_down) -> torch.Tensor:
    """``FusedSwiGLUExperts`` on quantised weights: gate and up (E, d_intermediate, d_model),
    down (E, d_out, d_intermediate), scales (E, ..., ...)."""
    _check_mlp(x, w_gate, s_gate, w_up, s_up, w_down, s_down, 3)
    check_routing(x, weights, indices)
    _no_grad(weights)
    k = weights.shape[-1]
    x2d = x.reshape(-1, x.shape[-1]).contiguous()
    y = _launch.fp8_experts(x2d, weights.reshape(-1, k).contiguous(), _launch.expert_indices(indices, w_gate.shape[0]),
                            *(t.contiguous() for t in (w_gate, s_gate, w_up, s_up, w_down, s_down)))
    return y.view(x.shape[:-1] + (w_down.shape[1],))


class _Quantised(nn.Module):
    """Holds quantised weights as buffers ``<name>`` and ``<name>_scale``."""

    def _keep(self, **weights) -> None:
        for name, w in weights.items():
            q, s = fp8_quantize_weight(w)
            self.register_buffer(name, q)
            self.register_buffer(name + "_scale", s)

    def _weights(self):
        return (self.w_gate, self.w_gate_scale, self.w_up, self.w_up_scale, self.w_down, self.w_down_scale)


class Fp8SwiGLUMLP(_Quantised):
    """Serving form of a ``SwiGLUMLP``: its weights, quantised once."""

    def __init__(self, mlp: SwiGLUMLP):
        super().__init__()
        self._keep(w_gate=mlp.w_gate, w_up=mlp.w_up, w_down=mlp.w_down)

    @torch.no_grad()
    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return fp8_swiglu_mlp(x, *self._weights())


class Fp8SwiGLUMoE(_Quantised):
    """Serving form of a ``SwiGLUMoE``: the experts' weights quantised once; the router, whose
    product is small, stays in 16 bits."""

    def __init__(self, moe: SwiGLUMoE):
        super().__init__()
        self._keep(w_gate=moe.w_gate, w_up=moe.w_up, w_down=moe.w_down)
        self.register_buffer("w_router", moe.w_router.detach().clone())
        self.register_buffer("balance_bias", None if moe.balance_bias is None else moe.balance_bias.detach().clone())
        self.top_k, self.routing = moe.top_k, dict(moe.routing)

    @torch.no_grad()
    def forward(self, x: torch.Tensor) -> torch.Tensor:
        weights, indices = route(RouterLogits.apply(x, self.w_router), self.top_k, bias=self.balance_bias, **self.routing)
        return fp8_swiglu_experts(x, weights, indices, *self._weights())
