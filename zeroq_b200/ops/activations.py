"""GELU (erf form) and SwiGLU, forward and backward (``csrc/elementwise.cu``).

``swiglu(gate, up) = silu(gate) * up``.  Both kernels read bf16 and compute in
fp32; the erf and exp calls are CUDA's own functions.

With ``saved="8bit"`` (``csrc/act8.cu``; bf16, fp16 and fp32) the outputs are the same and
the inputs are kept for the backward in the 8 bits of :mod:`zeroq_b200.ops.act8`: 1.03 bytes
an element instead of 2 or 4, and gradients at the kept values.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from . import _ext
from .act8 import check_saved, kept_values, quantize_reference

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


class _Kept(torch.autograd.Function):
    """``fn(*xs)`` in PyTorch whose backward differentiates at the inputs kept in 8 bits."""

    @staticmethod
    def forward(ctx, fn, *xs):
        ctx.fn, ctx.n = fn, len(xs)
        ctx.save_for_backward(*(t for x in xs for t in quantize_reference(x)))
        return fn(*(x.float() for x in xs)).to(xs[0].dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        kept = ctx.saved_tensors
        with torch.enable_grad():
            xs = [kept_values(kept[2 * i], kept[2 * i + 1], g.shape[-1]).view(g.shape).requires_grad_()
                  for i in range(ctx.n)]
            y = ctx.fn(*xs)
        return (None,) + tuple(d.to(g.dtype) for d in torch.autograd.grad(y, xs, g.float()))


def _check_kept(name, *xs):
    for x in xs:
        if x.dtype not in _FLOATS or x.dim() < 1:
            raise TypeError(f"{name}: 8 bits are kept of bf16, fp16 or fp32 [..., D], got {x.dtype} {tuple(x.shape)}")
        if x.shape != xs[0].shape or x.dtype != xs[0].dtype or x.device != xs[0].device:
            raise ValueError(f"{name}: inputs of one shape, type and device, got {x.dtype} {tuple(x.shape)} "
                             f"and {xs[0].dtype} {tuple(xs[0].shape)}")


class _Gelu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        y = torch.empty_like(x)
        _ext.ext().gelu_fwd(x.contiguous(), y)
        ctx.save_for_backward(x)
        return y

    @staticmethod
    def backward(ctx, g):
        (x,) = ctx.saved_tensors
        dx = torch.empty_like(x)
        _ext.ext().gelu_bwd(g.contiguous(), x.contiguous(), dx)
        return dx


def gelu(x: torch.Tensor, saved: str = "full") -> torch.Tensor:
    """``saved="8bit"``: ``x`` is kept for the backward in 8 bits."""
    if check_saved("gelu", saved):
        _check_kept("gelu", x)
        if torch.is_grad_enabled() and x.requires_grad:
            return _ext.ext().gelu8(x) if x.is_cuda and x.numel() else _Kept.apply(F.gelu, x)
    if x.is_cuda and x.dtype == torch.bfloat16:
        return _Gelu.apply(x)
    return F.gelu(x.float()).to(x.dtype)


class _SwiGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up):
        y = torch.empty_like(gate)
        _ext.ext().swiglu_fwd(gate.contiguous(), up.contiguous(), y)
        ctx.save_for_backward(gate, up)
        return y

    @staticmethod
    def backward(ctx, g):
        gate, up = ctx.saved_tensors
        dg = torch.empty_like(gate)
        du = torch.empty_like(up)
        _ext.ext().swiglu_bwd(g.contiguous(), gate.contiguous(), up.contiguous(), dg, du)
        return dg, du


def swiglu(gate: torch.Tensor, up: torch.Tensor, saved: str = "full") -> torch.Tensor:
    """``saved="8bit"``: ``gate`` and ``up`` are kept for the backward in 8 bits."""
    if check_saved("swiglu", saved):
        _check_kept("swiglu", gate, up)
        if torch.is_grad_enabled() and (gate.requires_grad or up.requires_grad):
            if gate.is_cuda and gate.numel():
                return _ext.ext().swiglu8(gate, up)
            return _Kept.apply(lambda g, u: F.silu(g) * u, gate, up)
    if gate.is_cuda and gate.dtype == torch.bfloat16:
        return _SwiGLU.apply(gate, up)
    return (F.silu(gate.float()) * up.float()).to(gate.dtype)
