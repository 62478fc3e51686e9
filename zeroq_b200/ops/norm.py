"""RMSNorm and layer norm, each with an optional fused residual add.

``add_rmsnorm(h, delta, w)`` returns ``(h + delta, rmsnorm(h + delta) * w)`` in
one kernel (``csrc/elementwise.cu``); its backward adds the incoming residual
gradient to the norm's input gradient in the same kernel and writes one row of
per-CTA weight-gradient partial sums, reduced here.  On CPU the PyTorch
expressions below are used; they are also the numerics oracle.

``layer_norm`` and ``add_layer_norm`` are the same pair with the mean taken off and a bias
(``csrc/layernorm.cu``); with ``saved="8bit"`` the backward reads the normalised rows' input
from the 8 bits of :mod:`zeroq_b200.ops.act8`.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _ext
from .act8 import check_saved, kept_values, quantize_reference


def rmsnorm_reference(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    r = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    return (xf * r * w.float()).to(x.dtype)


class _AddRMSNorm(torch.autograd.Function):
    """``(h + delta, rmsnorm(h + delta))`` in one kernel."""

    @staticmethod
    def forward(ctx, h, delta, w, eps):
        D = h.shape[-1]
        h2 = h.reshape(-1, D).contiguous()
        d2 = delta.reshape(-1, D).contiguous()
        M = h2.shape[0]
        hout = torch.empty_like(h2)
        y = torch.empty_like(h2)
        rstd = torch.empty(M, dtype=torch.float32, device=h.device)
        _ext.ext().add_rmsnorm_fwd(h2, d2, w, hout, y, rstd, float(eps))
        ctx.save_for_backward(hout, w, rstd)
        ctx.shape = h.shape
        return hout.view(h.shape), y.view(h.shape)

    @staticmethod
    def backward(ctx, g_h, g_y):
        hout, w, rstd = ctx.saved_tensors
        dx, dw = _norm_bwd(g_y, g_h, hout, w, rstd, ctx.needs_input_grad[2])
        dx = dx.view(ctx.shape)
        return dx, dx, None if dw is None else dw.to(w.dtype), None


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, eps):
        D = x.shape[-1]
        x2 = x.reshape(-1, D).contiguous()
        y = torch.empty_like(x2)
        rstd = torch.empty(x2.shape[0], dtype=torch.float32, device=x.device)
        _ext.ext().add_rmsnorm_fwd(x2, None, w, x2, y, rstd, float(eps))
        ctx.save_for_backward(x2, w, rstd)
        ctx.shape = x.shape
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, g_y):
        x2, w, rstd = ctx.saved_tensors
        dx, dw = _norm_bwd(g_y, None, x2, w, rstd, ctx.needs_input_grad[1])
        return dx.view(ctx.shape), None if dw is None else dw.to(w.dtype), None


def _norm_bwd(g_y, g_h, x2, w, rstd, want_dw: bool = True):
    """``(dx, dw)``; ``dw`` is None when not wanted or when it was added straight
    into ``w``'s bound fp32 gradient (a parameter bound by ``FlatParams``)."""
    D = x2.shape[-1]
    gy2 = g_y.reshape(-1, D).contiguous() if g_y is not None else torch.zeros_like(x2)
    gh2 = g_h.reshape(-1, D).contiguous() if g_h is not None else None
    dx = torch.empty_like(x2)
    grid = min(x2.shape[0], _num_sms(x2.device) * 2)
    dw_part = torch.empty(grid, D, dtype=torch.float32, device=x2.device)
    E = _ext.ext()
    E.rmsnorm_bwd(gy2, x2, w, rstd, gh2, dx, dw_part)
    if not want_dw:
        return dx, None
    # the per-CTA partial rows fold into the gradient in one column-sum kernel
    direct = (getattr(w, "_zq_flat_grad", False) and w.grad is not None
              and w.grad.dtype == torch.float32 and w.grad.is_contiguous() and D % 4 == 0
              and w.grad.data_ptr() % 16 == 0)
    if direct:
        E.colsum_accum(dw_part, w.grad)
        return dx, None
    dw = torch.zeros(D, dtype=torch.float32, device=x2.device)
    if D % 4 == 0:
        E.colsum_accum(dw_part, dw)
    else:
        dw = dw_part.sum(0)
    return dx, dw


_SMS = {}


def _num_sms(device) -> int:
    i = device.index if device.index is not None else torch.cuda.current_device()
    if i not in _SMS:
        _SMS[i] = torch.cuda.get_device_properties(i).multi_processor_count
    return _SMS[i]


def add_rmsnorm(h: torch.Tensor, delta: Optional[torch.Tensor], w: torch.Tensor,
                eps: float = 1e-6):
    """Returns ``(h_new, y)`` with ``h_new = h + delta`` (or ``h``) and
    ``y = h_new / rms(h_new) * w``."""
    if h.is_cuda and h.dtype == torch.bfloat16:
        if delta is None:
            return h, _RMSNorm.apply(h, w, eps)
        return _AddRMSNorm.apply(h, delta, w, eps)
    hn = h + delta if delta is not None else h
    return hn, rmsnorm_reference(hn, w, eps)


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    return add_rmsnorm(x, None, w, eps)[1]


_LN_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
#: columns of a row that the kernels take at most
MAX_LAYER_NORM = 16384


class _AddLayerNormReference(torch.autograd.Function):
    """``(h + delta, layer norm of it)`` in PyTorch, every output rounded once (the oracle;
    in 64 bits for 64-bit inputs)."""

    @staticmethod
    def forward(ctx, h, delta, w, b, eps, keep8):
        hn = h.clone() if delta is None else h + delta
        wide = torch.float64 if h.dtype == torch.float64 else torch.float32
        x = hn.to(wide)
        mu = x.mean(-1, keepdim=True)
        r = torch.rsqrt((x - mu).square().mean(-1, keepdim=True) + eps)
        y = (x - mu) * r
        ctx.save_for_backward(mu, r, w, *(quantize_reference(hn) if keep8 else (hn,)))
        ctx.types = (wide, w is not None and w.dtype, b is not None and b.dtype, delta is not None)
        y = y if w is None else y * w.to(wide)
        y = y if b is None else y + b.to(wide)
        return hn, y.to(h.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_h, g_y):
        mu, r, w, *kept = ctx.saved_tensors
        wide, wt, bt, residual = ctx.types
        dy = g_y.to(wide)
        x = kept_values(*kept, dy.shape[-1]).view(dy.shape) if len(kept) == 2 else kept[0].to(wide)
        n = (x - mu) * r
        a = dy if w is None else dy * w.to(wide)
        dx = r * (a - a.mean(-1, keepdim=True) - n * (a * n).mean(-1, keepdim=True))
        dx = (dx + g_h.to(wide)).to(g_y.dtype)
        rows = lambda t: t.sum(tuple(range(t.dim() - 1))) if t.dim() > 1 else t  # noqa: E731
        return (dx, dx if residual else None, rows(dy * n).to(wt) if wt else None,
                rows(dy).to(bt) if bt else None, None, None)


def add_layer_norm(h: torch.Tensor, delta: Optional[torch.Tensor], weight: Optional[torch.Tensor] = None,
                   bias: Optional[torch.Tensor] = None, eps: float = 1e-5, saved: str = "full"):
    """Returns ``(h_new, y)`` with ``h_new = h + delta`` (or ``h``), rounded to the type, and
    ``y = (h_new - mean) / sqrt(var + eps) * weight + bias`` over the last dimension.

    ``h [..., D]`` bf16, fp16 or fp32, ``D`` up to 16384 on the GPU; ``weight`` and ``bias``
    ``[D]`` of one type (fp32, bf16 or fp16), either may be left out.  ``saved="8bit"``: the
    backward reads ``h_new`` from 8 bits.  Statistics, sums and the weights' gradients are
    formed in 32 bits; those gradients are the same bits from run to run."""
    keep8 = check_saved("layer_norm", saved)
    if h.dim() < 1 or not h.is_floating_point():
        raise ValueError(f"layer_norm: floating-point [..., D], got {h.dtype} {tuple(h.shape)}")
    D = h.shape[-1]
    if delta is not None and (delta.shape != h.shape or delta.dtype != h.dtype or delta.device != h.device):
        raise ValueError(f"layer_norm: delta {delta.dtype} {tuple(delta.shape)} must be like h {h.dtype} {tuple(h.shape)}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and (p.shape != (D,) or not p.is_floating_point() or p.device != h.device):
            raise ValueError(f"layer_norm: {name} must be [{D}] on {h.device}, got {p.dtype} {tuple(p.shape)} on {p.device}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"layer_norm: weight {weight.dtype} and bias {bias.dtype} are of one type")
    if keep8 and h.dtype not in _LN_FLOATS:
        raise TypeError(f"layer_norm: 8 bits are kept of bf16, fp16 or fp32, got {h.dtype}")
    param = weight if weight is not None else bias
    if h.is_cuda and h.numel() and h.dtype in _LN_FLOATS and (param is None or param.dtype in _LN_FLOATS):
        if D > MAX_LAYER_NORM:
            raise ValueError(f"layer_norm: at most {MAX_LAYER_NORM} columns on the GPU, got {D}")
        out = _ext.ext().layer_norm(h, delta, weight, bias, float(eps), keep8)
        return (out[0], out[1]) if delta is not None else (h, out[0])
    hn, y = _AddLayerNormReference.apply(h, delta, weight, bias, float(eps), keep8)
    return (h if delta is None else hn), y


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, saved: str = "full") -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension
    (:func:`add_layer_norm` without the addition)."""
    return add_layer_norm(x, None, weight, bias, eps, saved)[1]
