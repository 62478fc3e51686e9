"""Activations kept in 8 bits for the backward pass.

A group of 128 consecutive elements of a row (the last of a row may be short) shares a
32-bit step; an element is a signed 8-bit code.  With ``a`` the group's largest size:
``code = round(x * inv)``, ``inv = 127 / a`` in 32 bits (ties to even, the product not
rounded before), ``step = a * (1 / 127)`` in 32 bits; an element reads back as
``code * step``, at most ``a / 254`` off.  1.03 bytes an element.  A group whose largest
size is below ``2^-119`` reads back as zeros; one that holds a NaN or an infinity reads
back as NaN throughout, so that it does not go unnoticed.

* :func:`quantize_activation`, :func:`dequantize_activation` - the two ways;
* :func:`checkpoint_8bit` - an activation checkpoint whose inputs are kept that way;
* ``gelu``, ``swiglu``, ``layer_norm`` with ``saved="8bit"`` - the outputs are those of the
  exact inputs, the backward reads the kept ones.

CUDA tensors run ``csrc/act8.cu``; on CPU the PyTorch form below is used (the oracle).
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _ext

GROUP = 128
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


class Activation8(NamedTuple):
    """``codes`` int8 ``[M, D up to a multiple of 16]`` (columns past ``D`` undefined) and ``steps``
    fp32 ``[M, ceil(D / 128)]`` of a tensor of ``shape`` ``[..., D]`` and ``dtype``."""

    codes: torch.Tensor
    steps: torch.Tensor
    shape: tuple
    dtype: torch.dtype

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + 4 * self.steps.numel()


def check_saved(name: str, saved: str) -> bool:
    """Whether ``saved`` asks for 8 bits."""
    if saved not in ("full", "8bit"):
        raise ValueError(f"{name}: saved is 'full' or '8bit', got {saved!r}")
    return saved == "8bit"


def _rows(x: torch.Tensor) -> tuple:
    return (math.prod(x.shape[:-1]), x.shape[-1])


def quantize_reference(x: torch.Tensor):
    """``(codes, steps)`` in PyTorch (any device)."""
    M, D = _rows(x)
    wide, groups = (D + 15) // 16 * 16, (D + GROUP - 1) // GROUP
    v = torch.zeros(M, groups * GROUP, dtype=torch.float32, device=x.device)
    v[:, :D] = x.detach().reshape(M, D)
    v = v.view(M, groups, GROUP)
    a = v.abs().amax(-1, keepdim=True) if groups else v.new_zeros(M, 0, 1)   # (NaN where there is one)
    bad, zero = ~torch.isfinite(a), a < 2.0 ** -119
    inv = torch.full_like(a, 127.0) / torch.where(bad | zero, torch.ones_like(a), a)
    inv = torch.where(bad | zero, torch.zeros_like(a), inv)
    codes = torch.round(v.double() * inv.double()).nan_to_num(0.0).to(torch.int8)
    step = a * torch.tensor(1.0 / 127.0, dtype=torch.float32, device=x.device)
    step = torch.where(zero, torch.zeros_like(a), torch.where(bad, torch.full_like(a, float("nan")), step))
    kept = torch.zeros(M, wide, dtype=torch.int8, device=x.device)
    kept[:, :D] = codes.reshape(M, groups * GROUP)[:, :D]
    return kept, step.reshape(M, groups)


def kept_values(codes: torch.Tensor, steps: torch.Tensor, D: int) -> torch.Tensor:
    """``code * step`` of ``[M, D]`` in 32 bits, in PyTorch (any device)."""
    return codes[:, :D].float() * steps.repeat_interleave(GROUP, dim=1)[:, :D]


def quantize_activation(x: torch.Tensor) -> Activation8:
    """``x [..., D]`` in 8 bits (no gradient passes).  bf16, fp16 or fp32."""
    if not isinstance(x, torch.Tensor) or x.dtype not in _FLOATS:
        raise TypeError(f"quantize_activation: a bf16, fp16 or fp32 tensor, got {getattr(x, 'dtype', type(x).__name__)}")
    if x.dim() < 1:
        raise ValueError("quantize_activation: [..., D], got a single number")
    if x.is_cuda and x.numel():
        codes, steps = _ext.ext().act8_quantize(x.detach())
    else:
        codes, steps = quantize_reference(x)
    return Activation8(codes, steps, tuple(x.shape), x.dtype)


def dequantize_activation(kept: Activation8) -> torch.Tensor:
    """The tensor of ``kept.shape`` and ``kept.dtype`` that was kept."""
    if not isinstance(kept, Activation8):
        raise TypeError(f"dequantize_activation: an Activation8, got {type(kept).__name__}")
    shape = tuple(kept.shape)
    M, D = math.prod(shape[:-1]), shape[-1]
    if (kept.codes.dtype != torch.int8 or tuple(kept.codes.shape) != (M, (D + 15) // 16 * 16)
            or kept.steps.dtype != torch.float32 or tuple(kept.steps.shape) != (M, (D + GROUP - 1) // GROUP)
            or kept.steps.device != kept.codes.device):
        raise ValueError(f"dequantize_activation: codes {tuple(kept.codes.shape)} and steps {tuple(kept.steps.shape)} "
                         f"do not belong to a tensor of shape {shape}")
    if kept.codes.is_cuda and M * D:
        return _ext.ext().act8_dequantize(kept.codes.contiguous(), kept.steps.contiguous(), list(shape), kept.dtype)
    return kept_values(kept.codes, kept.steps, D).to(kept.dtype).view(shape)


def checkpoint_8bit(fn, *args, **kwargs):
    """``fn(*args, **kwargs)`` now, and again in the backward from its inputs kept in 8 bits.

    Like ``torch.utils.checkpoint.checkpoint`` (without reentrance; ``preserve_rng_state`` is
    this function's): nothing that ``fn`` saves is held until the backward, only its inputs,
    given by place or by name.  Held in 8 bits are the activations: of the bf16, fp16 and fp32
    tensors that take a gradient and are no parameters the first (the hidden states) and those of
    its shape.  Everything else is held as it is - attention masks, whose lowest values would take a
    group's step or make it NaN, position tables and biases, another sequence's states - and
    costs nothing where layers share it.  The outputs are those of the exact inputs; the
    gradients are those of ``fn`` at the kept ones."""
    from torch.utils.checkpoint import checkpoint

    preserve = kwargs.pop("preserve_rng_state", True)
    if not torch.is_grad_enabled():
        return fn(*args, **kwargs)

    def activation(t):
        return (isinstance(t, torch.Tensor) and not isinstance(t, torch.nn.Parameter) and t.dtype in _FLOATS
                and t.dim() >= 1 and t.requires_grad)

    n, names = len(args), list(kwargs)
    inputs = [*args, *kwargs.values()]
    shape = next((t.shape for t in inputs if activation(t)), None)
    in8 = [activation(t) and t.shape == shape for t in inputs]
    kept = [quantize_activation(t) if m else t for t, m in zip(inputs, in8)]
    exact = [inputs]        # for the call now; given up behind it
    del args, kwargs, inputs

    def run():
        if exact:
            v = exact[0]
        else:
            v = [dequantize_activation(k).requires_grad_() if m else k for k, m in zip(kept, in8)]
        return fn(*v[:n], **dict(zip(names, v[n:])))

    out = checkpoint(run, use_reentrant=False, preserve_rng_state=preserve)
    exact.clear()
    return out
