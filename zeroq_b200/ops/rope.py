"""Rotary position embedding (rotate-half convention: pairs ``(i, i + D/2)``).

``apply_rope(q, k, theta)`` rotates ``q [B,S,Hq,D]`` and ``k [B,S,Hk,D]`` by
position-dependent angles ``pos * theta^(-2i/D)``; the backward is the rotation
by the negated angle.  CUDA tensors run ``csrc/elementwise.cu``'s kernel, which
computes the angles in fp32 per element (no cos/sin table in HBM).

``rotary_embedding(q, k, positions, ...)`` is the general form: an explicit position
for every token (packed documents, continued sequences), half or interleaved pairs,
a rotary width below the head's, and :class:`RopeScaling` for contexts longer than
the model was trained on.  CUDA tensors run ``csrc/rotary.cu``.
"""

from __future__ import annotations

import array
import functools
import math
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _ext


def rope_reference(x: torch.Tensor, theta: float, sign: float = 1.0) -> torch.Tensor:
    B, S, H, D = x.shape
    half = D // 2
    inv = theta ** (-torch.arange(0, half, dtype=torch.float64, device=x.device) * 2.0 / D)
    pos = torch.arange(S, dtype=torch.float64, device=x.device)
    ang = (pos[:, None] * inv[None, :]).float()
    cos = torch.cos(ang)[None, :, None, :]
    sin = torch.sin(ang)[None, :, None, :] * sign
    xf = x.float()
    x1, x2 = xf[..., :half], xf[..., half:]
    return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], dim=-1).to(x.dtype)


_TABLES = {}


def rope_table(S: int, D: int, theta: float, device) -> torch.Tensor:
    """fp32 ``[S, D/2, 2]`` (cos, sin) of the angles ``pos * theta^(-2i/D)``; the
    angle is formed in fp64 and rounded to fp32 before cos/sin, as in
    :func:`rope_reference`.  Cached per (S, D, theta, device)."""
    key = (S, D, float(theta), str(device))
    t = _TABLES.get(key)
    if t is None:
        half = D // 2
        inv = theta ** (-torch.arange(0, half, dtype=torch.float64, device=device) * 2.0 / D)
        pos = torch.arange(S, dtype=torch.float64, device=device)
        ang = (pos[:, None] * inv[None, :]).float()
        t = torch.stack([torch.cos(ang), torch.sin(ang)], dim=-1).contiguous()
        _TABLES[key] = t
    return t


class _Rope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, theta):
        cs = rope_table(q.shape[1], q.shape[3], theta, q.device)
        qo = torch.empty_like(q)
        ko = torch.empty_like(k)
        _ext.ext().rope(q.contiguous(), qo, cs, 1.0)
        _ext.ext().rope(k.contiguous(), ko, cs, 1.0)
        ctx.cs = cs
        return qo, ko

    @staticmethod
    def backward(ctx, gq, gk):
        dq = torch.empty_like(gq)
        dk = torch.empty_like(gk)
        _ext.ext().rope(gq.contiguous(), dq, ctx.cs, -1.0)
        _ext.ext().rope(gk.contiguous(), dk, ctx.cs, -1.0)
        return dq, dk, None


def apply_rope(q: torch.Tensor, k: torch.Tensor, theta: float = 10000.0):
    if q.is_cuda and q.dtype == torch.bfloat16:
        return _Rope.apply(q, k, theta)
    return rope_reference(q, theta), rope_reference(k, theta)


def rope_rows(x: torch.Tensor, cs: torch.Tensor, sign: float = 1.0) -> torch.Tensor:
    """Rotate the rows of ``x [M, H*D]`` (row m at position m % S, heads of
    ``D = 2 * cs.shape[1]``) by the table ``cs [S, D/2, 2]`` (``sign=-1``: the
    inverse rotation, i.e. the backward).  No autograd."""
    S, half = cs.shape[0], cs.shape[1]
    D = 2 * half
    M, N = x.shape
    x4 = x.reshape(M // S, S, N // D, D)
    if x.is_cuda and x.dtype == torch.bfloat16:
        out = torch.empty_like(x4)
        _ext.ext().rope(x4.contiguous(), out, cs, float(sign))
        return out.view(M, N)
    xf = x4.float()
    c = cs[..., 0][None, :, None, :].float()
    s_ = cs[..., 1][None, :, None, :].float() * sign
    x1, x2 = xf[..., :half], xf[..., half:]
    return torch.cat([x1 * c - x2 * s_, x2 * c + x1 * s_], dim=-1).to(x.dtype).view(M, N)


class RopeSpec:
    """The rotary table ``cs`` of one layer's q/k projections, shared with the
    attention that consumes their outputs.  A projection given a spec returns its
    output rotated (in the GEMM epilogue where it can); when the attention backward
    writes dQ/dK already rotated back it sets ``grads_unrotated``, and the
    projections then skip their own inverse rotation."""

    def __init__(self, cs: torch.Tensor):
        self.cs = cs
        self.grads_unrotated = False


def rope_table_of(rope) -> torch.Tensor:
    return rope.cs if isinstance(rope, RopeSpec) else rope


def rope_grad_done(rope) -> bool:
    return isinstance(rope, RopeSpec) and rope.grads_unrotated


class _RopeRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, rope):
        ctx.rope = rope
        return rope_rows(x, rope_table_of(rope), 1.0)

    @staticmethod
    def backward(ctx, g):
        if rope_grad_done(ctx.rope):
            return g, None
        return rope_rows(g.contiguous(), rope_table_of(ctx.rope), -1.0), None


def rope_rows_autograd(x: torch.Tensor, rope) -> torch.Tensor:
    return _RopeRows.apply(x, rope)


# ---------------------------------------------------------------------------
# explicit positions, pair layouts, part of the head, context scaling
# ---------------------------------------------------------------------------
@dataclass(frozen=True)
class RopeScaling:
    """How the frequencies ``w_i = theta^(-2i/R)`` change for contexts ``factor`` times
    longer than the ``original_max_position`` tokens a model was trained on.

    * ``linear``: ``w_i / factor`` (positions are interpolated).
    * ``ntk``: theta becomes ``theta * factor^(R/(R-2))``: the fastest pair keeps its
      frequency, the slowest is divided by ``factor``.
    * ``yarn``: pairs that turn more than ``beta_fast`` times within the original
      context keep their frequency, those that turn less than ``beta_slow`` times are
      divided by ``factor``, with a linear ramp over the pair index between them; cos
      and sin are multiplied by ``attention_factor`` (default ``0.1 ln(factor) + 1``).
      (Peng et al., "YaRN: Efficient Context Window Extension", 2023.)
    """

    kind: str
    factor: float = 1.0
    original_max_position: int = 4096
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attention_factor: Optional[float] = None

    def __post_init__(self):
        if self.kind not in ("linear", "ntk", "yarn"):
            raise ValueError(f"RopeScaling: unknown kind {self.kind!r} (linear, ntk or yarn)")
        if not (math.isfinite(self.factor) and self.factor >= 1.0):
            raise ValueError(f"RopeScaling: factor must be at least 1, got {self.factor}")
        if self.original_max_position < 1 or not 0 < self.beta_slow <= self.beta_fast:
            raise ValueError("RopeScaling: original_max_position >= 1 and 0 < beta_slow <= beta_fast")


@functools.lru_cache(maxsize=256)
def _rope_frequencies(rotary_dim: int, theta: float, scaling: Optional[RopeScaling]) -> Tuple[tuple, float]:
    """(frequency of each pair in radians per position, factor of cos and sin), 64 bits."""
    R, s = rotary_dim, 1.0 if scaling is None else scaling.factor
    kind = None if scaling is None else scaling.kind
    if kind == "ntk" and R > 2:
        theta = theta * s ** (R / (R - 2))
    freq = [theta ** (-2.0 * i / R) for i in range(R // 2)]
    if kind == "linear":
        return tuple(f / s for f in freq), 1.0
    if kind != "yarn":
        return tuple(freq), 1.0

    def pair_of(turns):   # the (fractional) pair that turns so many times within the original context
        return R * math.log(scaling.original_max_position / (turns * 2 * math.pi)) / (2 * math.log(theta))

    low = max(0, math.floor(pair_of(scaling.beta_fast)))
    high = min(R - 1, math.ceil(pair_of(scaling.beta_slow)))
    out = []
    for i, f in enumerate(freq):
        ramp = min(1.0, max(0.0, (i - low) / max(high - low, 0.001)))
        out.append(f * (1.0 - ramp) + f / s * ramp)
    factor = scaling.attention_factor
    return tuple(out), (0.1 * math.log(s) + 1.0 if factor is None else float(factor))


@functools.lru_cache(maxsize=256)
def _rope_turns(rotary_dim: int, theta: float, scaling: Optional[RopeScaling]) -> Tuple[bytes, float]:
    """The frequencies in turns per position, as the bytes (64-bit numbers) that the
    kernel's parameters are filled from.  (No tensor: a cached one could be a tracer's.)"""
    freq, factor = _rope_frequencies(rotary_dim, theta, scaling)
    return array.array("d", [f / (2 * math.pi) for f in freq]).tobytes(), factor


def rotary_reference(x: torch.Tensor, positions: torch.Tensor, theta: float = 10000.0,
                     rotary_dim: Optional[int] = None, interleaved: bool = False,
                     scaling: Optional[RopeScaling] = None) -> torch.Tensor:
    """PyTorch form of :func:`rotary_embedding` for one tensor ``[..., S, H, D]``."""
    R = x.shape[-1] if rotary_dim is None else rotary_dim
    freq, factor = _rope_frequencies(R, float(theta), scaling)
    ang = positions.double()[..., None, None] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    dt = torch.float64 if x.dtype == torch.float64 else torch.float32
    cos, sin = (torch.cos(ang) * factor).to(dt), (torch.sin(ang) * factor).to(dt)
    xf = x.to(dt)
    if interleaved:
        a, b = xf[..., 0:R:2], xf[..., 1:R:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = xf[..., : R // 2], xf[..., R // 2: R]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([y, xf[..., R:]], dim=-1).to(x.dtype)


_ROTARY_TYPES = frozenset((torch.bfloat16, torch.float16, torch.float32, torch.float64))


def rotary_embedding(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
                     theta: float = 10000.0, rotary_dim: Optional[int] = None, interleaved: bool = False,
                     scaling: Optional[RopeScaling] = None):
    """Rotate ``q [..., S, Hq, D]`` and ``k [..., S, Hk, D]`` (or ``None``) by their tokens'
    positions; returns new tensors ``(q', k')``, differentiable in q and k.

    ``positions``: whole numbers, ``q.shape[:-2]`` or ``[S]`` (shared by the rows before
    it).  Pair ``i`` of the first ``rotary_dim`` columns (default: all) turns by
    ``position * w_i`` with ``w_i = theta^(-2i/rotary_dim)`` changed by ``scaling``;
    pairs are columns ``(i, i + rotary_dim/2)``, or ``(2i, 2i + 1)`` with ``interleaved``.
    The other columns pass through.  Angles are formed in 64 bits, so positions may be
    far; the products are in 32 bits with one rounding.  bf16, fp16 or fp32, any strides."""
    qs, dtype, device = tuple(q.shape), q.dtype, q.device
    if len(qs) < 3:
        raise ValueError(f"rotary_embedding: q must be [..., S, H, D], got {qs}")
    D, rows = qs[-1], qs[:-2]
    R = D if rotary_dim is None else int(rotary_dim)
    if R < 2 or R % 2 or R > D or R > 256:
        raise ValueError(f"rotary_embedding: rotary_dim must be even, at most the head's {D} and at most 256, got {R}")
    if k is not None:
        ks = tuple(k.shape)
        if ks[:-2] != rows or ks[-1] != D or k.dtype != dtype or k.device != device:
            raise ValueError(f"rotary_embedding: k {ks} {k.dtype} does not go with q {qs} {dtype}")
    if dtype not in _ROTARY_TYPES:
        raise TypeError(f"rotary_embedding: bf16, fp16 or fp32 tensors, got {dtype}")
    if positions.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"rotary_embedding: positions must be int32 or int64, got {positions.dtype}")
    if positions.device != device:
        raise ValueError("rotary_embedding: positions must be on q's device")
    ps = tuple(positions.shape)
    if ps != rows and ps != rows[-1:]:
        raise ValueError(f"rotary_embedding: positions {ps} must be {rows} or {rows[-1:]}")
    if not theta > 1.0:
        raise ValueError(f"rotary_embedding: theta must be above 1, got {theta}")
    if device.type != "cuda" or dtype == torch.float64:
        args = (positions, float(theta), R, interleaved, scaling)
        return rotary_reference(q, *args), None if k is None else rotary_reference(k, *args)
    turns, factor = _rope_turns(R, float(theta), scaling)
    if len(ps) != 1 or not positions.is_contiguous():
        positions = positions.reshape(-1).contiguous()
    out = _ext.ext().rotary_embedding(q, k, positions, turns, bool(interleaved), factor)
    return (out[0], None) if k is None else (out[0], out[1])
