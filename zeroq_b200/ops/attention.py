"""Causal (GQA-capable) flash attention, forward and backward.

Tensors keep the projection layout ``[B, S, H, D]`` so no transposes surround
the kernels.  Forward and backward run on the 5th-generation tensor cores
(``csrc/attention_sm100.cu``): the forward with TMA-fed Q/K/V tiles, S and O
accumulated in tensor memory and softmax in registers, writing ``O`` and the
row log-sum-exp ``L``; the backward as a ``delta = rowsum(dO * O)`` pass, a dQ
kernel per query tile and a dK/dV kernel per key tile, both recomputing P from
``L`` with S, dP, P and dS in tensor memory, no atomics.  The kernels are built
for 128-wide heads; narrower heads (``D`` = 64 and other multiples of 16) are
zero-padded to 128 - padded columns change no score and come out zero - so
every head size up to 128 runs on the same kernels (at 128-wide cost).

CPU tensors, ``S`` not a multiple of 128 and heads wider than 128 use PyTorch's
SDPA (the oracle).

``flash_attention_varlen`` is attention over packed sequences of any lengths
(``csrc/attention_varlen_sm100.cu``): ``[T, H, D]`` rows, divided by a
:class:`~zeroq_b200.ops.packed.PackedSequences`, bf16 or fp16, with its backward.
"""

from __future__ import annotations

import math
from typing import Optional, Union

import torch
import torch.nn.functional as F

from . import _ext
from .packed import PackedSequences


def attention_reference(q, k, v, causal: bool = True, scale=None):
    B, S, Hq, D = q.shape
    Hk = k.shape[2]
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    qt = q.transpose(1, 2).float()
    kt = k.transpose(1, 2).float()
    vt = v.transpose(1, 2).float()
    if Hk != Hq:
        rep = Hq // Hk
        kt = kt.repeat_interleave(rep, dim=1)
        vt = vt.repeat_interleave(rep, dim=1)
    o = F.scaled_dot_product_attention(qt, kt, vt, is_causal=causal, scale=scale)
    return o.transpose(1, 2).to(q.dtype)


def _tma_ok(t: torch.Tensor) -> bool:
    return (t.stride(-1) == 1 and all(st % 8 == 0 for st in t.stride()[:-1])
            and t.data_ptr() % 16 == 0)


def _pad128(t: torch.Tensor) -> torch.Tensor:
    """``[B, S, H, D]`` (D < 128) zero-padded to ``[B, S, H, 128]``."""
    out = t.new_zeros(*t.shape[:-1], 128)
    out[..., : t.shape[-1]] = t
    return out


def _tc_ok(q: torch.Tensor) -> bool:
    D = q.shape[-1]
    return q.shape[1] % 128 == 0 and q.shape[1] > 0 and D <= 128 and D % 16 == 0


class _FlashAttn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal, scale, rope=None):
        D = q.shape[-1]
        ctx.d = D
        if D < 128:   # narrower heads run zero-padded on the 128-wide kernels
            q, k, v = _pad128(q), _pad128(k), _pad128(v)
        # the tcgen05 kernels read q/k/v through TMA maps and take strided views
        # (column slices of a fused q/k/v projection) as they are
        q, k, v = (t if _tma_ok(t) else t.contiguous() for t in (q, k, v))
        B, S, Hq, _ = q.shape
        o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        lse = torch.empty(B, Hq, S, dtype=torch.float32, device=q.device)
        _ext.ext().attn_fwd_tc(q, k, v, o, lse, bool(causal), float(scale))
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.causal, ctx.scale = causal, scale
        ctx.rope = rope if (rope is not None and hasattr(rope, "grads_unrotated")) else None
        return o if D == 128 else o[..., :D]

    @staticmethod
    def backward(ctx, do):
        q, k, v, o, lse = ctx.saved_tensors
        D = ctx.d
        do = do.contiguous() if D == 128 else _pad128(do)
        dq, dk = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
        dv = _like_token_pitched(v) if D == 128 else None
        if dv is None:
            dv = torch.empty(v.shape, dtype=v.dtype, device=v.device)
        rope = ctx.rope
        cs = rope.cs if (rope is not None and D == 128 and rope.cs.shape[0] == q.shape[1]) else None
        _ext.ext().attn_bwd_tc(do, q, k, v, o, lse, dq, dk, dv, bool(ctx.causal), float(ctx.scale),
                               None, cs)
        if cs is not None:
            rope.grads_unrotated = True  # dQ/dK are gradients of the pre-rotation q/k
        if D < 128:
            dq, dk, dv = dq[..., :D], dk[..., :D], dv[..., :D]
        return dq, dk, dv, None, None, None


def _like_token_pitched(v: torch.Tensor):
    """For ``v`` a column slice of a token-pitched 2-D buffer (the fused q/k/v
    projection's output ``[B*S, Nq+Nk+Nv]``), a gradient with the same layout in a
    fresh buffer of that width: the backward writes dV straight into the slice
    the fused projection's backward reads, so no copy assembles its gradient."""
    B, S, H, D = v.shape
    P = v.stride(1)
    if (v.stride(3) != 1 or v.stride(2) != D or P <= H * D or v.stride(0) != S * P
            or P % 8 or v.storage_offset() + H * D > P):
        return None
    buf = torch.empty(B * S * P, dtype=v.dtype, device=v.device)
    return buf.as_strided(v.shape, v.stride(), v.storage_offset())


def flash_attention(q, k, v, causal: bool = True, scale=None, rope=None):
    """``rope``: the :class:`~zeroq_b200.ops.rope.RopeSpec` with which q and k were
    rotated by their projections; the backward then writes dQ/dK rotated back
    (tcgen05 path) and marks the spec so the projections do not rotate again."""
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    if q.is_cuda and q.dtype == torch.bfloat16 and _tc_ok(q):
        return _FlashAttn.apply(q, k, v, causal, scale, rope)
    return attention_reference(q, k, v, causal, scale)


# ---------------------------------------------------------------------------
# packed sequences
# ---------------------------------------------------------------------------
def attention_varlen_reference(q, k, v, seqs: PackedSequences, causal: bool = True, scale=None):
    """PyTorch form of :func:`flash_attention_varlen`, a sequence at a time, in 32 bits
    (64 for 64-bit inputs); differentiable."""
    D, share = q.shape[-1], q.shape[1] // k.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    dt = torch.float64 if q.dtype == torch.float64 else torch.float32
    parts, end = [], 0
    for a, b in seqs.bounds():
        qs, ks, vs = (t[a:b].to(dt).transpose(0, 1) for t in (q, k, v))
        ks, vs = (t.repeat_interleave(share, dim=0) for t in (ks, vs))
        s = (qs @ ks.transpose(1, 2)) * scale
        if causal:
            s = s.masked_fill(torch.ones(b - a, b - a, dtype=torch.bool, device=q.device).triu(1), -math.inf)
        parts.append((torch.softmax(s, -1) @ vs).transpose(0, 1).to(q.dtype))
        end = b
    parts.append(q.new_zeros(q.shape[0] - end, *q.shape[1:]))
    return torch.cat(parts)


def flash_attention_varlen(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                           seqs: Union[PackedSequences, torch.Tensor], causal: bool = True,
                           scale: Optional[float] = None) -> torch.Tensor:
    """Attention of each sequence of a packed row over itself.

    ``q [T, Hq, D]``, ``k`` and ``v`` ``[T, Hk, D]`` with ``Hq`` a multiple of ``Hk``
    (query head ``h`` reads kv head ``h // (Hq / Hk)``), any strides with a unit head-dim
    stride; ``D`` a multiple of 8 up to 128; bf16 or fp16 on the GPU.  ``seqs``: the
    :class:`~zeroq_b200.ops.packed.PackedSequences` of the ``T`` rows, or its
    ``cu_seqlens`` (then its tables are built for this call).  ``causal``: a row sees its
    sequence's rows up to itself, otherwise all of them.  ``scale`` (positive) defaults
    to ``1/sqrt(D)``.  Rows of no sequence get an output and gradients of zero, whatever
    they hold, and another sequence's rows do not enter.  Within a sequence a key behind the
    mask weighs 0 (which times an infinite or NaN value is NaN, as in any product of P and V).
    P and dS are rounded to the inputs' type before their products;
    scores, softmax statistics and accumulators are in 32 bits."""
    qs, ks, dtype, device = tuple(q.shape), tuple(k.shape), q.dtype, q.device
    if len(qs) != 3 or len(ks) != 3 or tuple(v.shape) != ks or ks[0] != qs[0] or ks[2] != qs[2]:
        raise ValueError(f"flash_attention_varlen: q [T, Hq, D], k and v [T, Hk, D], got {qs}, {ks}, {tuple(v.shape)}")
    T, Hq, D = qs
    if ks[1] < 1 or Hq < 1 or Hq % ks[1]:
        raise ValueError(f"flash_attention_varlen: {Hq} query heads do not share {ks[1]} kv heads evenly")
    if not (k.dtype == v.dtype == dtype) or not (k.device == v.device == device):
        raise TypeError("flash_attention_varlen: q, k and v of one type on one device")
    if D < 1:
        raise ValueError("flash_attention_varlen: heads of no width")
    if not isinstance(seqs, (PackedSequences, torch.Tensor)):
        raise TypeError(f"flash_attention_varlen: seqs are PackedSequences or a cu_seqlens tensor, got {type(seqs).__name__}")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"flash_attention_varlen: scale must be positive, got {scale}")
    cu = None
    if not isinstance(seqs, PackedSequences):
        if (device.type == "cuda" and seqs.dtype == torch.int32 and seqs.device == device and seqs.dim() == 1
                and seqs.numel() and seqs.is_contiguous()):
            cu = seqs          # its plan is built by the same call
        else:
            seqs = PackedSequences(seqs, T, device=device)
    if cu is None and (seqs.total != T or seqs.device != device):
        raise ValueError(f"flash_attention_varlen: the sequences divide {seqs.total} rows on {seqs.device}, "
                         f"q has {T} on {device}")
    if device.type != "cuda" or T == 0:
        seqs = seqs if cu is None else PackedSequences(cu, T)
        return attention_varlen_reference(q, k, v, seqs, causal, scale)
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"flash_attention_varlen: bf16 or fp16 on the GPU, got {dtype}")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError(f"flash_attention_varlen: head width a multiple of 8 up to 128 on the GPU, got {D}")
    if cu is not None:
        return _ext.ext().attn_varlen_cu(q, k, v, cu, bool(causal), scale)
    return _ext.ext().attn_varlen(q, k, v, seqs.plan, seqs.n, bool(causal), scale)
