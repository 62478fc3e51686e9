"""Embedding lookup with scaling; its gradient is summed by sorted tokens.

``embedding(ids, weight, scale)`` stands beside ``torch.nn.functional.embedding``: rows of
the table times ``scale``, rounded once, and a zero row for an id outside the table (a
padded batch).  CUDA tensors run ``csrc/embedding.cu``: the backward sorts the tokens by id
on the device and adds every row's gradients in 32 bits in token order, so that a gradient
is the same bits from run to run.  On CPU the PyTorch form below is used; it is also the
numerics oracle.
"""

from __future__ import annotations

import torch

from . import _ext

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def embedding_reference(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """PyTorch form of :func:`embedding` (any device, differentiable)."""
    V, wide = weight.shape[0], weight if weight.dtype == torch.float64 else weight.float()
    there = (ids >= 0) & (ids < V)
    if V == 0:
        return wide.new_zeros(*ids.shape, weight.shape[1]).to(weight.dtype)
    rows = wide.index_select(0, torch.where(there, ids, torch.zeros_like(ids)).reshape(-1).long())
    rows, there = rows.view(*ids.shape, weight.shape[1]), there[..., None]
    none = torch.zeros_like(rows)
    # (twice: 0 by a scale that is not finite is NaN, by a negative one -0, and so it is on the way back)
    return torch.where(there, torch.where(there, rows, none) * scale, none).to(weight.dtype)


def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``scale * weight[ids]`` of shape ``[*ids.shape, D]``, in ``weight``'s type.

    ``ids``: int32 or int64 of any shape; an id outside ``[0, V)`` gives a row of zeros and
    takes no gradient.  ``weight [V, D]``: bf16, fp16 or fp32 on the GPU.  Differentiable in
    ``weight`` (a dense gradient, each row's sum formed in 32 bits and rounded once)."""
    if not isinstance(ids, torch.Tensor) or not isinstance(weight, torch.Tensor):
        raise TypeError("embedding: ids and weight are tensors")
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"embedding: ids must be int32 or int64, got {ids.dtype}")
    if weight.dim() != 2 or not weight.is_floating_point():
        raise ValueError(f"embedding: weight must be floating-point [V, D], got {weight.dtype} {tuple(weight.shape)}")
    if ids.device != weight.device:
        raise ValueError(f"embedding: ids on {ids.device}, weight on {weight.device}")
    if not weight.is_cuda or weight.dtype not in _FLOATS or ids.numel() == 0 or weight.numel() == 0:
        return embedding_reference(ids, weight, scale)
    return _ext.ext().embedding_lookup(ids, weight, float(scale))
