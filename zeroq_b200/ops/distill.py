"""Distillation from a teacher's top logits, mixed with the hard targets.

``distillation_loss`` stands beside :func:`~zeroq_b200.ops.cross_entropy.cross_entropy`
and takes the same (vocab-padded) logits.  CUDA tensors run ``csrc/distill.cu``: the
forward forms the gradient of the mean in the same launch, so a training step reads
the logits once and writes their gradient once.  On CPU the PyTorch form below is
used; it is also the numerics oracle.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _ext

#: entries of a row that the kernel takes at most
MAX_TEACHER_ENTRIES = 1024


def distillation_reference(logits, teacher_ids, teacher_logits, targets=None, temperature: float = 1.0,
                           alpha: float = 1.0, vocab: Optional[int] = None, ignore_index: int = -100,
                           reduction: str = "mean") -> torch.Tensor:
    """PyTorch form of :func:`distillation_loss` (any device, differentiable)."""
    vocab = logits.shape[-1] if vocab is None else vocab
    z = logits[:, :vocab]
    z = z if z.dtype == torch.float64 else z.float()
    z = z - z.detach().amax(-1, keepdim=True)   # before the scale too: logits far from 0 keep their differences
    ids = teacher_ids.long()
    there = (ids >= 0) & (ids < vocab)
    t = teacher_logits.to(z.dtype).masked_fill(~there, float("-inf"))
    some = (t > float("-inf")).any(-1, keepdim=True)
    if t.shape[-1]:   # (the largest taken off before the scale: entries near the type's lowest value stay finite)
        t = (t - t.amax(-1, keepdim=True)) / temperature
    p = torch.softmax(torch.where(some, t, torch.zeros_like(t)), -1)
    p = torch.where(some & (p != 0), p, torch.zeros_like(p))
    at = torch.where(there, ids, torch.zeros_like(ids))
    log_q = torch.log_softmax(z / temperature, -1).gather(1, at)
    log_q = torch.where(p != 0, log_q, torch.zeros_like(log_q))   # 0 · log 0 = 0
    loss = alpha * temperature ** 2 * (torch.special.xlogy(p, p) - p * log_q).sum(-1)
    counted = torch.ones_like(loss, dtype=torch.bool)
    if targets is not None:
        y = targets.long()
        counted = (y != ignore_index) & (y >= 0) & (y < vocab)
        if alpha < 1.0:
            label = torch.where(counted, y, torch.zeros_like(y))
            loss = loss - (1.0 - alpha) * torch.log_softmax(z, -1).gather(1, label[:, None])[:, 0]
    loss = torch.where(counted, loss, torch.zeros_like(loss))
    return loss if reduction == "none" else loss.sum() / counted.sum().clamp_min(1)


def distillation_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                      targets: Optional[torch.Tensor] = None, temperature: float = 1.0, alpha: float = 1.0,
                      vocab: Optional[int] = None, ignore_index: int = -100,
                      reduction: str = "mean") -> torch.Tensor:
    """``alpha * T^2 * KL(p || softmax(z / T)) + (1 - alpha) * CE(z, target)`` of each row.

    ``logits [M, V_pad]`` (columns past ``vocab`` are padding and get a gradient of 0);
    ``teacher_ids [M, K]`` and ``teacher_logits [M, K]``: the teacher's top entries, whose
    softmax at temperature ``T`` is ``p`` (log-probabilities do as well: a row's shift
    drops out).  An id outside ``[0, vocab)`` is no entry; a row without entries has no
    first term; entries with the same id add up.  ``targets [M]``: rows whose target is
    ``ignore_index`` or outside the vocabulary count nothing; they may be left out with
    ``alpha = 1``, then every row counts.

    ``reduction="mean"``: the mean over the counted rows (0 if there are none), whose
    backward may run once; ``"none"``: the rows' losses, fp32 ``[M]``.  Differentiable in
    ``logits``.  bf16, fp16 or fp32 on the GPU, a row of up to 1.5 MB."""
    if logits.dim() != 2 or teacher_ids.dim() != 2 or teacher_ids.shape[0] != logits.shape[0]:
        raise ValueError(f"distillation_loss: logits [M, V] and teacher_ids [M, K], got {tuple(logits.shape)} "
                         f"and {tuple(teacher_ids.shape)}")
    if teacher_logits.shape != teacher_ids.shape:
        raise ValueError(f"distillation_loss: teacher_logits {tuple(teacher_logits.shape)} must be like "
                         f"teacher_ids {tuple(teacher_ids.shape)}")
    M, K = teacher_ids.shape
    vocab = logits.shape[-1] if vocab is None else int(vocab)
    if not 0 < vocab <= logits.shape[-1]:
        raise ValueError(f"distillation_loss: vocab must be 1 to {logits.shape[-1]}, got {vocab}")
    if not (temperature > 0 and temperature < float("inf")) or not 0.0 <= alpha <= 1.0:
        raise ValueError("distillation_loss: temperature above 0 and alpha in [0, 1]")
    if targets is None and alpha < 1.0:
        raise ValueError("distillation_loss: alpha below 1 needs targets")
    if targets is not None and targets.shape != (M,):
        raise ValueError(f"distillation_loss: targets must be [{M}], got {tuple(targets.shape)}")
    if reduction not in ("mean", "none"):
        raise ValueError(f"distillation_loss: reduction is 'mean' or 'none', got {reduction!r}")
    if teacher_ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"distillation_loss: teacher_ids must be int32 or int64, got {teacher_ids.dtype}")
    if targets is not None and targets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"distillation_loss: targets must be int32 or int64, got {targets.dtype}")
    if not logits.is_floating_point() or not teacher_logits.is_floating_point():
        raise TypeError("distillation_loss: logits and teacher_logits are floating-point")
    if any(t is not None and t.device != logits.device for t in (teacher_ids, teacher_logits, targets)):
        raise ValueError("distillation_loss: all tensors on one device")
    if K > MAX_TEACHER_ENTRIES:
        raise ValueError(f"distillation_loss: at most {MAX_TEACHER_ENTRIES} teacher entries a row, got {K}")
    if targets is not None and 0 <= ignore_index < vocab:   # an id of the vocabulary marks the rows that count nothing
        targets = targets.masked_fill(targets == ignore_index, -1)
        ignore_index = -1
    if not logits.is_cuda or logits.dtype == torch.float64 or M == 0:
        return distillation_reference(logits, teacher_ids, teacher_logits.detach(), targets, temperature, alpha,
                                      vocab, ignore_index, reduction)
    teacher = teacher_logits.detach()
    if teacher.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        teacher = teacher.float()
    W = logits.shape[1]
    if logits.stride(1) != 1 or not W <= logits.stride(0) <= 2 * W:
        logits = logits.contiguous()
    if logits.data_ptr() % 16:
        logits = logits.clone(memory_format=torch.contiguous_format)
    # fp16: a gradient formed before the upstream factor (a loss scale) is known would
    # underflow, so its rows take the form that reads the logits again
    return _ext.ext().distill_loss(logits, teacher_ids, teacher, targets, vocab, int(ignore_index), float(temperature),
                                   float(alpha), reduction == "mean", logits.dtype != torch.float16)
