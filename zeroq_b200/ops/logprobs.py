"""Log probabilities of given tokens, with the entropy and the top alternatives of each row.

``token_logprobs`` stands beside :func:`~zeroq_b200.ops.cross_entropy.cross_entropy` and
:func:`~zeroq_b200.ops.distill.distillation_loss` and takes the same (vocab-padded) logits:
the quantities of policy training and scoring, and (its top alternatives) a teacher's
entries.  CUDA tensors run ``csrc/logprobs.cu``, one pass over the logits each way; on CPU
the PyTorch form below is used (the oracle).
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _ext

#: alternatives of a row that the kernel takes at most
MAX_TOP = 256


class TokenLogprobs(NamedTuple):
    """fp32 ``logprobs [M]`` (None without targets), ``entropy [M]``, ``top_logprobs [M, k]``;
    int64 ``top_ids [M, k]``, best first."""

    logprobs: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_logprobs: torch.Tensor
    top_ids: torch.Tensor


def _top_ids(z: torch.Tensor, k: int) -> torch.Tensor:
    if k == 0:
        return torch.empty(z.shape[0], 0, dtype=torch.int64, device=z.device)
    return torch.sort(z + 0.0, dim=-1, descending=True, stable=True).indices[:, :k]   # (NaN is the largest)


def token_logprobs_reference(logits, targets=None, top_k: int = 0, temperature: float = 1.0,
                             vocab: Optional[int] = None, ignore_index: int = -100) -> TokenLogprobs:
    """PyTorch form of :func:`token_logprobs` in 64 bits (any device, differentiable)."""
    vocab = logits.shape[-1] if vocab is None else vocab
    out = torch.float64 if logits.dtype == torch.float64 else torch.float32
    z = logits[:, :vocab].double()
    counted = (z > float("-inf")).any(-1) | z.isnan().any(-1)
    if targets is not None:
        y = targets.long()
        counted = counted & (y != ignore_index) & (y >= 0) & (y < vocab)
    z = torch.where(counted[:, None], z, torch.zeros_like(z))
    l = torch.log_softmax((z - z.detach().amax(-1, keepdim=True)) / temperature, -1)
    # p log p is 0 where p is, and takes no gradient there
    here = (l.detach().exp() != 0)   # (or NaN)
    safe = torch.where(here, l, torch.zeros_like(l))
    entropy = -(torch.where(here, safe.exp(), torch.zeros_like(l)) * safe).sum(-1)
    zero = torch.zeros_like(entropy)
    ids = _top_ids(z.detach(), top_k)
    top = torch.where(counted[:, None], l.gather(1, ids), torch.zeros_like(l[:, :1]))
    ids = torch.where(counted[:, None], ids, torch.full_like(ids, -1))
    logp = None
    if targets is not None:
        at = torch.where(counted, y, torch.zeros_like(y))
        logp = torch.where(counted, l.gather(1, at[:, None])[:, 0], zero).to(out)
    return TokenLogprobs(logp, torch.where(counted, entropy, zero).to(out), top.to(out), ids)


def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, top_k: int = 0,
                   temperature: float = 1.0, vocab: Optional[int] = None, ignore_index: int = -100) -> TokenLogprobs:
    """``log softmax(z / temperature)`` of each row at its target, the row's entropy, and the
    ``top_k`` largest logits' log probabilities and ids (the lowest id first among equals).

    ``logits [M, V_pad]`` (columns past ``vocab`` are padding and get a gradient of 0);
    ``targets [M]``, int32 or int64: a row whose target is ``ignore_index`` or outside the
    vocabulary counts nothing and is not read: zeros, ids -1 (no entry of
    :func:`~zeroq_b200.ops.distill.distillation_loss`), no gradient.  A row without a logit
    above -inf is taken the same way.  Without ``targets`` every row counts and ``logprobs``
    is None.  NaN or +inf make a row's numbers NaN; for the alternatives NaN is the largest.

    Differentiable in ``logits`` through all three outputs.  Temperatures of 1e-6 to 1e6; bf16, fp16 or fp32 on the GPU, a
    vocabulary of up to 2^22 and up to 256 alternatives."""
    if not isinstance(logits, torch.Tensor) or logits.dim() != 2 or not logits.is_floating_point():
        raise ValueError("token_logprobs: logits must be floating-point [M, V], got "
                         f"{getattr(logits, 'dtype', type(logits).__name__)} {tuple(getattr(logits, 'shape', ()))}")
    M = logits.shape[0]
    vocab = logits.shape[-1] if vocab is None else int(vocab)
    if not 0 < vocab <= logits.shape[-1]:
        raise ValueError(f"token_logprobs: vocab must be 1 to {logits.shape[-1]}, got {vocab}")
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"token_logprobs: temperature must be 1e-6 to 1e6, got {temperature}")
    if not 0 <= top_k <= min(vocab, MAX_TOP):
        raise ValueError(f"token_logprobs: top_k must be 0 to {min(vocab, MAX_TOP)}, got {top_k}")
    if targets is not None:
        if targets.shape != (M,):
            raise ValueError(f"token_logprobs: targets must be [{M}], got {tuple(targets.shape)}")
        if targets.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"token_logprobs: targets must be int32 or int64, got {targets.dtype}")
        if targets.device != logits.device:
            raise ValueError(f"token_logprobs: logits on {logits.device}, targets on {targets.device}")
        if 0 <= ignore_index < vocab:   # an id of the vocabulary marks the rows that count nothing
            targets = targets.masked_fill(targets == ignore_index, -1)
            ignore_index = -1
    if not logits.is_cuda or logits.dtype == torch.float64 or M == 0:
        return token_logprobs_reference(logits, targets, top_k, temperature, vocab, ignore_index)
    W = logits.shape[1]
    if (logits.stride(1) != 1 and W > 1) or (M > 1 and not W <= logits.stride(0) <= 2 * W):
        logits = logits.contiguous()
    logp, entropy, top, ids = _ext.ext().token_logprobs(logits, targets, int(top_k), vocab, float(temperature))
    return TokenLogprobs(logp if targets is not None else None, entropy, top, ids)
