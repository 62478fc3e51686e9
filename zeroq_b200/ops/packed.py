"""Packed rows: several sequences behind one another in one row of tokens.

:class:`PackedSequences` holds the division ``cu_seqlens`` of ``total`` rows and what the
kernels derive from it: the tile tables of the attention kernels and every row's
position in its sequence.  Both are built on the device by one kernel, without a copy
to the host, so a division may change from step to step (also in a captured graph:
the tables are built again at each replay).  Make one for a batch and give it to
every layer.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _ext


class PackedSequences:
    """Sequence ``i`` holds rows ``[cu_seqlens[i], cu_seqlens[i + 1])`` of ``total``;
    rows behind the last sequence are padding.  Sequences may be empty.

    ``cu_seqlens``: int32 or int64 ``[n + 1]``.  On the CPU it is checked here (it starts
    at 0, does not fall and ends within ``total``) and copied to ``device``; on the GPU
    it is not read by the host - values out of order are clamped by the kernel, and the
    result for such a division is undefined.  The tables are those of the values that it
    had here: make another one for another division.  A fixed ``n`` with empty sequences
    at the end is fine (a graph's static ``cu_seqlens``); each costs 60 bytes of tables, a few
    rows' worth of the attention backward's statistics and empty blocks in its launches."""

    def __init__(self, cu_seqlens: torch.Tensor, total: int, device: Optional[torch.device] = None):
        if not isinstance(cu_seqlens, torch.Tensor) or not hasattr(total, "__index__"):
            raise TypeError(f"PackedSequences: cu_seqlens a tensor and total a whole number, got {type(cu_seqlens).__name__} "
                            f"and {type(total).__name__}")
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
            raise ValueError(f"PackedSequences: cu_seqlens must be [n + 1], got {tuple(cu_seqlens.shape)}")
        if cu_seqlens.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"PackedSequences: cu_seqlens must be int32 or int64, got {cu_seqlens.dtype}")
        if not 0 <= total < 1 << 30:
            raise ValueError(f"PackedSequences: total must be 0 to 2^30 - 1, got {total}")
        device = cu_seqlens.device if device is None else torch.device(device)
        if not cu_seqlens.is_cuda:
            c = cu_seqlens.tolist()
            if c[0] != 0 or any(b < a for a, b in zip(c, c[1:])) or c[-1] > total:
                raise ValueError(f"PackedSequences: cu_seqlens must rise from 0 to at most total={total}")
        self.total = int(total)
        self.n = cu_seqlens.numel() - 1
        if cu_seqlens.dtype != torch.int32 or cu_seqlens.device != device or not cu_seqlens.is_contiguous():
            cu_seqlens = cu_seqlens.to(device=device, dtype=torch.int32).contiguous()
        elif not cu_seqlens.is_cuda:
            cu_seqlens = cu_seqlens.clone()   # bounds() goes on reading it
        self.cu_seqlens = cu_seqlens
        self.device = cu_seqlens.device   # with its index: "cuda" is the current device
        self.plan = None
        if cu_seqlens.is_cuda:
            self.plan, self.positions = _ext.ext().packed_sequences(self.cu_seqlens, self.total)
        else:
            self.positions = torch.zeros(self.total, dtype=torch.int32)
            for a, b in self.bounds():
                self.positions[a:b] = torch.arange(b - a, dtype=torch.int32)

    def bounds(self):
        """``[(first row, end row)]`` of the sequences (on the GPU read from there, int32
        ``cu_seqlens`` from the caller's own tensor as it is by now)."""
        c = self.cu_seqlens.tolist()
        return list(zip(c, c[1:]))
