"""Low-rank adapters for the MMDiT's block linears, several of them in one batch: every
sequence of a step names its adapter, the shared projection stays one GEMM, and
b200attn.lora_add adds each sequence's part (include/b200_lora.h)."""
from __future__ import annotations

from typing import Dict, Optional, Sequence, Tuple

import b200attn

# The linears of a block, by the names of the reference's VarBuilder paths.
TARGETS = ("attn.to_q", "attn.to_k", "attn.to_v", "attn.to_out.0", "img_mlp.gate_layer",
           "img_mlp.proj", "img_mlp.out")


class AdapterBank:
    """Adapters 0 .. E - 1.  adapters: one dict per adapter from a linear's name
    ("transformer_blocks.3.attn.to_q") to its pair (A [rank, in], B [out, rank]); scales: one
    factor per adapter (alpha / rank; 1 if not given).  An adapter may leave linears out;
    lower ranks are padded with zeros."""

    def __init__(self, adapters: Sequence[Dict[str, Tuple]], scales: Optional[Sequence[float]] = None,
                 device="cuda"):
        import torch
        if not adapters:
            raise ValueError("a bank holds at least one adapter")
        scales = [1.0] * len(adapters) if scales is None else list(scales)
        if len(scales) != len(adapters):
            raise ValueError("one scale per adapter")
        self.count = len(adapters)
        self.scale = torch.tensor(scales, dtype=torch.float32, device=device)
        self.linears: Dict[str, Tuple] = {}
        for name in sorted({n for a in adapters for n in a}):
            parts = name.split(".", 2)
            if len(parts) != 3 or parts[0] != "transformer_blocks" or parts[2] not in TARGETS:
                raise ValueError(f"{name} is not a block linear")
            pairs = [a.get(name) for a in adapters]
            shapes = {(p[0].shape[1], p[1].shape[0]) for p in pairs if p is not None}
            if len(shapes) != 1 or any(p is not None and p[0].shape[0] != p[1].shape[1] for p in pairs):
                raise ValueError(f"{name}: the adapters' shapes do not fit together")
            (k, n), = shapes
            rank = -(-max(p[0].shape[0] for p in pairs if p is not None) // 8) * 8
            if rank > b200attn.LORA_MAX_RANK:
                raise ValueError(f"{name}: rank {rank} is over {b200attn.LORA_MAX_RANK}")
            a = torch.zeros((self.count, rank, k), dtype=torch.bfloat16, device=device)
            b = torch.zeros((self.count, n, rank), dtype=torch.bfloat16, device=device)
            for e, p in enumerate(pairs):
                if p is not None:
                    a[e, :p[0].shape[0]] = p[0]
                    b[e, :, :p[1].shape[1]] = p[1]
            self.linears[name] = (a, b)


class BatchAdapters:
    """The adapters of one batch: `rows` rows per sequence, adapter ids[b] (None or negative:
    none) for sequence b."""

    def __init__(self, bank: AdapterBank, ids: Sequence[Optional[int]], rows: int):
        import torch
        ids = [-1 if i is None else int(i) for i in ids]
        if any(i >= bank.count for i in ids):
            raise ValueError(f"the bank has {bank.count} adapters")
        self.bank, self.rows = bank, rows
        dev = bank.scale.device
        self._who = torch.tensor(ids, dtype=torch.int32, device=dev)
        self._start = torch.arange(len(ids) + 1, dtype=torch.int32, device=dev) * rows
        self._from = {0: self._start}

    def add(self, name: str, x, y, first_row: int = 0) -> None:
        """y += the adapters' part of the linear `name` for x, in place; x and y are the
        batch's rows from first_row on."""
        ab = self.bank.linears.get(name)
        if ab is None:
            return
        start = self._from.get(first_row)
        if start is None:  # rows before the chunk are limited away by the operator
            start = self._from[first_row] = self._start - first_row
        b200attn.lora_add(x, ab[0], ab[1], y, start, self._who, scale=self.bank.scale)
