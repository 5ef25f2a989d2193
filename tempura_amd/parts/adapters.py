"""Room for low-rank adapters beside a part's projections (``ops.adapter_linear``).

A part that takes adapters names the checkpoint tensors that they may stand beside (``adapter_targets``) and, once the model
was given room (``enable_adapters``), keeps one ``AdapterSlots`` a product: the pairs (A, B) of up to ``slots`` adapters, those of
the matrices that were stacked into the product side by side.  A step whose context holds ``adapter_ids`` (int32 [tokens], the slot of
each token's request or -1) adds each row's share; any other step runs as it would without.
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple

import torch

from ..kernels import ops


class AdapterSlots:
    """``rows[i]``: the product's columns that stacked matrix i has, ``k`` its inputs.  ``interleaved``: two matrices whose columns
    alternate by eights."""

    def __init__(self, slots: int, rank: int, k: int, rows: Sequence[int], dtype: torch.dtype, device, interleaved: bool = False):
        self.rank = -(-int(rank) // 8) * 8      # (a multiple of 8: the kernels read the tensors here as they are)
        self.rows, self.k, self.interleaved = list(rows), int(k), bool(interleaved)
        n = sum(self.rows)
        self.a = torch.zeros((slots, len(self.rows) * self.rank, self.k), dtype=dtype, device=device)
        self.b = torch.zeros((slots, n, self.rank), dtype=dtype, device=device)
        self.scales = torch.zeros((slots,), dtype=torch.float32, device=device)
        ends = [sum(self.rows[: i + 1]) for i in range(len(self.rows))]
        self.handle = ops.Adapters(self.a, self.b, self.scales, None if self.interleaved else ends, self.interleaved)

    def fault(self, i: int, pair: Tuple[torch.Tensor, torch.Tensor]) -> Optional[str]:
        """Why a pair (A, B) cannot stand beside matrix i, or None."""
        a, b = pair
        if a.dim() != 2 or b.dim() != 2 or a.shape[0] != b.shape[1] or a.shape[0] < 1:
            return f"A {tuple(a.shape)} and B {tuple(b.shape)} are no pair"
        if a.shape[1] != self.k or b.shape[0] != self.rows[i]:
            return f"A {tuple(a.shape)} and B {tuple(b.shape)} beside a matrix of {self.rows[i]} x {self.k}"
        if a.shape[0] > self.rank:
            return f"rank {a.shape[0]} where there is room for {self.rank}"
        return None

    def set(self, slot: int, pairs: Sequence[Optional[Tuple[torch.Tensor, torch.Tensor]]], scale: float) -> None:
        """Fill a slot (a matrix without a pair: nothing is added beside it)."""
        a = torch.zeros(self.a.shape[1:], dtype=self.a.dtype)
        b = torch.zeros(self.b.shape[1:], dtype=self.b.dtype)
        first = 0
        for i, pair in enumerate(pairs):
            if pair is not None:
                rank = pair[0].shape[0]
                a[i * self.rank: i * self.rank + rank] = pair[0].to(a.dtype)
                into = b.view(-1, 2, 8, self.rank)[:, i] if self.interleaved else b[first: first + self.rows[i]]
                into[..., :rank] = pair[1].to(b.dtype).reshape(*into.shape[:-1], rank)
            first += self.rows[i]
        self.a[slot].copy_(a)
        self.b[slot].copy_(b)
        self.scales[slot] = float(scale)


#: checkpoint tensor name -> (product, which of its stacked matrices)
Targets = Dict[str, Tuple[str, int]]


class TakesAdapters:
    """Mixed into a part with ``adapter_targets``; ``adapters`` is None until the model was given room for some."""

    adapters: Optional[Dict[str, AdapterSlots]] = None

    def adapter_targets(self) -> Targets:
        return {}

    def adapter_products(self) -> Dict[str, dict]:
        """product -> the arguments of its ``AdapterSlots`` behind slots and rank."""
        return {}

    def adapter_rows(self, name: str, b: torch.Tensor) -> torch.Tensor:
        """The rows of B beside the tensor ``name`` in the order in which the part keeps that tensor's rows (A's columns: ``adapter_columns``)."""
        return b

    def enable_adapters(self, slots: int, rank: int) -> None:
        self.adapters = {p: AdapterSlots(slots, rank, dtype=self.dtype, device=self.device, **kw) for p, kw in self.adapter_products().items()}
        # (rows whose norm a product finishes come as they are to one that adds adapters: the norms run by themselves)
        self.split_norm = False

    def set_adapter(self, slot: int, pairs: Dict[str, Tuple[torch.Tensor, torch.Tensor]], scale: float) -> None:
        """Fill a slot from pairs by checkpoint tensor name; products without a pair are cleared."""
        targets = self.adapter_targets()
        for product, room in self.adapters.items():
            mine: List[Optional[Tuple[torch.Tensor, torch.Tensor]]] = [None] * len(room.rows)
            for name, (p, i) in targets.items():
                if p == product and name in pairs:
                    a, b = pairs[name]
                    mine[i] = (a, self.adapter_rows(name, b))
            room.set(slot, mine, scale)

    def adapters_of(self, ctx):
        """The step's slots by token, or None where this part adds nothing."""
        return getattr(ctx, "adapter_ids", None) if self.adapters is not None else None

    def product(self, x, w, which: str, ids, ctx, residual=None) -> torch.Tensor:
        return ops.adapter_linear(x, w, self.adapters[which].handle, ids, residual=residual, max_run=ctx.max_q_len)
