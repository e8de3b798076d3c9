"""Low-rank adapters on a part's products: which projections a packed matrix holds, and the adapters' matrices beside it."""

from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from .. import kernels as K
from .base import Runtime

RANK_UNIT = 8       # ranks are stored in multiples of this (16-byte pieces of bfloat16), zeros behind an adapter's own


def largest_rank(slices: int) -> int:
    """The largest rank that a product of so many packed projections has room for."""
    return min(K.LORA_MAX_RANK, K.LORA_MAX_PACKED // slices) // RANK_UNIT * RANK_UNIT


@dataclass
class AdaptedProduct:
    """A product of a part that takes adapters: ``modules`` are the checkpoint's names of the projections that its matrix packs and
    ``rows`` their numbers of outputs; ``order``: the packed matrix's rows as places in the projections one after another (None: in
    that order)."""
    name: str
    modules: Sequence[str]
    rows: Sequence[int]
    inputs: int
    order: Optional[torch.Tensor] = None


@dataclass
class TokenAdapters:
    """Which tokens of a step use which adapter: see ``kernels.lora_add``."""
    order: torch.Tensor
    start: torch.Tensor
    ids: torch.Tensor


class LowRank:
    """The adapters of one product: A [E, slices * R, inputs], B [E, outputs, R].  R is ``rank``, or what the kernel takes of so many
    packed projections where that is less."""

    def __init__(self, product: AdaptedProduct, capacity: int, rank: int, rt: Runtime):
        self.slices = len(product.modules)
        if self.slices > K.LORA_MAX_SLICES:
            raise ValueError(f"{product.modules[0]}: adapters take up to {K.LORA_MAX_SLICES} packed projections, not {self.slices}")
        self.product, self.rank, self.rt = product, min(-(-rank // RANK_UNIT) * RANK_UNIT, largest_rank(self.slices)), rt
        N = sum(product.rows)
        which = torch.repeat_interleave(torch.arange(self.slices), torch.tensor(list(product.rows)))
        self.order = torch.arange(N) if product.order is None else product.order.cpu()
        self.col_slice = None
        if self.slices > 1:
            packed = which[self.order]
            if N % 8 or not bool((packed.view(-1, 8) == packed.view(-1, 8)[:, :1]).all()):
                raise ValueError(f"{product.modules[0]}: adapters take packed projections in tiles of 8 outputs of one projection each")
            self.col_slice = packed.view(-1, 8)[:, 0].to(torch.uint8).to(rt.device)
        self.a = torch.zeros(capacity, self.slices * self.rank, product.inputs, dtype=rt.dtype, device=rt.device)
        self.b = torch.zeros(capacity, N, self.rank, dtype=rt.dtype, device=rt.device)
        self.scale = torch.zeros(capacity, dtype=torch.float32, device=rt.device)
        self.ranks = torch.zeros(capacity, dtype=torch.int32, device=rt.device)

    def check(self, pairs: Dict[str, Tuple[torch.Tensor, torch.Tensor]]) -> None:
        for module, n in zip(self.product.modules, self.product.rows):
            if module in pairs:
                a, b = pairs[module]
                if a.shape[1] != self.product.inputs or b.shape[0] != n:
                    raise ValueError(f"{module}: an adapter of {b.shape[0]} x {a.shape[1]} for a projection of {n} x {self.product.inputs}")
                if a.shape[0] > self.rank:
                    raise ValueError(f"{module}: an adapter of rank {a.shape[0]}; there is room for {self.rank}")

    def put(self, index: int, pairs: Dict[str, Tuple[torch.Tensor, torch.Tensor]], scale: float) -> None:
        """Adapter ``index``'s matrices; projections that it does not adapt get zeros."""
        R, first, rank = self.rank, 0, 0
        a = torch.zeros_like(self.a[index])
        b = torch.zeros(sum(self.product.rows), R, dtype=self.b.dtype, device=self.b.device)
        for s, (module, n) in enumerate(zip(self.product.modules, self.product.rows)):
            if module in pairs:
                ma, mb = pairs[module]
                r = ma.shape[0]
                a[s * R:s * R + r], b[first:first + n, :r] = ma.to(a), mb.to(b)
                rank = max(rank, r)
            first += n
        self.a[index], self.b[index] = a, b[self.order.to(b.device)]
        self.scale[index], self.ranks[index] = scale, rank

    def add(self, x: torch.Tensor, y: torch.Tensor, tokens: TokenAdapters) -> None:
        """y += scale B (A x) for the tokens that have an adapter."""
        K.lora_add(x, self.a, self.b, self.scale, self.ranks, tokens.order, tokens.start, tokens.ids, y, col_slice=self.col_slice,
                   slices=self.slices, status=self.rt.status)

    def bytes(self) -> int:
        return self.a.nbytes + self.b.nbytes
