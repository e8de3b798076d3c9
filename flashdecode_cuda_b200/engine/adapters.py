"""The low-rank adapters of a model: requests of one batch may each use one of them, or none.

``Adapters`` keeps, beside every product of the model that takes adapters, room for ``capacity`` adapters of ranks up to ``rank``
(allocated once, so that captured decode steps go on using the same memory when an adapter is added or replaced).  A sequence's
adapter is chosen when its slot is admitted; a step sorts its tokens by adapter on the host, and every product is followed by one
``kernels.lora_add`` for all of them.
"""

from __future__ import annotations

import itertools
import weakref
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from .. import kernels as K
from ..parts.lowrank import LowRank
from ..weights.adapters import Adapter

_made = itertools.count(1)


class Caches(weakref.WeakSet):
    """The caches whose sequences a model runs: adapters that they use stay.  A copied model has its own."""

    def __deepcopy__(self, memo):
        return Caches()

    def use(self, adapter: int) -> bool:
        return any(cache.adapter(slot) == adapter for cache in self for slot in cache.active_slots())


class _Held(list):
    """(a list that can be referred to weakly)"""


class Adapters:
    def __init__(self, model, capacity: int, rank: int):
        if not model.bound:
            raise RuntimeError("the model has no weights yet: adapters come after bind()")
        if capacity < 1 or rank < 1:
            raise ValueError("capacity and rank must be >= 1")
        if rank > K.LORA_MAX_RANK:
            raise ValueError(f"adapters of ranks up to {K.LORA_MAX_RANK} are taken, not {rank}")
        self.capacity, self.rank = capacity, rank
        self.made = next(_made)                      # a captured step belongs to the memory of one of these
        self.names: List[Optional[str]] = [None] * capacity
        self._waiting = weakref.WeakValueDictionary()
        self.products: Dict[str, LowRank] = {}       # by module
        built: List[Tuple[object, Dict[str, LowRank]]] = []
        for part in {id(p): p for p in model.all_parts()}.values():
            mine = {p.name: LowRank(p, capacity, rank, model.rt) for p in part.adapted_products()}
            for low in mine.values():
                for module in low.product.modules:
                    self.products[module] = low
            if mine:
                built.append((part, mine))
        if not built:
            raise ValueError("no part of this model takes low-rank adapters")
        for part, mine in built:
            part.lora = mine
        model.adapters = self

    @staticmethod
    def give_back(model) -> None:
        """The model has no adapters and no room for any again."""
        for part in model.all_parts():
            part.lora = None
        model.adapters = None

    def index(self, name: Optional[str]) -> int:
        """The number under which sequences use the adapter (-1 for None)."""
        if name is None:
            return -1
        try:
            return self.names.index(name)
        except ValueError:
            raise KeyError(f"there is no adapter {name!r}; there are {[n for n in self.names if n]}") from None

    def hold(self, requests: Sequence) -> Sequence:
        """Requests that are fed bit by bit: the adapters that they name stay until nobody has them any more."""
        held = _Held(requests)
        if any(r.adapter >= 0 for r in held):
            self._waiting[id(held)] = held
        return held

    def held(self, index: int) -> bool:
        return any(r.adapter == index for requests in self._waiting.values() for r in requests)

    def put(self, name: str, pairs: Adapter, scale: float) -> int:
        """Add an adapter, or replace the one of that name.  Its matrices take effect with the next step."""
        if not name:
            raise ValueError("an adapter needs a name")
        unknown = sorted(set(pairs) - set(self.products))
        if unknown:
            raise ValueError(f"adapter {name!r}: this model takes no adapter on {unknown[0]}" +
                             (f" and {len(unknown) - 1} more modules" if len(unknown) > 1 else ""))
        lows = list({id(low): low for low in self.products.values()}.values())
        for low in lows:
            low.check(pairs)
        if name in self.names:
            index = self.names.index(name)
        elif None in self.names:
            index = self.names.index(None)
        else:
            raise ValueError(f"adapter {name!r}: there is room for {self.capacity} adapters")
        for low in lows:
            low.put(index, pairs, scale)
        self.names[index] = name
        return index

    def remove(self, name: str) -> None:
        """Its place may be used again; no live sequence may use it any more."""
        self.names[self.index(name)] = None

    def bytes(self) -> int:
        return sum(low.bytes() for low in {id(low): low for low in self.products.values()}.values())
