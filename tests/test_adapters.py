"""Low-rank adapters without a GPU: the room for them, what is refused before anything is changed."""

import copy
from types import SimpleNamespace

import pytest
import torch

from flashdecode_cuda_b200 import kernels as K
from flashdecode_cuda_b200.cache import KVGroupSpec, PagedCache
from flashdecode_cuda_b200.engine.adapters import Adapters, Caches
from flashdecode_cuda_b200.parts.lowrank import AdaptedProduct, LowRank, largest_rank

RT = SimpleNamespace(device=torch.device("cpu"), dtype=torch.float32, status=None)


class Part:
    lora = None

    def adapted_products(self):
        return [AdaptedProduct("qkv", ["q_proj", "k_proj", "v_proj"], [32, 16, 16], 24), AdaptedProduct("o", ["o_proj"], [24], 32),
                AdaptedProduct("gate_up", ["gate_proj", "up_proj"], [40, 40], 24)]


def model():
    parts = [Part(), Part()]
    return SimpleNamespace(bound=True, rt=RT, all_parts=lambda: parts[:1], adapters=None, parts=parts, caches=Caches())


def pair(n, k, rank):
    g = torch.Generator().manual_seed(n + rank)
    return torch.randn(rank, k, generator=g), torch.randn(n, rank, generator=g)


def test_room_is_what_the_kernel_takes():
    for slices, most in ((1, 256), (2, 256), (3, 168), (4, 128)):
        assert largest_rank(slices) == most
        product = AdaptedProduct("p", [f"m{i}" for i in range(slices)], [8] * slices, 16)
        for rank in (1, 8, most - 7, most, most + 1, 256):
            low = LowRank(product, 2, rank, RT)
            assert low.rank == min(-(-rank // 8) * 8, most) and low.rank <= K.LORA_MAX_RANK and low.rank * slices <= K.LORA_MAX_PACKED
            assert low.a.shape == (2, slices * low.rank, 16) and low.b.shape == (2, 8 * slices, low.rank)
    with pytest.raises(ValueError, match="up to 4 packed"):
        LowRank(AdaptedProduct("p", list("abcde"), [8] * 5, 16), 2, 8, RT)


def test_a_rank_that_a_product_cannot_take_is_refused_when_the_adapter_is_added():
    m = model()
    ad = Adapters(m, 2, 256)
    assert {k: low.rank for k, low in ad.products.items()} == {"q_proj": 168, "k_proj": 168, "v_proj": 168, "o_proj": 256, "gate_proj": 256, "up_proj": 256}
    assert ad.put("wide", {"o_proj": pair(24, 32, 256), "q_proj": pair(32, 24, 168)}, 1.0) == 0
    kept = [(low.a.clone(), low.b.clone(), low.ranks.clone()) for low in ad.products.values()]
    with pytest.raises(ValueError, match="k_proj: an adapter of rank 169; there is room for 168"):
        ad.put("wider", {"o_proj": pair(24, 32, 2), "k_proj": pair(16, 24, 169)}, 1.0)
    assert ad.names == ["wide", None]
    assert all(torch.equal(x, y) for low, k in zip(ad.products.values(), kept) for x, y in zip((low.a, low.b, low.ranks), k))
    assert ad.put("small", {"k_proj": pair(16, 24, 4)}, 1.0) == 1
    with pytest.raises(ValueError, match="up to 256"):
        Adapters(model(), 2, 257)


def engine(m):
    from flashdecode_cuda_b200.engine.api import Engine
    eng = object.__new__(Engine)
    eng.model, eng.cache, eng._own_cache = m, None, None
    return eng


def named(pairs):
    return {f"{m}.lora_{h}.weight": t for m, ab in pairs.items() for h, t in zip("AB", ab)}


def test_a_refused_first_adapter_leaves_no_room_behind():
    """Room is allocated once; that of an adapter that was not taken would be too small for the next one."""
    m = model()
    eng = engine(m)
    for bad in ({"lm_head": pair(9, 24, 4)}, {"q_proj": pair(31, 24, 4)}, {"q_proj": pair(32, 24, 200), "o_proj": pair(24, 32, 2)}):
        with pytest.raises(ValueError):
            eng.add_adapter("x", named(bad), 1.0)
        assert m.adapters is None and all(p.lora is None for p in m.parts)
    with pytest.raises(ValueError, match="needs a name"):
        eng.add_adapter("", named({"q_proj": pair(32, 24, 4)}), 1.0)
    assert m.adapters is None
    assert eng.add_adapter("x", named({"o_proj": pair(24, 32, 40)}), 1.0) == 0 and m.adapters.rank == 40
    with pytest.raises(ValueError, match="takes no adapter"):
        eng.add_adapter("y", named({"lm_head": pair(9, 24, 4)}), 1.0)
    assert m.adapters.names[0] == "x" and m.parts[0].lora is not None       # room that is used stays


def test_a_dropped_model_goes_at_once():
    """Adapters do not keep their model, nor it itself through them."""
    import gc
    import weakref

    class Model(SimpleNamespace):
        pass
    m = Model(**vars(model()))
    Adapters(m, 2, 8)
    seen = weakref.ref(m), weakref.ref(m.adapters)
    gc.disable()
    try:
        del m
        assert seen[0]() is None and seen[1]() is None
    finally:
        gc.enable()


def small_cache():
    return PagedCache([KVGroupSpec(1, 1, 8, None)], [], 8, 4, 2, 4, torch.float32, "cpu")


def test_an_adapter_of_a_live_sequence_stays_whatever_the_cache():
    m = model()
    eng = engine(m)
    for name in ("x", "y"):
        eng.add_adapter(name, named({"q_proj": pair(32, 24, 4)}), 1.0)
    mine, other = small_cache(), small_cache()
    m.caches.add(mine)                           # as a model does with the caches that it makes or runs
    slot = mine.admit(1)
    with pytest.raises(RuntimeError, match="in use"):
        eng.remove_adapter("y")
    mine.release(slot)
    other.admit(1)
    eng.cache = other                            # the engine's own
    with pytest.raises(RuntimeError, match="in use"):
        eng.remove_adapter("y")
    assert not m.caches.use(0) and copy.deepcopy(m.caches) is not m.caches and len(copy.deepcopy(m.caches)) == 0
    eng.cache = None
    del other                                    # a cache that is gone holds nothing
    eng.remove_adapter("y")
    assert m.adapters.names[:2] == ["x", None]


def test_an_adapter_that_a_stream_waits_for_stays():
    """A stream's requests have their adapters' numbers before their sequences start."""
    m = model()
    eng = engine(m)
    for name in ("x", "y"):
        eng.add_adapter(name, named({"q_proj": pair(32, 24, 4)}), 1.0)
    eng.device = torch.device("cpu")
    eng.cache = None
    cache = small_cache()
    eng.run = lambda slots, tokens, requests, steps: [3] * len(slots)
    stream = eng.stream([[1], [2], [1]], 2, cache, max_batch=1, adapter=[None, "y", None])
    for _ in range(2):                           # not begun; then its second request still waits
        with pytest.raises(RuntimeError, match="stream"):
            eng.remove_adapter("y")
        next(stream)
    eng.remove_adapter("x")
    next(stream)                                 # the second request's first token
    with pytest.raises(RuntimeError, match="live sequence"):
        eng.remove_adapter("y")
    assert len(list(stream)) == 3
    eng.remove_adapter("y")
    eng.add_adapter("y", named({"q_proj": pair(32, 24, 4)}), 1.0)
    stream = eng.stream([[1], [2]], 2, cache, adapter="y")
    del stream                                   # never begun
    eng.remove_adapter("y")
