"""Requests of one batch that differ, through the entry points: beam search and low-rank adapters, alone and together, against the
plain implementation (whose weights get an adapter's product added), and on every architecture against the engine's own
whole-sequence logits."""

import json
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import bifatar_helpers
import botusun_helpers
import flashdecode_cuda_b200 as fd
import gulozen_helpers
import lonasun_helpers
import nizazen_helpers
import revelix_helpers
from flashdecode_cuda_b200.cache import PagedCache
from flashdecode_cuda_b200.weights import write_adapter
from helpers import TINY, TOL, prompts_for, raw_config, rel_err, weights_of, write_folder
from plain import qwen2_plain as P
from test_beam import by_hand, by_hand_uncut

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("requests")
    return {n: write_folder(tmp, n, seed=9) for n in TINY}


def adapter_for(folder, seed, rank, keep=lambda module: True):
    """(A, B) for the projections of a model folder, about as large as the weights they are added to."""
    g = torch.Generator().manual_seed(seed)
    out = {}
    for name, w in sorted(weights_of(folder).items()):
        module = name[:-len(".weight")]
        if module.endswith("_proj") and keep(module):
            n, k = w.shape
            out[module] = ((torch.randn(rank, k, generator=g) * k ** -0.5).bfloat16(),
                           (0.02 * k ** 0.5 * torch.randn(n, rank, generator=g) * rank ** -0.5).bfloat16())
    return out


def as_tensors(pairs):
    return {f"{m}.lora_{h}.weight": t for m, ab in pairs.items() for h, t in zip("AB", ab)}


def merged(folder, pairs, scale):
    w = {k: v.double() for k, v in weights_of(folder).items()}
    for m, (a, b) in (pairs or {}).items():
        w[f"{m}.weight"] = w[f"{m}.weight"] + scale * (b.double() @ a.double())
    return w


class Language:
    """The plain implementation as the language of the search by hand, one set of weights per adapter."""

    def __init__(self, raw, weights):
        self.raw, self.weights, self.seen = raw, weights, {}

    def logp(self, text, adapter=-1):
        key = (tuple(text), adapter)
        if key not in self.seen:
            self.seen[key] = torch.log_softmax(P.logits(self.raw, self.weights[adapter], list(text))[-1].double(), 0)
        return self.seen[key]


# ------------------------------------------------------------------------------------------------------------------ beams
@pytest.mark.parametrize("name,beams,n,penalty", [("A", 1, 6, 1.0), ("B", 4, 8, 1.0), ("C", 3, 10, 0.5), ("D", 2, 5, 2.0)])
def test_beam_search_equals_the_search_by_hand(folders, name, beams, n, penalty):
    eng = fd.load(folders[name], device="cuda", dtype="float32")
    raw = raw_config(folders[name])
    lang = Language(raw, {-1: weights_of(folders[name])})
    # lengths on both sides of a cache block's end, and a window that gives blocks back (C)
    prompts = prompts_for(raw["vocab_size"], [3, 30, 1, 17], seed=2)
    stop = [int(t) for t in lang.logp(prompts[0]).topk(3).indices[1:]]
    for graphs in (True, False):
        eng.use_graphs = graphs
        got = eng.beam_search(prompts, n, num_beams=beams, length_penalty=penalty, num_return=beams, stop_token_ids=stop,
                              block_size=16, max_batch=3 * beams)
        eng.model.check_status()
        for p, r in zip(prompts, got):
            want = by_hand(lang, p, n, beams, penalty, stop)
            assert [h.tokens for h in r.hypotheses] == [t for _, t, _ in want]
            assert [h.finish_reason for h in r.hypotheses] == [why for _, _, why in want]
            assert all(abs(h.score - s) < 1e-4 for h, (s, _, _) in zip(r.hypotheses, want))
        assert not eng.cache.active_slots()
        eng.cache.check_invariants()
        assert eng.cache.blocks_in_use() == [0] * len(eng.cache.groups)


def test_many_beams_with_several_stop_tokens(folders):
    """More candidates than one selection gives: a request's rows are selected from in parts."""
    eng = fd.load(folders["B"], device="cuda", dtype="float32")
    raw = raw_config(folders["B"])
    lang = Language(raw, {-1: weights_of(folders["B"])})
    prompt = prompts_for(raw["vocab_size"], [7], seed=12)[0]
    stop = [int(t) for t in lang.logp(prompt).topk(6).indices]
    (got,) = eng.beam_search([prompt], 3, num_beams=30, num_return=30, stop_token_ids=stop)
    want, counts = by_hand_uncut(lang, prompt, 3, 30, stop)
    assert counts == [30] * len(counts)
    assert [h.tokens for h in got.hypotheses] == [t for _, t, _ in want]
    assert all(abs(h.score - s) < 1e-4 for h, (s, _, _) in zip(got.hypotheses, want))
    eng.model.check_status()


def test_one_beam_is_greedy_and_requests_may_differ(folders):
    eng = fd.load(folders["B"], device="cuda", dtype="float32")
    prompts = prompts_for(384, [5, 40, 12], seed=3)
    greedy = eng.generate(prompts, [4, 9, 7])
    beams = eng.beam_search(prompts, [4, 9, 7], num_beams=[1, 1, 1])
    assert [r.tokens for r in beams] == [r.tokens for r in greedy]
    mixed = eng.beam_search(prompts, [4, 9, 7], num_beams=[1, 5, 2])
    alone = [eng.beam_search([p], m, num_beams=b)[0] for p, m, b in zip(prompts, [4, 9, 7], [1, 5, 2])]
    assert [r.tokens for r in mixed] == [r.tokens for r in alone]
    assert eng.beam_search([], 4) == []
    for bad in (dict(num_beams=0), dict(num_beams=65), dict(num_return=5), dict(num_beams=[1, 2]), dict(adapter="x"), dict(max_batch=2)):
        with pytest.raises((ValueError, KeyError)):
            eng.beam_search(prompts, 4, **bad)
    eng.model.check_status()


ARCHITECTURES = [(lonasun_helpers, "X"), (lonasun_helpers, "Z"), (nizazen_helpers, "P"), (nizazen_helpers, "S"), (revelix_helpers, "P"),
                 (revelix_helpers, "Q"), (botusun_helpers, "A"), (botusun_helpers, "C"), (gulozen_helpers, "A"), (gulozen_helpers, "B"),
                 (bifatar_helpers, "U"), (bifatar_helpers, "W")]


@pytest.mark.parametrize("H,name", ARCHITECTURES, ids=[f"{h.__name__[:-8]}-{n}" for h, n in ARCHITECTURES])
def test_beams_of_every_architecture_score_what_their_text_scores(tmp_path, H, name):
    """A hypothesis is fed again as one prompt: its score is the sum of the log-probabilities there, whatever its beam's slots
    were copied from."""
    eng = fd.load(H.write_folder(tmp_path, name, seed=1), device="cuda", dtype="float32")
    model = eng.model
    prompts = prompts_for(model.vocab_size, [13, 4], seed=4)
    got = eng.beam_search(prompts, 14, num_beams=4, num_return=4, length_penalty=1.0, block_size=16)
    model.check_status()
    eng.cache.check_invariants()
    for p, r in zip(prompts, got):
        assert len(r.hypotheses) == 4 and len({tuple(h.tokens) for h in r.hypotheses}) == 4
        for h in r.hypotheses:
            cache = model.new_cache(max_tokens=64)
            logits = model.step(cache, [cache.admit()], [p + h.tokens[:-1]], "all").double().cpu()
            lp = torch.log_softmax(logits, 1)
            total = sum(float(lp[len(p) - 1 + i, t]) for i, t in enumerate(h.tokens))
            # a logit of a step and of a whole prompt are apart by at most 1e-4 of the largest; a log-probability by twice that
            tol = 2e-4 * float(logits.abs().max())
            assert abs(h.score - total / len(h.tokens)) <= tol, (h.score, total / len(h.tokens))
    model.check_status()


# --------------------------------------------------------------------------------------------------------------- adapters
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B", "C", "E"])
def test_adapters_equal_merged_weights(folders, name, dtype):
    folder = folders[name]
    raw = raw_config(folder)
    eng = fd.load(folder, device="cuda", dtype=dtype)
    one, two = adapter_for(folder, 1, 8), adapter_for(folder, 2, 3, lambda m: "q_proj" in m or "up_proj" in m)
    eng.add_adapter("one", as_tensors(one), scale=0.5)
    eng.add_adapter("two", as_tensors(two), scale=2.0)
    weights = [merged(folder, one, 0.5), merged(folder, None, 1.0), merged(folder, two, 2.0), merged(folder, one, 0.5)]
    model = eng.model
    lengths = [20, 7, 1, 33] if name != "E" else [150, 70, 1, 33]
    prompts = prompts_for(raw["vocab_size"], lengths, seed=5)
    more = prompts_for(raw["vocab_size"], [3] * 4, seed=6)
    cache = model.new_cache(max_tokens=64 * 16)
    slots = [cache.admit(a) for a in (0, -1, 1, 0)]
    rows = [model.step(cache, slots, prompts, "last").double().cpu()]
    for i in range(3):
        rows.append(model.step(cache, slots, [[m[i]] for m in more], "last").double().cpu())
    model.check_status()
    for j, (p, m, w) in enumerate(zip(prompts, more, weights)):
        want = P.logits(raw, w, p + m)
        for i, r in enumerate(rows):
            assert rel_err(r[j], want[len(p) - 1 + i]) < TOL[dtype], (j, i)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_the_largest_ranks(folders, dtype):
    """Ranks of 256, and of 168 where three projections are one product, beside an adapter of a small rank."""
    folder = folders["B"]
    raw = raw_config(folder)
    eng = fd.load(folder, device="cuda", dtype=dtype)
    wide = {m: ab for rank, part in ((168, "self_attn"), (256, "mlp"), (256, "o_proj"))
            for m, ab in adapter_for(folder, rank, rank, lambda m: part in m).items()}
    small = adapter_for(folder, 3, 4)
    eng.add_adapter("wide", as_tensors(wide), scale=0.5)
    eng.add_adapter("small", as_tensors(small), scale=0.5)
    weights = [merged(folder, wide, 0.5), merged(folder, small, 0.5)]
    prompts = prompts_for(raw["vocab_size"], [20, 9], seed=15)
    cache = eng.model.new_cache(max_tokens=64 * 4)
    slots = [cache.admit(0), cache.admit(1)]
    first = eng.model.step(cache, slots, prompts, "last").double().cpu()
    second = eng.model.step(cache, slots, [[5], [6]], "last").double().cpu()
    eng.model.check_status()
    for j, w in enumerate(weights):
        want = P.logits(raw, w, prompts[j] + [5 + j])
        assert rel_err(first[j], want[len(prompts[j]) - 1]) < TOL[dtype] and rel_err(second[j], want[len(prompts[j])]) < TOL[dtype]
    with pytest.raises(ValueError, match="q_proj: an adapter of rank 176"):
        eng.add_adapter("wider", as_tensors(adapter_for(folder, 1, 176, lambda m: "q_proj" in m)), scale=1.0)


def test_adapters_in_generation_and_with_beams(folders):
    folder = folders["B"]
    raw = raw_config(folder)
    eng = fd.load(folder, device="cuda", dtype="float32")
    pairs = [adapter_for(folder, s, r) for s, r in ((3, 4), (4, 16))]
    for i, p in enumerate(pairs):
        eng.add_adapter(f"a{i}", as_tensors(p), scale=1.0)
    weights = {-1: weights_of(folder), 0: merged(folder, pairs[0], 1.0), 1: merged(folder, pairs[1], 1.0)}
    prompts = prompts_for(raw["vocab_size"], [9, 9, 9, 22, 1], seed=7)
    prompts[1] = prompts[2] = prompts[0]                    # the same prompt with three sets of weights
    who = [None, "a0", "a1", "a1", None]
    index = [-1, 0, 1, 1, -1]
    want = [P.generate(raw, weights[e], p, 10) for p, e in zip(prompts, index)]
    assert len({tuple(w) for w in want[:3]}) == 3
    for graphs in (True, False):
        eng.use_graphs = graphs
        assert [r.tokens for r in eng.generate(prompts, 10, adapter=who, max_batch=4)] == want
    eng.use_graphs = True
    # graphs with and without adapters live side by side over one cache
    assert [r.tokens for r in eng.generate(prompts, 10)] == [P.generate(raw, weights[-1], p, 10) for p in prompts]
    assert [r.tokens for r in eng.generate(prompts[:2], 10, adapter="a1")] == [P.generate(raw, weights[1], p, 10) for p in prompts[:2]]
    lang = Language(raw, weights)
    got = eng.beam_search(prompts, 8, num_beams=3, num_return=3, adapter=who, block_size=16)
    for p, e, r in zip(prompts, index, got):
        assert [h.tokens for h in r.hypotheses] == [t for _, t, _ in by_hand(lang, p, 8, 3, 1.0, (), False, e)]
    # another adapter under the same name: captured steps use it too
    eng.add_adapter("a0", as_tensors(pairs[1]), scale=1.0)
    assert [r.tokens for r in eng.generate(prompts[:3], 10, adapter="a0")] == [P.generate(raw, weights[1], p, 10) for p in prompts[:3]]
    streamed = {}
    for step in eng.stream(prompts[:3], 10, adapter=["a1", None, "a1"]):
        for i, t, _ in step:
            streamed.setdefault(i, []).append(t)
    assert streamed[0] == P.generate(raw, weights[1], prompts[0], 10) and streamed[1] == P.generate(raw, weights[-1], prompts[1], 10)
    eng.model.check_status()


def test_more_adapters_than_rows_and_padded_batches(folders):
    """Steps of three sequences run in a graph of four rows; eight adapters have room."""
    folder = folders["D"]
    raw = raw_config(folder)
    eng = fd.load(folder, device="cuda", dtype="float32")
    eng.enable_adapters(max_adapters=8, max_rank=8)
    pairs = [adapter_for(folder, 20 + i, 1 + i) for i in range(8)]
    for i, p in enumerate(pairs):
        eng.add_adapter(str(i), as_tensors(p), scale=1.0)
    prompts = prompts_for(raw["vocab_size"], [4] * 11, seed=8)
    who = [7, 2, 5, 0, 1, 3, 4, 6, 7, 0, None]
    want = [P.generate(raw, merged(folder, None if e is None else pairs[e], 1.0), p, 5) for p, e in zip(prompts, who)]
    names = [None if e is None else str(e) for e in who]
    assert [r.tokens for r in eng.generate(prompts, 5, adapter=names)] == want
    assert [r.tokens for r in eng.generate(prompts[:3], 5, adapter=names[:3])] == want[:3]
    assert [r.tokens for r in eng.generate(prompts, 5, adapter=names, max_batch=3)] == want
    eng.model.check_status()


def test_adapter_refusals(folders, tmp_path):
    eng = fd.load(folders["B"], device="cuda", dtype="bfloat16")
    good = adapter_for(folders["B"], 1, 4)
    with pytest.raises(KeyError, match="no adapters"):
        eng.generate([[1, 2]], 2, adapter="x")
    with pytest.raises(KeyError):
        eng.remove_adapter("x")
    with pytest.raises(ValueError, match="scale"):
        eng.add_adapter("x", as_tensors(good))
    eng.enable_adapters(max_adapters=2, max_rank=4)
    with pytest.raises(RuntimeError, match="already"):
        eng.enable_adapters()
    with pytest.raises(ValueError, match="takes no adapter"):
        eng.add_adapter("x", {"lm_head.lora_A.weight": torch.zeros(2, 96), "lm_head.lora_B.weight": torch.zeros(384, 2)}, 1.0)
    first = sorted(good)[0]
    a, b = good[first]
    with pytest.raises(ValueError, match="projection of"):
        eng.add_adapter("x", as_tensors({first: (a[:, 1:], b)}), 1.0)
    with pytest.raises(ValueError, match="room for"):
        eng.add_adapter("x", as_tensors(adapter_for(folders["B"], 1, 9)), 1.0)
    with pytest.raises(ValueError, match="come together"):
        eng.add_adapter("x", {f"{first}.lora_A.weight": a}, 1.0)
    with pytest.raises(ValueError, match="not a tensor"):
        eng.add_adapter("x", {f"{first}.weight": a}, 1.0)
    folder = write_adapter(tmp_path / "ad", good, alpha=8.0)
    assert eng.add_adapter("x", folder) == 0 and eng.add_adapter("y", folder) == 1 and eng.add_adapter("x", folder) == 0
    assert eng.model.adapters.products[first].scale.tolist() == [2.0, 2.0]
    with pytest.raises(ValueError, match="2 adapters"):
        eng.add_adapter("z", folder)
    with pytest.raises(KeyError, match="no adapter 'z'"):
        eng.generate([[1, 2]], 2, adapter=["z"])
    with pytest.raises(ValueError, match="3 adapters for 1"):
        eng.generate([[1, 2]], 2, adapter=["x", "y", None])
    eng.cache = eng.new_cache(max_tokens=128)
    slot = eng.admit(1)
    with pytest.raises(RuntimeError, match="in use"):
        eng.remove_adapter("y")
    eng.release(slot)
    eng.remove_adapter("y")
    assert eng.add_adapter("z", folder) == 1
    lonasun = fd.load(lonasun_helpers.write_folder(tmp_path, "Z"), device="cuda", dtype="float32")
    with pytest.raises(ValueError, match="no part"):
        lonasun.enable_adapters()


def test_adapters_of_sequences_in_any_cache_stay(folders):
    eng = fd.load(folders["B"], device="cuda", dtype="float32")
    for i in range(2):
        eng.add_adapter(str(i), as_tensors(adapter_for(folders["B"], i, 4)), scale=1.0)
    mine = eng.model.new_cache(max_tokens=128)
    first = eng.model.new_cache(max_tokens=128)
    by_hand_made = PagedCache(*eng.model._layout[:2], 8, 2, 4, 16, torch.float32, "cuda")
    for cache, step in ((mine, False), (by_hand_made, True)):
        slot = cache.admit(1)
        if step:
            eng.model.step(cache, [slot], [[1, 2, 3]])
        with pytest.raises(RuntimeError, match="in use"):
            eng.remove_adapter("1")
        cache.release(slot)
    slot = first.admit(0)
    eng.remove_adapter("1")
    eng.model.check_status()


def test_command_line(folders, tmp_path):
    folder = folders["B"]
    raw = raw_config(folder)
    pairs = adapter_for(folder, 5, 4)
    ad = write_adapter(tmp_path / "adapter", pairs, alpha=4.0)
    cmd = [sys.executable, "-m", "flashdecode_cuda_b200", "generate", "--model", str(folder), "--prompt-ids", "5,6,7", "--prompt-ids", "9",
           "--max-new-tokens", "6", "--dtype", "float32", "--stop-ids", "383", "--adapter", str(ad), "--beams", "3", "--length-penalty", "0.5"]
    out = subprocess.run(cmd, capture_output=True, text=True, cwd=ROOT, check=True).stdout.splitlines()
    lang = Language(raw, {0: merged(folder, pairs, 1.0)})
    for line, p in zip(out, ([5, 6, 7], [9])):
        got = json.loads(line)
        score, tokens, why = by_hand(lang, p, 6, 3, 0.5, (383,), False, 0)[0]
        assert got["tokens"] == tokens and abs(got["score"] - score) < 1e-4 and got["finish_reason"] == why
