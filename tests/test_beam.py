"""Beam search without a GPU: the cache's forks (blocks shared, none lost or written to by two), the loop's decisions against a
search that enumerates, refusals."""

import itertools
import math
import random

import pytest
import torch

from flashdecode_cuda_b200.cache import IdAllocator, KVGroupSpec, PagedCache, PoolExhausted, StateSpec
from flashdecode_cuda_b200.engine.beam import BeamBackend, BeamLoop, BeamRequest


def make(num_blocks=40, slots=8, per_seq=8, bs=4, window=None, states=True, keys_only=False):
    groups = [KVGroupSpec(2, 2, 8, None)]
    if window:
        groups.append(KVGroupSpec(1, 1, 8, window, v_head_dim=6))
    if keys_only:
        groups.append(KVGroupSpec(2, 1, 4, keys_only=True))
    st = [StateSpec("a", (2, 3)), StateSpec("b", (5,), torch.bfloat16)] if states else []
    return PagedCache(groups, st, num_blocks, slots, per_seq, bs, torch.float32, "cpu")


def write(c, slot, value):
    """One token whose keys, values and state are ``value``."""
    c.reserve([(slot, 1)])
    pos = c.length(slot)
    for gi, g in enumerate(c.groups):
        b, o = c.slot_of(slot, pos, gi)
        assert g.alloc.holders(b) == 1, "a shared block is written to"
        g.keys[:, b, :, o] = value
        if g.values is not g.keys:
            g.values[:, b, :, o] = value
    for t in c.states.values():
        t[slot] = value
    c.advance(slot, 1)


def holds(c, slot, values, window=None):
    for gi, g in enumerate(c.groups):
        for layer in range(g.spec.n_layers):
            k, v = c.gather(slot, gi, layer)
            first = g.spec.first_needed(len(values))
            for p in range(first, len(values)):
                if not (bool((k[p] == values[p]).all()) and bool((v[p] == values[p]).all())):
                    return False
    return not values or all(bool((t[slot] == torch.tensor(values[-1]).to(t.dtype)).all()) for t in c.states.values())


def test_ids_with_several_holders():
    a = IdAllocator(3)
    x, y = a.allocate(2)
    a.share([x])
    assert a.holders(x) == 2 and a.num_used == 2
    a.free([x])
    assert a.in_use(x) and a.num_used == 2 and a.num_free == 1
    a.free([x, y])
    assert a.num_used == 0
    with pytest.raises(ValueError, match="not in use"):
        a.share([x])
    with pytest.raises(ValueError, match="double free"):
        a.free([x])


@pytest.mark.parametrize("length", [1, 3, 4, 5, 8, 11])
@pytest.mark.parametrize("window", [None, 6])
def test_fork_shares_full_blocks_and_copies_the_last(length, window):
    c = make(window=window, keys_only=True)
    a, b, d = c.admit(), c.admit(), c.admit(5)
    for i in range(length):
        write(c, a, 10 + i)
    for i in range(7):
        write(c, b, 50 + i)
    c.fork([(a, b), (a, d)])
    c.check_invariants()
    values = [10 + i for i in range(length)]
    assert [c.length(s) for s in (a, b, d)] == [length] * 3 and c.adapter(d) == -1
    assert all(holds(c, s, values) for s in (a, b, d))
    n = length // 4
    assert c.slots[a].blocks[0][:n] == c.slots[b].blocks[0][:n] == c.slots[d].blocks[0][:n]
    if length % 4:
        assert len({c.slots[s].blocks[0][n] for s in (a, b, d)}) == 3
    for i, s in enumerate((a, b, d)):           # they go on apart
        for j in range(6):
            write(c, s, 100 * (i + 1) + j)
        c.check_invariants()
    for i, s in enumerate((a, b, d)):
        assert holds(c, s, values + [100 * (i + 1) + j for j in range(6)])
    for s in (b, a, d):
        c.release(s)
        c.check_invariants()
    assert c.blocks_in_use() == [0] * len(c.groups)
    c.sync()
    assert all(torch.equal(g.table, torch.from_numpy(g.table_host)) and int((g.table >= 0).sum()) == 0 for g in c.groups)


def test_fork_refusals_change_nothing():
    c = make(num_blocks=4, slots=4)
    a, b = c.admit(), c.admit()
    for i in range(6):
        write(c, a, i)                           # 2 blocks
    for i in range(5):
        write(c, b, i)                           # 2 more: the pool is full
    version = c.lengths_version
    d = c.admit()
    for pairs in ([(a, d), (b, d)], [(a, b), (b, d)], [(a, a)]):
        with pytest.raises(ValueError, match="destination"):
            c.fork(pairs)
    with pytest.raises(ValueError, match="no sequence"):
        c.fork([(a, 3)])
    with pytest.raises(PoolExhausted):
        c.fork([(a, d)])
    c.check_invariants()
    assert c.length(d) == 0 and c.blocks_in_use() == [4] and c.lengths_version == version + 1
    c.fork([(a, b)])                             # b's own blocks serve
    c.check_invariants()
    assert c.blocks_in_use() == [3] and holds(c, b, list(range(6)))
    c.fork([])


def test_reorder_keeps_first_children_in_place():
    c = make(num_blocks=64, slots=8, per_seq=16)
    s = [c.admit() for _ in range(3)]
    t = [c.admit() for _ in range(2)]
    for i, slot in enumerate(s + t):
        for j in range(5):
            write(c, slot, 10 * i + j)
    got, other = c.reorder([(s, [s[1], s[1], s[2]]), (t, [t[0], t[1]])])
    assert got == [s[1], s[0], s[2]] and other == t
    c.check_invariants()
    assert [holds(c, x, [10 * p + j for j in range(5)]) for x, p in zip(got, (1, 1, 2))] == [True] * 3
    # more beams than before: free slots; fewer: slots go back
    got, other = c.reorder([(got, [got[0]] * 4), (other, [other[1]])])
    c.check_invariants()
    assert len(set(got)) == 4 and other == [t[1]] and len(c.active_slots()) == 5
    assert all(holds(c, x, [10 + j for j in range(5)]) for x in got)
    assert c.reorder([(got, []), (other, other)]) == [[], other] and c.active_slots() == other
    with pytest.raises(ValueError, match="one request"):
        c.reorder([(other, []), (other, other)])
    with pytest.raises(ValueError, match="one request"):
        c.reorder([(other, [other[0] + 1])])
    for _ in range(7):
        c.admit()
    with pytest.raises(PoolExhausted):
        c.reorder([(other, other * 2)])
    c.check_invariants()


def test_many_random_reorders():
    rng = random.Random(4)
    c = make(num_blocks=80, slots=12, per_seq=12, window=7, keys_only=True)
    requests = [[c.admit(i)] for i in range(3)]
    texts = {r[0]: [] for r in requests}
    for step in range(30):
        for r in requests:
            for slot in r:
                v = rng.randrange(1, 200)
                write(c, slot, v)
                texts[slot] = texts[slot] + [v]
        c.check_invariants()
        moves = [(r, [rng.choice(r) for _ in range(rng.randint(1, 4))]) for r in requests]
        placed = c.reorder(moves)
        texts = {s: texts[p] for (_, parents), row in zip(moves, placed) for p, s in zip(parents, row)}
        requests = placed
        c.check_invariants()
        for i, r in enumerate(requests):
            assert all(holds(c, s, texts[s]) and c.adapter(s) == i for s in r)
        if step % 9 == 8:                        # an end, and a beginning
            for s in requests[0]:
                c.release(s)
            requests[0] = [c.admit(0)]
            texts[requests[0][0]] = []


# ---------------------------------------------------------------------------------------------------------------- the loop
class Table(BeamBackend):
    """A language of V tokens whose log-probabilities depend on all tokens so far (and on the adapter), by a seeded draw."""

    def __init__(self, V=7, slots=16, tokens=4096, peak=1.5):
        self.V, self.slots, self.tokens, self.peak = V, slots, tokens, peak
        self.text, self.who, self.calls = {}, {}, 0

    def logp(self, text, adapter=-1):
        g = torch.Generator().manual_seed(hash((tuple(text), adapter)) & 0x7fffffff)
        return torch.log_softmax(self.peak * torch.randn(self.V, generator=g, dtype=torch.float64), 0)

    def beam_capacity(self):
        return self.slots, self.tokens

    def beam_tokens_held(self, r):
        return len(r.prompt) + r.num_beams * r.max_new_tokens

    def admit(self, adapter=-1):
        s = min(set(range(self.slots)) - set(self.text))
        self.text[s], self.who[s] = [], adapter
        return s

    def release(self, slot):
        del self.text[slot]

    def reorder(self, beams):
        out, old = [], dict(self.text)
        who = dict(self.who)
        for slots, _ in beams:
            for s in slots:
                del self.text[s]
        for slots, parents in beams:
            row = []
            for p in parents:
                s = self.admit(who[p])
                self.text[s] = old[p]
                row.append(s)
            out.append(row)
        return out

    def select(self, slots, tokens, scores, start, k):
        assert len(set(slots)) == len(slots)
        self.calls += 1
        S, R, T = [], [], []
        for s, t in zip(slots, tokens):
            self.text[s] = self.text[s] + list(t)
        for lo, hi in zip(start[:-1], start[1:]):
            c = [(-(scores[b] + float(lp)), b, v) for b in range(lo, hi)
                 for v, lp in enumerate(self.logp(self.text[slots[b]], self.who[slots[b]]))]
            c = sorted(c)[:k]
            pad = k - len(c)
            S.append([-x for x, _, _ in c] + [-math.inf] * pad)
            R.append([b for _, b, _ in c] + [-1] * pad)
            T.append([v for _, _, v in c] + [-1] * pad)
        return S, R, T


def by_hand(lang, prompt, n, beams, penalty=1.0, stop=(), early=False, adapter=-1):
    """Beam search over whole texts, written out."""
    live, done = [(0.0, [])], []
    for step in range(1, n + 1):
        c = []
        for i, (s, t) in enumerate(live):
            c += [(s + float(lp), i, v, t) for v, lp in enumerate(lang.logp(prompt + t, adapter))]
        c = sorted(c, key=lambda x: (-x[0], x[1], x[2]))[:2 * beams]
        live = []
        for rank, (s, _, v, t) in enumerate(c):
            if v in stop:
                if rank < beams:
                    done.append((s / step ** penalty, t + [v], "stop"))
            elif len(live) < beams:
                live.append((s, t + [v]))
        done = sorted(done, key=lambda h: -h[0])[:beams]
        if not live:
            break
        if step == n:
            done = sorted(done + [(s / n ** penalty, t, "length") for s, t in live], key=lambda h: -h[0])[:beams]
            break
        if len(done) == beams:
            best = max(s for s, _ in live) / (n if penalty > 0 else step + 1) ** penalty
            if early or best <= done[-1][0]:
                break
    return done


@pytest.mark.parametrize("beams,n,penalty,stop,early", [(1, 6, 1.0, (), False), (3, 5, 1.0, (2,), False), (4, 8, 0.6, (1, 5), False),
                                                        (4, 8, 2.0, (3,), True), (2, 7, 0.0, (0,), False), (5, 6, -1.0, (4,), False), (9, 4, 1.0, (6,), False)])
def test_loop_against_the_search_by_hand(beams, n, penalty, stop, early):
    lang = Table(slots=2 * beams + 1)
    prompts = [[1, 2, 3], [4], [5, 5], [0, 6, 1, 2]]
    reqs = [BeamRequest(p, n, beams, penalty, stop, early, adapter=i % 2 - 1, request_id=i) for i, p in enumerate(prompts)]
    got = BeamLoop(lang, max_batch=2 * beams).run(reqs)
    for i, (p, r) in enumerate(zip(prompts, got)):
        want = by_hand(lang, p, n, beams, penalty, stop, early, i % 2 - 1)
        assert r.request_id == i and [h.tokens for h in r.hypotheses] == [t for _, t, _ in want]
        assert [h.finish_reason for h in r.hypotheses] == [why for _, _, why in want]
        assert all(abs(h.score - s) < 1e-12 for h, (s, _, _) in zip(r.hypotheses, want))
    assert not lang.text                         # every slot was given back


def test_wide_beams_find_the_best_text_of_all():
    lang = Table(V=4, slots=64, peak=1.0)
    (r,) = BeamLoop(lang).run([BeamRequest([2], 3, 64, 0.0)])
    best = max(itertools.product(range(4), repeat=3), key=lambda t: sum(float(lang.logp([2] + list(t[:i]))[t[i]]) for i in range(3)))
    assert r.tokens == list(best) and len(r.hypotheses) == 64


def test_unequal_requests_in_one_batch():
    lang = Table(slots=9)
    reqs = [BeamRequest([1], 3, 2, request_id=0), BeamRequest([2, 2], 7, 4, stop_token_ids=(3,), request_id=1), BeamRequest([3], 1, 3, request_id=2)]
    got = BeamLoop(lang, 9).run(reqs)
    for r, q in zip(got, reqs):
        assert [h.tokens for h in r.hypotheses] == [t for _, t, _ in by_hand(lang, q.prompt, q.max_new_tokens, q.num_beams, 1.0, q.stop_token_ids)]
    assert lang.calls <= 7 and not lang.text


def test_what_is_refused_and_errors_give_slots_back():
    for bad in (dict(prompt=[]), dict(max_new_tokens=0), dict(num_beams=0), dict(num_beams=65)):
        with pytest.raises(ValueError):
            BeamRequest(**{**dict(prompt=[1], max_new_tokens=2), **bad})
    lang = Table(slots=3)
    with pytest.raises(ValueError, match="need 4 slots"):
        BeamLoop(lang).run([BeamRequest([1], 2, 4)])
    with pytest.raises(ValueError, match="max_batch"):
        BeamLoop(lang, 0)

    class Breaks(Table):
        def select(self, *a):
            if self.calls == 2:
                raise RuntimeError("broken")
            return super().select(*a)

        def reorder(self, beams):
            if getattr(self, "full", False):
                raise PoolExhausted("full")
            return super().reorder(beams)
    lang = Breaks()
    with pytest.raises(RuntimeError, match="broken"):
        BeamLoop(lang).run([BeamRequest([1], 5, 3), BeamRequest([2], 5, 2)])
    assert not lang.text
    lang = Breaks()
    lang.full = True
    with pytest.raises(PoolExhausted):
        BeamLoop(lang).run([BeamRequest([1], 5, 3)])
    assert not lang.text

    class Nothing(Table):
        def select(self, slots, tokens, scores, start, k):
            n = len(start) - 1
            return [[-math.inf] * k] * n, [[-1] * k] * n, [[-1] * k] * n
    lang = Nothing()
    with pytest.raises(RuntimeError, match="no continuation"):
        BeamLoop(lang).run([BeamRequest([1], 5, 3)])
    assert not lang.text


# ------------------------------------------------------------------------------------------------------ adapters on the host
def test_adapter_files_and_names(tmp_path):
    from flashdecode_cuda_b200.weights import AdapterError, pair_up, read_adapter, write_adapter
    a, b = torch.randn(3, 10).bfloat16(), torch.randn(7, 3).bfloat16()
    folder = write_adapter(tmp_path / "x", {"model.layers.0.self_attn.q_proj": (a, b)}, alpha=6.0)
    pairs, scale = read_adapter(folder)
    assert scale == 2.0 and list(pairs) == ["model.layers.0.self_attn.q_proj"]
    assert torch.equal(pairs["model.layers.0.self_attn.q_proj"][0], a) and torch.equal(pairs["model.layers.0.self_attn.q_proj"][1], b)
    assert list(pair_up({"m.q.lora_A.default.weight": a, "m.q.lora_B.default.weight": b})) == ["m.q"]
    import json
    config = json.loads((folder / "adapter_config.json").read_text())
    for change in (dict(bias="all"), dict(use_dora=True), dict(modules_to_save=["lm_head"]), dict(r=4), dict(r=None), dict(lora_alpha=None),
                   dict(rank_pattern={"q_proj": 8})):
        (folder / "adapter_config.json").write_text(json.dumps({**config, **change}))
        with pytest.raises(AdapterError):
            read_adapter(folder)
    (folder / "adapter_config.json").write_text(json.dumps({**config, "use_rslora": True, "modules_to_save": None, "bias": "none"}))
    assert abs(read_adapter(folder)[1] - 6.0 / 3 ** 0.5) < 1e-12
    for bad in ({}, {"m.lora_A.weight": a}, {"m.lora_A.weight": a, "m.lora_B.weight": torch.zeros(7, 4)}, {"m.weight": a}):
        with pytest.raises(AdapterError):
            pair_up(bad)


def test_tokens_by_adapter():
    from types import SimpleNamespace

    from flashdecode_cuda_b200.engine.model import Model
    c = make(slots=8)
    slots = [c.admit(a) for a in (3, -1, 0, 3, -1)]
    fake = SimpleNamespace(adapters=SimpleNamespace(capacity=4))
    assert Model.adapter_segments(SimpleNamespace(adapters=None), c, slots, 5) == 0
    assert Model.adapter_segments(fake, c, [slots[1], slots[4]], 2) == 0
    n = Model.adapter_segments(fake, c, slots, 8)
    assert n == 4 and Model.adapter_segments(fake, c, slots[:1], 1) == 1
    got = Model.token_adapters(fake, c, slots, [2, 1, 1, 3, 2], 12, n).tolist()         # nine tokens and three of padding
    order, start, ids = got[:12], got[12:17], got[17:]
    assert sorted(order) == list(range(12)) and order[:6] == [3, 0, 1, 4, 5, 6]
    assert start == [0, 1, 6, 6, 6] and ids == [0, 3, -1, -1]


# ------------------------------------------------------------------------------------------------------ several stop tokens
class Ending(Table):
    """A language that likes to end: tokens 0, 1, ... of ``ends`` have the largest log-probabilities."""

    def __init__(self, ends, **kw):
        super().__init__(**kw)
        self.ends, self.live = ends, []

    def logp(self, text, adapter=-1):
        lp = super().logp(text, adapter)
        return torch.log_softmax(lp + 3.0 * (torch.arange(self.V) < self.ends), 0)

    def select(self, slots, tokens, scores, start, k):
        self.live.append(len(slots))
        assert all(hi - lo <= 64 for lo, hi in zip(start[:-1], start[1:])) and k <= 128
        return super().select(slots, tokens, scores, start, k)


def by_hand_uncut(lang, prompt, n, beams, stop):
    """The search over all candidates of every step."""
    live, done, counts = [(0.0, [])], [], []
    for step in range(1, n + 1):
        c = sorted(((s + float(lp), i, v, t) for i, (s, t) in enumerate(live) for v, lp in enumerate(lang.logp(prompt + t))),
                   key=lambda x: (-x[0], x[1], x[2]))
        live = []
        for rank, (s, _, v, t) in enumerate(c):
            if v in stop:
                if rank < beams:
                    done.append((s / step, t + [v], "stop"))
            elif len(live) < beams:
                live.append((s, t + [v]))
        counts.append(len(live))
        done = sorted(done, key=lambda h: -h[0])[:beams]
        if step == n:
            done = sorted(done + [(s / n, t, "length") for s, t in live], key=lambda h: -h[0])[:beams]
        elif len(done) == beams and max(s for s, _ in live) / n <= done[-1][0]:
            break
    return done, counts


@pytest.mark.parametrize("beams,n,V,ends", [(1, 6, 7, 2), (4, 6, 9, 3), (3, 5, 12, 6), (8, 4, 20, 7), (64, 3, 14, 3), (40, 3, 30, 5), (63, 3, 70, 65)])
def test_beams_go_on_whatever_the_number_of_stop_tokens(beams, n, V, ends):
    lang = Ending(ends, V=V, slots=beams)
    stop = tuple(range(ends)) * 2                # named twice: still so many
    (r,) = BeamLoop(lang).run([BeamRequest([1], n, beams, stop_token_ids=stop)])
    want, counts = by_hand_uncut(Ending(ends, V=V), [1], n, beams, stop)
    assert [h.tokens for h in r.hypotheses] == [t for _, t, _ in want]
    assert [h.finish_reason for h in r.hypotheses] == [why for _, _, why in want]
    assert lang.live == [1] + counts[:len(lang.live) - 1] and counts[-1] == min(beams, counts[-2] * (V - ends))


def test_more_stop_tokens_than_a_selection_has_room_for_are_refused():
    BeamRequest([1], 2, 64, stop_token_ids=tuple(range(64)))
    with pytest.raises(ValueError, match="64 beams and 65 stop tokens"):
        BeamRequest([1], 2, 64, stop_token_ids=tuple(range(65)))


# ------------------------------------------------------------------------------------------------- nothing to go on with
class Dies(Table):
    """After ``when`` tokens a text that begins with 9 has no candidate any more."""
    when = 3

    def select(self, slots, tokens, scores, start, k):
        S, R, T = super().select(slots, tokens, scores, start, k)
        for i, (lo, hi) in enumerate(zip(start[:-1], start[1:])):
            if hi > lo and self.text[slots[lo]][0] == 9 and len(self.text[slots[lo]]) >= self.when:
                S[i], R[i], T[i] = [-math.inf] * k, [-1] * k, [-1] * k
        return S, R, T


def test_a_request_without_continuations_does_not_end_the_others():
    from flashdecode_cuda_b200.engine.beam import NoContinuation
    lang = Dies(slots=9)
    reqs = [BeamRequest([1, 2], 4, 3, request_id=5), BeamRequest([9], 4, 2, request_id=6), BeamRequest([3], 6, 3, stop_token_ids=(2,), request_id=7)]
    with pytest.raises(NoContinuation, match="request 6: no continuation") as e:
        BeamLoop(lang, 6).run(reqs)
    results = e.value.results
    assert e.value.failed == [6] and [r.request_id for r in results] == [5, 6, 7] and results[1].hypotheses == [] and not lang.text
    for r, q in ((results[0], reqs[0]), (results[2], reqs[2])):
        assert [h.tokens for h in r.hypotheses] == [t for _, t, _ in by_hand(lang, q.prompt, q.max_new_tokens, q.num_beams, 1.0, q.stop_token_ids)]


def test_what_is_finished_stays_where_nothing_goes_on():
    lang = Dies()
    lp = lang.logp([9])
    stop = int(lp.argmax())
    lang.when = 2                                # the prompt and one more
    (r,) = BeamLoop(lang).run([BeamRequest([9], 6, 3, stop_token_ids=(stop,))])
    assert [(h.tokens, h.finish_reason) for h in r.hypotheses] == [([stop], "stop")] and abs(r.hypotheses[0].score - float(lp[stop])) < 1e-12
    assert not lang.text


def test_a_request_without_room_is_refused_before_others_have_run():
    lang = Table(slots=4)
    for bad in (BeamRequest([1], 3, 5, request_id=1), BeamRequest([1] * 5000, 3, 2, request_id=1)):
        with pytest.raises(ValueError, match="request 1: "):
            BeamLoop(lang).run([BeamRequest([1], 3, 4), bad])
    assert lang.calls == 0 and not lang.text
