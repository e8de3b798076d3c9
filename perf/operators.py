"""Operators for requests of one batch that differ: several beams each, low-rank adapters of their own.

A serving batch runs one step for everybody; what a request asks for beside that - keep several hypotheses, use an
adapter - must cost little more than its own bytes.  The cases stand for such steps.  The projections' sizes are those of the
dense presets (``config/presets``), the cache sizes too; the recurrent states are of the sizes that the Revelix comparison in
``bench.py`` has.  Vocabularies, contexts and batches reach from one short request to a full server.

``beam``    selection of the best continuations of every request over its beams and the whole vocabulary
``blocks``  the partly filled last cache blocks of sequences that go on as several beams, copied for all layers at once
``states``  the recurrent states of such sequences, copied between cache slots for all layers at once
``lora``    the low-rank terms of the tokens' adapters, added beside a shared projection
"""

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _beam(name, requests, most, ragged, vocab, k):
    return dict(name=name, op="beam", requests=requests, most=most, ragged=ragged, vocab=vocab, k=k)


def _blocks(name, planes, heads, block, dim, copies, dtype):
    return dict(name=name, op="blocks", planes=planes, heads=heads, block=block, dim=dim, copies=copies, dtype=dtype)


def _states(name, layers, heads, dk, dv, conv, slots, copies):
    return dict(name=name, op="states", layers=layers, heads=heads, dk=dk, dv=dv, conv=conv, slots=slots, copies=copies)


def _lora(name, dtype, seqs, shortest, longest, adapters, rank, slices, tiled, K, N):
    return dict(name=name, op="lora", dtype=dtype, seqs=seqs, shortest=shortest, longest=longest, adapters=adapters, rank=rank,
                slices=slices, tiled=tiled, K=K, N=N)


def listed():
    return [
        # one user, four beams: what a step of beam search adds to a decode step's latency
        _beam("beam-1x4", 1, 4, False, 151936, 8),
        # a few requests that keep unequal numbers of beams, an odd vocabulary
        _beam("beam-7-ragged", 7, 8, True, 50257, 16),
        # a full server of translations
        _beam("beam-64x8", 64, 8, False, 152064, 16),
        # four beams of one request of the smallest preset, three of which go on from another one
        _blocks("blocks-3", 56, 2, 64, 128, 3, "bf16"),
        # a full server of the largest preset, most beams replaced
        _blocks("blocks-90", 96, 8, 64, 128, 90, "bf16"),
        # the same for a recurrent model: one request
        _states("states-3", 6, 4, 128, 128, 4099, 8, 3),
        # ... and a full server
        _states("states-60", 24, 16, 128, 128, 12288, 96, 60),
        # one user with an adapter on the q/k/v projection: latency
        _lora("lora-1", "bf16", 1, 1, 1, 2, 16, 3, False, 1536, 2048),
        # a decode step of 48 requests of twelve adapters (some of none) on the gate/up projection
        _lora("lora-48", "bf16", 48, 1, 1, 12, 64, 2, True, 3584, 37888),
        # short prompts of four adapters packed into one step, on the output projection
        _lora("lora-5-prompts", "bf16", 5, 101, 700, 4, 32, 1, False, 3584, 3584),
        # long prompts, on the down projection of the largest preset
        _lora("lora-4-long", "bf16", 4, 1900, 2048, 3, 64, 1, False, 13824, 5120),
        # the 32-bit path: a decode step
        _lora("lora-24-fp32", "fp32", 24, 1, 1, 5, 16, 1, False, 8960, 1536),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["beam", "beam", "blocks", "states", "lora", "lora", "lora"])
    if op == "beam":
        most = _log(rng, 1, 32)
        vocab = _log(rng, 300, 160000)
        requests = _log(rng, 1, max(1, min(128, 64 * 8 * 152064 // (most * vocab))))
        c = _beam("", requests, most, rng.random() < 0.5, vocab, min(64, 2 * most + rng.randrange(3)))
    elif op == "blocks":
        planes, heads, dim = 2 * rng.randint(2, 48), rng.randint(1, 8), 16 * rng.randint(1, 16)
        block = rng.choice([16, 32, 48, 64, 128])
        copies = _log(rng, 1, max(1, min(120, 96 * 8 * 64 * 128 * 90 // (planes * heads * block * dim * 2))))
        c = _blocks("", planes, heads, block, dim, copies, rng.choice(["bf16", "fp32"]))
    elif op == "states":
        layers, heads, dk, dv = rng.randint(1, 24), rng.randint(1, 16), 16 * rng.randint(2, 8), 16 * rng.randint(2, 8)
        slots = _log(rng, 2, 96)
        c = _states("", layers, heads, dk, dv, _log(rng, 7, 20001), slots, _log(rng, 1, max(1, slots // 2)))
    else:
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        slices, tiled = rng.choice([(1, False), (1, False), (3, False), (2, True)])
        rank = rng.choice([4, 8, 16, 24, 32, 64] if dtype == "bf16" else [2, 8, 16, 33])
        K, N = 8 * _log(rng, 32, 1700), 8 * _log(rng, 24, 2300)
        if rng.random() < 0.2 and slices == 1:
            K, N = K + rng.randrange(1, 8), N + rng.randrange(1, 8)
        seqs = _log(rng, 1, 64)
        if rng.random() < 0.5:
            short = long = 1
        else:
            cap = 4 * 2048 * (13824 + 2 * 5120) // (K + 2 * N) // seqs
            if dtype == "fp32":
                cap //= 8
            long = _log(rng, 2, max(2, min(2048, cap)))
            short = rng.randint(1, long)
        c = _lora("", dtype, seqs, short, long, _log(rng, 1, 24), rank, slices, tiled, K, N)
    c.pop("name")
    return c


# ---------------------------------------------------------------------------------------------------------------- inputs

def _shape(case):
    """What belongs to whom, in plain numbers: the same for every seed."""
    rng = random.Random(",".join(f"{k}={v}" for k, v in sorted(case.items()) if k != "name"))
    if case["op"] == "beam":
        beams = [rng.randint(1, case["most"]) if case["ragged"] else case["most"] for _ in range(case["requests"])]
        return dict(start=np.concatenate([[0], np.cumsum(beams)]).astype(np.int32))
    if case["op"] == "blocks":
        return dict(count=[rng.randint(1, case["block"]) for _ in range(case["copies"])])
    lengths = [rng.randint(case["shortest"], case["longest"]) for _ in range(case["seqs"])]
    # some requests use no adapter (-1), unless there is but one
    who = [rng.randrange(case["adapters"]) if case["seqs"] == 1 or rng.random() > 0.15 else -1 for _ in lengths]
    ranks = [case["rank"] if i == 0 else rng.randint(max(1, case["rank"] // 4), case["rank"]) for i in range(case["adapters"])]
    token = np.repeat(np.asarray(who, dtype=np.int32), lengths)
    # the tokens in the order of their adapters, and where each adapter's begin
    order = np.argsort(token, kind="stable").astype(np.int32)
    ids, first = np.unique(token[order], return_index=True)
    start = np.concatenate([first, [len(token)]]).astype(np.int32)
    return dict(token=token, order=order, ids=ids.astype(np.int32), start=start, ranks=ranks)


def _places(count, copies, seed):
    """Where copies come from and go to: no place twice among the latter, none of them among the former."""
    rng = random.Random(seed * 1000003 + 17)
    ids = list(range(count))
    rng.shuffle(ids)
    return [rng.choice(ids[copies:]) for _ in range(copies)], ids[:copies]


def _column_slices(case):
    """Which of the packed projections each tile of 8 columns belongs to: q, k and v one after another in unequal shares, or gate
    and up in turns."""
    tiles = case["N"] // 8
    if case["slices"] == 1:
        return None
    if case["tiled"]:
        return np.arange(tiles, dtype=np.uint8) % case["slices"]
    bounds = [tiles - 2 * (tiles // 8), tiles - tiles // 8]
    return np.searchsorted(bounds, np.arange(tiles), side="right").astype(np.uint8)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 7919 + 3)

    def up(v, dtype=torch.int32):
        return torch.as_tensor(np.asarray(v)).to(device=DEV, dtype=dtype)

    if case["op"] == "beam":
        h = _shape(case)
        n, V, k, R = int(h["start"][-1]), case["vocab"], case["k"], case["requests"]
        logits = torch.randn(n, V, generator=g, device=DEV) * 3.0
        # a stop token that may not come yet, and some banned ones
        logits[:, torch.randint(0, V, (3,), generator=g, device=DEV)] = -math.inf
        scores = -20.0 * torch.rand(n, generator=g, device=DEV)
        most = case["most"]
        rows = np.full((R, most), -1, dtype=np.int64)
        for r in range(R):
            rows[r, :h["start"][r + 1] - h["start"][r]] = np.arange(h["start"][r], h["start"][r + 1])
        return dict(op="beam", logits=logits, scores=scores, start=up(h["start"]), rows=up(rows, torch.int64), k=k,
                    out=(torch.empty(R, k, device=DEV), torch.empty(R, k, dtype=torch.int32, device=DEV),
                         torch.empty(R, k, dtype=torch.int32, device=DEV)))
    if case["op"] == "blocks":
        src, dst = _places(2 * case["copies"] + 3, case["copies"], seed)
        pool = torch.randn(case["planes"], 2 * case["copies"] + 3, case["heads"], case["block"], case["dim"], generator=g, device=DEV,
                           dtype=DTYPES[case["dtype"]])
        return dict(op="blocks", pool=pool, src=up(src), dst=up(dst), count=up(_shape(case)["count"]))
    if case["op"] == "states":
        slots = case["slots"]
        src, dst = _places(slots, case["copies"], seed)
        states = []
        for _ in range(case["layers"]):
            states.append(torch.randn(slots, case["heads"], case["dk"], case["dv"], generator=g, device=DEV))
            states.append(torch.randn(slots, case["conv"], generator=g, device=DEV))
        return dict(op="states", states=states, src=up(src), dst=up(dst))
    h = _shape(case)
    dt, K, N, R, S, E = DTYPES[case["dtype"]], case["K"], case["N"], case["rank"], case["slices"], case["adapters"]
    T = len(h["token"])
    x = torch.randn(T, K, generator=g, device=DEV, dtype=dt)
    y = torch.randn(T, N, generator=g, device=DEV, dtype=dt)
    # an adapter of a smaller rank than the widest has zeros behind it
    ranks = up(h["ranks"])
    inside = torch.arange(R, device=DEV)[None, :] < ranks[:, None]
    a = torch.randn(E, S, R, K, generator=g, device=DEV, dtype=dt) * K ** -0.5 * inside[:, None, :, None]
    b = torch.randn(E, N, R, generator=g, device=DEV, dtype=dt) * R ** -0.5 * inside[:, None, :]
    cols = _column_slices(case)
    return dict(op="lora", x=x, y=y, a=a.to(dt).view(E, S * R, K), b=b.to(dt), scale=0.5 + torch.rand(E, generator=g, device=DEV), ranks=ranks,
                cols=None if cols is None else up(cols, torch.uint8), order=up(h["order"]), start=up(h["start"]), ids=up(h["ids"]),
                token=up(h["token"], torch.int64), runs=list(zip(h["ids"].tolist(), h["start"][:-1].tolist(), h["start"][1:].tolist())),
                slices=S, out=torch.empty(T, N, device=DEV, dtype=dt))


# ------------------------------------------------------------------------------------------------------------ plain forms

def _plain_beam(s):
    """64 bits: which of two candidates of different beams comes first hangs on the difference of two long sums."""
    x = s["logits"].double()
    top = x.amax(1, keepdim=True)
    lse = top + (x - top).exp().sum(1, keepdim=True).log()
    cand = s["scores"].double()[:, None] + x - lse
    V, rows = cand.shape[1], s["rows"]
    R, B = rows.shape
    flat = torch.where((rows >= 0)[:, :, None], cand[rows.clamp(min=0)], -math.inf).view(R, B * V)
    k = min(s["k"], B * V)
    # everything that reaches the k-th value (more than k where values tie), the lowest places first
    best = flat.topk(k, dim=1).values
    least = best[:, -1:]
    place = torch.arange(B * V, device=flat.device)
    above = (flat > least).sum(1, keepdim=True)
    tied = flat == least
    taken = (flat > least) | (tied & (tied.cumsum(1) <= k - above))
    at = torch.where(taken, place, B * V).topk(k, dim=1, largest=False, sorted=True).values
    value, by = flat.gather(1, at).sort(dim=1, descending=True, stable=True)
    at = at.gather(1, by)
    found = value > -math.inf
    out_s, out_r, out_t = (o.fill_(v) for o, v in zip(s["out"], (-math.inf, -1, -1)))
    out_s[:, :k] = torch.where(found, value, -math.inf).float()
    out_r[:, :k] = torch.where(found, rows.gather(1, at // V), -1).int()
    out_t[:, :k] = torch.where(found, at % V, -1).int()
    return dict(scores=out_s, rows=out_r, tokens=out_t)


def _plain_blocks(s):
    pool, src, dst = s["pool"], s["src"].long(), s["dst"].long()
    inside = torch.arange(pool.shape[3], device=pool.device)[None, :] < s["count"][:, None]
    pool.index_copy_(1, dst, torch.where(inside[None, :, None, :, None], pool.index_select(1, src), pool.index_select(1, dst)))
    return pool


def _plain_states(s):
    src, dst = s["src"].long(), s["dst"].long()
    for st in s["states"]:
        st.index_copy_(0, dst, st.index_select(0, src))
    return s["states"]


def _plain_lora(s):
    x, y, a, b, S = s["x"], s["y"], s["a"], s["b"], s["slices"]
    R, N = b.shape[2], b.shape[1]
    cols = None if s["cols"] is None else s["cols"].long().repeat_interleave(8)
    if x.shape[0] <= 64:
        # few tokens: each with its own matrices
        i = s["token"].clamp(min=0)
        h = torch.bmm(a[i].float(), x.float()[:, :, None]).view(-1, S, R)
        if cols is None:
            d = torch.bmm(b[i].float(), h[:, 0, :, None])[:, :, 0]
        else:
            d = torch.zeros(x.shape[0], N, device=x.device)
            for j in range(S):
                d = torch.where(cols == j, torch.bmm(b[i].float(), h[:, j, :, None])[:, :, 0], d)
        d = torch.where((s["token"] >= 0)[:, None], d * s["scale"][i][:, None], 0.0)
        return (y.float() + d).to(y.dtype)
    out = y.clone()
    for e, lo, hi in s["runs"]:
        if e < 0:
            continue
        t = s["order"][lo:hi].long()
        h = x[t].float() @ a[e].float().t()
        w = b[e].float()
        if cols is None:
            d = h @ w.t()
        else:
            d = torch.zeros(len(t), N, device=x.device)
            for j in range(S):
                d[:, cols == j] = h[:, j * R:(j + 1) * R] @ w[cols == j].t()
        out[t] = (y[t].float() + s["scale"][e] * d).to(y.dtype)
    return out


# ------------------------------------------------------------------------------------------------- the framework's calls

def _own(s):
    from flashdecode_cuda_b200 import kernels as K
    if s["op"] == "beam":
        scores, rows, tokens = s["out"]
        K.beam_select(s["logits"], s["scores"], s["start"], scores, rows, tokens)
        return dict(scores=scores, rows=rows, tokens=tokens)
    if s["op"] == "blocks":
        K.copy_blocks(s["pool"], s["src"], s["dst"], s["count"])
        return s["pool"]
    if s["op"] == "states":
        K.copy_states(s["states"], s["src"], s["dst"])
        return s["states"]
    K.lora_add(s["x"], s["a"], s["b"], s["scale"], s["ranks"], s["order"], s["start"], s["ids"], s["y"], s["out"], col_slice=s["cols"],
               slices=s["slices"])
    return s["out"]


def run(state):
    if own:
        return _own(state)
    return {"beam": _plain_beam, "blocks": _plain_blocks, "states": _plain_states, "lora": _plain_lora}[state["op"]](state)


def work(case):
    op = case["op"]
    if op == "beam":
        n = int(_shape(case)["start"][-1])
        return {"bytes": n * case["vocab"] * 4 + n * 4 + case["requests"] * case["k"] * 12, "flops": 4 * n * case["vocab"]}
    if op == "blocks":
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": 2 * case["planes"] * case["heads"] * case["dim"] * size * sum(_shape(case)["count"]), "flops": 0}
    if op == "states":
        return {"bytes": 2 * case["copies"] * case["layers"] * 4 * (case["heads"] * case["dk"] * case["dv"] + case["conv"]), "flops": 0}
    h, size, T = _shape(case), 2 if case["dtype"] == "bf16" else 4, 0
    weights = flops = tokens = 0
    for e, n in zip(h["ids"].tolist(), np.diff(h["start"]).tolist()):
        T += n
        if e >= 0:
            one = h["ranks"][e] * (case["slices"] * case["K"] + case["N"])
            tokens, weights, flops = tokens + n, weights + one, flops + 2 * n * one
    return {"bytes": size * (tokens * case["K"] + 2 * T * case["N"] + weights), "flops": flops}


# -------------------------------------------------------------------------------------------------- from the definitions

def exact(case, seed):
    if case["op"] in ("blocks", "states"):
        return None                                    # copied, not computed
    s = prepare(case, seed)
    if case["op"] == "beam":
        found = []
        start = s["start"].tolist()
        for lo, hi in zip(start[:-1], start[1:]):
            p = torch.log_softmax(s["logits"][lo:hi].double(), dim=1) + s["scores"][lo:hi].double()[:, None]
            v = p.flatten().sort(descending=True, stable=True).values[:s["k"]]
            found.append(torch.nn.functional.pad(v, (0, s["k"] - v.numel()), value=-math.inf))
        return dict(scores=torch.stack(found), rows=None, tokens=None)
    R, S, N = s["b"].shape[2], s["slices"], s["b"].shape[1]
    out = s["y"].double()
    column = np.zeros(N, dtype=np.int64) if s["cols"] is None else np.repeat(_column_slices(case).astype(np.int64), 8)
    places = torch.as_tensor(column, device=DEV)[:, None] * R + torch.arange(R, device=DEV)[None, :]       # [N, R]
    for e in range(case["adapters"]):
        t = torch.nonzero(s["token"] == e)[:, 0]
        if t.numel():
            whole = torch.zeros(N, S * R, device=DEV, dtype=torch.float64).scatter_(1, places, s["b"][e].double())
            out[t] += s["scale"][e].double() * (s["x"][t].double() @ (whole @ s["a"][e].double()).t()) if N * s["x"].shape[1] <= 1 << 25 \
                else s["scale"][e].double() * ((s["x"][t].double() @ s["a"][e].double().t()) @ whole.t())
    return out
