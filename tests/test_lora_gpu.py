"""Low-rank adapters beside a shared projection, against 64-bit products."""

import pytest
import torch

from flashdecode_cuda_b200 import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def plan(token):
    """order, start, ids of the tokens' adapters (a list, -1: none)."""
    t = torch.tensor(token, dtype=torch.int32)
    order = torch.argsort(t, stable=True).int()
    ids, n = torch.unique_consecutive(t[order.long()], return_counts=True)
    start = torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)]).int()
    return order.to(DEV), start.to(DEV), ids.int().to(DEV)


def make(dtype, T, Kd, N, E, R, S=1, tiled=False, seed=0, ranks=None):
    g = torch.Generator().manual_seed(seed)
    dt = DT[dtype]
    ranks = torch.tensor([max(1, R - 3 * e) for e in range(E)] if ranks is None else ranks, dtype=torch.int32)
    inside = torch.arange(R)[None] < ranks[:, None]
    x = torch.randn(T, Kd, generator=g).to(dt)
    a = (torch.randn(E, S, R, Kd, generator=g) * Kd ** -0.5 * inside[:, None, :, None]).to(dt).view(E, S * R, Kd)
    b = (torch.randn(E, N, R, generator=g) * R ** -0.5 * inside[:, None]).to(dt)
    y = torch.randn(T, N, generator=g).to(dt)
    scale = 0.5 + torch.rand(E, generator=g)
    cols = None
    if S > 1:
        tiles = torch.arange(N // 8)
        cols = (tiles % S if tiled else torch.clamp(tiles * (S + 1) // (N // 8), max=S - 1)).to(torch.uint8)
    return dict(x=x, a=a, b=b, scale=scale, ranks=ranks, y=y), cols, S


def expected(d, cols, S, token):
    """The exact result and, with absolute values, what the errors are counted against."""
    N, R = d["b"].shape[1:]
    col = torch.zeros(N, dtype=torch.int64) if cols is None else cols.long().repeat_interleave(8)
    out, size, hsize = d["y"].double().clone(), torch.zeros(d["y"].shape, dtype=torch.float64), torch.zeros(d["y"].shape, dtype=torch.float64)
    for t, e in enumerate(token):
        if e < 0:
            continue
        a, b, x = d["a"][e].double(), d["b"][e].double(), d["x"][t].double()
        h, ha = (a @ x).view(S, R), (a.abs() @ x.abs()).view(S, R)
        sc = float(d["scale"][e].double())
        out[t] += sc * (b * h[col]).sum(1)
        size[t] = sc * (b.abs() * ha[col]).sum(1)                 # |B| |A| |x|
        hsize[t] = sc * (b.abs() * h[col].abs()).sum(1)           # |B| |h|
    return out, size, hsize


def tolerance(dtype, d, out, size, hsize):
    """Per element.  32-bit sums: a chain of at most K / 32 + 64 additions for A x (a lane's share of a row, the lanes, the chunks
    and the CTAs of a cluster) and R + 8 for B h, each off by 2^-24 of what is added up in absolute values.  bfloat16: h as two
    numbers of 8 bits each is off by 2^-17, and the result is rounded once, 2^-8."""
    Kd, R = d["x"].shape[1], d["b"].shape[2]
    tol = (Kd / 32 + 64 + R + 8) * 2.0 ** -24 * size + 2.0 ** -23 * out.abs()
    if dtype == "bfloat16":
        tol = tol + 2.0 ** -16 * hsize + 2.0 ** -8 * (out.abs() + tol)
    return tol + 1e-30


def run(d, cols, S, token, in_place=False, **kw):
    u = {k: v.to(DEV) for k, v in d.items()}
    order, start, ids = plan(token)
    out = u["y"] if in_place else torch.full_like(u["y"], 9.0)
    K.lora_add(u["x"], u["a"], u["b"], u["scale"], u["ranks"], order, start, ids, u["y"], None if in_place else out,
               col_slice=None if cols is None else cols.to(DEV), slices=S, **kw)
    return out.cpu()


def check(dtype, T, Kd, N, E, R, S=1, tiled=False, token=None, seed=0, ranks=None, in_place=False):
    d, cols, S = make(dtype, T, Kd, N, E, R, S, tiled, seed, ranks)
    if token is None:
        g = torch.Generator().manual_seed(seed + 1)
        token = torch.randint(-1, E, (T,), generator=g).tolist()
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = run(d, cols, S, token, in_place, status=st)
    assert int(st.item()) == 0
    want, size, hsize = expected(d, cols, S, token)
    err = (got.double() - want).abs()
    tol = tolerance(dtype, d, want, size, hsize)
    assert bool((err <= tol).all()), float((err / tol).max())
    none = [t for t, e in enumerate(token) if e < 0]
    assert torch.equal(got[none], d["y"][none])
    return got


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T,Kd,N,E,R", [
    (1, 64, 64, 1, 4), (1, 1536, 2048, 2, 16), (3, 8, 8, 3, 1), (17, 100, 52, 2, 3), (33, 1001, 333, 4, 7), (5, 1, 1, 1, 1),
    (64, 3584, 1024, 9, 64), (40, 520, 4104, 5, 24), (2, 2048, 4096, 2, 256), (16, 192, 320, 1, 8), (130, 256, 264, 3, 16),
    (300, 640, 776, 2, 32), (129, 1024, 512, 1, 64), (513, 136, 1032, 4, 40), (257, 96, 200, 3, 128), (400, 72, 80, 2, 12)])
def test_plain(dtype, T, Kd, N, E, R):
    check(dtype, T, Kd, N, E, R)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("S,tiled", [(3, False), (2, True), (4, True)])
@pytest.mark.parametrize("T,Kd,N,R", [(1, 256, 384, 16), (21, 1536, 2048, 16), (9, 72, 64, 5), (140, 320, 640, 24), (300, 128, 1088, 64), (6, 40, 32, 128)])
def test_packed_projections(dtype, S, tiled, T, Kd, N, R):
    check(dtype, T, Kd, N, 3, R, S, tiled)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T", [7, 200])
def test_in_place_and_out_of_place_agree(dtype, T):
    token = [(i * 7) % 4 - 1 for i in range(T)]
    a = check(dtype, T, 512, 648, 3, 16, token=token)
    b = check(dtype, T, 512, 648, 3, 16, token=token, in_place=True)
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T", [12, 260])
def test_ranks_of_zero_and_one(dtype, T):
    check(dtype, T, 264, 136, 4, 16, ranks=[16, 0, 1, 15])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_runs_of_prompts(dtype):
    """Sequences one after another, as prompts come; one adapter in two places; one without."""
    check(dtype, 700, 384, 520, 3, 32, token=[2] * 150 + [-1] * 60 + [0] * 257 + [2] * 1 + [1] * 232)


def test_a_token_does_not_depend_on_the_others_in_float32():
    d, cols, S = make("float32", 40, 1500, 900, 3, 12)
    token = [i % 3 for i in range(40)]
    whole = run(d, cols, S, token)
    for t in (0, 13, 39):
        one = {**d, "x": d["x"][t:t + 1], "y": d["y"][t:t + 1]}
        assert torch.equal(run(one, cols, S, token[t:t + 1])[0], whole[t])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("offset", [1, 2, 4])
def test_tensors_that_begin_anywhere(dtype, offset):
    d, cols, S = make(dtype, 150, 64, 72, 2, 16)
    token = [i % 2 for i in range(150)]
    want = run(d, cols, S, token)
    u = {}
    for k, v in d.items():
        if k in ("x", "a", "b", "y"):
            flat = torch.zeros(v.numel() + offset, dtype=v.dtype, device=DEV)
            u[k] = flat[offset:].view(v.shape)
            u[k].copy_(v)
        else:
            u[k] = v.to(DEV)
    order, start, ids = plan(token)
    out = torch.zeros(150 * 72 + offset, dtype=DT[dtype], device=DEV)[offset:].view(150, 72)
    K.lora_add(u["x"], u["a"], u["b"], u["scale"], u["ranks"], order, start, ids, u["y"], out)
    exact, size, hsize = expected(d, cols, S, token)
    assert bool(((out.cpu().double() - exact).abs() <= tolerance(dtype, d, exact, size, hsize)).all())
    assert bool(((want.double() - exact).abs() <= tolerance(dtype, d, exact, size, hsize)).all())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T", [6, 200])
def test_tokens_behind_the_last_segment_and_empty_segments(dtype, T):
    d, cols, S = make(dtype, T, 128, 96, 3, 8)
    u = {k: v.to(DEV) for k, v in d.items()}
    used = T - 2
    order = torch.arange(T, dtype=torch.int32, device=DEV)
    up = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    start, ids = up([0, 0, used // 2, used // 2, used, used, used]), up([1, 2, 0, 1, -1, 0])
    out = torch.full_like(u["y"], 5.0)
    K.lora_add(u["x"], u["a"], u["b"], u["scale"], u["ranks"], order, start, ids, u["y"], out)
    token = [2] * (used // 2) + [1] * (used - used // 2)
    want, size, hsize = expected(d, cols, S, token + [-1] * 2)
    got = out.cpu()
    assert bool(((got.double() - want).abs() <= tolerance(dtype, d, want, size, hsize))[:used].all())
    assert bool((got[used:] == 5.0).all())
    # no segment at all: nothing is written
    out.fill_(5.0)
    K.lora_add(u["x"], u["a"], u["b"], u["scale"], u["ranks"], order, up([0]), up([]), u["y"], out)
    assert bool((out == 5.0).all())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T", [6, 200])
def test_what_does_not_exist_is_skipped_and_reported(dtype, T):
    d, cols, S = make(dtype, T, 128, 96, 3, 8)
    u = {k: v.to(DEV) for k, v in d.items()}
    up = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    base = list(range(T))
    h = T // 2
    for order, start, ids in ((base, [0, h, T], [3, 1]), (base, [0, h, T], [-2, 1]), ([T] + base[1:], [0, h, T], [0, 1]),
                              ([-1] + base[1:], [0, h, T], [0, 1]), (base, [0, h, T + 1], [0, 1]), (base, [0, h, h - 1], [0, 1]),
                              (base, [-3, h, T], [0, 1])):
        st = torch.zeros(1, dtype=torch.int32, device=DEV)
        out = torch.full_like(u["y"], 5.0)
        K.lora_add(u["x"], u["a"], u["b"], u["scale"], u["ranks"], up(order), up(start), up(ids), u["y"], out, status=st)
        assert int(st.item()) == K.STATUS_BAD_INDEX, (start, ids)
    # the good segment of a call with a bad one is computed
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = torch.full_like(u["y"], 5.0)
    K.lora_add(u["x"], u["a"], u["b"], u["scale"], u["ranks"], up(base), up([0, h, T]), up([7, 1]), u["y"], out, status=st)
    want, size, hsize = expected(d, cols, S, [-1] * h + [1] * (T - h))
    got = out.cpu()
    assert bool(((got.double() - want).abs() <= tolerance(dtype, d, want, size, hsize))[h:].all()) and bool((got[:h] == 5.0).all())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T", [5, 300])
def test_infinities_stay_with_their_token(dtype, T):
    d, cols, S = make(dtype, T, 256, 264, 2, 16)
    token = [i % 2 for i in range(T)]
    want = run(d, cols, S, token)
    d["x"][3, 7] = float("inf")
    got = run(d, cols, S, token)
    others = [t for t in range(T) if t != 3]
    assert torch.equal(got[others], want[others]) and not bool(torch.isfinite(got[3].float()).any())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T", [4, 200])
def test_other_streams_and_graph_replay(dtype, T):
    d, cols, S = make(dtype, T, 512, 768, 3, 16)
    token = [i % 3 for i in range(T)]
    want = run(d, cols, S, token)
    u = {k: v.to(DEV) for k, v in d.items()}
    order, start, ids = plan(token)
    outs = [torch.zeros_like(u["y"]) for _ in range(2)]
    torch.cuda.synchronize()
    for o, s in zip(outs, (torch.cuda.Stream(), torch.cuda.Stream())):
        with torch.cuda.stream(s):
            for _ in range(4):
                K.lora_add(u["x"], u["a"], u["b"], u["scale"], u["ranks"], order, start, ids, u["y"], o)
    torch.cuda.synchronize()
    assert all(torch.equal(o.cpu(), want) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.lora_add(u["x"], u["a"], u["b"], u["scale"], u["ranks"], order, start, ids, u["y"], outs[0])
    # another step: the same numbers of tokens and segments, other adapters
    token2 = [(i + 1) % 3 for i in range(T)]
    want2 = run(d, cols, S, token2)
    o2, s2, i2 = plan(token2)
    order.copy_(o2), start.copy_(s2), ids.copy_(i2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0].cpu(), want2)


def test_refusals():
    f = lambda *s: torch.zeros(*s, device=DEV)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)
    ok = dict(x=f(4, 16), a=f(2, 8, 16), b=f(2, 24, 8), scale=f(2), ranks=i(2), order=i(4), start=i(2), ids=i(1), y=f(4, 24))
    K.lora_add(**ok)
    for bad in (dict(x=f(4, 16).bfloat16()), dict(x=f(4, 16).half(), a=f(2, 8, 16).half(), b=f(2, 24, 8).half(), y=f(4, 24).half()),
                dict(a=f(2, 8, 17)), dict(a=f(2, 9, 16)), dict(a=f(3, 8, 16)), dict(y=f(4, 25)), dict(out=f(3, 24)),
                dict(scale=f(3)), dict(scale=f(2).bfloat16()), dict(ranks=i(2).long()), dict(order=i(5)), dict(start=i(1)), dict(start=i(3)),
                dict(ids=i(1).float()), dict(slices=2), dict(slices=2, a=f(2, 16, 16)), dict(col_slice=torch.zeros(4, dtype=torch.uint8, device=DEV)),
                dict(col_slice=i(3)), dict(x=f(16, 4).t()), dict(scale=f(2).cpu()), dict(a=f(2, 257, 16), b=f(2, 24, 257)),
                dict(slices=5, a=f(2, 40, 16), col_slice=torch.zeros(3, dtype=torch.uint8, device=DEV)),
                dict(slices=4, a=f(2, 4 * 136, 16), b=f(2, 24, 136), col_slice=torch.zeros(3, dtype=torch.uint8, device=DEV))):
        with pytest.raises(K.KernelError):
            K.lora_add(**{**ok, **bad})


@pytest.mark.parametrize("form", [1, 2])
@pytest.mark.parametrize("T,Kd,N,E,R,S,tiled", [
    (1, 64, 64, 1, 16, 1, False), (128, 64, 128, 1, 16, 1, False), (130, 72, 136, 1, 8, 1, False), (300, 1000, 264, 3, 24, 1, False),
    (129, 4096, 1024, 2, 64, 1, False), (257, 640, 520, 2, 128, 1, False), (140, 328, 384, 2, 16, 3, False), (260, 512, 648, 3, 64, 3, False),
    (135, 704, 512, 2, 40, 2, True), (270, 128, 136, 2, 96, 2, True), (20, 2048, 4096, 5, 32, 2, True), (900, 256, 1288, 4, 16, 4, True),
    (129, 8, 8, 1, 8, 1, False)])
def test_both_forms(form, T, Kd, N, E, R, S, tiled):
    K.lora_set_form(form)
    try:
        check("bfloat16", T, Kd, N, E, R, S, tiled)
        check("bfloat16", T, Kd, N, E, R, S, tiled, token=[(i // 150) % E for i in range(T)], in_place=True, seed=3)
    finally:
        K.lora_set_form(0)


@pytest.mark.parametrize("form", [1, 2])
@pytest.mark.parametrize("T", [300, 1500])
def test_both_forms_on_other_streams_and_in_graphs(form, T):
    K.lora_set_form(form)
    try:
        d, cols, S = make("bfloat16", T, 512, 776, 3, 32, 2, True)
        tokens = [[(i // 70) % 4 - 1 for i in range(T)], [2 - (i // 200) % 3 for i in range(T)]]
        wants = [run(d, cols, S, t) for t in tokens]
        u = {k: v.to(DEV) for k, v in d.items()}
        plans = [[p.clone() for p in plan(t)] for t in tokens]
        # two graphs that share nothing, and whose replays overlap
        graphs, outs, cs = [], [], cols.to(DEV)
        for p in plans:
            out, graph = torch.zeros_like(u["y"]), torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                K.lora_add(u["x"], u["a"], u["b"], u["scale"], u["ranks"], *p, u["y"], out, col_slice=cs, slices=S)
            graphs.append(graph), outs.append(out)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        for _ in range(4):
            for graph, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o.cpu(), w) for o, w in zip(outs, wants))
    finally:
        K.lora_set_form(0)


def test_rows_that_lie_here_and_there():
    """Prompts' tiles whose tokens are no neighbours: one by one, in runs of odd lengths, backwards."""
    T = 1100
    g = torch.Generator().manual_seed(11)
    K.lora_set_form(2)
    try:
        for token in (torch.randint(0, 2, (T,), generator=g).tolist(), [(i // 37) % 2 for i in range(T)], [(i // 300) % 3 - 1 for i in range(T)]):
            check("bfloat16", T, 456, 328, 2, 24, token=token)
        d, cols, S = make("bfloat16", T, 456, 328, 2, 24)
        u = {k: v.to(DEV) for k, v in d.items()}
        up = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
        out = torch.zeros_like(u["y"])
        K.lora_add(u["x"], u["a"], u["b"], u["scale"], u["ranks"], up(list(range(T - 1, -1, -1))), up([0, 500, T]), up([1, 0]), u["y"], out)
        want, size, hsize = expected(d, cols, S, [0] * (T - 500) + [1] * 500)
        assert bool(((out.cpu().double() - want).abs() <= tolerance("bfloat16", d, want, size, hsize)).all())
    finally:
        K.lora_set_form(0)


def test_an_output_over_the_input_is_refused():
    x = torch.zeros(3, 16, device=DEV)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)
    with pytest.raises(K.KernelError, match="out is x"):
        K.lora_add(x, torch.zeros(1, 4, 16, device=DEV), torch.zeros(1, 16, 4, device=DEV), torch.zeros(1, device=DEV), i(1), i(3), i(2), i(1),
                   torch.zeros(3, 16, device=DEV), x)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_an_output_that_shares_memory_in_part_is_refused(dtype):
    dt = DT[dtype]
    z, i = (lambda *s: torch.zeros(*s, device=DEV, dtype=dt)), (lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV))
    both = z(7, 16)
    call = lambda x, y, out: K.lora_add(x, z(1, 4, 16), z(1, 16, 4), torch.zeros(1, device=DEV), i(1), i(3), i(2), i(1), y, out)
    for x, y, out in [(z(3, 16), both[:3], both[1:4]), (z(3, 16), both[1:4], both[:3]), (both[:3], z(3, 16), both[2:5]), (both[4:], both[2:5], both[2:5])]:
        with pytest.raises(K.KernelError, match="shares memory"):
            call(x, y, out)
    both.fill_(2.0)
    call(both[:3], both[3:6], both[3:6])                         # neighbours share nothing
    call(z(3, 16), both[:3], both[3:6])
    assert bool((both == 2).all())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("E", [7, 8, 14, 15, 17, 33, 34])
def test_one_token_of_each_of_many_adapters(dtype, E):
    # one token to a tile, as many clusters as run at once and one more
    check(dtype, E, 1024, 2056, E, 8, token=list(range(E)))
    check(dtype, E, 4096, 520, E, 16, token=list(range(E)), in_place=True)


@pytest.mark.parametrize("T", [15 * 128, 15 * 128 + 1, 33 * 128, 33 * 128 + 1])
def test_as_many_large_tiles_as_run_at_once_and_one_more(T):
    K.lora_set_form(2)
    try:
        check("bfloat16", T, 520, 136, 1, 8, token=[0] * T)
        check("bfloat16", T, 520, 136, 3, 8, token=[min(t * 4 // T, 2) for t in range(T)], in_place=True, seed=2)
    finally:
        K.lora_set_form(0)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("N", [1, 7, 8, 12, 136, 4872])
@pytest.mark.parametrize("form", [1, 2])
def test_rows_without_an_adapter_come_out_as_they_are(dtype, N, form):
    # every token but a few, here and there; rows on and off the 16-byte boundary; an adapter of rank zero with a scale that is no number
    T, Kd, R = 413, 64, 8
    for off in (0, 1):
        g = torch.Generator().manual_seed(N + off)
        y = torch.randn(T * N + off, generator=g).to(DT[dtype]).to(DEV)[off:].view(T, N)
        out = torch.full((T * N + off,), 9.0, dtype=DT[dtype], device=DEV)[off:].view(T, N)
        token = torch.randint(-1, 2, (T,), generator=g).tolist()
        x = torch.randn(T, Kd, generator=g).to(DT[dtype]).to(DEV)
        K.lora_set_form(form)
        try:
            K.lora_add(x, torch.zeros(2, R, Kd, dtype=DT[dtype], device=DEV), torch.zeros(2, N, R, dtype=DT[dtype], device=DEV),
                       torch.tensor([1.0, float("inf")], device=DEV), torch.tensor([R, 0], dtype=torch.int32, device=DEV), *plan(token), y, out)
        finally:
            K.lora_set_form(0)
        assert torch.equal(out, y)


@pytest.mark.parametrize("Kd,N,R,S", [(1536, 512, 16, 1), (4100, 304, 12, 2), (260, 100, 33, 1), (600, 1030, 4, 1), (96, 300, 8, 1)])
def test_a_float32_token_has_the_same_bits_in_any_step(Kd, N, R, S):
    T = 1300
    d, cols, S = make("float32", T, Kd, N, 3, R, S)
    token = [(t * 5) % 4 - 1 for t in range(T)]
    want = run(d, cols, S, token)
    for some in ([0], [5, 1299, 700], list(range(3, 560)), list(range(0, 1300, 2))):
        part = dict(d, x=d["x"][some], y=d["y"][some])
        assert torch.equal(run(part, cols, S, [token[t] for t in some]), want[some])


@pytest.mark.parametrize("tokens", ["neighbours", "here and there"])
@pytest.mark.parametrize("Kd,C", [(64, 1), (192, 2), (520, 8)])
@pytest.mark.parametrize("kept", [1, 2])
def test_waits_that_run_out_in_tiles_of_128(kept, Kd, C, tokens):
    """One copy never leaves.  For the sums over K: its whole cluster stores nothing, whichever of its CTAs waited.  For b: the columns
    before it are right, those from there on are left as they were.  The status says so, and the next call is right."""
    T, N, R = 300, 20 * 128, 16
    d, cols, S = make("bfloat16", T, Kd, N, 2, R)
    token = [i * 2 // T for i in range(T)] if tokens == "neighbours" else [(i * 5 // 3) % 2 for i in range(T)]
    K.lora_set_form(2)
    try:
        want = run(d, cols, S, token)
        st = torch.zeros(1, dtype=torch.int32, device=DEV)
        K.tc_test_hook(wait_ns=1_000_000, skip_last=kept)
        got = run(d, cols, S, token, status=st)
        assert int(st.item()) == K.STATUS_WAIT_TIMEOUT
        done = 0 if kept == 1 else (20 - C) * 128                # of 20 tiles each CTA's last is not computed
        assert torch.equal(got[:, :done], want[:, :done]) and bool((got[:, done:] == 9.0).all())
        K.tc_test_hook()
        st.zero_()
        assert torch.equal(run(d, cols, S, token, status=st), want) and int(st.item()) == 0
    finally:
        K.tc_test_hook()
        K.lora_set_form(0)


@pytest.mark.parametrize("form", [0, 2])
@pytest.mark.parametrize("T", [3, 2600])
def test_more_rows_of_b_than_a_copy_can_name(T, form):
    """2^31 rows of b (34 GB): steps of any length are taken, by the form that can name them."""
    E, N, R, Kd = 1 << 17, 1 << 14, 8, 64
    g = torch.Generator().manual_seed(T)
    x, y = torch.randn(T, Kd, generator=g).bfloat16().to(DEV), torch.randn(T, N, generator=g).bfloat16().to(DEV)
    a, b = torch.empty(E, R, Kd, dtype=torch.bfloat16, device=DEV), torch.empty(E, N, R, dtype=torch.bfloat16, device=DEV)
    for e in (0, E - 1):
        a[e], b[e] = (torch.randn(R, Kd, generator=g) / 8).bfloat16(), torch.randn(N, R, generator=g).bfloat16()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = torch.empty_like(y)
    K.lora_set_form(form)
    try:
        K.lora_add(x, a, b, torch.ones(E, device=DEV), torch.full((E,), R, dtype=torch.int32, device=DEV), i32(list(range(T))),
                   i32([0, T // 2, T]), i32([E - 1, 0]), y, out, status=st)
    finally:
        K.lora_set_form(0)
    assert int(st.item()) == 0
    for t in (0, T // 2, T - 1):
        e = E - 1 if t < T // 2 else 0
        small = dict(x=x[t:t + 1].cpu(), a=a[e:e + 1].cpu(), b=b[e:e + 1].cpu(), y=y[t:t + 1].cpu(), scale=torch.ones(1))
        want, size, hsize = expected(small, None, 1, [0])
        assert bool(((out[t:t + 1].cpu().double() - want).abs() <= tolerance("bfloat16", small, want, size, hsize)).all())


@pytest.mark.parametrize("dtype,form", [("float32", 0), ("bfloat16", 0), ("bfloat16", 1), ("bfloat16", 2)])
@pytest.mark.parametrize("T", [5, 16, 300])
def test_an_infinite_sum_gives_what_the_formula_gives(dtype, form, T):
    """Adapters of rank 1: A x is +inf or -inf for a token with an infinity, and so is every output, with B's sign; NaN where B is zero."""
    Kd, N, R = 256, 264, 8
    d, cols, S = make(dtype, T, Kd, N, 2, R, ranks=[1, 1])
    d["b"][:, 5] = 0.0
    d["x"][2, 7], d["x"][T - 1, 30] = float("inf"), -float("inf")
    if form == 0 and dtype == "bfloat16":
        Kd = 255                                                 # sizes for the CUDA cores
        d["x"], d["a"] = d["x"][:, :Kd].contiguous(), d["a"][:, :, :Kd].contiguous()
    token = [i % 2 for i in range(T)]
    K.lora_set_form(form)
    try:
        got = run(d, cols, S, token)
    finally:
        K.lora_set_form(0)
    for t in (2, T - 1):
        e = token[t]
        h = (d["a"][e, 0].double() * d["x"][t].double()).sum()
        want = d["y"][t].double() + float(d["scale"][e]) * d["b"][e, :, 0].double() * h
        assert bool(h.isinf()) and bool(want[5].isnan()) and int(want.isinf().sum()) == N - 1
        assert torch.equal(got[t].double().nan_to_num(nan=0.5, posinf=1.0, neginf=-1.0), want.nan_to_num(nan=0.5, posinf=1.0, neginf=-1.0))


@pytest.mark.parametrize("dtype,form", [("float32", 0), ("bfloat16", 1), ("bfloat16", 2)])
def test_the_same_call_gives_the_same_bits(dtype, form):
    """Sums over a cluster's CTAs are added in the order of their ranks."""
    d, cols, S = make(dtype, 700, 4104, 1032, 3, 40)
    token = [(i // 90) % 3 for i in range(700)]
    K.lora_set_form(form)
    try:
        first = run(d, cols, S, token)
        assert all(torch.equal(run(d, cols, S, token), first) for _ in range(10))
    finally:
        K.lora_set_form(0)
