"""Beam search's kernels: the selection over beams and vocabulary against 64-bit log-softmaxes, the copies of cache blocks and
states against indexing."""

import math

import pytest
import torch

from flashdecode_cuda_b200 import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"

# How far the kernel's normaliser may be from the exact one.  With p_i the softmax and d_i = max - x_i: every difference is off by
# at most d_i 2^-24, which moves the sum by at most 2^-24 sum p_i d_i <= 2^-24 ln V of itself (ln V < 12); every 32-bit exponential by two
# steps, 2^-22; the 32-bit sum of 16 of them by at most 5 roundings on the way up (pairs, fours, and three fours added in turn): 5 2^-24.
LSE_ERR = (12 + 4 + 5) * 2.0 ** -24


def select(logits, scores, start, k, **kw):
    R = len(start) - 1
    out = (torch.full((R, k), 7.0, device=DEV), torch.full((R, k), 7, dtype=torch.int32, device=DEV),
           torch.full((R, k), 7, dtype=torch.int32, device=DEV))
    K.beam_select(logits.to(DEV), scores.to(DEV), torch.tensor(start, dtype=torch.int32, device=DEV), *out, **kw)
    return [o.cpu() for o in out]


def plain(logits, scores, start, k):
    """(score, row, token) lists per request, k + 1 long so that the last gap can be seen."""
    out = []
    x = logits.double()
    x = x - x.amax(1, keepdim=True)                      # NaN where a row has no normaliser
    norm = x.exp().sum(1).log()
    V = x.shape[1]
    for lo, hi in zip(start[:-1], start[1:]):
        c = (scores[lo:hi].double() - norm[lo:hi])[:, None] + x[lo:hi]
        alive = torch.isfinite(scores[lo:hi].double() - norm[lo:hi])
        c = torch.where(alive[:, None] & (c > -math.inf), c, -math.inf).flatten()
        v, i = c.sort(descending=True, stable=True)
        out.append([(float(a), lo + int(j) // V, int(j) % V) for a, j in zip(v[:k + 1], i[:k + 1]) if float(a) > -math.inf])
    return out


def check(logits, scores, start, k):
    got = select(logits, scores, start, k)
    want = plain(logits, scores, start, k)
    for r, w in enumerate(want):
        # the order is only told where neighbours of different rows are further apart than both normalisers may be off
        for (a, ra, _), (b, rb, _) in zip(w, w[1:]):
            assert ra == rb or a - b > 2 * LSE_ERR or a == b, "choose other inputs: a near-tie between beams"
        w = w[:k]
        assert got[1][r].tolist() == [i for _, i, _ in w] + [-1] * (k - len(w))
        assert got[2][r].tolist() == [i for _, _, i in w] + [-1] * (k - len(w))
        for a, (b, _, _) in zip(got[0][r].tolist(), w):
            assert abs(a - b) <= LSE_ERR + 2.0 ** -24 * abs(b)
        assert all(v == -math.inf for v in got[0][r].tolist()[len(w):])


@pytest.mark.parametrize("V", [1, 5, 127, 128, 129, 1000, 4099, 50257, 151936])
@pytest.mark.parametrize("beams,k", [([1], 1), ([4], 8), ([3, 1, 5, 2], 10), ([17, 33, 64], 128)])
def test_selection(V, beams, k):
    if sum(beams) * V > 6_000_000:
        beams = [2, 3]
    g = torch.Generator().manual_seed(V + k)
    start = [0]
    for b in beams:
        start.append(start[-1] + b)
    n = start[-1]
    logits = 3.0 * torch.randn(n, V, generator=g)
    scores = -20.0 * torch.rand(n, generator=g)
    check(logits, scores, start, k)


def test_rows_of_wide_range():
    """Peaked rows, far offsets, large and tiny values."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(6, 3001, generator=g)
    x[1] *= 40
    x[2] += 5000.0
    x[3] -= 5000.0
    x[4] *= 1e-3
    x[5, 77] = 60.0
    check(x, torch.tensor([-1.0, -2.5, 0.0, -3.0, -100.0, -7.0]), [0, 2, 6], 16)


def test_masks_and_rows_without_candidates():
    g = torch.Generator().manual_seed(4)
    x = torch.randn(9, 777, generator=g)
    x[0, 5:] = -math.inf                                 # five candidates
    x[1] = -math.inf                                     # nothing left
    x[2, 3] = math.nan                                   # no normaliser
    x[3, 9] = math.inf
    x[4] = torch.finfo(torch.float32).min                # masked by the type's lowest value: uniform
    x[5, ::2] = torch.finfo(torch.float32).min
    s = torch.tensor([-1.0, -1.0, -1.0, -1.0, -3.0, -2.0, -math.inf, math.nan, -0.5])
    check(x, s, [0, 9], 20)
    check(x, s, [0, 2, 3, 4, 6, 8, 9], 20)               # among them requests whose rows all have no candidate
    got = select(x, s, [1, 4, 4, 6], 6)                  # a request without rows; rows of no request
    assert got[1][0].tolist() == [-1] * 6 and got[1][1].tolist() == [-1] * 6 and got[1][2][0] == 5
    assert got[0][1].tolist() == [-math.inf] * 6 and got[2][1].tolist() == [-1] * 6


@pytest.mark.parametrize("V", [50, 900, 20011, 151936])
def test_ties_go_to_the_lowest_row_and_token(V):
    x = torch.zeros(3, V)
    check(x, torch.zeros(3), [0, 3], 40)                 # all equal, in rows that are equal
    check(x, torch.tensor([-1.0, 0.0, 0.0]), [0, 3], 40)
    y = torch.zeros(2, V)
    y[:, V // 2] = 1.0
    y[:, V // 3] = 1.0
    y[1] = y[0]
    check(y, torch.zeros(2), [0, 2], 8)
    # few different values: the last taken ones are tied with thousands
    g = torch.Generator().manual_seed(V)
    z = torch.randint(0, 5, (1, V), generator=g).float().repeat(4, 1)
    check(z, torch.zeros(4), [0, 1, 4], 64)


def test_one_long_run_of_the_best():
    """The best lie side by side, in a few groups."""
    x = torch.linspace(0, 20, 30011)[None].repeat(2, 1)
    x[1] = x[1].flip(0) + 1e-3
    check(x, torch.tensor([0.0, -0.3]), [0, 1, 2], 100)
    check(x, torch.tensor([0.0, -0.30003]), [0, 2], 1)


def test_bad_ranges_are_reported_and_refused_calls_change_nothing():
    g = torch.Generator().manual_seed(5)
    x, s = torch.randn(70, 300, generator=g), torch.zeros(70)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    for start in ([0, 65], [-1, 2], [3, 1], [60, 71]):
        st.zero_()
        got = select(x, s, start, 4, status=st)
        assert int(st.item()) == K.STATUS_BAD_INDEX and got[1][0].tolist() == [-1] * 4
    st.zero_()
    select(x, s, [0, 64, 70], 4, status=st)
    assert int(st.item()) == 0


def test_two_streams_and_graph_replay():
    """Calls without a workspace of their own do not share one; a captured call reads what is there when it is replayed."""
    g = torch.Generator().manual_seed(6)
    a, b = torch.randn(4, 40000, generator=g).to(DEV), torch.randn(4, 40000, generator=g).to(DEV)
    start = torch.tensor([0, 4], dtype=torch.int32, device=DEV)
    sc = torch.zeros(4, device=DEV)
    want = [select(x.cpu(), torch.zeros(4), [0, 4], 8) for x in (a, b)]
    outs = [[torch.empty(1, 8, device=DEV), torch.empty(1, 8, dtype=torch.int32, device=DEV), torch.empty(1, 8, dtype=torch.int32, device=DEV)]
            for _ in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for x, o, st in zip((a, b), outs, streams):
            with torch.cuda.stream(st):
                K.beam_select(x, sc, start, *o)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(p.cpu(), q) for p, q in zip(o, w))
    x, o = a.clone(), outs[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.beam_select(x, sc, start, *o)
    for src, w in ((b, want[1]), (a, want[0])):
        x.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p.cpu(), q) for p, q in zip(o, w))


# ---------------------------------------------------------------------------------------------------------------- copies
@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float32, 64), (torch.bfloat16, 6), (torch.uint8, 5), (torch.bfloat16, 256)])
@pytest.mark.parametrize("planes,heads,size", [(1, 1, 1), (5, 3, 16), (4, 2, 64)])
def test_copy_blocks(dtype, dim, planes, heads, size):
    g = torch.Generator().manual_seed(planes + dim)
    pool = torch.randint(0, 200, (planes, 13, heads, size, dim), generator=g).to(dtype).to(DEV)
    src, dst = [3, 3, 7, 1, 9], [0, 12, 4, 5, 6]
    count = [size, 0, 1, max(1, size // 2), size - 1]
    want = pool.clone()
    for s, d, c in zip(src, dst, count):
        want[:, d, :, :c] = pool[:, s, :, :c]
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    up = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    K.copy_blocks(pool, up(src), up(dst), up(count), st)
    assert torch.equal(pool, want) and int(st.item()) == 0
    # outside the pool: skipped and reported, the others done
    for s, d, c in ((13, 0, 1), (-1, 0, 1), (2, 13, 1), (2, -1, 1), (2, 0, size + 1), (2, 0, -1)):
        st.zero_()
        want[:, 11, :, :size] = pool[:, 8, :, :size]
        K.copy_blocks(pool, up([s, 8]), up([d, 11]), up([c, size]), st)
        assert torch.equal(pool, want) and int(st.item()) == K.STATUS_BAD_INDEX


def test_copy_blocks_beyond_32_bits():
    """A pool whose offsets pass 2^31 elements."""
    pool = torch.zeros(2, 40, 4, 64, 128 * 1024, dtype=torch.uint8, device=DEV)        # 2 x 40 x 32 MB
    pool[1, 37, :, :5] = 3
    K.copy_blocks(pool, *(torch.tensor([v], dtype=torch.int32, device=DEV) for v in (37, 39, 4)))
    assert int(pool[1, 39].sum(dtype=torch.int64)) == 3 * 4 * 4 * 128 * 1024 and int(pool[0, 39].max()) == 0


@pytest.mark.parametrize("slots,shapes", [(4, [(3,)]), (9, [(2, 16, 8), (5, 7), (12,), (1,)]), (6, [(40000,)] * 70)])
def test_copy_states(slots, shapes):
    g = torch.Generator().manual_seed(slots)
    types = [torch.float32, torch.bfloat16, torch.uint8]
    states = [torch.randint(0, 200, (slots, *s), generator=g).to(types[i % 3]).to(DEV) for i, s in enumerate(shapes)]
    src, dst = [1, 1, 3], [0, 2, slots - 1] if slots > 4 else [0, 2, 2]
    if slots == 4:
        src, dst = [1, 3], [0, 2]
    want = [t.clone() for t in states]
    for w, t in zip(want, states):
        for s, d in zip(src, dst):
            w[d] = t[s]
    up = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    K.copy_states(states, up(src), up(dst), st)
    assert all(torch.equal(a, b) for a, b in zip(states, want)) and int(st.item()) == 0
    for s, d in ((slots, 0), (-1, 0), (1, slots), (1, -5)):
        st.zero_()
        K.copy_states(states, up([s]), up([d]), st)
        assert all(torch.equal(a, b) for a, b in zip(states, want)) and int(st.item()) == K.STATUS_BAD_INDEX
    K.copy_states(states, up([]), up([]), st)
    K.copy_states([], up([1]), up([0]), st)


def test_refusals():
    f = lambda *s: torch.zeros(*s, device=DEV)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)
    ok = dict(logits=f(4, 10), scores=f(4), row_start=i(3), out_scores=f(2, 3), out_rows=i(2, 3), out_tokens=i(2, 3))
    K.beam_select(**ok)
    for bad in (dict(logits=f(4, 10).bfloat16()), dict(scores=f(3)), dict(row_start=i(2)), dict(row_start=i(3).long()),
                dict(out_rows=i(2, 4)), dict(out_tokens=f(2, 3)), dict(logits=f(4, 20)[:, ::2]), dict(scores=f(4).cpu()),
                dict(out_scores=f(2, 129), out_rows=i(2, 129), out_tokens=i(2, 129)), dict(scratch=f(1)),
                dict(scratch=torch.zeros(3, dtype=torch.uint8, device=DEV))):
        with pytest.raises(K.KernelError):
            K.beam_select(**{**ok, **bad})
    with pytest.raises(K.KernelError):
        K.copy_blocks(f(2, 3, 4), i(1), i(1), i(1))
    with pytest.raises(K.KernelError):
        K.copy_blocks(f(2, 3, 4, 5, 6), i(1), i(2), i(1))
    with pytest.raises(K.KernelError):
        K.copy_blocks(f(2, 3, 4, 5, 6), i(1), i(1).long(), i(1))
    with pytest.raises(K.KernelError):
        K.copy_states([f(3, 4), f(4, 4)], i(1), i(1))
    with pytest.raises(K.KernelError):
        K.copy_states([f(3, 4).t()], i(1), i(1))
    with pytest.raises(K.KernelError):
        K.copy_states([f(3, 4).cpu()], i(1), i(1))


@pytest.mark.parametrize("form", [1, 2])
@pytest.mark.parametrize("V,beams,k", [(1, [3], 4), (130, [2, 0, 64, 1], 128), (4096, [4, 4], 8), (50257, [1, 8, 3], 16), (151936, [4], 8), (700, [1] * 150, 3)])
def test_both_forms(form, V, beams, k):
    K.beam_select_set_form(form)
    try:
        g = torch.Generator().manual_seed(V * 3 + k)
        start = [0]
        for b in beams:
            start.append(start[-1] + b)
        n = start[-1]
        x = 3.0 * torch.randn(n, V, generator=g)
        x[:, V // 2] = -math.inf
        check(x, -20.0 * torch.rand(n, generator=g), start, k)
        x.zero_()                                        # constant rows: the exact cuts
        check(x, torch.zeros(n), start, k)
    finally:
        K.beam_select_set_form(0)


def test_two_kernels_in_a_graph_and_a_workspace_of_the_callers():
    K.beam_select_set_form(2)
    try:
        g = torch.Generator().manual_seed(8)
        a, b = (torch.randn(6, 50257, generator=g).to(DEV) for _ in range(2))
        start, sc = torch.tensor([0, 2, 6], dtype=torch.int32, device=DEV), torch.zeros(6, device=DEV)
        want = [select(x.cpu(), torch.zeros(6), [0, 2, 6], 8) for x in (a, b)]
        outs = [torch.empty(2, 8, device=DEV)] + [torch.empty(2, 8, dtype=torch.int32, device=DEV) for _ in range(2)]
        scratch = torch.full((K.beam_select_scratch_bytes(6, 50257),), 255, dtype=torch.uint8, device=DEV)
        x = a.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            K.beam_select(x, sc, start, *outs, scratch=scratch)
        for src, w in ((b, want[1]), (a, want[0]), (b, want[1])):
            x.copy_(src)
            scratch.fill_(255)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p.cpu(), q) for p, q in zip(outs, w))
    finally:
        K.beam_select_set_form(0)


def test_largest_vocabulary_and_beyond():
    x = torch.zeros(2, K.BEAM_MAX_VOCAB)
    x[0, -1], x[1, -129], x[1, 70000] = 3.0, 2.0, 2.0
    check(x, torch.zeros(2), [0, 2], 4)
    with pytest.raises(K.KernelError, match="vocabulary"):
        select(torch.zeros(1, K.BEAM_MAX_VOCAB + 1), torch.zeros(1), [0, 1], 4)


@pytest.mark.parametrize("form", [1, 2])
@pytest.mark.parametrize("V,beams,k", [(335, [26, 25], 53), (1191, [29, 3, 64], 59), (14151, [22], 55), (16384, [40], 128), (16385, [30], 64), (324, [10] * 5, 21), (40000, [12, 13], 128)])
def test_many_rows_of_nearly_the_same_score(form, V, beams, k):
    # the best come from all rows: groups of many rows to read again, and more entries than are ranked at once
    K.beam_select_set_form(form)
    try:
        g = torch.Generator().manual_seed(V + 7 * k)
        start = [0]
        for b in beams:
            start.append(start[-1] + b)
        n = start[-1]
        x, scores = torch.randn(n, V, generator=g), 0.1 * torch.rand(n, generator=g)
        check(x, scores, start, k)
        check(torch.round(2.0 * x) / 2.0, scores, start, k)          # ties within every row
    finally:
        K.beam_select_set_form(0)


def test_exponentials_of_far_entries():
    """Rows of a few zeros and very many entries of one value d, at which the product d log2 e has the largest roundings: what a normaliser
    is off by is what exp(d) is.  Zeros where every warp begins, so that all of them count from 0.  Bound: exp(d) is off by 4 2^-24 of
    itself, the sum of 16 equal ones by one rounding (8 of them are exact, 12 not; 16 again), which is another."""
    V = 1 << 22
    x = torch.empty(1, V, device=DEV)
    zeros = (torch.arange(0, V, 2048 * 128)[:, None] + torch.arange(0, 64, 4) * 128).flatten().to(DEV)
    d = torch.linspace(-8.75, -8.4, 20001)
    log2e = torch.tensor(math.log2(math.e), dtype=torch.float64)
    off = (d * log2e.float()).double() - d.double() * log2e
    order = off.argsort()
    K.beam_select_set_form(1)
    try:
        for v in d[torch.cat([order[:12], order[-12:]])].tolist():
            x.fill_(v)
            x[0, zeros] = 0.0
            tail = (V - len(zeros)) * math.exp(v)
            lse = math.log(len(zeros) + tail)
            s = torch.tensor([lse])                              # the best candidate's score is then what both are off by
            got = select(x, s, [0, 1], 1)
            share = tail / (len(zeros) + tail)
            assert abs(float(got[0]) - (float(s) - lse)) <= 5 * 2.0 ** -24 * share + 2.0 ** -40, v
    finally:
        K.beam_select_set_form(0)


@pytest.mark.parametrize("form", [0, 1, 2])
@pytest.mark.parametrize("requests", [1, 5, 400])
def test_requests_without_any_row(form, requests):
    K.beam_select_set_form(form)
    try:
        st = torch.zeros(1, dtype=torch.int32, device=DEV)
        got = select(torch.zeros(0, 1000), torch.zeros(0), [0] * (requests + 1), 6, status=st)
        assert bool((got[0] == -math.inf).all()) and bool((got[1] == -1).all()) and bool((got[2] == -1).all()) and int(st.item()) == 0
        got = select(torch.zeros(0, 1000), torch.zeros(0), [0] * requests + [1], 6, status=st)
        assert bool((got[1] == -1).all()) and int(st.item()) == K.STATUS_BAD_INDEX
    finally:
        K.beam_select_set_form(0)


def test_outputs_over_inputs_or_each_other_are_refused():
    """Scores written over the ones that are read would be the natural thing to do with as many candidates as beams."""
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)
    x, scores, start = torch.randn(4, 100, device=DEV), torch.zeros(4, device=DEV), torch.tensor([0, 2, 4], dtype=torch.int32, device=DEV)
    both = torch.zeros(12, device=DEV)
    ints = both.view(torch.int32)
    for s, out in ((scores, (scores.view(2, 2), i(2, 2), i(2, 2))), (both[:4], (both[2:6].view(2, 2), i(2, 2), i(2, 2))),
                   (both[3:7], (torch.zeros(2, 2, device=DEV), i(2, 2), ints[:4].view(2, 2))),
                   (scores, (x[3, 90:94].view(2, 2), i(2, 2), i(2, 2))), (scores, (both[:4].view(2, 2), ints[3:7].view(2, 2), i(2, 2))),
                   (scores, (both[:4].view(2, 2), ints[4:8].view(2, 2), ints[7:11].view(2, 2)))):
        with pytest.raises(K.KernelError, match="share"):
            K.beam_select(x, s, start, *out)
    K.beam_select(x, both[:4], start, both[4:8].view(2, 2), ints[8:12].view(2, 2), i(2, 2))          # neighbours share nothing
    want = select(x.cpu(), torch.zeros(4), [0, 2, 4], 2)
    assert torch.equal(both[4:8].view(2, 2).cpu(), want[0]) and torch.equal(ints[8:12].view(2, 2).cpu(), want[1])
