"""Beam search over batches of unequal prompts.

davidjoyme/flashdecode-cuda decodes one greedy sequence per row (engine/model.py:315-329).  Here a request keeps up to
``num_beams`` unfinished sequences.  Each step feeds the last token of every beam of every request; the best continuations of each
request over its beams and the vocabulary are selected on the device (``kernels.beam_select``), and the beams that go on take over the
cached keys, values and states of the ones they continue (``PagedCache.reorder``).  Only the selected candidates come to the host.

The rules.  A request's candidates are taken in their order: one that ends with a stop token becomes a finished
hypothesis if it is among the first num_beams, any other becomes a beam until there are num_beams.  (With m stop tokens, num_beams
of the best (1 + m) num_beams candidates go on, so that many are asked for.)  A hypothesis of n new tokens scores
(sum of its tokens' log-probabilities) / n ** length_penalty.  The best num_beams hypotheses are kept.  A request ends when
num_beams are finished and no beam can still do better (with ``early_stopping``: when num_beams are finished), or at
``max_new_tokens``, where its beams become hypotheses too, or with what is finished when no continuation has a finite
log-probability.  A request that has nothing finished then fails: ``NoContinuation``, raised when all others are done.

The loop's decisions need no GPU: it talks to a ``BeamBackend``, which in tests is a fake.
"""

from __future__ import annotations

from dataclasses import dataclass, field
from typing import List, Optional, Sequence, Tuple

from .. import kernels as K


@dataclass
class BeamRequest:
    prompt: List[int]
    max_new_tokens: int
    num_beams: int = 4
    length_penalty: float = 1.0
    stop_token_ids: Tuple[int, ...] = ()
    early_stopping: bool = False
    adapter: int = -1
    request_id: int = 0

    def __post_init__(self):
        if len(self.prompt) == 0:
            raise ValueError("a request needs at least one prompt token")
        if self.max_new_tokens < 1:
            raise ValueError("max_new_tokens must be >= 1")
        if not (1 <= self.num_beams <= K.BEAM_MAX_ROWS):
            raise ValueError(f"num_beams must lie in 1..{K.BEAM_MAX_ROWS}, got {self.num_beams}")
        self.stops = len(set(self.stop_token_ids))
        if self.num_beams + self.stops > K.BEAM_MAX_CANDIDATES:
            raise ValueError(f"{self.num_beams} beams and {self.stops} stop tokens; {K.BEAM_MAX_CANDIDATES} in all are taken")

    def candidates(self, rows: int) -> int:
        """How many of the best candidates of ``rows`` beams hold all that may be taken: each beam has at most ``stops`` that end."""
        return max(2 * self.num_beams, self.num_beams + rows * self.stops)

    def cuts(self, rows: int) -> List[int]:
        """``rows`` beams in parts whose candidates one selection can give (one part but for many beams with several stop tokens)."""
        part = rows
        if self.candidates(rows) > K.BEAM_MAX_CANDIDATES:
            part = (K.BEAM_MAX_CANDIDATES - self.num_beams) // self.stops
        return [min(part, rows - at) for at in range(0, rows, part)]


@dataclass
class Hypothesis:
    tokens: List[int]
    score: float                     # normalised by the length
    finish_reason: str               # "stop" (a stop token, kept in tokens) or "length"


@dataclass
class BeamResult:
    request_id: int
    hypotheses: List[Hypothesis] = field(default_factory=list)      # best first

    @property
    def tokens(self) -> List[int]:
        return self.hypotheses[0].tokens


class NoContinuation(RuntimeError):
    """Requests for which no continuation had a finite log-probability before a hypothesis was finished.  ``results``: those of all
    requests; of these ones without hypotheses."""

    def __init__(self, failed: Sequence[int], results: List[BeamResult]):
        super().__init__(", ".join(f"request {i}" for i in failed) + ": no continuation has a finite log-probability")
        self.failed, self.results = list(failed), results


class BeamBackend:
    """What the loop needs from an engine."""

    def beam_capacity(self) -> Tuple[int, int]:
        """(slots, tokens) that a batch may hold when nothing else is live."""
        raise NotImplementedError

    def beam_tokens_held(self, request: BeamRequest) -> int:
        """Cache tokens that the request's beams may occupy in all."""
        raise NotImplementedError

    def admit(self, adapter: int = -1) -> int:
        raise NotImplementedError

    def release(self, slot: int) -> None:
        raise NotImplementedError

    def reorder(self, beams: Sequence[Tuple[Sequence[int], Sequence[int]]]) -> List[List[int]]:
        raise NotImplementedError

    def select(self, slots: Sequence[int], tokens: Sequence[Sequence[int]], scores: Sequence[float], row_start: Sequence[int],
               k: int) -> Tuple[List[List[float]], List[List[int]], List[List[int]]]:
        """Feed ``tokens[i]`` to ``slots[i]``; the k best continuations per request: scores, rows and tokens."""
        raise NotImplementedError


class _Beam:
    """An unfinished sequence: its new tokens as a chain that beams share."""
    __slots__ = ("slot", "score", "token", "before", "length")

    def __init__(self, slot: int, score: float, token: Optional[int], before: Optional["_Beam"]):
        self.slot, self.score, self.token, self.before = slot, score, token, before
        self.length = 0 if before is None else before.length + 1

    def tokens(self) -> List[int]:
        out, b = [], self
        while b.before is not None:
            out.append(b.token)
            b = b.before
        return out[::-1]


class _Live:
    def __init__(self, index: int, request: BeamRequest, slot: int):
        self.index, self.request = index, request
        self.slots = [slot]              # what the request holds in the cache
        self.beams = [_Beam(slot, 0.0, None, None)]
        self.finished: List[Hypothesis] = []

    def finish(self, beam: _Beam, reason: str) -> None:
        r = self.request
        h = Hypothesis(beam.tokens(), beam.score / beam.length ** r.length_penalty, reason)
        self.finished.append(h)
        self.finished.sort(key=lambda h: -h.score)               # stable: of equal ones the first found stays first
        del self.finished[r.num_beams:]

    def take(self, scores: List[float], parents: List[_Beam], tokens: List[int]) -> None:
        """The candidates in their order; ``beams`` are the unfinished sequences then, their slots still the parents'."""
        r, beams = self.request, []
        for i, (score, parent, token) in enumerate(zip(scores, parents, tokens)):
            beam = _Beam(parent.slot, score, token, parent)
            if token in r.stop_token_ids:
                if i < r.num_beams:
                    self.finish(beam, "stop")
            else:
                beams.append(beam)
                if len(beams) == r.num_beams:
                    break
        self.beams = beams

    def over(self) -> bool:
        r = self.request
        if not self.beams:
            return True
        if self.beams[0].length >= r.max_new_tokens:
            for b in self.beams:
                self.finish(b, "length")
            return True
        if len(self.finished) < r.num_beams:
            return False
        if r.early_stopping:
            return True
        # sums of log-probabilities only fall: the best a beam can come to is its sum, at the length that favours it most
        length = r.max_new_tokens if r.length_penalty > 0 else self.beams[0].length + 1
        return max(b.score for b in self.beams) / length ** r.length_penalty <= self.finished[-1].score


class BeamLoop:
    def __init__(self, backend: BeamBackend, max_batch: int = 64):
        """``max_batch``: beams (cache slots) that run together."""
        if max_batch < 1:
            raise ValueError("max_batch must be >= 1")
        self.backend, self.max_batch = backend, max_batch

    def _start(self, waiting: List[Tuple[int, BeamRequest]], slots: int, tokens: int) -> int:
        n = 0
        for _, r in waiting:
            need = self.backend.beam_tokens_held(r)
            if r.num_beams > slots or need > tokens:             # (each has room alone)
                break
            n, slots, tokens = n + 1, slots - r.num_beams, tokens - need
        return n

    def run(self, requests: Sequence[BeamRequest]) -> List[BeamResult]:
        """The requests' results in their order; ``NoContinuation`` has them too."""
        slots, tokens = self.backend.beam_capacity()
        slots = min(slots, self.max_batch)
        for r in requests:                                       # before any of them has run
            need = self.backend.beam_tokens_held(r)
            if r.num_beams > slots or need > tokens:
                raise ValueError(f"request {r.request_id}: {r.num_beams} beams of {len(r.prompt)} prompt + {r.max_new_tokens} new tokens "
                                 f"need {r.num_beams} slots and {need} cache tokens; there are {slots} and {tokens}")
        results = [BeamResult(r.request_id) for r in requests]
        waiting = list(enumerate(requests))
        while waiting:
            n = self._start(waiting, slots, tokens)
            batch, waiting = waiting[:n], waiting[n:]
            live: List[_Live] = []
            try:
                for i, r in batch:
                    live.append(_Live(i, r, self.backend.admit(r.adapter) if r.adapter >= 0 else self.backend.admit()))
                first = True
                while live:
                    live = self._step(live, first, results)
                    first = False
            finally:
                for l in live:                                   # only on an error
                    for s in l.slots:
                        self.backend.release(s)
        failed = [r.request_id for r in results if not r.hypotheses]
        if failed:
            raise NoContinuation(failed, results)
        return results

    def _step(self, live: List[_Live], first: bool, results: List[BeamResult]) -> List[_Live]:
        beams = [b for l in live for b in l.beams]
        start, first_part = [0], []
        for l in live:
            first_part.append(len(start) - 1)
            for n in l.request.cuts(len(l.beams)):
                start.append(start[-1] + n)
        first_part.append(len(start) - 1)
        feed = [list(l.request.prompt) for l in live] if first else [[b.token] for b in beams]
        k = min(K.BEAM_MAX_CANDIDATES, max(l.request.candidates(len(l.beams)) for l in live))
        scores, rows, tokens = self.backend.select([b.slot for b in beams], feed, [b.score for b in beams], start, k)
        still, moves = [], []
        for l, lo, hi in zip(live, first_part, first_part[1:]):
            found = [c for part in range(lo, hi) for c in zip(scores[part], rows[part], tokens[part]) if c[1] >= 0]
            if hi - lo > 1:
                found.sort(key=lambda c: -c[0])                  # stable: the lower rows first where scores tie
            l.take([c[0] for c in found], [beams[c[1]] for c in found], [c[2] for c in found])
            if l.over():
                l.beams = []
                results[l.index].hypotheses = l.finished
            else:
                still.append(l)
            moves.append((l.slots, [b.slot for b in l.beams]))
        placed = self.backend.reorder(moves)
        for l, row in zip(live, placed):
            l.slots = list(row)
            for b, s in zip(l.beams, row):
                b.slot = s
        return still
