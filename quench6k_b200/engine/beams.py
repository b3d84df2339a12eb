"""Beam search above the step function.

A prompt runs once; its cache and states are then copied to the other beams (a page has one owner: a search holds a prompt's pages once for
each of its beams).  Every further step runs one token of each beam
of all prompts as one batch (a decode step like any other: it replays the recording of its size), chooses the best continuations
of each prompt on the device (ops.beam_select), and lets the beams that die go on from ones that live (ModelRunner.reorder): only
the positions since the two parted are copied.  A beam that lives stays where it is.

(The reference has no beam search: its sampler works on one sequence, crates/cli/src/flint.rs:339-353.)
"""
from __future__ import annotations

import itertools
import math
from dataclasses import dataclass, field
from typing import List, Optional, Sequence, Tuple

import torch

from .. import ops
from ..cache import OutOfPages, OutOfSlots
from ..sampling.params import BeamParams
from .batch import StepEntry
from .runner import ModelRunner

STOP, LENGTH = "stop", "length"


@dataclass
class BeamOutput:
    tokens: List[int]
    score: float                          # the sum of log-probabilities over the length to the power length_penalty
    logprob: float                        # the sum itself
    finish_reason: str


@dataclass
class _Search:
    """One prompt's beams.  Beam b is request rids[b] of the runner, its tokens and the sum of their log-probabilities."""
    prompt: List[int]
    rids: List[Tuple]
    tokens: List[List[int]] = field(default_factory=list)
    sums: List[float] = field(default_factory=list)
    same: List[List[int]] = field(default_factory=list)       # positions below same[a][b] of beams a and b hold the same in the cache
    ended: List[BeamOutput] = field(default_factory=list)     # best first, at most `width`
    done: bool = False


def _worth(total: float, length: int, params: BeamParams) -> float:
    return total / float(length) ** params.length_penalty


def choose(search: _Search, candidates: Sequence[Tuple[float, int, int]], params: BeamParams, cached: int):
    """One step of one prompt on the host: candidates (sum, beam, token) in descending order become ended continuations and the
    next beams.  Returns (parents, first): for every beam the one it goes on from and the first cached position in which they
    differ; `cached` positions are held.  A beam without a continuation of its own has the sum -infinity from here on."""
    W, stops = params.width, set(params.stop_tokens)
    live: List[Tuple[float, int, int]] = []
    for rank, (total, beam, token) in enumerate(candidates):
        if total == -math.inf or len(live) == W:
            break
        tokens = search.tokens[beam] + [token]
        if token in stops:
            if rank < W:                                    # a continuation that ends must be among the best `width` to count
                search.ended.append(BeamOutput(tokens, _worth(total, len(tokens), params), total, STOP))
        else:
            live.append((total, beam, token))
    search.ended.sort(key=lambda o: -o.score)               # (stable: among equals the earlier one)
    del search.ended[W:]
    # the first continuation of a beam stays in its place, the others take the places of beams that die
    parents, places, late = [-1] * W, [None] * W, []
    for c in live:
        if parents[c[1]] < 0:
            parents[c[1]], places[c[1]] = c[1], c
        else:
            late.append(c)
    free = [b for b in range(W) if parents[b] < 0]
    for b, c in zip(free, late):
        parents[b], places[b] = c[1], c
    for b in range(W):
        if parents[b] < 0:
            parents[b] = b
    first = [search.same[b][p] if p != b else cached for b, p in enumerate(parents)]
    search.same = [[cached if parents[a] == parents[b] else search.same[parents[a]][parents[b]] for b in range(W)] for a in range(W)]
    search.tokens = [search.tokens[c[1]] + [c[2]] if c else search.tokens[b] + [0] for b, c in enumerate(places)]
    search.sums = [c[0] if c else -math.inf for c in places]
    # nothing that still lives can become worth more: a sum only falls, and is divided by at most the longest length (or, with a
    # penalty below zero, by the present one)
    best, length = max(search.sums), len(search.tokens[0])
    if best == -math.inf:
        search.done = True
    elif len(search.ended) == W:
        reach = _worth(best, params.max_tokens if params.length_penalty > 0 else length, params)
        search.done = params.early_stopping or search.ended[-1].score >= reach
    if not search.done and length >= params.max_tokens:
        for total, tokens in zip(search.sums, search.tokens):
            if total > -math.inf:
                search.ended.append(BeamOutput(tokens, _worth(total, len(tokens), params), total, LENGTH))
        search.ended.sort(key=lambda o: -o.score)
        del search.ended[W:]
        search.done = True
    return parents, first


class BeamSearch:
    _numbers = itertools.count()

    def __init__(self, runner: ModelRunner, max_batch_tokens: int = 2048):
        self.runner, self.max_batch_tokens = runner, max_batch_tokens

    # ------------------------------------------------------------------ room
    def _pages(self, length: int, params: BeamParams) -> List[int]:
        """Pages that a prompt's beams hold at most, for each cache group."""
        m, longest = self.runner.manager, length + params.max_tokens
        portion = min(length, self.max_batch_tokens)
        out = []
        for g in m.groups:
            held = longest if g.kind == "full" else min(longest, g.window + portion)
            out.append(params.width * (-(-held // m.page_size) + (0 if g.kind == "full" else 2)))
        return out

    def _batches(self, prompts, params: BeamParams):
        """The prompts in order, as many at a time as the slots and the pages hold."""
        m = self.runner.manager
        room, slots = [p.num_free for p in m.pools], m.slots.num_free // params.width
        if slots == 0:
            raise OutOfSlots(f"{params.width} beams need as many request slots, {m.slots.num_free} are free")
        batch, used = [], [0] * len(room)
        for i, p in enumerate(prompts):
            need = self._pages(len(p), params)
            if any(n > r for n, r in zip(need, room)):
                raise OutOfPages(f"{params.width} beams of {len(p)} + {params.max_tokens} tokens need {need} pages of the cache groups, {room} are free")
            if batch and (len(batch) == slots or any(u + n > r for u, n, r in zip(used, need, room))):
                yield batch
                batch, used = [], [0] * len(room)
            batch.append(i)
            used = [u + n for u, n in zip(used, need)]
        if batch:
            yield batch

    # ------------------------------------------------------------------ running
    def run(self, prompts: Sequence[Sequence[int]], params: BeamParams) -> List[List[BeamOutput]]:
        params.validate()
        vocab = self.runner.vocab_size
        prompts = [[int(t) for t in p] for p in prompts]
        for p in prompts:
            if not p:
                raise ValueError("a prompt needs at least one token")
            if any(not 0 <= t < vocab for t in p):
                raise ValueError(f"a token id outside 0..{vocab - 1}")
        results: List[Optional[List[BeamOutput]]] = [None] * len(prompts)
        for batch in list(self._batches(prompts, params)):
            searches = [_Search(prompts[i], [("beam", next(self._numbers), b) for b in range(params.width)]) for i in batch]
            try:
                self._run(searches, params)
            finally:
                for s in searches:
                    for rid in s.rids:
                        if self.runner.has_request(rid):
                            self.runner.end_request(rid)
            for i, s in zip(batch, searches):
                results[i] = s.ended[:params.num_return or params.width]
        return results

    def _select(self, logits: torch.Tensor, sums: List[List[float]], params: BeamParams):
        """[[(sum, beam, token)]] of each search's best continuations, best first."""
        width = len(sums[0])
        count = min(params.width * (1 + len(set(params.stop_tokens))), width * self.runner.vocab_size)
        scores = torch.tensor(sums, dtype=torch.float32).to(logits.device, non_blocking=True)
        values, beams, tokens = ops.beam_select(logits, scores, count)
        host = torch.stack((values.view(torch.int32), beams, tokens)).cpu()          # one copy
        values = host[0].view(torch.float32).tolist()
        return [list(zip(v, b, t)) for v, b, t in zip(values, host[1].tolist(), host[2].tolist())]

    def _start(self, s: _Search, params: BeamParams) -> torch.Tensor:
        """Runs the prompt; the logits of its last token [1, V]."""
        r, logits = self.runner, None
        r.add_request(s.rids[0])
        for at in range(0, len(s.prompt), self.max_batch_tokens):
            part = s.prompt[at:at + self.max_batch_tokens]
            logits = r.step([StepEntry(s.rids[0], part, [len(part) - 1] if at + len(part) == len(s.prompt) else [])])
        return logits

    def _fork(self, searches: List[_Search], params: BeamParams) -> None:
        """The other beams take over what the first one holds."""
        r = self.runner
        for s in searches:
            for rid in s.rids[1:]:
                r.add_request(rid)
                for at in range(0, len(s.prompt), self.max_batch_tokens):
                    r.assume_cached(rid, min(self.max_batch_tokens, len(s.prompt) - at))
        if params.width > 1:
            zeros = [[0] * params.width for _ in searches]
            r.reorder([s.rids for s in searches], zeros, zeros)

    def _run(self, searches: List[_Search], params: BeamParams) -> None:
        W, r = params.width, self.runner
        for s in searches:
            logits = self._start(s, params)
            s.tokens, s.sums = [[] for _ in range(W)], [0.0] + [-math.inf] * (W - 1)
            s.same = [[len(s.prompt)] * W for _ in range(W)]
            # all beams go on from the prompt: their places are given out as they come
            choose(s, [(v, 0, t) for v, _, t in self._select(logits, [[0.0]], params)[0]], params, len(s.prompt))
        live = [s for s in searches if not s.done]
        self._fork(live, params)
        while live:
            entries = [StepEntry(rid, [toks[-1]], [0]) for s in live for rid, toks in zip(s.rids, s.tokens)]
            logits = r.step(entries)
            picked = self._select(logits, [s.sums for s in live], params)
            moves = [choose(s, c, params, len(s.prompt) + len(s.tokens[0])) for s, c in zip(live, picked)]
            on = [(s, m) for s, m in zip(live, moves) if not s.done]
            for s in live:
                if s.done:
                    for rid in s.rids:
                        r.end_request(rid)
            if on:
                r.reorder([s.rids for s, _ in on], [m[0] for _, m in on], [m[1] for _, m in on])
            live = [s for s, _ in on]
