"""The host's half of beam search without a GPU: the choice of one step over a cache that is only copied where `choose` says so,
against a search that keeps whole sequences; the room that a search asks for; the options' checks."""
import math
import random

import pytest

from quench6k_b200 import BeamParams
from quench6k_b200.cache import GroupSpec, OutOfPages, OutOfSlots, PyCacheManager
from quench6k_b200.engine.beams import BeamSearch, _Search, choose


def logprobs(tokens, vocab, seed):
    """A model of sorts: log-probabilities of the next token that depend on the last three tokens."""
    r = random.Random(repr((seed, tokens[-3:])))
    w = [r.gauss(0.0, 1.5) for _ in range(vocab)]
    z = math.log(sum(math.exp(x) for x in w))
    return [x - z for x in w]


def plain_search(prompt, vocab, seed, params):
    """Whole sequences, nothing shared: [(tokens, worth, reason)] best first."""
    worth = lambda total, n: total / n ** params.length_penalty
    beams, ended = [([], 0.0)], []
    while True:
        every = sorted(((total + lp, b, t) for b, (toks, total) in enumerate(beams) for t, lp in enumerate(logprobs(prompt + toks, vocab, seed))),
                       key=lambda c: (-c[0], c[1], c[2]))
        after = []
        for rank, (total, b, t) in enumerate(every):
            if len(after) == params.width:
                break
            toks = beams[b][0] + [t]
            if t in params.stop_tokens:
                if rank < params.width:
                    ended.append((toks, worth(total, len(toks)), "stop"))
            else:
                after.append((toks, total))
        ended = sorted(ended, key=lambda e: -e[1])[:params.width]
        beams = after
        if not beams:
            return ended
        n = len(beams[0][0])
        reach = worth(max(b[1] for b in beams), params.max_tokens if params.length_penalty > 0 else n)
        if len(ended) == params.width and (params.early_stopping or ended[-1][1] >= reach):
            return ended
        if n >= params.max_tokens:
            return sorted(ended + [(toks, worth(total, n), "length") for toks, total in beams], key=lambda e: -e[1])[:params.width]


def shared_search(prompt, vocab, seed, params):
    """The same through `choose`, with a cache of a list for each beam: a step appends the token that a beam ran, a beam that goes
    on from another takes over its positions from `first` on and no others."""
    W = params.width
    s = _Search(prompt, [("b", b) for b in range(W)], [[] for _ in range(W)], [0.0] + [-math.inf] * (W - 1), [[len(prompt)] * W for _ in range(W)])
    count = W * (1 + len(params.stop_tokens))

    def best(rows):
        every = sorted(((s.sums[b] + lp, b, t) for b, row in enumerate(rows) for t, lp in enumerate(row)), key=lambda c: (-c[0], c[1], c[2]))
        return every[:count]

    choose(s, best([logprobs(prompt, vocab, seed)]), params, len(prompt))
    caches = [list(prompt) for _ in range(W)]
    copied = 0
    while not s.done:
        for b in range(W):
            caches[b].append(s.tokens[b][-1])
            if s.sums[b] > -math.inf:
                assert caches[b] == prompt + s.tokens[b], "a beam runs on a cache that is not its own"
        parents, first = choose(s, best([logprobs(c, vocab, seed) for c in caches]), params, len(caches[0]))
        before = [list(c) for c in caches]
        for b, (p, f) in enumerate(zip(parents, first)):
            if p != b:
                caches[b][f:] = before[p][f:]
                copied += len(before[p]) - f
    return [(o.tokens, o.score, o.finish_reason) for o in s.ended], copied


@pytest.mark.parametrize("early", [False, True])
@pytest.mark.parametrize("penalty", [1.0, 0.0, 2.0, -0.5])
@pytest.mark.parametrize("width,vocab,stops", [(1, 7, [0]), (2, 5, []), (3, 9, [1, 4]), (4, 12, [2]), (8, 20, [0]), (4, 3, [1]), (5, 2, [0])])
def test_search_that_copies_only_where_beams_part(width, vocab, stops, penalty, early):
    for seed in range(6):
        params = BeamParams(width=width, max_tokens=9, stop_tokens=stops, length_penalty=penalty, early_stopping=early)
        prompt = [random.Random(seed).randrange(vocab) for _ in range(3)]
        got, _ = shared_search(prompt, vocab, seed, params)
        want = plain_search(prompt, vocab, seed, params)
        assert [(t, r) for t, _, r in got] == [(t, r) for t, _, r in want]
        assert all(abs(a[1] - b[1]) < 1e-9 for a, b in zip(got, want))


def test_less_is_copied_than_the_sequences_hold():
    params = BeamParams(width=4, max_tokens=30)
    _, copied = shared_search(list(range(10)), 15, 1, params)
    assert 0 < copied < 4 * sum(range(30)) / 4


def test_one_token():
    params = BeamParams(width=3, max_tokens=1)
    got, copied = shared_search([1, 2], 8, 0, params)
    assert copied == 0 and got == plain_search([1, 2], 8, 0, params) and all(r == "length" for _, _, r in got)


def test_options_that_are_refused():
    for bad in (dict(width=0), dict(width=33), dict(max_tokens=0), dict(num_return=5), dict(num_return=0), dict(width=32, stop_tokens=[1, 2, 3, 4])):
        with pytest.raises(ValueError):
            BeamParams(**bad).validate()
    BeamParams(width=32, stop_tokens=[1, 2, 3]).validate()


class _Runner:
    """Just what the room's count reads."""

    def __init__(self, pages, slots, groups=(GroupSpec("full"),)):
        self.manager = PyCacheManager(list(groups), 4, [pages] * len(groups), slots)
        self.vocab_size = 50


def test_powers_of_a_length_that_are_no_numbers_are_refused():
    for bad in (float("inf"), float("nan"), 400.0, -400.0):
        with pytest.raises(ValueError, match="length_penalty"):
            BeamParams(length_penalty=bad, max_tokens=64).validate()
    BeamParams(length_penalty=400.0, max_tokens=1).validate()


def test_prompts_run_as_many_at_a_time_as_fit():
    # two beams of 6 + 4 tokens: 3 pages each
    params = BeamParams(width=2, max_tokens=4)
    batches = lambda pages, slots, n: list(BeamSearch(_Runner(pages, slots))._batches([[1] * 6] * n, params))
    assert batches(100, 8, 5) == [[0, 1, 2, 3], [4]]
    assert batches(12, 100, 5) == [[0, 1], [2, 3], [4]]
    assert batches(6, 2, 2) == [[0], [1]]
    with pytest.raises(OutOfPages):
        batches(5, 8, 1)
    with pytest.raises(OutOfSlots):
        batches(100, 1, 1)


def test_a_window_needs_fewer_pages():
    windows = _Runner(100, 8, (GroupSpec("sliding", 8), GroupSpec("full"), GroupSpec("chunked", 8)))
    need = BeamSearch(windows, max_batch_tokens=8)._pages(400, BeamParams(width=2, max_tokens=4))
    assert need == [2 * (4 + 2), 2 * 101, 2 * (4 + 2)]


def test_prompts_that_are_refused():
    for prompts in ([[]], [[1, 50]], [[-1]]):
        with pytest.raises(ValueError):
            BeamSearch(_Runner(100, 8)).run(prompts, BeamParams())
