"""Beam search through the engine, against a search that runs every sequence from its first token: no cache, no state and no page
is shared there, so a beam that went on from the wrong one, or from too late a position, shows."""
import pytest
import torch

import gunenex_configs
import gunenex_helpers
import helpers
import kipedra_configs
import kipedra_helpers
import kitodra_configs
import kitodra_helpers
import kodatar_configs
import kodatar_helpers
import pedotar_configs
import pedotar_helpers
import sigusun_configs
import sigusun_helpers

pytestmark = pytest.mark.gpu

ARCHITECTURES = {
    "flint": lambda folder: helpers.make_model_folder(folder, "B", seed=7, init_std=0.2),             # windows, sinks, a shared expert
    "flint_order": lambda folder: helpers.make_model_folder(folder, "C", seed=3, init_std=0.2),       # layers run twice, borrowed pages
    "pedotar": lambda folder: pedotar_helpers.make_folder(folder, pedotar_configs.get("P1"), seed=7, init_std=0.06),
    "kipedra": lambda folder: kipedra_helpers.make_folder(folder, kipedra_configs.get("K1"), seed=7, init_std=0.08),
    "sigusun": lambda folder: sigusun_helpers.make_folder(folder, sigusun_configs.get("G1"), seed=7, init_std=0.08),
    "kitodra": lambda folder: kitodra_helpers.make_folder(folder, kitodra_configs.get("T1"), seed=7, init_std=0.08),
    "gunenex": lambda folder: gunenex_helpers.make_folder(folder, gunenex_configs.get("G1"), seed=7, init_std=0.08),
    "kodatar": lambda folder: kodatar_helpers.make_folder(folder, kodatar_configs.get("K1"), seed=7, init_std=0.08),
}


def engine(folder, **kw):
    from quench6k_b200 import Engine
    return Engine.from_folder(str(folder), **{"dtype": "float32", "num_pages": 400, "max_requests": 16, "max_batch_tokens": 7, **kw})


def whole_sequences(eng, prompt, params):
    """[(tokens, worth)] best first, and the smallest distance of two scores that an order depended on."""
    from quench6k_b200.engine import StepEntry
    worth = lambda total, n: total / n ** params.length_penalty
    runner, stops, nearest = eng.runner, set(params.stop_tokens), float("inf")
    beams, ended = [([], 0.0)], []
    while True:
        every = []
        for b, (toks, total) in enumerate(beams):
            runner.add_request("whole")
            seq = prompt + toks
            logits = runner.step([StepEntry("whole", seq, [len(seq) - 1])])
            runner.end_request("whole")
            every += [(total + lp, b, t) for t, lp in enumerate(torch.log_softmax(logits[0].double(), 0).tolist())]
        every.sort(key=lambda c: (-c[0], c[1], c[2]))
        count = params.width * (1 + len(stops))
        nearest = min([nearest] + [a[0] - b[0] for a, b in zip(every[:count], every[1:count + 1])])
        after = []
        for rank, (total, b, t) in enumerate(every):
            if len(after) == params.width:
                break
            toks = beams[b][0] + [t]
            if t in stops:
                if rank < params.width:
                    ended.append((toks, worth(total, len(toks))))
            else:
                after.append((toks, total))
        ended, beams = sorted(ended, key=lambda e: -e[1])[:params.width], after
        n = len(beams[0][0])
        if len(ended) == params.width and ended[-1][1] >= worth(beams[0][1], params.max_tokens):
            return ended, nearest
        if n >= params.max_tokens:
            return sorted(ended + [(toks, worth(total, n)) for toks, total in beams], key=lambda e: -e[1])[:params.width], nearest


def prompt_of(eng, n, seed, *params):
    """A random prompt of n tokens none of whose searches (`params`) depends on scores closer than 1e-4: the sums of a model's float32
    arithmetic may be taken in two orders, which moves a score by far less."""
    graphs, eng.runner.cuda_graphs = eng.runner.cuda_graphs, False
    try:
        for s in range(seed, seed + 40):
            prompt = helpers.random_tokens(n, eng.runner.vocab_size, s)
            if all(whole_sequences(eng, prompt, p)[1] > 1e-4 for p in params):
                return prompt
    finally:
        eng.runner.cuda_graphs = graphs
    raise AssertionError("no prompt whose scores lie apart")


def compare(eng, prompts, params):
    got = eng.beam_search(prompts, params)
    torch.cuda.synchronize()
    eng.runner.manager.check()
    assert len(eng.runner.manager.requests) == 0
    eng.runner.cuda_graphs = False
    for prompt, outs in zip(prompts, got):
        want, _ = whole_sequences(eng, prompt, params)
        assert [o.tokens for o in outs] == [t for t, _ in want]
        assert all(abs(o.score - s) < 1e-4 for o, (_, s) in zip(outs, want))
    return got


@pytest.mark.parametrize("name", sorted(ARCHITECTURES))
def test_beams_of_every_architecture(name, tmp_path):
    from quench6k_b200 import BeamParams
    cfg, _ = ARCHITECTURES[name](str(tmp_path))
    eng = engine(tmp_path)
    params = BeamParams(width=4, max_tokens=10)
    compare(eng, [prompt_of(eng, n, 60 + n, params) for n in (13, 30)], params)


@pytest.mark.parametrize("graphs", [True, False])
def test_beams_that_end(graphs, tmp_path):
    """Stop tokens, several prompts in one batch, more prompts than the slots hold at a time."""
    from quench6k_b200 import BeamParams
    ARCHITECTURES["flint"](str(tmp_path))
    eng = engine(tmp_path, max_requests=7)
    eng.runner.cuda_graphs = graphs
    first = eng.beam_search([helpers.random_tokens(n, eng.runner.vocab_size, 10 + n) for n in (3, 17)], BeamParams(width=3, max_tokens=8))
    stops = [first[0][0].tokens[3], first[1][1].tokens[2]]            # tokens that such searches come across
    params = BeamParams(width=3, max_tokens=8, stop_tokens=stops, length_penalty=0.7)
    outs = compare(eng, [prompt_of(eng, n, 10 + n, params) for n in (3, 17, 9)], params)
    reasons = [o.finish_reason for out in outs for o in out]
    assert "stop" in reasons and "length" in reasons
    assert all((o.tokens[-1] in stops) == (o.finish_reason == "stop") for out in outs for o in out)


def test_one_beam_is_greedy(tmp_path):
    from quench6k_b200 import BeamParams, SamplingParams
    ARCHITECTURES["flint"](str(tmp_path))
    eng = engine(tmp_path)
    prompts = [helpers.random_tokens(n, eng.runner.vocab_size, 90 + n) for n in (5, 21)]
    greedy = eng.generate(prompts, SamplingParams(max_tokens=10, temperature=0.0))
    beams = eng.beam_search(prompts, BeamParams(width=1, max_tokens=10))
    assert [b[0].tokens for b in beams] == [g.tokens for g in greedy]
    assert eng.beam_search(prompts, BeamParams(width=3, max_tokens=10, num_return=2))[0].__len__() == 2


def test_searches_that_are_refused_leave_nothing_behind(tmp_path):
    from quench6k_b200 import BeamParams, SamplingParams
    from quench6k_b200.cache import OutOfPages, OutOfSlots
    ARCHITECTURES["flint"](str(tmp_path))
    eng = engine(tmp_path, num_pages=20, max_requests=4)
    prompt = helpers.random_tokens(20, eng.runner.vocab_size, 1)
    with pytest.raises(OutOfPages):
        eng.beam_search([prompt * 5], BeamParams(width=4, max_tokens=8))
    with pytest.raises(OutOfSlots):
        eng.beam_search([prompt], BeamParams(width=5, max_tokens=8))
    with pytest.raises(ValueError):
        eng.beam_search([prompt], BeamParams(width=0))
    eng.add_request(prompt, SamplingParams(max_tokens=2))
    with pytest.raises(RuntimeError):
        eng.beam_search([prompt], BeamParams(width=2, max_tokens=2))
    while eng.has_unfinished():
        eng.step()
    assert len(eng.beam_search([prompt], BeamParams(width=2, max_tokens=3))[0]) == 2
    eng.runner.manager.check()


def test_reorder_refuses_what_does_not_fit(tmp_path):
    ARCHITECTURES["flint"](str(tmp_path))
    runner = engine(tmp_path).runner
    for rid in "abc":
        runner.add_request(rid)
        runner.assume_cached(rid, 5 if rid != "c" else 6)
    for groups, parents, first in (([["a", "b"]], [[0]], [[0, 0]]), ([["a", "b"]], [[0, 2]], [[0, 0]]), ([["a", "c"]], [[0, 0]], [[0, 0]]), ([["a", "a"]], [[0, 0]], [[0, 0]])):
        with pytest.raises(ValueError):
            runner.reorder(groups, parents, first)
    runner.reorder([["a", "b"]], [[1, 0]], [[2, 2]])
