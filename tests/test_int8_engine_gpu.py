"""Engines whose weights are kept in 8 bits: the kernels against the same engine with the products written out in plain tensor
operations, recordings against eager steps, and what is refused."""
import pytest
import torch

import helpers
import kipedra_configs
import kipedra_helpers
import kitodra_configs
import kitodra_helpers
import kodatar_configs
import kodatar_helpers

pytestmark = pytest.mark.gpu


def plain_quantize_rows(x):
    x = x.float()
    a = x.abs().amax(1)
    u = torch.where(a > 0, torch.reciprocal(a) * 127, torch.zeros_like(a))
    return torch.round(x * u[:, None]).to(torch.int8), a * torch.reciprocal(torch.full_like(a, 127.0))


def plain_gemm_i8(a, a_scale, w, w_scale, out=None, accumulate=False, w2=None, w2_scale=None, act=None, offsets=None, a_rows=None, early=False):
    if a_rows is not None:
        a, a_scale = a[a_rows.long()], a_scale[a_rows.long()]
    rows = a.shape[0]
    if offsets is not None:
        g = torch.bucketize(torch.arange(rows, device=a.device), offsets[1:].long(), right=True).clamp(max=w.shape[0] - 1)
    else:
        g, w, w_scale = torch.zeros(rows, dtype=torch.long, device=a.device), w[None], w_scale[None]
        w2, w2_scale = (w2[None], w2_scale[None]) if w2 is not None else (None, None)
    return plain_pairs(a, a_scale, g, w, w_scale, w2, w2_scale, act, out, accumulate)


def plain_pairs(a, a_scale, g, w, w_scale, w2, w2_scale, act, out=None, accumulate=False):
    def product(w, t):
        y = torch.empty((a.shape[0], w.shape[1]), dtype=torch.float32, device=a.device)
        for e in g.unique().tolist():
            mine = g == e
            y[mine] = (a[mine].double() @ w[e].double().T).float() * (a_scale[mine][:, None] * t[e][None, :])
        return y

    y = product(w, w_scale)
    if w2 is not None or act is not None:
        z = y.double()
        gate = {None: z * torch.sigmoid(z), "silu": z * torch.sigmoid(z), "relu2": z.clamp(min=0) ** 2,
                "gelu_tanh": 0.5 * z * (1 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z ** 3)))}.get(act if not isinstance(act, tuple) else None)
        if isinstance(act, tuple):
            z = z.clamp(max=act[1])
            gate = z * torch.sigmoid(1.702 * z)
        if w2 is not None:
            u = product(w2, w2_scale).double()
            gate = gate * (u.clamp(-act[1], act[1]) + 1 if isinstance(act, tuple) else u)
        y = gate.to(torch.bfloat16)
    if out is not None:
        out.copy_(out + y if accumulate else y)
        return out
    return y


def plain_linear_i8(x, w, w_scale, out=None, accumulate=False, w2=None, w2_scale=None, act=None, pair_expert=None, pair_div=1, weights_are_old=False):
    q, s = plain_quantize_rows(x)
    if pair_expert is None:
        return plain_gemm_i8(q, s, w, w_scale, out, accumulate, w2, w2_scale, act)
    row = torch.arange(pair_expert.numel(), device=x.device) // pair_div
    return plain_pairs(q[row], s[row], pair_expert.long().clamp(0, w.shape[0] - 1), w, w_scale, w2, w2_scale, act)


MODELS = {
    "flint_D": lambda f: helpers.make_model_folder(f, "D", seed=5, init_std=0.1),                       # routed experts, an LM head of its own
    "flint_B": lambda f: helpers.make_model_folder(f, "B", seed=7, init_std=0.15),                      # a dense layer, a shared expert, a tied head
    "kipedra": lambda f: kipedra_helpers.make_folder(f, kipedra_configs.get("K1"), seed=7, init_std=0.08),      # experts without a gate
    "kitodra": lambda f: kitodra_helpers.make_folder(f, kitodra_configs.get("T1"), seed=7, init_std=0.08),      # the clamped gate
    "kodatar": lambda f: kodatar_helpers.make_folder(f, kodatar_configs.get("K1"), seed=7, init_std=0.08),      # identity experts, a gated shared expert
}


def logits_of(folder, requests, **kw):
    """Prompt portions of several sizes, then single tokens; FP32 logits of every position."""
    from quench6k_b200.engine import ModelRunner, StepEntry
    runner = ModelRunner.from_folder(str(folder), num_pages=200, max_requests=8, weights="int8", **kw)
    out = []
    for rid, toks in requests.items():
        runner.add_request(rid)
        at = 0
        for n in (len(toks) - 12, 7, 1, 1, 1, 1, 1):
            out.append(runner.step([StepEntry(rid, toks[at:at + n], list(range(n)))]).clone())
            at += n
    return torch.cat(out), runner


@pytest.mark.parametrize("name", sorted(MODELS))
def test_the_engines_products(name, tmp_path, monkeypatch):
    from quench6k_b200 import ops
    from quench6k_b200.parts.linear import Int8Matrix
    MODELS[name](str(tmp_path))
    import json
    vocab = json.load(open(tmp_path / "config.json"))
    vocab = vocab.get("vocab_size") or vocab["vocab"]
    requests = {"a": helpers.random_tokens(45, vocab, 2), "b": helpers.random_tokens(29, vocab, 3)}
    calls = {}
    for f in ("linear_i8", "gemm_i8"):
        real = getattr(ops, f)
        monkeypatch.setattr(ops, f, lambda *a, _f=f, _real=real, **kw: (calls.__setitem__(_f, calls.get(_f, 0) + 1), _real(*a, **kw))[1])
    got, runner = logits_of(tmp_path, requests)
    assert calls.get("linear_i8"), "no product went through the 8-bit kernels"
    assert any(isinstance(v, Int8Matrix) for b in runner.model.blocks for _, part in b.parts() for v in vars(part).values())
    for f, plain in (("linear_i8", plain_linear_i8), ("gemm_i8", plain_gemm_i8), ("quantize_rows", plain_quantize_rows)):
        monkeypatch.setattr(ops, f, plain)
    want, _ = logits_of(tmp_path, requests, cuda_graphs=False)
    # the same numbers up to roundings of activations to bfloat16 that fall the other way, which then pass through the layers (and now and then to
    # another expert): the bound of the bfloat16 comparisons of whole models
    off = (got - want).abs().amax(1) / want.abs().max()
    assert bool(torch.isfinite(got).all()) and float(off.quantile(0.9)) < 4e-2, f"{off}"
    assert ops.tc_status() == 0


def test_recorded_steps_give_the_tokens_of_eager_ones(tmp_path):
    from quench6k_b200 import Engine, SamplingParams
    MODELS["flint_D"](str(tmp_path))
    prompts = [helpers.random_tokens(n, 1000, 5 + n) for n in (5, 17, 40)]
    tokens = []
    for graphs in (True, False):
        eng = Engine.from_folder(str(tmp_path), num_pages=100, weights="int8")
        eng.runner.cuda_graphs = graphs
        tokens.append([o.tokens for o in eng.generate(prompts, SamplingParams(max_tokens=24, temperature=0.0))])
        assert (eng.runner.graph_replays > 0) == graphs
    assert tokens[0] == tokens[1]


def test_a_search_on_8_bit_weights(tmp_path):
    """Everything together: products in 8 bits under recorded decode steps, selection, reordering; and half the bytes."""
    from quench6k_b200 import BeamParams, Engine
    MODELS["flint_D"](str(tmp_path))
    eng = Engine.from_folder(str(tmp_path), num_pages=300, weights="int8")
    prompts = [helpers.random_tokens(n, 1000, 50 + n) for n in (33, 6)]
    outs = eng.beam_search(prompts, BeamParams(width=4, max_tokens=16))
    assert all(len(o) == 4 and len({tuple(x.tokens) for x in o}) == 4 and all(a.score >= b.score for a, b in zip(o, o[1:])) for o in outs)
    eng.runner.cuda_graphs = False
    again = eng.beam_search(prompts, BeamParams(width=4, max_tokens=16))
    assert [[x.tokens for x in o] for o in outs] == [[x.tokens for x in o] for o in again]
    part = eng.runner.model.blocks[0].ffn
    assert part.w_up.q.dtype == torch.int8 and part.w_up.q.element_size() * 2 == torch.bfloat16.itemsize


def test_what_is_refused(tmp_path):
    from quench6k_b200 import Engine
    MODELS["flint_D"](str(tmp_path))
    with pytest.raises(ValueError, match="bfloat16"):
        Engine.from_folder(str(tmp_path), dtype="float32", weights="int8")
    with pytest.raises(ValueError, match="int8"):
        Engine.from_folder(str(tmp_path), weights="int4")


def in_32_bits(folder, config, helper):
    """The model's folder again with its matrices stored in 32 bits; the stored tensors by name."""
    import os
    from quench6k_b200.weights.safetensors_io import write_safetensors
    _, weights = helper(folder, config)
    for i, (name, t) in enumerate(weights.items()):
        if t.dtype == torch.bfloat16:
            weights[name] = torch.randn(t.shape, generator=torch.Generator().manual_seed(i)) * 0.1
    write_safetensors(os.path.join(folder, "model.safetensors"), weights.items())
    return weights


@pytest.mark.parametrize("name", ["flint_D", "gunenex"])
def test_matrices_stored_in_32_bits_are_rounded_once(name, tmp_path):
    """The 8 bits of every matrix are those of its stored values, not of their bfloat16 roundings."""
    import gunenex_configs
    import gunenex_helpers
    from test_int8_gpu import quantized
    from quench6k_b200.engine import ModelRunner
    from quench6k_b200.parts.attention import Attention
    from quench6k_b200.parts.linear import Int8Matrix
    source = {"flint_D": lambda f: in_32_bits(f, "D", helpers.make_model_folder),
              "gunenex": lambda f: in_32_bits(f, gunenex_configs.get("G1"), gunenex_helpers.make_folder)}[name](str(tmp_path))
    model = ModelRunner.from_folder(str(tmp_path), num_pages=4, max_requests=2, weights="int8").model

    def check(matrix, stored):
        q, scale = quantized(stored.reshape(-1, stored.shape[-1]).numpy())
        assert isinstance(matrix, Int8Matrix) and tuple(matrix.shape) == tuple(stored.shape)
        assert torch.equal(matrix.q.cpu().view(q.shape), torch.from_numpy(q)) and torch.equal(matrix.scale.cpu().view(-1), torch.from_numpy(scale))

    seen = 0
    for spec, block in zip(model.spec.layers, model.blocks):
        parts = [(spec.prefix + model.spec.sub_names[sub], part) for sub, part in block.parts()]
        parts += [(pre + part.names[side], inner) for pre, part in parts if hasattr(part, "sides") for side, inner in part.sides.items()]
        for pre, part in parts:
            stored = lambda n: source[pre + n]
            if isinstance(part, Attention):
                rows = [stored(part.names[x]) for x in ("q", "k", "v") if not (x == "v" and part.values_are_keys)]
                if part.head_gate:
                    rows += [stored(part.names["gate"]), torch.zeros(part.ng - part.Hq, part.D)]
                check(part.w_qkv, torch.cat(rows))
                check(part.w_o, stored(part.names["o"]))
                seen += 1
            elif hasattr(part, "w_down"):
                for attr, key in (("w_up", "up"), ("w_gate", "gate"), ("w_down", "down")):
                    if isinstance(getattr(part, attr), Int8Matrix):        # (rows that are no multiple of 16 long stay as they are)
                        check(getattr(part, attr), stored(part.names[key]))
                        seen += 1
    if model.spec.head_name is not None:
        check(model.head, source[model.spec.head_name])
    assert seen >= (8 if name == "flint_D" else 2)


def with_rows_in_8_bits(config):
    """The configuration with feed-forwards whose widths the 8-bit products take."""
    if isinstance(config, dict):
        return {k: -(-v // 16) * 16 if k == "ff" else with_rows_in_8_bits(v) for k, v in config.items()}
    return [with_rows_in_8_bits(v) for v in config] if isinstance(config, list) else config


ROUTED = {
    **{name: MODELS[name] for name in ("flint_D", "flint_B")},
    "kipedra": lambda f: kipedra_helpers.make_folder(f, with_rows_in_8_bits(kipedra_configs.get("K1")), seed=7, init_std=0.08),
    "kitodra": lambda f: kitodra_helpers.make_folder(f, with_rows_in_8_bits(kitodra_configs.get("T1")), seed=7, init_std=0.08),
    "kodatar": lambda f: kodatar_helpers.make_folder(f, with_rows_in_8_bits(kodatar_configs.get("K1")), seed=7, init_std=0.08),
}


class Checked:
    """ops.linear_i8 and ops.gemm_i8 whose every result is compared with the formula in 64 bits on the call's own operands; `seen`: how many
    results of each form were."""

    def __init__(self, ops, monkeypatch):
        self.seen, self.quantize = {}, ops.quantize_rows
        for name in ("linear_i8", "gemm_i8"):
            real = getattr(ops, name)
            monkeypatch.setattr(ops, name, lambda *a, _real=real, _f=getattr(self, name), **kw: _f(_real, *a, **kw))

    def linear_i8(self, real, x, w, w_scale, out=None, accumulate=False, w2=None, w2_scale=None, act=None, pair_expert=None, pair_div=1, weights_are_old=False):
        base = out.clone() if accumulate else None
        y = real(x, w, w_scale, out=out, accumulate=accumulate, w2=w2, w2_scale=w2_scale, act=act, pair_expert=pair_expert, pair_div=pair_div, weights_are_old=weights_are_old)
        q, s = self.quantize(x)
        if pair_expert is None:
            self.check("one row" if x.shape[0] == 1 else "rows", y, base, q, s, [(w, w_scale), (w2, w2_scale)], act)
        else:
            e = pair_expert.long()
            row = torch.arange(e.numel(), device=x.device) // pair_div
            self.groups("pairs", y, q[row], s[row], [e == g for g in range(w.shape[0])], w, w_scale, w2, w2_scale, act)
        return y

    def gemm_i8(self, real, a, a_scale, w, w_scale, w2=None, w2_scale=None, act=None, offsets=None, a_rows=None, early=False):
        y = real(a, a_scale, w, w_scale, w2=w2, w2_scale=w2_scale, act=act, offsets=offsets, a_rows=a_rows, early=early)
        if a_rows is not None:
            a, a_scale = a[a_rows.long()], a_scale[a_rows.long()]
        at = torch.arange(a.shape[0], device=a.device)
        self.groups("grouped, picked" if a_rows is not None else "grouped", y, a, a_scale, [(at >= offsets[g]) & (at < offsets[g + 1]) for g in range(w.shape[0])],
                    w, w_scale, w2, w2_scale, act)
        return y

    def groups(self, form, y, q, s, members, w, w_scale, w2, w2_scale, act):
        for g, mine in enumerate(members):
            self.check(form, y[mine], None, q[mine], s[mine], [(w[g], w_scale[g]), (w2, w2_scale) if w2 is None else (w2[g], w2_scale[g])], act)

    def check(self, form, y, base, q, s, mats, act):
        from test_int8_gpu import BF16_HALF, HALF, STORED, gated64, product64
        if y.numel() == 0:
            return
        g = product64(q, s, *mats[0])
        if mats[1][0] is None and act is None:
            want, allowed = g if base is None else g + base.double(), STORED * g.abs()
            if base is not None:
                allowed = allowed + HALF * 1.01 * want.abs()
        else:
            u = torch.ones_like(g) if mats[1][0] is None else product64(q, s, *mats[1])
            want = gated64(g, u, act)
            # of the result: its rounding to bfloat16; three roundings of the gate's argument, which move silu by 1 + |g| times as much, and three of the other factor;
            # an exponential off by 3 + 1.2 |g| units of two half steps; ten half steps of the gate's other arithmetic
            allowed = want.abs() * (BF16_HALF * 1.01 + HALF * (3 * (1 + g.abs()) + 3 + 2 * (3 + 1.2 * g.abs()) + 10)) + 1e-30
            if act not in (None, "silu"):          # sums that nearly cancel: a rounding counts in full
                allowed = allowed + 8 * HALF * g.abs() * (u.abs() + 1)
        off = (y.double() - want).abs()
        assert bool((off <= allowed).all()), f"{form}, {tuple(y.shape)}, act {act}: off by {float((off / allowed).max()):.3g} of what is allowed"
        self.seen[form] = self.seen.get(form, 0) + y.numel()


@pytest.mark.parametrize("name", sorted(ROUTED))
def test_every_product_of_a_models_steps(name, tmp_path, monkeypatch):
    """Prompts, portions and single tokens: each product alone, so that a wrong one shows whatever the layers behind it make of it."""
    import json
    from quench6k_b200 import ops
    from quench6k_b200.parts.ffn import RoutedExperts
    ROUTED[name](str(tmp_path))
    vocab = json.load(open(tmp_path / "config.json"))
    vocab = vocab.get("vocab_size") or vocab["vocab"]
    checked = Checked(ops, monkeypatch)
    got, runner = logits_of(tmp_path, {"a": helpers.random_tokens(45, vocab, 2), "b": helpers.random_tokens(29, vocab, 3)}, cuda_graphs=False)
    experts = [part for b in runner.model.blocks for _, part in b.parts() if isinstance(part, RoutedExperts)]
    assert experts and all(part.int8 for part in experts)
    # pair by pair where a part hands its rows on unsummed: not where it has a shared expert's to add to them (all layers of flint_B)
    forms = {"one row", "rows", "grouped, picked", "grouped"} | ({"pairs"} if any(part.shared is None for part in experts) else set())
    assert set(checked.seen) >= forms, checked.seen
    assert bool(torch.isfinite(got).all()) and ops.tc_status() == 0
