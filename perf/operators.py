"""Operators that a serving program calls one by one, each in its plain form and as the framework's kernel.

Products in 8-bit integers: rows are taken to 8 bits with a scale of their own (`quantize`), and multiply weights that were
taken to 8 bits channel by channel when they were loaded (`product`, `pairs` and `experts`).  Beam search: the best
continuations of a request's beams over beams and vocabulary (`select`), and the cache pages and fixed-size states that follow
the beams that live on (`pages`, `slots`).

`own` chooses between the plain forms and the framework's calls; `exact` restates each operator in 64 bits.
"""
import math
import zlib

import torch

own = False

DEV = "cuda:0"
F32, F64 = torch.float32, torch.float64
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # a decode step's rows before one product: latency
        {"name": "quantize_step", "kind": "quantize", "rows": 32, "cols": 2048, "dtype": "bf16"},
        # the hidden rows of a prompt portion before the down projection: bandwidth
        {"name": "quantize_portion", "kind": "quantize", "rows": 8192, "cols": 8192, "dtype": "bf16"},
        # one user's decode step, the down projection of a dense feed-forward: latency and the weights' bytes
        {"name": "product_one_row", "kind": "product", "rows": 1, "n": 2048, "k": 8192, "gated": False},
        # eight requests of four beams each against the head: the weights' bytes
        {"name": "product_head_beams", "kind": "product", "rows": 32, "n": 151936, "k": 2048, "gated": False},
        # a portion of a prompt through gate and up, no size of the rows a multiple of a tile: the tensor cores
        {"name": "product_portion", "kind": "product", "rows": 1522, "n": 8192, "k": 2048, "gated": True},
        # a prompt portion through routed experts, rows gathered by expert, the experts' shares uneven
        {"name": "experts_portion", "kind": "experts", "tokens": 2048, "experts": 256, "top": 8, "n": 512, "k": 2048},
        # one request's four beams: latency
        {"name": "select_one", "kind": "select", "requests": 1, "width": 4, "vocab": 32768, "count": 8, "banned": 0},
        # a batch of wide searches over a long vocabulary, some tokens ruled out: the logits' bytes
        {"name": "select_batch", "kind": "select", "requests": 16, "width": 8, "vocab": 151936, "count": 16, "banned": 200},
        # a step of eight searches in which some beams die: the positions since the beams parted
        {"name": "pages_step", "kind": "pages", "layers": 24, "heads": 4, "dim": 128, "page": 16, "requests": 8, "width": 4,
         "length": 1789, "since": 21, "dtype": "bf16"},
        # a search begins: the prompt's pages go to every beam
        {"name": "pages_fork", "kind": "pages", "layers": 24, "heads": 4, "dim": 128, "page": 16, "requests": 2, "width": 4,
         "length": 4096, "since": 4096, "dtype": "bf16"},
        # one request's beams, the states of two recurrent layers: latency
        {"name": "slots_one", "kind": "slots", "layers": 2, "values": 65536, "requests": 1, "width": 4},
        # a batch of searches, the states of eight retention layers: bandwidth
        {"name": "slots_batch", "kind": "slots", "layers": 8, "values": 262144, "requests": 16, "width": 4},
    ]


def _between(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["quantize", "product", "product", "pairs", "experts", "select", "select", "pages", "slots"])
    if kind == "quantize":
        cols = _between(rng, 1, 20000)
        return {"kind": kind, "rows": _between(rng, 1, (1 << 26) // cols), "cols": cols, "dtype": rng.choice(["bf16", "f32"])}
    if kind == "product":
        k, n = 16 * _between(rng, 1, 640), _between(rng, 1, 40000)
        return {"kind": kind, "rows": _between(rng, 1, max(1, min(4096, (1 << 34) // (k * n)))), "n": n, "k": k, "gated": rng.choice([False, True])}
    if kind == "pairs":
        experts, k = _between(rng, 2, 256), 16 * _between(rng, 2, 160)
        return {"kind": kind, "tokens": _between(rng, 1, 16), "experts": experts, "top": min(experts, _between(rng, 1, 8)),
                "n": _between(rng, 8, min(1024, (1 << 28) // (experts * k))), "k": k, "gated": rng.choice([False, True])}
    if kind == "experts":
        experts, k = _between(rng, 2, 256), 16 * _between(rng, 2, 128)
        return {"kind": kind, "tokens": _between(rng, 1, 2048), "experts": experts, "top": min(experts, _between(rng, 1, 8)),
                "n": _between(rng, 8, min(1024, (1 << 28) // (experts * k))), "k": k}
    if kind == "select":
        width, vocab = _between(rng, 1, 32), _between(rng, 40, 200000)
        return {"kind": kind, "requests": _between(rng, 1, max(1, min(64, 20000000 // (width * vocab)))), "width": width, "vocab": vocab,
                "count": min(width * rng.choice([1, 2, 3]), vocab), "banned": rng.choice([0, vocab // 50, vocab - 30])}
    width = _between(rng, 2, 16)
    if kind == "pages":
        layers, heads, dim = _between(rng, 1, 24), rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 96, 128, 192, 576])
        room = (1 << 29) // (width * layers * heads * dim * 2)                       # positions of one request's beams
        length = _between(rng, 1, min(4096, room))
        room = room // length
        return {"kind": kind, "layers": layers, "heads": heads, "dim": dim, "page": rng.choice([16, 32, 64]), "requests": _between(rng, 1, min(8, room)),
                "width": width, "length": length, "since": _between(rng, 1, length), "dtype": rng.choice(["bf16", "f32"])}
    layers, values = _between(rng, 1, 12), _between(rng, 100, 262144)
    return {"kind": kind, "layers": layers, "values": values, "requests": _between(rng, 1, max(1, min(16, (1 << 27) // (layers * values * width)))), "width": width}


# ----------------------------------------------------------------------------------------------- inputs
def _generator(*key):
    """A generator whose stream depends on every number of `key`."""
    seed = 0
    for k in key:
        seed = (seed * 1000003 + int(k) + 12345) % (2 ** 62)
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(gen, shape, std=1.0, dtype=F32):
    return (torch.randn(shape, generator=gen, device=DEV, dtype=F32) * std).to(dtype)


def _activations(gen, rows, cols, dtype):
    """Normed rows: a few channels of far larger values, as models have them."""
    x = torch.randn((rows, cols), generator=gen, device=DEV, dtype=F32)
    loud = torch.rand(cols, generator=gen, device=DEV) < 0.004
    return (x * torch.where(loud, 12.0, 1.0)).to(dtype)


def _weights(gen, *shape):
    """A matrix (or one for each expert) in 8 bits, and the scales of its channels."""
    q = torch.randint(-127, 128, shape, generator=gen, device=DEV, dtype=torch.int8)
    q[..., 0] = 127                                    # every channel's largest value is 127
    return q, torch.rand(shape[:-1], generator=gen, device=DEV) * 4e-4 + 2e-4


def _routing(gen, tokens, experts, top):
    """Experts by token, some chosen far more often than others."""
    liked = torch.randn(experts, generator=gen, device=DEV)
    return (torch.randn((tokens, experts), generator=gen, device=DEV) + 0.7 * liked).topk(top, dim=1).indices.int()


def _parents(gen, requests, width):
    """For every beam the beam that it goes on from: about half of them die, and go on from one that stays what it is."""
    keep = torch.rand((requests, width), generator=gen, device=DEV) < 0.5
    keep[:, 0] = True
    order = torch.argsort(keep.int(), dim=1, descending=True, stable=True)          # the beams that stay come first
    pick = (torch.rand((requests, width), generator=gen, device=DEV) * keep.sum(1, keepdim=True)).long()
    own_number = torch.arange(width, device=DEV).expand(requests, width)
    return torch.where(keep, own_number, order.gather(1, pick)).int().contiguous()


def prepare(case, seed):
    c, kind = case, case["kind"]
    gen = _generator(seed, zlib.crc32(repr(sorted((k, v) for k, v in c.items() if k != "name")).encode()))
    if kind == "quantize":
        return {"kind": kind, "x": _activations(gen, c["rows"], c["cols"], DTYPES[c["dtype"]])}
    if kind == "product":
        x = _activations(gen, c["rows"], c["k"], torch.bfloat16)
        return {"kind": kind, "x": x, "w": _weights(gen, c["n"], c["k"]), "w2": _weights(gen, c["n"], c["k"]) if c["gated"] else (None, None)}
    if kind == "pairs":
        sel = _routing(gen, c["tokens"], c["experts"], c["top"])
        shape = (c["experts"], c["n"], c["k"])
        return {"kind": kind, "x": _activations(gen, c["tokens"], c["k"], torch.bfloat16), "expert": sel.reshape(-1).contiguous(), "top": c["top"],
                "w": _weights(gen, *shape), "w2": _weights(gen, *shape) if c["gated"] else (None, None)}
    if kind == "experts":
        sel = _routing(gen, c["tokens"], c["experts"], c["top"]).reshape(-1)
        order = torch.argsort(sel, stable=True)                                       # rows by expert
        offsets = torch.zeros(c["experts"] + 1, dtype=torch.int32, device=DEV)
        offsets[1:] = torch.bincount(sel, minlength=c["experts"]).cumsum(0).int()
        shape = (c["experts"], c["n"], c["k"])
        return {"kind": kind, "x": _activations(gen, c["tokens"], c["k"], torch.bfloat16), "row_token": (order // c["top"]).int(), "offsets": offsets,
                "expert": sel[order].long(), "most": int(offsets.diff().max()), "w": _weights(gen, *shape), "w2": _weights(gen, *shape)}
    if kind == "select":
        rows = c["requests"] * c["width"]
        logits = _normal(gen, (rows, c["vocab"]), 2.5)
        if c["banned"]:                                                               # tokens that a grammar rules out
            logits[:, torch.randperm(c["vocab"], generator=gen, device=DEV)[:c["banned"]]] = -math.inf
        scores = -torch.rand((c["requests"], c["width"]), generator=gen, device=DEV) * 6.0 - 20.0
        return {"kind": kind, "logits": logits, "scores": scores.sort(dim=1, descending=True).values.contiguous(), "count": c["count"]}
    rows = c["requests"] * c["width"]
    if kind == "pages":
        blocks = -(-c["length"] // c["page"])
        pool = rows * blocks + 3
        values = torch.randint(-30000, 30000, (2 * c["layers"], c["heads"], pool, c["page"], c["dim"]), generator=gen, device=DEV,
                               dtype=torch.int16 if c["dtype"] == "bf16" else torch.int32).view(DTYPES[c["dtype"]])
        table = torch.randperm(pool, generator=gen, device=DEV)[:rows * blocks].int().view(rows, blocks).contiguous()
        parents = _parents(gen, c["requests"], c["width"])
        first = c["length"] - 1 - (torch.rand(rows, generator=gen, device=DEV) * c["since"]).int()
        first[::2] = c["length"] - c["since"]
        return {"kind": kind, "all": values, "pages": list(values.unbind(0)), "table": table, "parents": parents, "first": first,
                "lengths": torch.full((rows,), c["length"], dtype=torch.int32, device=DEV), "length": c["length"], "since": c["since"], "page": c["page"]}
    values = _normal(gen, (c["layers"], rows + 1, c["values"]))
    return {"kind": kind, "all": values, "states": list(values.unbind(0)), "parents": _parents(gen, c["requests"], c["width"]),
            "slots": torch.randperm(rows + 1, generator=gen, device=DEV)[:rows].int().contiguous()}


# ----------------------------------------------------------------------------------------------- one pass
def _to_8_bits(x):
    x = x.float()
    most = x.abs().amax(1, keepdim=True)
    return torch.round(x * torch.where(most > 0, 127.0 / most, 0.0)), most / 127.0


def _product(q, scale, w, w2):
    """Rows in 8 bits against one matrix, or a gate's and another's; with a leading dimension, each batch of rows against its own."""
    y = (q @ w[0].float().mT) * (scale * w[1].unsqueeze(-2))
    if w2[0] is None:
        return y
    return (y / (1.0 + torch.exp(-y)) * ((q @ w2[0].float().mT) * (scale * w2[1].unsqueeze(-2)))).to(torch.bfloat16)


def _best(total, count):
    """The largest of each row and where they stand, the lowest place first among equals."""
    values, at = torch.sort(total, dim=1, descending=True, stable=True)
    return values[:, :count], at[:, :count]


def run(state):
    s, kind = state, state["kind"]
    if own:
        from quench6k_b200 import ops
        if kind == "quantize":
            return ops.quantize_rows(s["x"])
        if kind == "product":
            return ops.linear_i8(s["x"], *s["w"], w2=s["w2"][0], w2_scale=s["w2"][1])
        if kind == "pairs":
            return ops.linear_i8(s["x"], *s["w"], w2=s["w2"][0], w2_scale=s["w2"][1], pair_expert=s["expert"], pair_div=s["top"])
        if kind == "experts":
            q, scale = ops.quantize_rows(s["x"])
            return ops.gemm_i8(q, scale, *s["w"], w2=s["w2"][0], w2_scale=s["w2"][1], offsets=s["offsets"], a_rows=s["row_token"])
        if kind == "select":
            return ops.beam_select(s["logits"], s["scores"], s["count"])
        if kind == "pages":
            if "set" not in s:                         # a program makes it once, with its cache
                s["set"] = ops.PageSet(s["pages"])
            ops.reorder_pages(s["set"], s["table"], s["parents"], s["first"], s["lengths"])
            return s["all"].view(torch.int16 if s["all"].element_size() == 2 else torch.int32)
        if "set" not in s:
            s["set"] = ops.SlotSet(s["states"])
        ops.reorder_slots(s["set"], s["slots"], s["parents"])
        return s["all"].view(torch.int32)

    if kind == "quantize":
        q, scale = _to_8_bits(s["x"])
        return q.to(torch.int8), scale.squeeze(1)
    if kind == "product":
        return _product(*_to_8_bits(s["x"]), s["w"], s["w2"])
    if kind == "pairs":
        token = torch.arange(s["expert"].numel(), device=DEV) // s["top"]
        q, scale = _to_8_bits(s["x"])
        e = s["expert"].long()                         # a matrix for every row
        w, w2 = ((m[0][e], m[1][e]) if m[0] is not None else m for m in (s["w"], s["w2"]))
        return _product(q[token].unsqueeze(1), scale[token].unsqueeze(1), w, w2).squeeze(1)
    if kind == "experts":
        q, scale = _to_8_bits(s["x"])
        token, e, offsets = s["row_token"].long(), s["expert"], s["offsets"].long()
        place = torch.arange(token.numel(), device=DEV) - offsets[e]                 # every expert's rows in a batch of `most`
        rows, scales = q.new_zeros((offsets.numel() - 1, s["most"], q.shape[1])), q.new_zeros((offsets.numel() - 1, s["most"], 1))
        rows[e, place], scales[e, place] = q[token], scale[token]
        return _product(rows, scales, s["w"], s["w2"])[e, place]
    if kind == "select":
        requests, width = s["scores"].shape
        x = s["logits"].double()                       # scores of different beams may lie next to each other
        most = x.amax(1, keepdim=True)
        x = x - (most + torch.log(torch.exp(x - most).sum(1, keepdim=True)))
        value, at = _best((x.view(requests, width, -1) + s["scores"].double().unsqueeze(2)).view(requests, -1), s["count"])
        vocab = s["logits"].shape[1]
        return value.float(), (at // vocab).int(), (at % vocab).int()
    requests, width = s["parents"].shape
    beam = torch.arange(requests * width, device=DEV)
    source = (s["parents"].long() + torch.arange(requests, device=DEV).unsqueeze(1) * width).view(-1)
    if kind == "pages":
        at = torch.arange(s["length"] - s["since"], s["length"], device=DEV)        # the positions that any beam takes over
        block, place = at // s["page"], at % s["page"]
        taken = torch.where(at >= s["first"].unsqueeze(1), source.unsqueeze(1), beam.unsqueeze(1))
        page_to, page_from = s["table"].long()[:, block], s["table"].long()[taken, block]
        s["all"][:, :, page_to, place] = s["all"][:, :, page_from, place]
        return s["all"].view(torch.int16 if s["all"].element_size() == 2 else torch.int32)
    slots = s["slots"].long()
    s["all"][:, slots] = s["all"][:, slots[source]]
    return s["all"].view(torch.int32)


# ----------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c, kind = case, case["kind"]
    size = {"bf16": 2, "f32": 4}.get(c.get("dtype"), 2)
    if kind == "quantize":
        return {"bytes": c["rows"] * c["cols"] * (size + 1) + 4 * c["rows"], "flops": 3 * c["rows"] * c["cols"]}
    if kind == "product":
        mats = 2 if c["gated"] else 1
        return {"bytes": mats * c["n"] * (c["k"] + 4) + 2 * c["rows"] * c["k"] + (2 if c["gated"] else 4) * c["rows"] * c["n"],
                "flops": 2 * mats * c["rows"] * c["n"] * c["k"]}
    if kind in ("pairs", "experts"):
        gated = kind == "experts" or c["gated"]
        mats, rows = (2 if gated else 1), c["tokens"] * c["top"]
        live = c["experts"] * (1.0 - (1.0 - 1.0 / c["experts"]) ** rows)              # experts that some row chose
        return {"bytes": int(mats * live * c["n"] * (c["k"] + 4)) + 2 * c["tokens"] * c["k"] + (2 if gated else 4) * rows * c["n"],
                "flops": 2 * mats * rows * c["n"] * c["k"]}
    rows = c["requests"] * c["width"]
    if kind == "select":
        return {"bytes": 4 * rows * c["vocab"] + 4 * rows + 12 * c["requests"] * c["count"], "flops": 3 * rows * c["vocab"]}
    # about half of the beams die: what they take over is written once, and read once for each request that has any
    if kind == "pages":
        span = 0.75 * c["since"]
        return {"bytes": int(2 * c["layers"] * c["heads"] * c["dim"] * size * span * (rows - c["requests"]) * 0.5 * 2), "flops": 0}
    return {"bytes": int(c["layers"] * c["values"] * 4 * (rows - c["requests"]) * 0.5 * 2), "flops": 0}


# ----------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind in ("pages", "slots"):
        return None                                    # values that move: nothing is computed

    def in_8_bits(x):
        # the two factors and the product that is rounded are 32-bit values by the operator's definition
        most = x.to(F64).abs().max(dim=1).values
        up, scale = (127.0 / most).to(F32), (most / 127.0).to(F32)
        return torch.round((x.to(F64) * up.to(F64)[:, None]).to(F32)).to(F64), scale.to(F64)

    def rows_times(q, scale, w, w_scale):
        return torch.einsum("rk,nk->rn", q, w.to(F64)) * scale[:, None] * w_scale.to(F64)[None, :]

    if kind == "quantize":
        q, scale = in_8_bits(s["x"])
        return q, scale
    if kind == "select":
        x, scores = s["logits"].to(F64), s["scores"].to(F64)
        total = torch.log_softmax(x, dim=1) + scores.reshape(-1, 1)
        return torch.topk(total.reshape(scores.shape[0], -1), s["count"], dim=1).values, None, None

    q, scale = in_8_bits(s["x"])
    if kind == "product":
        y = rows_times(q, scale, *s["w"])
        return y if s["w2"][0] is None else y * torch.sigmoid(y) * rows_times(q, scale, *s["w2"])
    token = s["row_token"].long() if kind == "experts" else torch.arange(s["expert"].numel(), device=DEV) // s["top"]
    parts = torch.empty((token.numel(), s["w"][0].shape[1]), dtype=F64, device=DEV)
    for e in s["expert"].unique().tolist():
        mine = torch.nonzero(s["expert"] == e).squeeze(1)
        y = rows_times(q[token[mine]], scale[token[mine]], s["w"][0][e], s["w"][1][e])
        if s["w2"][0] is not None:
            y = y * torch.sigmoid(y) * rows_times(q[token[mine]], scale[token[mine]], s["w2"][0][e], s["w2"][1][e])
        parts[mine] = y
    return parts
