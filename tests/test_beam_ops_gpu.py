"""Beam search's selection and the reordering of pages and slots against plain host implementations (64-bit scores, copies row by row)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -24


# ----------------------------------------------------------------------------------------------- selection
def selected(logits, scores, count):
    """Scores (64 bits), beams and tokens of each request's best continuations; what is not finite counts as -infinity."""
    requests, width = scores.shape
    V = logits.shape[1]
    x = logits.astype(np.float64)
    with np.errstate(all="ignore"):
        most = x.max(axis=1, keepdims=True)
        t = scores.astype(np.float64).reshape(-1, 1) + ((x - most) - np.log(np.exp(x - most).sum(axis=1, keepdims=True)))
        t = np.where(np.isfinite(t), t, -np.inf).reshape(requests, width * V)
    order = np.argsort(-t, axis=1, kind="stable")[:, :count + 1]
    best = np.take_along_axis(t, order, axis=1)
    # continuations of different beams further apart than the kernel's sums may be off: the order is then the same in any arithmetic
    apart = -np.diff(np.where(np.isfinite(best), best, -1e30), axis=1)
    gap = np.where((order[:, 1:] // V != order[:, :-1] // V) & np.isfinite(best[:, 1:]), apart, 1.0)
    assert float(gap.min(initial=1.0)) > 1.5e-5, "the inputs have scores too close to tell apart"
    order, best = order[:, :count], best[:, :count]
    return best, order // V, order % V


def check_select(logits, scores, count):
    from quench6k_b200 import ops
    got, beams, tokens = ops.beam_select(torch.from_numpy(logits).cuda(), torch.from_numpy(scores).cuda(), count)
    best, want_beams, want_tokens = selected(logits, scores, count)
    assert got.dtype == torch.float32 and beams.dtype == tokens.dtype == torch.int32
    np.testing.assert_array_equal(beams.cpu().numpy(), want_beams)
    np.testing.assert_array_equal(tokens.cpu().numpy(), want_tokens)
    got = got.cpu().numpy().astype(np.float64)
    finite = np.isfinite(best)
    np.testing.assert_array_equal(got[~finite], best[~finite])
    # one rounding of the score; the row's sum in half steps: 4 of an exponential and 20 of its argument (below 20 where a term
    # counts, rounded once) against its thread's maximum, the same 24 and 2 of a product from there to the warp's and again to
    # the block's, 31 + 1 + 5 + 8 additions one after the other of a tile, a thread, a warp and a block: 121
    assert float((np.abs(got[finite] - best[finite]) - HALF * np.abs(best[finite])).max(initial=0.0)) <= 121 * HALF


def logits_of(seed, rows, V, spread=3.0):
    return (np.random.default_rng(seed).standard_normal((rows, V)) * spread).astype(np.float32)


def scores_of(seed, requests, width):
    return np.sort(-np.random.default_rng([seed, 1]).random((requests, width)) * 8 - 3, axis=1)[:, ::-1].astype(np.float32).copy()


@pytest.mark.parametrize("requests,width,V,count", [(1, 1, 1, 1), (1, 1, 7, 7), (2, 3, 5, 15), (1, 4, 32768, 8), (3, 4, 8192, 8), (2, 2, 8193, 5), (5, 3, 1000, 9),
                                                    (1, 32, 300, 96), (2, 8, 50001, 16), (1, 1, 40000, 128), (1, 32, 20010, 128), (4, 5, 151936, 15), (40, 4, 513, 8)])
def test_selection(requests, width, V, count):
    check_select(logits_of(V + count, requests * width, V), scores_of(V, requests, width), count)


@pytest.mark.parametrize("V", [100, 9000, 30001])
def test_selection_among_equal_logits(V):
    """Coarse logits: most of the best are equal, within the slices and across them; the lowest token comes first."""
    x = np.round(logits_of(V, 6, V)).astype(np.float32)
    check_select(np.minimum(x, 4.0), scores_of(5, 2, 3), 40)
    check_select(np.zeros((3, V), dtype=np.float32), np.array([[-1.0, -1.5, -9.0]], dtype=np.float32), 100)


def test_beams_that_are_the_same_tie_to_the_lowest():
    x = logits_of(3, 1, 20000).repeat(4, axis=0)
    s = np.full((1, 4), -2.0, dtype=np.float32)
    from quench6k_b200 import ops
    _, beams, tokens = ops.beam_select(torch.from_numpy(x).cuda(), torch.from_numpy(s).cuda(), 10)
    order = np.argsort(-x[0], kind="stable")
    assert beams[0].tolist() == [0, 1, 2, 3, 0, 1, 2, 3, 0, 1]
    assert tokens[0].tolist() == [int(order[i // 4]) for i in range(10)]


def test_first_step_of_a_search():
    """All beams but one at -infinity: the others take part only when the first has nothing left."""
    x, s = logits_of(1, 4, 9000), np.array([[0.0, -np.inf, -np.inf, -np.inf]], dtype=np.float32)
    check_select(x, s, 8)
    check_select(logits_of(2, 4, 3), s, 8)


@pytest.mark.parametrize("allowed", [0, 1, 3, 30])
def test_tokens_that_are_ruled_out(allowed):
    """Fewer continuations than wanted: the rest follow in order of place with -infinity."""
    x = np.full((6, 10000), -np.inf, dtype=np.float32)
    keep = np.random.default_rng(allowed).permutation(10000)[:allowed]
    x[:, keep] = logits_of(7, 6, 10000)[:, keep]
    check_select(x, scores_of(2, 2, 3), 24)


def test_rows_and_scores_that_are_not_finite():
    x, s = logits_of(4, 8, 9001), scores_of(4, 2, 4)
    x[0, 17], x[1, 8999], x[2, :] = np.nan, np.inf, -np.inf
    x[5, 100:200] = -np.inf
    s[1, 2], s[1, 3] = np.nan, np.inf
    check_select(x, s, 12)
    check_select(x[:4], s[:1], 128)
    check_select(np.full((2, 40), np.nan, dtype=np.float32), s[:1, :2].copy(), 50)


def test_large_logits():
    """Rows far from zero, and one value that outweighs its row."""
    x = logits_of(9, 4, 12000) + np.array([[3e4], [-3e4], [0], [0]], dtype=np.float32)
    x[2, 7777] = 200.0
    x[3, 5] = -3e38
    check_select(x, scores_of(6, 1, 4), 16)


def test_tokens_masked_with_the_lowest_value():
    """float32's lowest value is finite: such tokens come after all others, in order of place, with their scores."""
    low = np.finfo(np.float32).min
    x = np.full((3, 20000), low, dtype=np.float32)
    x[0, 5000:5040] = logits_of(8, 1, 40)[0]
    x[1, 19999] = 2.0
    check_select(x, np.array([[-1.0, -4.5, -8.25]], dtype=np.float32), 50)
    check_select(x[2:], np.array([[-1.0]], dtype=np.float32), 20)
    check_select(-x[:1], np.array([[-1.0]], dtype=np.float32), 20)


@pytest.mark.parametrize("mask", [-6.5e4, -9.9e5, -1e6, -1e9, -1e10, -1e12, -1e20, -9e29, -2e30])
def test_tokens_masked_with_a_large_finite_value(mask):
    """Masks of any size leave a row's sum and its other tokens as they are; threads, tiles and whole parts of a row see nothing but the mask."""
    x = np.full((4, 30000), mask, dtype=np.float32)
    keep = np.random.default_rng(11).permutation(30000)[:60]
    x[:, keep] = logits_of(13, 4, 30000)[:, keep]
    x[3] = logits_of(14, 1, 30000)[0]
    x[3, 8192:] = mask
    check_select(x, scores_of(15, 1, 4), 24)
    check_select(x, scores_of(15, 2, 2), 24)
    check_select(x[:1], np.array([[-1.0]], dtype=np.float32), 80)         # every token that is left, then masked ones in order of place


@pytest.mark.parametrize("level", [1e6, 3e9, -1e10, 1e10, -1e15, 1e29])
def test_rows_of_a_large_level(level):
    """Logits that differ by whole steps of a large number: equal ones share the row, the others count for nothing."""
    step = np.spacing(np.float32(abs(level)))
    x = (np.float32(level) + np.random.default_rng(17).integers(-3, 1, (3, 9001)).astype(np.float32) * step * 64).astype(np.float32)
    check_select(x, np.array([[-1.0, -2.5, -7.25]], dtype=np.float32), 32)


@pytest.mark.parametrize("V", [70000, 70001])
def test_rows_whose_logits_ascend_or_descend(V):
    """Orders that hide the best from a threshold of the first logits, or show them all at once."""
    up = np.arange(V, dtype=np.float32) * 2.0 ** -10
    check_select(np.stack([up, up[::-1]]), np.array([[-1.0, -3.3]], dtype=np.float32), 30)


def test_many_rows_of_many_tiles():
    """More work than one round of the GPU: parts of several tiles."""
    check_select(logits_of(12, 96, 100000), scores_of(12, 12, 8), 16)


def test_no_requests():
    from quench6k_b200 import ops
    got, beams, tokens = ops.beam_select(torch.empty(0, 50, device="cuda"), torch.empty(0, 4, device="cuda"), 8)
    assert got.shape == beams.shape == tokens.shape == (0, 8)


def test_selections_in_two_recordings():
    from quench6k_b200 import ops
    xs = [torch.from_numpy(logits_of(30 + i, 8, 20000)).cuda() for i in range(2)]
    s = torch.from_numpy(scores_of(3, 2, 4)).cuda()
    want = [ops.beam_select(x, s, 8) for x in xs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.beam_select(x, s, 8))
        graphs.append(g)
    for i in (1, 0, 1, 0):
        graphs[i].replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(o, w))


# ----------------------------------------------------------------------------------------------- reordering
def moved_pages(tensors, table, parents, first, lengths):
    """Row by row from a copy of everything as it was."""
    groups, width = parents.shape
    page = tensors[0].shape[2]
    out = [t.clone() for t in tensors]
    for r in range(groups * width):
        p = int(parents[r // width, r % width])
        if not 0 <= p < width or p == r % width:
            continue
        src = r // width * width + p
        for at in range(max(0, int(first[r])), min(int(lengths[src]), table.shape[1] * page)):
            a, b = int(table[src, at // page]), int(table[r, at // page])
            for o, t in zip(out, tensors):
                if 0 <= a < t.shape[1] and 0 <= b < t.shape[1]:
                    o[:, b, at % page] = t[:, a, at % page]
    return out


def bits(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    if dtype == torch.bfloat16:
        return torch.randint(-30000, 30000, shape, generator=g, dtype=torch.int16).view(torch.bfloat16)
    return torch.randint(-2 ** 31, 2 ** 31 - 1, shape, generator=g, dtype=torch.int64).to(torch.int32).view(torch.float32) if dtype == torch.float32 else \
        torch.randint(-128, 127, shape, generator=g, dtype=torch.int8)


def same_bits(a, b):
    return torch.equal(a.cpu().contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def check_pages(tensors, table, parents, first, lengths):
    from quench6k_b200 import ops
    dev = [t.cuda() for t in tensors]
    i32 = lambda x: torch.as_tensor(x, dtype=torch.int32)
    table, parents, first, lengths = i32(table), i32(parents), i32(first), i32(lengths)
    ops.reorder_pages(dev, table.cuda(), parents.cuda(), first.cuda(), lengths.cuda())
    torch.cuda.synchronize()
    for got, want in zip(dev, moved_pages(tensors, table, parents, first, lengths)):
        assert same_bits(got, want)


def table_of(rows, blocks, pages, seed):
    return torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:rows * blocks].view(rows, blocks)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.bfloat16, 20), (torch.bfloat16, 5), (torch.float32, 64), (torch.float32, 3), (torch.int8, 9)])
@pytest.mark.parametrize("groups,width,parents", [(1, 1, [[0]]), (1, 2, [[1, 0]]), (2, 4, [[0, 0, 1, 1], [3, 2, 1, 0]]), (1, 5, [[4, 0, 1, 2, 3]]),
                                                  (2, 9, [[0] * 9, [8, 8, 8, 0, 0, 0, 1, 1, 1]])])
def test_pages_of_every_row_type(groups, width, parents, dtype, dim):
    rows, blocks = groups * width, 5
    tensors = [bits((3, rows * blocks + 2, 4, dim), dtype, 1), bits((1, rows * blocks + 2, 4, dim), dtype, 2)]
    g = torch.Generator().manual_seed(width)
    first = torch.randint(0, 19, (rows,), generator=g)
    check_pages(tensors, table_of(rows, blocks, rows * blocks + 2, 3), parents, first, torch.full((rows,), 19))


def test_pages_of_one_token_and_of_none():
    tensors = [bits((2, 12, 8, 16), torch.bfloat16, 4)]
    table = table_of(4, 3, 12, 5)
    check_pages(tensors, table, [[1, 1, 0, 2]], [0, 0, 0, 0], [1, 1, 1, 1])
    check_pages(tensors, table, [[1, 1, 0, 2]], [0, 0, 0, 0], [0, 0, 0, 0])
    check_pages(tensors, table, [[1, 1, 0, 2]], [30, 24, 23, 5], [24, 24, 24, 24])


def test_pages_that_a_row_does_not_hold_and_parents_outside_the_group():
    tensors = [bits((2, 20, 8, 16), torch.float32, 6)]
    table = table_of(6, 3, 20, 7)
    table[0, 0] = table[1, 0] = -1                       # a window has passed: neither holds the block
    table[3, 1], table[4, 2], table[5, 0] = -1, 20, 1 << 30
    check_pages(tensors, table, [[1, 0, 7], [1, -1, 0]], [0, 3, 0, 0, 0, -5], [24, 20, 24, 24, 24, 24])
    check_pages(tensors, table, [[1, 0, 0], [2, 0, 1]], [0, 3, 0, 0, 0, 2], [1000, 24, 9, 24, 25, 24])     # lengths behind the table's end


def test_rows_of_different_lengths():
    tensors = [bits((2, 40, 4, 24), torch.bfloat16, 8)]
    check_pages(tensors, table_of(8, 5, 40, 9), [[1, 0, 3, 3], [2, 2, 0, 1]], [0, 2, 4, 6, 8, 1, 3, 5], [20, 7, 11, 13, 5, 6, 18, 20])


@pytest.mark.parametrize("width", [16, 17, 32])
def test_widest_groups(width):
    tensors = [bits((2, width * 3, 4, 16), torch.bfloat16, 10)]
    g = torch.Generator().manual_seed(width)
    for parents in (torch.randperm(width, generator=g), torch.randint(0, width, (width,), generator=g)):
        check_pages(tensors, table_of(width, 3, width * 3, 11), parents.view(1, width), torch.randint(0, 12, (width,), generator=g), torch.full((width,), 12))


def test_tensors_of_different_shapes_types_and_more_than_one_launch_takes():
    tensors = [bits((1 + i % 3, 12, 4, (8, 3, 16)[i % 3]), (torch.bfloat16, torch.float32, torch.int8)[i % 3], i) for i in range(131)]
    check_pages(tensors, table_of(4, 3, 12, 12), [[1, 2, 3, 0]], [0, 1, 2, 3], [12, 12, 12, 12])


def test_many_positions():
    """More places than one round of the launch's threads."""
    rows, blocks = 4, 160
    tensors = [bits((2, rows * blocks, 16, 128), torch.bfloat16, 13) for _ in range(2)]
    check_pages(tensors, table_of(rows, blocks, rows * blocks, 14), [[3, 1, 1, 0]], [100, 0, 7, 2000], [2555, 2555, 2555, 2555])


def moved_slots(tensors, slots, parents):
    groups, width = parents.shape
    out = [t.clone() for t in tensors]
    for r in range(groups * width):
        p = int(parents[r // width, r % width])
        if 0 <= p < width:
            a, b = int(slots[r // width * width + p]), int(slots[r])
            for o, t in zip(out, tensors):
                if 0 <= a < t.shape[0] and 0 <= b < t.shape[0]:
                    o[b] = t[a]
    return out


@pytest.mark.parametrize("shapes", [[(9, 4, 16)], [(9,)], [(9, 3), (9, 5, 7), (11, 1)], [(9, 40000), (9, 100003)]])
@pytest.mark.parametrize("parents", [[[0, 0, 0, 0], [3, 0, 1, 2]], [[1, 0, 1, 2], [2, 9, -1, 0]], [[7, 6, 5, 4, 3, 2, 1, 0]]])
def test_slots(shapes, parents):
    from quench6k_b200 import ops
    tensors = [bits(s, (torch.float32, torch.bfloat16, torch.int8)[i % 3], i) for i, s in enumerate(shapes)]
    slots = torch.randperm(9, generator=torch.Generator().manual_seed(15))[:8].int()
    parents = torch.tensor(parents, dtype=torch.int32)
    dev = [t.cuda() for t in tensors]
    ops.reorder_slots(dev, slots.cuda(), parents.cuda())
    for got, want in zip(dev, moved_slots(tensors, slots, parents)):
        assert same_bits(got, want)
    slots[2], slots[5] = -1, 1000                        # nothing is held there
    dev = [t.cuda() for t in tensors]
    ops.reorder_slots(dev, slots.cuda(), parents.cuda())
    for got, want in zip(dev, moved_slots(tensors, slots, parents)):
        assert same_bits(got, want)


def test_reordering_in_a_recording():
    from quench6k_b200 import ops
    t = bits((2, 12, 8, 16), torch.bfloat16, 16)
    state = bits((5, 33), torch.float32, 17)
    table, parents = table_of(4, 3, 12, 18).int(), torch.tensor([[1, 0, 3, 3]], dtype=torch.int32)
    first, lengths, slots = torch.tensor([0, 5, 2, 0], dtype=torch.int32), torch.full((4,), 20, dtype=torch.int32), torch.tensor([4, 0, 2, 1], dtype=torch.int32)
    dev, dstate = t.cuda(), state.cuda()
    args = [x.cuda() for x in (table, parents, first, lengths, slots)]
    pages, states = ops.PageSet([dev]), ops.SlotSet([dstate])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.reorder_pages(pages, args[0], args[1], args[2], args[3])
        ops.reorder_slots(states, args[4], args[1])
    want, want_state = [t], [state]
    for _ in range(3):
        g.replay()
        want, want_state = moved_pages(want, table, parents, first, lengths), moved_slots(want_state, slots, parents)
    torch.cuda.synchronize()
    assert same_bits(dev, want[0]) and same_bits(dstate, want_state[0])


def test_refusals():
    from quench6k_b200 import ops
    x, s = torch.zeros(8, 50, device="cuda"), torch.zeros(2, 4, device="cuda")
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")
    pages = torch.zeros(2, 6, 4, 8, device="cuda")
    bad = [lambda: ops.beam_select(x, s, 0), lambda: ops.beam_select(x, s, 129), lambda: ops.beam_select(x[:, :1].contiguous(), s, 5), lambda: ops.beam_select(x[:6], s, 4),
           lambda: ops.beam_select(x.bfloat16(), s, 4), lambda: ops.beam_select(x, s.double(), 4), lambda: ops.beam_select(x[:, :40], s, 4),
           lambda: ops.beam_select(torch.zeros(33, 50, device="cuda"), torch.zeros(1, 33, device="cuda"), 4),
           lambda: ops.reorder_pages([pages], i32(7, 2), i32(2, 4), i32(8), i32(8)), lambda: ops.reorder_pages([pages], i32(8, 2), i32(2, 4), i32(7), i32(8)),
           lambda: ops.reorder_pages([pages], i32(8, 2).long(), i32(2, 4), i32(8), i32(8)), lambda: ops.reorder_pages([], i32(8, 2), i32(2, 4), i32(8), i32(8)),
           lambda: ops.reorder_pages([pages, torch.zeros(2, 6, 8, 8, device="cuda")], i32(8, 2), i32(2, 4), i32(8), i32(8)),
           lambda: ops.reorder_pages([pages[:, :, :, :4]], i32(8, 2), i32(2, 4), i32(8), i32(8)), lambda: ops.reorder_pages([pages], i32(33, 2), i32(1, 33), i32(33), i32(33)),
           lambda: ops.reorder_slots([pages], i32(7), i32(2, 4)), lambda: ops.reorder_slots([], i32(8), i32(2, 4)), lambda: ops.reorder_slots([pages], i32(8), i32(8))]
    for i, call in enumerate(bad):
        with pytest.raises(ops.KernelError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_reorderings_of_nothing_count_no_launch():
    from quench6k_b200 import ops
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")
    pages, states = [torch.ones(2, 3, 4, 8, device="cuda")], [torch.ones(5, 8, device="cuda")]
    before = ops.launch_count
    ops.reorder_pages(pages, i32(0, 3), i32(0, 2), i32(0), i32(0))
    ops.reorder_pages(pages, i32(2, 0), i32(1, 2), i32(2), i32(2))
    ops.reorder_slots(states, i32(0), i32(0, 2))
    assert ops.launch_count == before and bool((pages[0] == 1).all()) and bool((states[0] == 1).all())
    ops.reorder_pages(pages, i32(2, 3), i32(1, 2), i32(2), i32(2))
    ops.reorder_slots(states, torch.arange(2, dtype=torch.int32, device="cuda"), i32(1, 2))
    assert ops.launch_count == before + 2
