"""Rows and products in 8-bit integers against the formulas in NumPy (float32 steps where the definition has them) and 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -24                                       # half a step of float32
BF16_HALF = 2.0 ** -8


def quantized(x):
    """The definition in NumPy, value by value in float32: (q int8, scale float32) of float32 rows."""
    x = np.asarray(x, dtype=np.float32)
    a = np.abs(x).max(axis=1)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        u = np.float32(1) / a * np.float32(127)
        finite = np.isfinite(a)
        zero = ~finite | ~np.isfinite(u)
        q = np.rint(x * np.where(zero, np.float32(0), u)[:, None])
    q = np.where(zero[:, None], 0, np.nan_to_num(q)).astype(np.int8)
    return q, np.where(~finite, np.float32(np.nan), np.where(zero, np.float32(0), a * (np.float32(1) / np.float32(127)))).astype(np.float32)


def rows_of(seed, rows, cols, dtype, apart=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols + apart, generator=g) * 3).to(dtype)
    return x.cuda()[:, :cols], x[:, :cols].float().numpy()


def check_quantized(x_dev, x):
    from quench6k_b200 import ops
    q, scale = ops.quantize_rows(x_dev)
    want_q, want_scale = quantized(x)
    assert q.dtype == torch.int8 and scale.dtype == torch.float32
    np.testing.assert_array_equal(q.cpu().numpy(), want_q)
    np.testing.assert_array_equal(scale.cpu().numpy(), want_scale)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols,apart", [(1, 1, 0), (3, 7, 0), (2, 16, 0), (5, 255, 1), (4, 2048, 0), (33, 2049, 7), (1, 20000, 0), (7, 8192, 8),
                                             (600, 1000, 0), (2, 131056, 0), (1000, 64, 64), (3000, 40, 0)])
def test_rows_in_8_bits(rows, cols, apart, dtype):
    check_quantized(*rows_of(rows * 7 + cols, rows, cols, dtype, apart))


def test_rows_that_start_off_16_bytes():
    x = torch.randn(9, 100, generator=torch.Generator().manual_seed(1)).cuda()
    check_quantized(x[:, 3:90], x[:, 3:90].cpu().numpy())
    b = x.bfloat16()
    check_quantized(b[:, 1:98], b[:, 1:98].float().cpu().numpy())


def test_rows_of_zeros_ties_and_values_that_are_not_finite():
    x = torch.zeros(9, 40)
    x[1, 3] = float("nan")
    x[2, 5] = float("inf")
    x[3, 39], x[3, 0] = -float("inf"), 1.0
    x[4] = torch.arange(40) + 0.5                       # with 127 as the largest value the products are whole and a half
    x[4, 39] = 127.0
    x[5, 7] = 3.0e-38                                   # 127 over it is infinite
    x[6, 7] = 4.0e-37                                   # and here not
    x[7, 2] = torch.finfo(torch.float32).max
    x[8, 2] = -1e-45
    check_quantized(x.cuda(), x.numpy())


def test_no_rows():
    from quench6k_b200 import ops
    q, scale = ops.quantize_rows(torch.empty(0, 32, device="cuda"))
    assert q.shape == (0, 32) and scale.shape == (0,)
    y = ops.linear_i8(torch.empty(0, 32, device="cuda"), torch.zeros(5, 32, dtype=torch.int8, device="cuda"), torch.ones(5, device="cuda"))
    assert y.shape == (0, 5)


# ----------------------------------------------------------------------------------------------- products
def operands(seed, rows, n, k, experts=None, mats=1):
    """int8 rows and matrices with their scales, on the host."""
    g = torch.Generator().manual_seed(seed)
    ints = lambda *s: torch.randint(-127, 128, s, generator=g, dtype=torch.int8)
    lead = () if experts is None else (experts,)
    a, s = ints(rows, k), torch.rand(rows, generator=g) * 0.02 + 0.001
    return a, s, [(ints(*lead, n, k), torch.rand(*lead, n, generator=g) * 1e-3 + 1e-4) for _ in range(mats)]


def product64(a, s, w, t):
    """The scaled product in 64 bits (the integers are exact there)."""
    return (a.double() @ w.double().T) * (s.double()[:, None] * t.double()[None, :])


def gated64(g, u, act):
    if act is None or act == "silu":
        return g * torch.sigmoid(g) * u
    if act == "gelu_tanh":
        return 0.5 * g * (1 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g ** 3))) * u
    if act == "relu2":
        return g.clamp(min=0) ** 2 * u
    limit = act[1]
    g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return g * torch.sigmoid(1.702 * g) * (u + 1)


def near(got, want, rel, abs_=0.0):
    got, want = got.double().cpu(), want.double().cpu()
    assert got.shape == want.shape
    off = (got - want).abs()
    assert bool((off <= rel * want.abs() + abs_).all()), f"off by {float((off / (want.abs() + 1e-300)).max()):.3g} of a value, allowed {rel:.3g}"


# The sum leaves the integers with one rounding, the scales' product and the product with it have one each.
STORED = 3 * HALF * (1 + 1e-6)
# Of a gated result the rounding to bfloat16, and what the FP32 steps before it can move it: relative to the result |v f'(v) / f(v)| <= 1 + |v|
# times the gate's three roundings, the other product's three, and some ten of the gate's own arithmetic; |v| <= 200 in these tests.
GATED = BF16_HALF + (3 * 201 + 3 + 10 + 201) * HALF

SHAPES = [(1, 1, 16), (1, 2048, 2048), (2, 100, 48), (3, 17, 1024), (8, 64, 64), (9, 4097, 80), (16, 129, 4096), (17, 128, 128), (32, 1000, 2048), (33, 257, 272),
          (64, 384, 512), (100, 640, 1040), (129, 300, 144), (200, 129, 8192), (257, 512, 2064), (300, 7, 16), (1000, 1024, 256),
          (17, 512, 10240), (100, 200, 8208), (48, 2048, 8192), (250, 1100, 4112), (130, 90, 1168), (13, 17000, 2048), (8, 17000, 2048)]      # few tiles and long rows: K in slices


@pytest.mark.parametrize("rows,n,k", SHAPES)
def test_product(rows, n, k):
    from quench6k_b200 import ops
    a, s, ((w, t),) = operands(rows + n + k, rows, n, k)
    y = ops.gemm_i8(a.cuda(), s.cuda(), w.cuda(), t.cuda())
    assert y.dtype == torch.float32
    near(y, product64(a, s, w, t), STORED)


@pytest.mark.parametrize("rows,n,k", [(1, 300, 512), (12, 129, 64), (40, 256, 2048), (300, 520, 528), (30, 300, 8192)])
def test_product_added(rows, n, k):
    from quench6k_b200 import ops
    a, s, ((w, t),) = operands(rows, rows, n, k)
    base = torch.randn(rows, n, generator=torch.Generator().manual_seed(3))
    out = base.cuda()
    assert ops.gemm_i8(a.cuda(), s.cuda(), w.cuda(), t.cuda(), out=out, accumulate=True) is out
    y = product64(a, s, w, t)
    off = (out.double().cpu() - (base.double() + y)).abs()
    assert bool((off <= STORED * y.abs() + HALF * 1.01 * (base.double() + y).abs()).all())


@pytest.mark.parametrize("act", [None, "gelu_tanh", "relu2", ("clamped", 7.0)])
@pytest.mark.parametrize("rows,n,k", [(1, 512, 2048), (16, 130, 272), (70, 129, 512), (600, 300, 1040), (1200, 1024, 256), (40, 250, 8192), (200, 70, 4112)])
def test_gated_product(rows, n, k, act):
    from quench6k_b200 import ops
    a, s, ((w, t), (w2, t2)) = operands(rows * 3 + n, rows, n, k, mats=2)
    s = s * 0.02                                       # gates of a few units
    y = ops.gemm_i8(a.cuda(), s.cuda(), w.cuda(), t.cuda(), w2=w2.cuda(), w2_scale=t2.cuda(), act=act)
    assert y.dtype == torch.bfloat16
    g, u = product64(a, s, w, t), product64(a, s, w2, t2)
    assert float(g.abs().max()) < 200
    # the clamped form adds 1 to its second factor, and gelu's 1 + tanh cancels for negative gates: there an FP32 rounding of a sum near 1 counts in full
    near(y, gated64(g, u, act), GATED, abs_=float(8 * HALF * (g.abs() * (u.abs() + 1)).max()))


@pytest.mark.parametrize("rows,n,k,gated", [(129, 20000, 48, False), (193, 20000, 16, False), (961, 11000, 32, False), (2048, 8192, 144, False),
                                            (129, 11000, 48, True), (385, 11000, 48, True), (1290, 8192, 64, True), (1281, 8192, 128, True)])
def test_product_whose_last_tiles_are_cut(rows, n, k, gated):
    """More tiles than run at a time and few in the last round; some pieces of those have no row.  The memory behind the result stays as it was."""
    from quench6k_b200 import ops
    a, s, mats = operands(rows + k, rows, n, k, mats=2 if gated else 1)
    s = s * 0.02
    (w, t), more = mats[0], {}
    if gated:
        more = {"w2": mats[1][0].cuda(), "w2_scale": mats[1][1].cuda()}
    out = torch.full((rows + 300, n), 7.0, dtype=torch.bfloat16 if gated else torch.float32, device="cuda")
    ops.gemm_i8(a.cuda(), s.cuda(), w.cuda(), t.cuda(), out=out, **more)
    g = product64(a, s, w, t)
    if gated:
        u = product64(a, s, *mats[1])
        near(out[:rows], gated64(g, u, None), GATED, 1e-30)
    else:
        near(out[:rows], g, STORED)
    assert bool((out[rows:] == 7.0).all())


@pytest.mark.parametrize("act", ["silu", "relu2"])
@pytest.mark.parametrize("rows,n,k", [(5, 64, 128), (150, 300, 256), (20, 100, 6144)])
def test_activated_product(rows, n, k, act):
    from quench6k_b200 import ops
    a, s, ((w, t),) = operands(rows, rows, n, k)
    y = ops.gemm_i8(a.cuda(), s.cuda(), w.cuda(), t.cuda(), act=act)
    assert y.dtype == torch.bfloat16
    g = product64(a, s, w, t)
    near(y, gated64(g, torch.ones_like(g), act), GATED, 1e-30)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("counts,n,k", [([3, 0, 1, 17], 40, 64), ([0, 0, 0], 16, 32), ([1] * 9, 130, 272), ([130, 0, 257, 5, 64], 200, 512), ([0, 500, 3], 129, 128),
                                        ([20] * 64, 64, 256)])
def test_grouped_product(counts, n, k, gated):
    """Rows by group, gathered; rows behind the last group stay as they were."""
    from quench6k_b200 import ops
    total, behind = sum(counts), 4
    a, s, mats = operands(total + n, 50, n, k, experts=len(counts), mats=2 if gated else 1)
    if gated:
        s = s * 0.02
    g = torch.Generator().manual_seed(9)
    pick = torch.randint(0, 50, (total + behind,), generator=g, dtype=torch.int32)
    offsets = torch.tensor([0] + counts).cumsum(0).int()
    out = torch.full((total + behind, n), 77.0, dtype=torch.bfloat16 if gated else torch.float32, device="cuda")
    more = dict(w2=mats[1][0].cuda(), w2_scale=mats[1][1].cuda()) if gated else {}
    ops.gemm_i8(a.cuda(), s.cuda(), mats[0][0].cuda(), mats[0][1].cuda(), out=out, offsets=offsets.cuda(), a_rows=pick.cuda(), **more)
    assert bool((out[total:] == 77.0).all())
    for e in range(len(counts)):
        at = slice(int(offsets[e]), int(offsets[e + 1]))
        p = pick[at].long()
        y = product64(a[p], s[p], mats[0][0][e], mats[0][1][e])
        if gated:
            near(out[at], gated64(y, product64(a[p], s[p], mats[1][0][e], mats[1][1][e]), None), GATED, 1e-30)
        else:
            near(out[at], y, STORED)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("tokens,top,n,k", [(1, 8, 512, 2048), (3, 2, 33, 80), (16, 4, 128, 1024), (5, 1, 7, 16), (16, 8, 200, 512), (16, 8, 170, 2064)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_product_pair_by_pair(tokens, top, n, k, gated, dtype):
    """One row for each (token, expert); a pair that names no matrix is left as it was."""
    from quench6k_b200 import ops
    experts = 12
    _, _, mats = operands(tokens + n, 1, n, k, experts=experts, mats=2 if gated else 1)
    x, host = rows_of(tokens, tokens, k, dtype)
    e = torch.randint(0, experts + 3, (tokens, top), generator=torch.Generator().manual_seed(4), dtype=torch.int32).view(-1)
    e[0] = experts - 1
    if e.numel() > 2:
        e[1], e[2] = experts, -1
    out = torch.full((tokens * top, n), 77.0, dtype=torch.bfloat16 if gated else torch.float32, device="cuda")
    more = dict(w2=mats[1][0].cuda(), w2_scale=mats[1][1].cuda() * 0.02) if gated else {}
    ops.linear_i8(x, mats[0][0].cuda(), mats[0][1].cuda() * 0.02, out=out, pair_expert=e.cuda(), pair_div=top, **more)
    q, s = (torch.from_numpy(v) for v in quantized(host))
    for i, g in enumerate(e.tolist()):
        row = slice(i // top, i // top + 1)
        if not 0 <= g < experts:
            assert bool((out[i] == 77.0).all())
            continue
        y = product64(q[row], s[row], mats[0][0][g], mats[0][1][g] * 0.02)
        if gated:
            near(out[i:i + 1], gated64(y, product64(q[row], s[row], mats[1][0][g], mats[1][1][g] * 0.02), None), GATED, 1e-30)
        else:
            near(out[i:i + 1], y, STORED)


@pytest.mark.parametrize("old", [False, True])
@pytest.mark.parametrize("k", [16, 2032, 4096, 8192])
@pytest.mark.parametrize("bad", [False, True])
def test_one_row_taken_to_8_bits_inside_the_product(k, bad, old):
    """The same numbers as in two calls, for rows of zeros and rows that are not finite too."""
    from quench6k_b200 import ops
    _, _, ((w, t), (w2, t2)) = operands(k, 1, 333, k, mats=2)
    w, t, w2, t2 = w.cuda(), t.cuda() * 0.01, w2.cuda(), t2.cuda() * 0.01
    rows = [rows_of(3, 1, k, torch.bfloat16)[0].contiguous(), torch.zeros(1, k, dtype=torch.bfloat16, device="cuda")]
    if bad:
        rows[0][0, k - 1], rows[1][0, 0] = float("nan"), -float("inf")
    for x in rows:
        q, s = ops.quantize_rows(x)
        for more in ({}, {"w2": w2, "w2_scale": t2}, {"act": "relu2"}):
            assert torch.equal(ops.linear_i8(x, w, t, weights_are_old=old, **more).nan_to_num(7.0), ops.gemm_i8(q, s, w, t, **more).nan_to_num(7.0))


@pytest.mark.parametrize("rows", [1, 4, 7, 16, 17, 40, 130])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_product_of_rows_taken_to_8_bits_has_the_bits_of_the_two_calls(rows, dtype):
    from quench6k_b200 import ops
    x, _ = rows_of(rows, rows, 528, dtype, apart=16)
    _, _, ((w, t), (w2, t2)) = operands(5, 1, 700, 528, mats=2)
    w, t, w2, t2 = w.cuda(), t.cuda() * 0.01, w2.cuda(), t2.cuda() * 0.01
    q, s = ops.quantize_rows(x)
    assert torch.equal(ops.linear_i8(x, w, t), ops.gemm_i8(q, s, w, t))
    assert torch.equal(ops.linear_i8(x, w, t, w2=w2, w2_scale=t2), ops.gemm_i8(q, s, w, t, w2=w2, w2_scale=t2))


def test_largest_sums_are_exact():
    """The longest rows of the largest values: 131,056 products of 128 x 128 stay below 2^31."""
    from quench6k_b200 import ops
    k = 131056
    for rows in (2, 40):
        a = torch.full((rows, k), -128, dtype=torch.int8, device="cuda")
        w = torch.full((3, k), -128, dtype=torch.int8, device="cuda")
        w[1] = 127
        one = torch.ones(rows, device="cuda")
        y = ops.gemm_i8(a, one, w, torch.ones(3, device="cuda"))
        want = torch.tensor([128 * 128 * k, -128 * 127 * k, 128 * 128 * k], dtype=torch.float64).float()
        assert torch.equal(y.cpu(), want.expand(rows, 3))


@pytest.mark.parametrize("rows", [3, 50])
def test_a_row_that_is_not_finite_makes_its_results_nan_and_no_other(rows):
    from quench6k_b200 import ops
    x, _ = rows_of(2, rows, 256, torch.bfloat16)
    x = x.clone()
    x[1, 9] = float("inf")
    _, _, ((w, t),) = operands(6, 1, 200, 256)
    y = ops.linear_i8(x, w.cuda(), t.cuda())
    assert bool(y[1].isnan().all()) and not bool(y[[i for i in range(rows) if i != 1]].isnan().any())


@pytest.mark.parametrize("rows,n", [(5, 100), (12, 100), (12, 33000), (40, 100)])
def test_rows_that_are_picked(rows, n):
    """Without groups: some twice, some not at all."""
    from quench6k_b200 import ops
    a, s, ((w, t),) = operands(rows, 20, n, 1024)
    pick = torch.randint(0, 20, (rows,), generator=torch.Generator().manual_seed(rows), dtype=torch.int32)
    near(ops.gemm_i8(a.cuda(), s.cuda(), w.cuda(), t.cuda(), a_rows=pick.cuda()), product64(a[pick.long()], s[pick.long()], w, t), STORED)


@pytest.mark.parametrize("rows,n,launches,scratch", [(8, 100, 1, 0), (9, 100, 1, 0), (16, 100, 1, 0), (17, 100, 2, 17 * 1028), (9, 33000, 2, 9 * 1028)])
def test_picked_rows_take_the_launches_and_the_memory_that_are_counted(rows, n, launches, scratch, monkeypatch):
    from quench6k_b200 import ops
    a, s, ((w, t),) = operands(rows, 20, n, 1024)
    a, s, w, t = a.cuda(), s.cuda(), w.cuda(), t.cuda()
    pick = torch.randint(0, 20, (rows,), generator=torch.Generator().manual_seed(rows), dtype=torch.int32).cuda()
    out = torch.empty(rows, n, device="cuda")
    taken, empty = [], torch.empty
    monkeypatch.setattr(torch, "empty", lambda *size, **kw: (taken.append(size), empty(*size, **kw))[1])
    before = ops.launch_count
    ops.gemm_i8(a, s, w, t, out=out, a_rows=pick)
    assert ops.launch_count - before == launches and taken == ([(scratch,)] if scratch else [])


@pytest.mark.parametrize("rows,n", [(5, 100), (12, 33000), (40, 100)])
def test_a_picked_row_that_is_none_is_a_row_of_nan(rows, n):
    from quench6k_b200 import ops
    a, s, ((w, t),) = operands(rows, 20, n, 256)
    pick = torch.randint(0, 20, (rows,), generator=torch.Generator().manual_seed(rows), dtype=torch.int32)
    bad = torch.zeros(rows, dtype=torch.bool)
    pick[0], pick[2], pick[4] = -1, 20, 2 ** 31 - 1
    bad[[0, 2, 4]] = True
    y = ops.gemm_i8(a.cuda(), s.cuda(), w.cuda(), t.cuda(), a_rows=pick.cuda()).cpu()
    assert bool(y[bad].isnan().all())
    near(y[~bad], product64(a[pick[~bad].long()], s[pick[~bad].long()], w, t), STORED)


@pytest.mark.parametrize("rows", [4, 200])
def test_operands_whose_rows_lie_apart(rows):
    from quench6k_b200 import ops
    a, s, ((w, t),) = operands(8, rows, 65, 112)
    wide = torch.zeros(rows, 160, dtype=torch.int8)
    wide[:, 16:128] = a
    y = ops.gemm_i8(wide.cuda()[:, 16:128], s.cuda(), w.cuda(), t.cuda())
    near(y, product64(a, s, w, t), STORED)


@pytest.mark.parametrize("rows", [3, 90])
def test_products_in_two_recordings_and_on_another_stream(rows):
    """Two recorded calls replayed by turns, and a call on a stream of its own, give the bits of the eager call."""
    from quench6k_b200 import ops
    _, _, ((w, t),) = operands(11, 1, 300, 512)
    w, t = w.cuda(), t.cuda()
    xs = [rows_of(20 + i, rows, 512, torch.bfloat16)[0].contiguous() for i in range(2)]
    want = [ops.linear_i8(x, w, t) for x in xs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.linear_i8(x, w, t))
        graphs.append(g)
    for o in outs:
        o.zero_()
    for i in (0, 1, 0, 1):
        graphs[i].replay()
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        apart = ops.linear_i8(xs[0], w, t)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(apart, want[0])
    assert ops.tc_status() == 0


def test_refusals():
    from quench6k_b200 import ops
    a, s = torch.zeros(4, 32, dtype=torch.int8, device="cuda"), torch.zeros(4, device="cuda")
    w, t = torch.zeros(8, 32, dtype=torch.int8, device="cuda"), torch.zeros(8, device="cuda")
    bad = [lambda: ops.gemm_i8(a.float(), s, w, t), lambda: ops.gemm_i8(a, s[:3], w, t), lambda: ops.gemm_i8(a, s, w, t[:7]),
           lambda: ops.gemm_i8(a, s, w.view(2, 4, 32), t.view(2, 4)), lambda: ops.gemm_i8(a[:, :24], s, w[:, :24].contiguous(), t),
           lambda: ops.gemm_i8(a, s, w, t, accumulate=True), lambda: ops.gemm_i8(a, s, w, t, w2=w), lambda: ops.gemm_i8(a, s, w, t, w2=w[:4], w2_scale=t[:4]),
           lambda: ops.gemm_i8(a, s, w, t, out=torch.zeros(4, 8, dtype=torch.bfloat16, device="cuda")), lambda: ops.gemm_i8(a, s, w, t, act="tanh"),
           lambda: ops.gemm_i8(a, s, w, t, act=("clamped", 1.0)), lambda: ops.gemm_i8(a[:, 1:17], s, w[:, :16].contiguous(), t),
           lambda: ops.gemm_i8(a, s, w.view(2, 4, 32), t.view(2, 4), offsets=torch.zeros(2, dtype=torch.int32, device="cuda")),
           lambda: ops.gemm_i8(a, s, w, t, w2=w, w2_scale=t, out=torch.zeros(4, 8, device="cuda"), accumulate=True),
           lambda: ops.linear_i8(torch.zeros(4, 32, dtype=torch.float16, device="cuda"), w, t), lambda: ops.linear_i8(torch.zeros(4, 48, device="cuda"), w, t),
           lambda: ops.linear_i8(torch.zeros(4, 32, device="cuda"), w.view(2, 4, 32), t.view(2, 4), pair_expert=torch.zeros(9, dtype=torch.int32, device="cuda"), pair_div=2),
           lambda: ops.quantize_rows(torch.zeros(4, 0, device="cuda")), lambda: ops.quantize_rows(torch.zeros(4, 8, device="cuda").T),
           lambda: ops.quantize_rows(torch.zeros(4, device="cuda"))]
    for i, call in enumerate(bad):
        with pytest.raises(ops.KernelError):
            call()
            pytest.fail(f"call {i} was not refused")
