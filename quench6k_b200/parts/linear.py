"""Chooses the matrix-product kernel for an operand dtype and shape.

float32 operands always take the CUDA-core FP32 kernel (no reduced-precision matrix mode exists on
that path).  bfloat16 operands take the tcgen05 tensor-core kernel where the shape allows (K a
multiple of 8, rows starting on 16 bytes), the matrix-vector kernel or the mma.sync kernel for few tokens where the
library prefers them (steps of at most 16 tokens), and the CUDA-core kernel otherwise.

A matrix that is kept in 8 bits (Int8Matrix, what to_weight makes where the runtime asks for it) takes the products in 8-bit
integers instead, whatever the number of rows: the rows are taken to 8 bits with a scale each, the sums are exact.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import ops
from .base import to_operand


def _tc(a: torch.Tensor, w: torch.Tensor, rt) -> bool:
    return rt.tensor_cores and not rt.is_fp32 and ops.tc_supported(a, w)


class Int8Matrix:
    """A matrix [N, K] (or one for each group, [G, N, K]) in 8 bits with a scale for each of its rows."""

    def __init__(self, q: torch.Tensor, scale: torch.Tensor):
        self.q, self.scale = q, scale

    @property
    def shape(self):
        return self.q.shape

    def __getitem__(self, rows: slice) -> "Int8Matrix":
        """Neighbouring rows of it."""
        return Int8Matrix(self.q[rows], self.scale[rows])


def int8_rows_allowed(K: int) -> bool:
    return K % 16 == 0 and 0 < K < 131072


def to_weight(t: torch.Tensor, rt):
    """A stored matrix as the products consume it: in the operand dtype, or in 8 bits where the runtime keeps its weights so and
    the kernels take its rows.  Those 8 bits are the only rounding: a matrix stored in 32 bits does not pass through the operand dtype."""
    if not rt.int8_weights or not int8_rows_allowed(t.shape[-1]):
        return to_operand(t, rt)
    w = t.to(device=rt.device, dtype=t.dtype if t.dtype == torch.bfloat16 else torch.float32).contiguous()
    q, scale = ops.quantize_rows(w.view(-1, w.shape[-1]))
    return Int8Matrix(q.view(w.shape), scale.view(w.shape[:-1]))


def stacked_weight(rows: int, K: int, pieces, get, rt):
    """The same for one matrix [rows, K] of stored matrices, (first row, tensor name) each; rows that none of them covers are zeros.
    The tensors are fetched and put in their places one by one, so that no two copies of all of them are held at once."""
    if rt.int8_weights and int8_rows_allowed(K):
        w = Int8Matrix(torch.zeros((rows, K), dtype=torch.int8, device=rt.device), torch.zeros(rows, dtype=torch.float32, device=rt.device))
        for at, name in pieces:
            part = to_weight(get(name), rt)
            w.q[at:at + part.shape[0]].copy_(part.q)
            w.scale[at:at + part.shape[0]].copy_(part.scale)
            del part
        return w
    w = torch.zeros((rows, K), dtype=rt.dtype, device=rt.device)
    for at, name in pieces:
        part = get(name)
        w[at:at + part.shape[0]].copy_(part)
        del part
    return w


def matmul(a: torch.Tensor, w: torch.Tensor, rt, out: Optional[torch.Tensor] = None, accumulate: bool = False,
           partials_ok: bool = False) -> torch.Tensor:
    """FP32 out[r] (+)= a[r] @ w^T;  a: [M, K], w: [N, K].  partials_ok: the caller's next kernel
    can sum split-K partial products itself, so the result may come as [slices, M, N] (a view of
    the device's scratch buffer: consume it before the next kernel that uses scratch)."""
    if isinstance(w, Int8Matrix):
        return ops.linear_i8(a, w.q, w.scale, out=out, accumulate=accumulate, weights_are_old=True)
    if _tc(a, w, rt):
        if ops.gemv_preferred(a.shape[0], w.shape[0], w.shape[1]):       # a token or two: the matrix-vector kernel
            return ops.gemv(a, w, out=out, accumulate=accumulate)
        if ops.gemm_skinny_preferred(a.shape[0], w.shape[0], w.shape[1]):  # up to 16 tokens against many rows: mma.sync, K not split over blocks
            return ops.gemm_skinny(a, w, out=out, accumulate=accumulate)
        if partials_ok and out is None and not accumulate and w.shape[0] % 4 == 0:
            slices = ops.gemm_skinny_slices(a.shape[0], w.shape[0], w.shape[1])
            if slices:                                                   # a few tokens against few rows: the same kernel, K in slices
                return ops.gemm_skinny(a, w, slices=slices)
            return ops.gemm_tc(a, w, keep_partials=True)
        return ops.gemm_tc(a, w, out=out, accumulate=accumulate)
    return ops.gemm_simt(a, w, out=out, accumulate=accumulate)


def swiglu_matmul(a: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, rt, act=None) -> torch.Tensor:
    """y[r] = act(a[r] @ w_gate^T) * (a[r] @ w_up^T) in a's dtype; act None: silu."""
    if isinstance(w_gate, Int8Matrix):
        return ops.linear_i8(a, w_gate.q, w_gate.scale, w2=w_up.q, w2_scale=w_up.scale, act=act, weights_are_old=True)
    if _tc(a, w_gate, rt):
        # the kernel for one or two tokens takes activations without a constant
        if not ops.act_has_param(act) and ops.gemv_preferred(a.shape[0], w_gate.shape[0], w_gate.shape[1]):
            return ops.gemv(a, w_gate, w2=w_up, act=act)
        if ops.gemm_skinny_preferred(a.shape[0], w_gate.shape[0], w_gate.shape[1]):
            return ops.gemm_skinny(a, w_gate, w2=w_up, act=act)
        return ops.gemm_tc(a, w_gate, w2=w_up, act=act)
    return ops.gemm_simt(a, w_gate, w2=w_up, act=act)


class GroupPlan:
    """The permutation of a step's (token, slot) pairs by expert and the row tiles of the experts'
    groups, for whichever kernel runs them; on the tensor-core path also the gathered input rows."""

    def __init__(self, a: torch.Tensor, sel_e: torch.Tensor, num_groups: int, rt, tc: bool, live: int):
        """num_groups: expert numbers there are; live: those that have matrices (the pairs of the others get no tiles)."""
        self.live = live
        self.pairs, self.tc, self.xs = sel_e.numel(), tc, None
        if tc:
            avg = max(1, self.pairs // max(1, num_groups))
            want = avg + avg // 2
            self.bt_dual = ops.tc_token_tile(want, True)
            self.bt = self.bt_dual
            # permutation, tile list and the gathered input rows in three launches (the last one, a block per pair,
            # finishes the pair's rank and copies its row)
            if a.shape[1] * a.element_size() % 16 == 0:
                self.offsets, self.pair_row, self.row_token, self.tiles, self.xs = ops.moe_plan(sel_e, num_groups, self.bt, a, live=live)
            else:
                self.offsets, self.pair_row, self.row_token, self.tiles = ops.moe_plan(sel_e, num_groups, self.bt, live=live)
                self.xs = ops.gather_rows(a, self.row_token)
        else:
            self.offsets, self.pair_row, self.row_token, self.tiles = ops.moe_plan(sel_e, num_groups, ops.simt_tile_rows(), live=live)


class Int8Plan:
    """The same for products in 8-bit integers: the groups' first rows, the rows' tokens, and the input rows in 8 bits (they are
    gathered by the product)."""

    def __init__(self, a: torch.Tensor, sel_e: torch.Tensor, num_groups: int, live: int):
        self.pairs = sel_e.numel()
        offsets, self.pair_row, self.row_token = ops.moe_permute(sel_e, num_groups)
        self.offsets = offsets[:live + 1]              # the pairs of experts without matrices come last
        self.q, self.scale = ops.quantize_rows(a)


def group_plan(a: torch.Tensor, w: torch.Tensor, sel_e: torch.Tensor, rt, without: int = 0):
    """without: expert numbers beyond the last matrix of w, whose pairs take part in no product."""
    if isinstance(w, Int8Matrix):
        return Int8Plan(a, sel_e, w.shape[0] + without, w.shape[0])
    return GroupPlan(a, sel_e, w.shape[0] + without, rt, _tc(a, w, rt) and a.is_contiguous(), w.shape[0])


def grouped_swiglu(a: torch.Tensor, plan: GroupPlan, w_gate: torch.Tensor, w_up: torch.Tensor, rt, act=None) -> torch.Tensor:
    """y[row] = act(x w_gate^T) * (x w_up^T) for x = a[row_token[row]] with the weights of the row's group (act None: silu); [pairs, I]."""
    if isinstance(plan, Int8Plan):
        return ops.gemm_i8(plan.q, plan.scale, w_gate.q, w_gate.scale, w2=w_up.q, w2_scale=w_up.scale, act=act, offsets=plan.offsets, a_rows=plan.row_token)
    if plan.tc:
        return ops.gemm_tc(plan.xs, w_gate, w2=w_up, groups=plan.tiles, bt=plan.bt, rows=plan.pairs, act=act)
    return ops.gemm_simt(a, w_gate, w2=w_up, a_rows=plan.row_token, groups=plan.tiles, rows=plan.pairs, act=act)


def grouped_activated(a: torch.Tensor, plan: GroupPlan, w: torch.Tensor, rt, act: str) -> torch.Tensor:
    """y[row] = act(a[row_token[row]] @ w_g^T) in a's dtype with the weights of the row's group: the first product of
    experts that have no gate; [pairs, N]."""
    if isinstance(plan, Int8Plan):
        return ops.gemm_i8(plan.q, plan.scale, w.q, w.scale, act=act, offsets=plan.offsets, a_rows=plan.row_token)
    if plan.tc:
        return ops.gemm_tc(plan.xs, w, groups=plan.tiles, bt=plan.bt, rows=plan.pairs, act=act)
    return ops.gemm_simt(a, w, a_rows=plan.row_token, groups=plan.tiles, rows=plan.pairs, act=act)


def grouped_matmul(a: torch.Tensor, plan: GroupPlan, w: torch.Tensor, rt) -> torch.Tensor:
    """FP32 y[row] = a[row] @ w_g^T with the weights of the row's group; [pairs, N]."""
    if isinstance(plan, Int8Plan):
        q, scale = ops.quantize_rows(a)
        return ops.gemm_i8(q, scale, w.q, w.scale, offsets=plan.offsets, early=True)
    if plan.tc and ops.tc_supported(a, w):
        return ops.gemm_tc(a, w, groups=plan.tiles, bt=plan.bt, rows=plan.pairs)
    if plan.tc:
        return ops.gemm_simt(a, w, groups=ops.tile_list(plan.tiles[0][:plan.live + 1], plan.pairs, ops.simt_tile_rows()), rows=plan.pairs)
    return ops.gemm_simt(a, w, groups=plan.tiles, rows=plan.pairs)


_uniform = {}


def _uniform_groups(groups: int, rows_per_group: int, bm: int, device):
    """The tile list of `groups` groups of equal size, rows group-major; made once per shape (outside any recording) and kept:
    recorded CUDA graphs point at it."""
    key = (groups, rows_per_group, bm, str(device))
    if key not in _uniform:
        offsets = (torch.arange(groups + 1, dtype=torch.int32) * rows_per_group).to(device)
        _uniform[key] = ops.tile_list(offsets, groups * rows_per_group, bm)
    return _uniform[key]


def pair_products(a: torch.Tensor, sel_e: torch.Tensor, per_row: int, w: "Int8Matrix", w_up: Optional["Int8Matrix"] = None, act=None) -> torch.Tensor:
    """A step of few tokens: y[p] = a[p // per_row] @ w_e^T for the expert e of pair p, FP32 (or act of it, or the gated form with
    w_up, in bfloat16), straight from the selection."""
    more = {} if w_up is None else {"w2": w_up.q, "w2_scale": w_up.scale}
    return ops.linear_i8(a, w.q, w.scale, act=act, pair_expert=sel_e.view(-1), pair_div=per_row, **more)


def batched_matmul(a: torch.Tensor, w: torch.Tensor, rt, rows_per_group: int, rounded: bool = False) -> torch.Tensor:
    """FP32 y[g M + r] = a[g M + r] @ w[g]^T for G groups of M = rows_per_group rows each: one product per head, the rows
    laid out head by head.  a: [G M, K], w: [G, N, K].  rounded: y in bfloat16 (for a consumer that would round it first)."""
    G = w.shape[0]
    total = G * rows_per_group
    if _tc(a, w, rt) and a.is_contiguous():
        bt = ops.tc_token_tile(rows_per_group, False)
        return ops.gemm_tc(a, w, groups=_uniform_groups(G, rows_per_group, bt, a.device), bt=bt, rows=total, rounded=rounded)
    y = ops.gemm_simt(a, w, groups=_uniform_groups(G, rows_per_group, ops.simt_tile_rows(), a.device), rows=total)
    return ops.cast_columns(y, 0, y.shape[1], torch.bfloat16) if rounded else y
