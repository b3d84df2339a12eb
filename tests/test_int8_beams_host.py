"""Calls that are refused before any kernel is launched, seen without a GPU: operands on the host."""
import pytest
import torch

from quench6k_b200 import ops


def test_operands_on_the_host_are_refused():
    q, s = torch.zeros(4, 32, dtype=torch.int8), torch.ones(4)
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32)
    for call in (lambda: ops.quantize_rows(torch.zeros(4, 32)), lambda: ops.gemm_i8(q, s, q, s), lambda: ops.linear_i8(torch.zeros(4, 32), q, s),
                 lambda: ops.beam_select(torch.zeros(4, 32), torch.zeros(1, 4), 4), lambda: ops.PageSet([torch.zeros(1, 2, 4, 8)]),
                 lambda: ops.SlotSet([torch.zeros(4, 8)]), lambda: ops.reorder_pages([torch.zeros(1, 2, 4, 8)], i32(4, 1), i32(1, 4), i32(4), i32(4)),
                 lambda: ops.reorder_slots([torch.zeros(4, 8)], i32(4), i32(1, 4))):
        with pytest.raises(ops.KernelError, match="CUDA device only"):
            call()


def test_a_type_without_kernels_is_refused():
    with pytest.raises(ops.KernelError, match="float32 or bfloat16"):
        ops.quantize_rows(torch.zeros(4, 32, dtype=torch.float64))


def test_scratch_for_picked_rows():
    """Rows that the product of few rows reads where they are take none; others are brought side by side, with their scales."""
    assert [ops._gemm_i8_scratch(rows, 100, 1024, False, False) for rows in (0, 1, 8, 9, 12, 16)] == [0] * 6
    assert ops._gemm_i8_scratch(17, 100, 1024, False, False) == 17 * 1028
    # sixteen rows against 32 MB of weights and more go to the tiles
    assert ops._gemm_i8_scratch(12, 32768, 1024, False, False) == 12 * 1028 and ops._gemm_i8_scratch(12, 32767, 1024, False, False) == 0
    assert ops._gemm_i8_scratch(12, 16384, 1024, True, False) == 12 * 1028 and ops._gemm_i8_scratch(8, 32768, 1024, True, False) == 0
    assert ops._gemm_i8_scratch(3, 100, 1024, True, True) == 3 * 1028 and ops._gemm_i8_scratch(1 << 20, 100, 131056, False, True) == 131060 << 20
