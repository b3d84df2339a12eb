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
