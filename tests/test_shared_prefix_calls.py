"""What a call of the attention over a shared prefix counts, chooses, refuses and reports."""
from __future__ import annotations

import pytest
import torch

from test_answers_of_one_prompt import EVERY_WAY, attention_case, call_attention, ops, way  # noqa: F401  (ops, way: the fixtures)


@pytest.mark.gpu
@EVERY_WAY
def test_kernels_are_counted(ops, way):  # noqa: F811
    case = attention_case(31, torch.bfloat16, 8, 2, 64, 16, 100, [(20, 4), (6, 1), (9, 70)])
    before = ops.launch_count
    call_attention(ops, case)
    assert ops.launch_count - before == (2 if way[0] else 1)   # with the prefix once for all rows its kernel and the one that brings its parts in


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.bfloat16, 80)], ids=["float32", "head size 80"])
def test_kernels_of_the_general_way_are_counted(ops, dtype, dim):  # noqa: F811
    case = attention_case(32, dtype, 4, 2, dim, 16, 40, [(20, 4), (6, 1)])
    before = ops.launch_count
    call_attention(ops, case)
    assert ops.launch_count - before == 2
    empty = {**case, "qkv": case["qkv"][:0], "positions": case["positions"][:0], "seq_starts": case["seq_starts"] * 0}
    call_attention(ops, empty)
    assert ops.launch_count - before == 2
