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


def test_a_plan_is_for_the_switches_it_is_asked_with():
    from tinyllama_inference_engine_b200.ops import fast

    sizes = (8, 8, 12, 32, 8, 128, 64, 500)
    for prefix in (0, 1):
        for own in (0, 1):
            for _ in range(2):
                assert list(fast.shared_prefix_plan(*sizes, prefix, own)[0])[:2] == [prefix, own]
    assert list(fast.shared_prefix_plan(*sizes, None, None)[0]) == list(fast.shared_prefix_plan(*sizes)[0])


@pytest.mark.gpu
def test_a_switch_holds_for_sizes_seen_before(ops, monkeypatch):  # noqa: F811
    case = attention_case(33, torch.bfloat16, 8, 2, 64, 16, 100, [(20, 1), (6, 1)])
    for prefix, own, kernels in ((0, 0, 1), (1, 1, 2), (0, 1, 1), (1, 0, 2), (0, 0, 1)):
        monkeypatch.setattr(ops.fast, "use_prefix", prefix)
        monkeypatch.setattr(ops.fast, "use_own", own)
        before = ops.launch_count
        call_attention(ops, case)
        assert ops.launch_count - before == kernels, (prefix, own)


def test_tables_near_2_to_31_keys_are_refused():
    """The kernels count keys in 32-bit numbers and look up to 2,048 keys ahead of a request's last one."""
    from tinyllama_inference_engine_b200 import ops as plain
    from tinyllama_inference_engine_b200.errors import KernelError

    good = dict(qkv=torch.zeros(3, 4 * 64), pages=torch.zeros(4, 2, 1, 16, 64), positions=torch.zeros(3, dtype=torch.int32), seq_starts=torch.zeros(3, dtype=torch.int32), shared=16,
                out=torch.zeros(3, 4 * 64), q_heads=4, kv_heads=1, head_dim=64, page_size=16)
    one = torch.zeros(1, dtype=torch.int32)
    for width, message in (((1 << 27) - 1, "fewer than 2^31 keys"), ((1 << 27) - 256, "fewer than 2^31 keys"), ((1 << 27) - 257, "contiguous")):   # (the last is let past: what it lacks is something else)
        with pytest.raises(KernelError, match=message.replace("^", r"\^")):
            plain.shared_prefix_attention(block_table=one.expand(2, width), **good)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
def test_an_error_word_made_inside_a_capture_keeps_what_it_holds(ops, dtype, monkeypatch):  # noqa: F811
    """The first call of a process may be a captured one: the device's error word is no part of that graph, whose replays leave what other work has reported."""
    from tinyllama_inference_engine_b200.errors import KernelError

    case = attention_case(34, dtype, 8, 2, 64, 16, 40, [(20, 1), (6, 1)], poison=False)
    c = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in case.items()}
    out = torch.zeros(2, 512, dtype=dtype, device="cuda")
    device = torch.device("cuda:0")
    call_attention(ops, case)
    torch.cuda.synchronize()
    monkeypatch.setattr(ops, "_error_flags", {})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.shared_prefix_attention(c["qkv"], c["pages"], c["positions"], c["seq_starts"], c["table"], c["shared"], out, 8, 2, 64, 16)
    ops.check_device_errors(device)   # nothing has run
    ops.error_flag(device).fill_(4)
    graph.replay()
    with pytest.raises(KernelError, match="learned position vectors"):
        ops.check_device_errors(device)
    graph.replay()
    ops.check_device_errors(device)
    c["table"][0, 1] = 1 << 30
    for _ in range(2):   # what a replay reports is not lost to the next one
        graph.replay()
    c["table"].copy_(case["table"])
    graph.replay()
    with pytest.raises(KernelError, match="outside the pool"):
        ops.check_device_errors(device)
    assert torch.equal(out, call_attention(ops, case))
