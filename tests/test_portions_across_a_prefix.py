"""Portions whose first rows lie inside the shared prefix and whose last ones lie behind it: of a pair of row tiles one then has no key of the request's own."""
from __future__ import annotations

import re
from pathlib import Path

import pytest
import torch

from test_answers_of_one_prompt import U, attention_case, call_attention, compare_attention, ops, plain_attention, way  # noqa: F401  (ops, way: the fixtures)


def test_queries_have_landed_before_their_place_is_used():
    """The kernel that brings the prefix's parts in puts them where the queries lie.  A row tile without keys has waited for none of its products, so it waits for the copy."""
    from tinyllama_inference_engine_b200 import ops

    source = (Path(ops.__file__).parent.parent / "csrc" / "attention_prefix_tc.cu").read_text()
    softmax = source[source.index("} else if (warp >= kFirstSoftmaxWarp) {") :]
    use = softmax.index("reinterpret_cast<float4*>(sm.q[u])")
    assert re.search(r"if \(JOINS && mine == 0 && n > 0\) ok = warp_wait\(&sm\.q_full, 0, gave_up\);", softmax[:use])
    assert "sm.q[u]" not in softmax[:use]


def test_the_plan_takes_the_kernel_that_joins_here():
    from tinyllama_inference_engine_b200 import ops

    assert list(ops.fast.shared_prefix_plan(8 * 128, 8, -(-(4048 + 128) // 64), 32, 8, 128, 64, 4096)[0])[:2] == [1, 1]


@pytest.mark.gpu
@pytest.mark.parametrize("way", [(1, 1, 0, 0), (1, 1, 3, 0), (0, 1, 0, 0)], ids=lambda w: "-".join(map(str, w)), indirect=True)
@pytest.mark.parametrize("heads", [(8, 2, 128), (16, 2, 64), (72, 2, 128)], ids=lambda h: f"{h[0]}-{h[1]}x{h[2]}")
@pytest.mark.parametrize("page_size,shared", [(64, 330), (16, 385)])
def test_portions_that_begin_inside_the_prefix(ops, way, heads, page_size, shared):  # noqa: F811
    tile = 128 // (heads[0] // heads[1])   # rows of a row tile
    entries = [(tile, 2 * tile), (1, tile + 1), (tile // 2, 2 * tile + tile // 2), (0, 2 * tile), (2 * tile, 2 * tile), (3, 3)]
    case = attention_case(21, torch.bfloat16, *heads, page_size, shared, entries, front=1, behind=1)
    compare_attention(call_attention(ops, case), case, *plain_attention(case))


@pytest.mark.gpu
@pytest.mark.parametrize("way", [(1, 1, 0, 0), (1, 1, 2, 0)], ids=lambda w: "-".join(map(str, w)), indirect=True)
def test_row_tiles_that_see_nothing(ops, way):  # noqa: F811
    """Negative positions leave a row tile without any key, in the prefix or behind it."""
    case = attention_case(22, torch.bfloat16, 8, 2, 128, 32, 170, [(64, 64), (64, 64), (40, 64)])
    case["positions"][:32] = -1      # the first of the first portion's two row tiles
    case["positions"][96:128] = -7   # the second of the second's
    got = call_attention(ops, case)
    assert (got[:32] == 0).all() and (got[96:128] == 0).all()
    compare_attention(got, case, *plain_attention(case))


@pytest.mark.gpu
def test_portions_across_a_long_prefix(ops):  # noqa: F811
    """As the plan runs them: 8 portions of 128 rows, 32 heads over 8 of 128, the first 48 rows of each before the end of 4,096 shared keys.  Every call's bits are the same."""
    heads, kv_heads, dim, page_size, shared, rows = 32, 8, 128, 64, 4096, 128
    case = attention_case(23, torch.bfloat16, heads, kv_heads, dim, page_size, shared, [(80, rows)] * 8)
    first = call_attention(ops, case)
    for _ in range(20):
        assert torch.equal(call_attention(ops, case), first)
    # The kernel that shares nothing.  Each of the two may be off by two roundings to 8 bits (weights and output), and by 2 (128 + 3) u of scores whose products sum to 60 at most, 2 (4,176 + 8) u of the
    # sums and 2^-21 of the exponentials (u = 2^-24): together less than 2^-9, all of the largest value.
    token_seq = torch.arange(8, dtype=torch.int32, device="cuda").repeat_interleave(rows)
    plain = torch.empty_like(first)
    ops.paged_attention(case["qkv"].cuda(), case["pages"].cuda(), case["positions"].cuda(), token_seq, case["table"].cuda(), plain, heads, kv_heads, dim, page_size)
    reach = max(float(k[1].float().abs().max()) for k in case["keys"])
    assert float((first.float() - plain.float()).abs().max()) <= 2 * reach * (2 * 2.0 ** -8 + 2.0 ** -9)
    for entry in (0, 7):   # some rows against 64 bits
        for row in (0, 47, 48, 127):
            t = entry * rows + row
            n = int(case["positions"][t]) + 1
            for h in (0, 31):
                q = case["qkv"][t, h * dim : (h + 1) * dim].double()
                k, v = (case["keys"][entry][i, h // 4, :n].double() for i in (0, 1))
                want = torch.softmax(k @ q * dim ** -0.5, 0) @ v
                products = float((k.abs() @ q.abs()).max()) * dim ** -0.5
                assert products <= 60
                off = float(v.abs().max()) * (2 * (dim + 3) * U * products + 2 * (n + 8) * U + 2.0 ** -21 + 2.0 ** -8) + want.abs() * 2.0 ** -8
                assert ((first[t, h * dim : (h + 1) * dim].cpu().double() - want).abs() <= off).all()
