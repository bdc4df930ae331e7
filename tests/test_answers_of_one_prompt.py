"""Attention over a prefix that a batch shares, and the choice of tokens with top-k, top-p and min-p, against plain functions in 64 bits.

Tolerances.  u = 2^-24 is half a step of a 32-bit float, 2^-8 half a step of bfloat16, both relative.
A score is a sum of D products, off by (D + 3) u sum|q k| scale at most, and its weight by that much relatively (twice: in the numerator and in the
denominator); a weight's own exponential by 2^-21; a sum of n weights or weighted values by (n + 8) u.  All of that multiplies max|v|.
bfloat16 kernels may round a weight before it meets its value (2^-8 max|v|), and round the output (2^-8 |out|).
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

U = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    from tinyllama_inference_engine_b200 import ops as module

    assert torch.cuda.is_available(), "these tests need the GPU"
    return module


# --- attention ------------------------------------------------------------------------------------------------------------------
def attention_case(seed, dtype, heads, kv_heads, dim, page_size, shared, entries, front=0, behind=0, wider=0, poison=True):
    """``entries``: (tokens behind the shared ones, rows of this step) per request.  Slots that hold no token are NaN, and so are rows in front and behind."""
    g = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    whole = shared // page_size
    own = [max(0, -(-(shared + h) // page_size) - whole) for h, _ in entries]
    total = whole + sum(own) + 2
    order = torch.randperm(total, generator=g).int()
    table = torch.full((len(entries), whole + max(own) + 1), -1, dtype=torch.int32)
    table[:, :whole] = order[:whole]
    pages = torch.full((total, 2, kv_heads, page_size, dim), float("nan") if poison else 0.0)
    prefix = randn(2, kv_heads, shared, dim)
    keys = []
    at = whole
    for i, ((held, _), n) in enumerate(zip(entries, own)):
        table[i, whole : whole + n] = order[at : at + n]
        at += n
        context = torch.cat([prefix, randn(2, kv_heads, held, dim)], 2)
        keys.append(context.to(dtype))
        for j in range(context.shape[2]):
            pages[table[i, j // page_size].item(), :, :, j % page_size] = context[:, :, j]
    rows = sum(r for _, r in entries)
    qkv = torch.full((front + rows + behind, heads * dim + wider), float("nan"))
    qkv[front : front + rows] = randn(rows, heads * dim + wider) * 2
    positions = [-5] * front + [shared + h - r + i for h, r in entries for i in range(r)] + [10 ** 6] * behind
    starts = front + np.concatenate([[0], np.cumsum([r for _, r in entries])])
    return {"qkv": qkv.to(dtype), "pages": pages.to(dtype), "positions": torch.tensor(positions, dtype=torch.int32), "seq_starts": torch.tensor(starts, dtype=torch.int32),
            "table": table, "keys": keys, "shared": shared, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page_size": page_size}


def plain_attention(case, scale=None):
    """Every row and head for itself in 64 bits; also what each output may be off by (without the output's own rounding)."""
    heads, dim, group = case["heads"], case["dim"], case["heads"] // case["kv_heads"]
    scale = dim ** -0.5 if scale is None else scale
    starts = case["seq_starts"].tolist()
    out = torch.full((case["qkv"].shape[0], heads, dim), float("nan"), dtype=torch.float64)
    off = torch.zeros_like(out)
    for b in range(len(starts) - 1):
        for t in range(starts[b], starts[b + 1]):
            n = min(int(case["positions"][t]) + 1, case["keys"][b].shape[2])
            for h in range(heads):
                q = case["qkv"][t, h * dim : (h + 1) * dim].double()
                k, v = case["keys"][b][0, h // group, : max(0, n)].double(), case["keys"][b][1, h // group, : max(0, n)].double()
                if n <= 0:
                    out[t, h] = 0
                    continue
                out[t, h] = torch.softmax(k @ q * scale, 0) @ v
                reach = float((k.abs() @ q.abs()).max()) * scale
                off[t, h] = float(v.abs().max()) * (2 * (dim + 3) * U * reach + 2 * (n + 8) * U + 2.0 ** -21)
                if case["qkv"].dtype == torch.bfloat16:
                    off[t, h] += float(v.abs().max()) * 2.0 ** -8
    return out.flatten(1), off.flatten(1)


def call_attention(ops, case, scale=None, out=None):
    c = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in case.items()}
    if out is None:
        out = torch.full((c["qkv"].shape[0], c["heads"] * c["dim"]), 7.0, dtype=c["qkv"].dtype, device="cuda")
    ops.shared_prefix_attention(c["qkv"], c["pages"], c["positions"], c["seq_starts"], c["table"], c["shared"], out, c["heads"], c["kv_heads"], c["dim"], c["page_size"], scale)
    return out


def compare_attention(got, case, want, off):
    first, end = int(case["seq_starts"][0]), int(case["seq_starts"][-1])
    got = got.cpu().double()
    if got.shape[0] > end or first > 0:
        assert (torch.cat([got[:first], got[end:]]) == 7.0).all(), "rows of no entry were written"
    got, want, off = got[first:end], want[first:end], off[first:end]
    off = off + want.abs() * (2.0 ** -8 if case["qkv"].dtype == torch.bfloat16 else U)
    assert not torch.isnan(got).any()
    worst = ((got - want).abs() - off).max()
    assert float(worst) <= 0, (float(worst), float((got - want).abs().max()))


HEADS = [(32, 4, 64), (8, 8, 128), (8, 2, 128), (6, 2, 64), (64, 1, 64), (5, 1, 80), (4, 2, 256), (2, 1, 16)]
SHAPES = {   # page size, shared, [(tokens behind, rows)]
    "one request, one token behind": (16, 33, [(1, 1)]),
    "answers of several lengths": (64, 130, [(1, 1), (64, 1), (7, 1), (129, 1), (40, 1)]),
    "the prefix ends with a page": (32, 128, [(5, 1), (33, 1)]),
    "nothing shared": (64, 0, [(9, 1), (70, 1)]),
    "one shared token": (16, 1, [(3, 1), (1, 1)]),
    "only the prefix": (64, 100, [(0, 1), (0, 1), (4, 1)]),
    "portions of several rows": (64, 70, [(37, 37), (5, 2), (130, 100), (1, 1)]),
    "entries without rows": (48, 100, [(3, 0), (20, 20), (0, 0), (2, 1), (7, 0)]),
    "rows inside the prefix": (16, 90, [(0, 50), (3, 10), (2, 2)]),
    "long": (128, 1300, [(700, 1), (3, 1), (260, 5)]),
}


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("heads", HEADS, ids=lambda h: f"{h[0]}-{h[1]}x{h[2]}")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
def test_attention_over_a_shared_prefix(ops, dtype, heads, shape):
    page_size, shared, entries = SHAPES[shape]
    case = attention_case(len(shape), dtype, *heads, page_size, shared, entries)
    compare_attention(call_attention(ops, case), case, *plain_attention(case))


# (prefix once for all rows, own keys on the tensor cores): every way that the bfloat16 kernels can be put together, whatever the sizes would choose
WAYS = {"row by row": (0, 0), "prefix once, own by rows": (1, 0), "prefix once, own by entries": (1, 1), "all by entries": (0, 1)}


@pytest.fixture
def way(request, ops, monkeypatch):
    prefix, own, parts, ctas = request.param
    monkeypatch.setattr(ops.fast, "use_prefix", prefix)
    monkeypatch.setattr(ops.fast, "use_own", own)
    if parts:
        monkeypatch.setattr(ops.fast, "prefix_tc_parts", lambda rows, kv_heads, group, head_dim, shared: (max(1, min(parts, -(-shared // ops.fast.PREFIX_TC_KEYS[head_dim]))), 1.0))
    if ctas:
        monkeypatch.setattr(ops.fast, "prefix_rows_ctas", lambda *_: ctas)
    ops.fast.shared_prefix_plan.cache_clear()
    yield request.param
    ops.fast.shared_prefix_plan.cache_clear()


EVERY_WAY = pytest.mark.parametrize("way", [(*w, 0, 0) for w in WAYS.values()], ids=WAYS.keys(), indirect=True)
TC_HEADS = [h for h in HEADS if h[2] in (64, 128)] + [(72, 2, 128), (128, 1, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("heads", TC_HEADS, ids=lambda h: f"{h[0]}-{h[1]}x{h[2]}")
@EVERY_WAY
def test_every_way_to_put_the_kernels_together(ops, way, heads, shape):
    page_size, shared, entries = SHAPES[shape]
    case = attention_case(len(shape) + 1, torch.bfloat16, *heads, page_size, shared, entries)
    compare_attention(call_attention(ops, case), case, *plain_attention(case))


@pytest.mark.gpu
@pytest.mark.parametrize("way", [(1, 0, 32, 1), (1, 0, 7, 2), (1, 1, 3, 0), (0, 0, 0, 1), (0, 0, 0, 4), (0, 0, 0, 8), (1, 0, 1, 8)], ids=lambda w: "-".join(map(str, w)), indirect=True)
@pytest.mark.parametrize("heads", [(16, 2, 64), (12, 4, 128)], ids=lambda h: f"{h[0]}-{h[1]}x{h[2]}")
@pytest.mark.parametrize("shape", ["long", "answers of several lengths", "rows inside the prefix"])
def test_runs_of_the_prefix_and_ctas_of_a_row(ops, way, heads, shape):
    page_size, shared, entries = SHAPES[shape]
    case = attention_case(len(shape) + 2, torch.bfloat16, *heads, page_size, 3 * shared + 5, entries, front=1, behind=1, wider=16)
    compare_attention(call_attention(ops, case), case, *plain_attention(case))


@pytest.mark.gpu
@pytest.mark.parametrize("way", [(0, 0, 0, 1), (1, 0, 5, 1), (0, 0, 0, 2)], ids=lambda w: "-".join(map(str, w)), indirect=True)
@pytest.mark.parametrize("warps", [2, 4, 16])
@pytest.mark.parametrize("heads", [(5, 5, 64), (12, 4, 128), (34, 2, 128)], ids=lambda h: f"{h[0]}-{h[1]}x{h[2]}")
def test_warps_of_a_row(ops, way, warps, heads, monkeypatch):
    monkeypatch.setattr(ops.fast, "prefix_rows_warps", lambda *_: (0.0, warps))
    case = attention_case(16, torch.bfloat16, *heads, 32, 333, [(5, 1), (0, 1), (400, 3), (40, 0), (31, 30)], front=1, behind=1, wider=8)
    compare_attention(call_attention(ops, case), case, *plain_attention(case))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("heads,page_size,wider", [((8, 2, 64), 24, 0), ((8, 2, 128), 64, 3), ((160, 1, 64), 16, 0), ((7, 7, 176), 1, 0), ((4, 2, 240), 40, 0)])
def test_sizes_of_the_general_kernel(ops, dtype, heads, page_size, wider):
    case = attention_case(11, dtype, *heads, page_size, 210, [(31, 1), (1, 1), (64, 33), (0, 0), (95, 2)], front=1, behind=2, wider=wider)
    compare_attention(call_attention(ops, case), case, *plain_attention(case))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128, 96])
def test_rows_of_no_entry_strides_and_scale(ops, dtype, dim):
    case = attention_case(3, dtype, 8, 2, dim, 64, 90, [(20, 3), (1, 1), (64, 40)], front=3, behind=2, wider=24)
    want, off = plain_attention(case, 0.21)
    compare_attention(call_attention(ops, case, 0.21), case, want, off)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
def test_a_row_without_a_key_is_zero(ops, dtype):
    case = attention_case(4, dtype, 8, 2, 64, 16, 40, [(20, 2), (6, 1)])
    case["positions"][0] = -1
    case["positions"][2] = -100
    want, off = plain_attention(case)
    got = call_attention(ops, case)
    assert (got[0] == 0).all() and (got[2] == 0).all()
    compare_attention(got, case, want, off)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_later_keys_and_values_that_are_no_numbers_stay_out(ops, dtype, bad):
    """A row of a portion does not see its request's later tokens, whatever stands there; the rows that do see them show it."""
    for dim in (64, 128):
        case = attention_case(5, dtype, 8, 2, dim, 64, 75, [(30, 30), (90, 20)])
        clean = call_attention(ops, case)
        for plane in (0, 1):
            spoiled = {**case, "pages": case["pages"].clone()}
            place = 75 + 19   # request 0: its rows 19 and behind see this key
            spoiled["pages"][int(case["table"][0, place // 64]), plane, :, place % 64, 5] = bad
            got = call_attention(ops, spoiled)
            assert torch.equal(got[:19], clean[:19]) and torch.equal(got[30:], clean[30:])
            if plane == 1:
                column = got[19:30].float().view(11, 8, dim)[:, :, 5]
                assert (torch.isnan(column) if math.isnan(bad) else column == bad).all()
                other = torch.arange(dim) != 5
                assert torch.equal(got[19:30].view(11, 8, dim)[:, :, other], clean[19:30].view(11, 8, dim)[:, :, other])


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dim", [64, 128])
@EVERY_WAY
def test_numbers_that_are_none_in_every_way(ops, way, dim, bad):
    """Behind a row's position they stay out, in the prefix and behind it; a value among a row's keys shows in its column alone, a key or a query in its heads."""
    case = attention_case(12, torch.bfloat16, 8, 2, dim, 32, 200, [(0, 150), (40, 3), (3, 1)])
    clean = call_attention(ops, case)
    position = case["positions"].cuda()
    for place in (7, 130, 199):
        page, slot = case["table"][:, place // 32].long(), place % 32   # every entry's: key 199 lies in a page that each has a copy of
        sees = position >= place
        spoiled = {**case, "pages": case["pages"].clone()}
        spoiled["pages"][page, 1, 1, slot, 9] = bad
        got = call_attention(ops, spoiled).view(-1, 8, dim)
        touched = torch.zeros(got.shape, dtype=torch.bool, device="cuda")
        touched[:, 4:, 9] = sees[:, None]
        assert torch.equal(got[~touched], clean.view(-1, 8, dim)[~touched])
        column = got[touched].float()
        assert (torch.isnan(column) if math.isnan(bad) else column == bad).all()
        spoiled["pages"][page] = case["pages"][page]
        spoiled["pages"][page, 0, 1, slot, 9] = bad
        got = call_attention(ops, spoiled).view(-1, 8, dim)
        touched[:, 4:] = sees[:, None, None]
        assert torch.equal(got[~touched], clean.view(-1, 8, dim)[~touched])
        if math.isnan(bad):
            assert torch.isnan(got[touched]).all()
    spoiled = {**case, "qkv": case["qkv"].clone()}
    spoiled["qkv"][151, 3 * dim + 2] = bad
    got = call_attention(ops, spoiled).view(-1, 8, dim)
    touched = torch.zeros(got.shape, dtype=torch.bool, device="cuda")
    touched[151, 3] = True
    assert torch.equal(got[~touched], clean.view(-1, 8, dim)[~touched]) and torch.isnan(got[151, 3]).all()


@pytest.mark.gpu
@EVERY_WAY
def test_rows_without_keys_and_bad_pages_in_every_way(ops, way):
    from tinyllama_inference_engine_b200.errors import KernelError

    for dim in (64, 128):
        case = attention_case(13, torch.bfloat16, 8, 2, dim, 16, 100, [(20, 4), (6, 1), (30, 0), (9, 70)])
        for row, at in ((0, -1), (3, -100), (4, -2147483648), (30, -1)):
            case["positions"][row] = at
        got = call_attention(ops, case)
        assert (got[[0, 3, 4, 30]] == 0).all()
        compare_attention(got, case, *plain_attention(case))
        for entry, page, message in ((0, 2, "outside the pool"), (3, 8, "outside the pool"), (1, None, "beyond the block table")):
            case = attention_case(14, torch.bfloat16, 8, 2, dim, 16, 100, [(20, 4), (6, 1), (30, 0), (70, 70)], poison=False)
            if page is None:
                case["table"] = case["table"].clamp(min=0)
                case["positions"][4] = 2147483647
            else:
                case["table"][entry, page] = 1 << 30
            call_attention(ops, case)
            with pytest.raises(KernelError, match=message):
                ops.check_device_errors(torch.device("cuda:0"))


@pytest.mark.gpu
@EVERY_WAY
def test_every_way_in_a_graph_beside_another_stream(ops, way):
    case = attention_case(15, torch.bfloat16, 8, 2, 128, 64, 300, [(30, 1), (70, 4), (1, 1)])
    want, off = plain_attention(case)
    c = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in case.items()}
    outs = [torch.full((6, 8 * 128), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
    call = lambda out: ops.shared_prefix_attention(c["qkv"], c["pages"], c["positions"], c["seq_starts"], c["table"], 300, out, 8, 2, 128, 64)  # noqa: E731
    call(outs[0])
    graphs = []
    for out in outs[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(out)
            call(out)   # (the second waits for the first)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(3):
        for out in outs:
            out.fill_(7.0)
        torch.cuda.synchronize()
        for i in range(3):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay() if i < 2 else call(outs[2])
        torch.cuda.synchronize()
        for out in outs:
            compare_attention(out, case, want, off)
            assert torch.equal(out, outs[0])


@pytest.mark.gpu
def test_pages_outside_the_pool_are_reported(ops):
    from tinyllama_inference_engine_b200.errors import KernelError

    for dim in (64, 128, 80):
        for dtype in (torch.float32, torch.bfloat16):
            for value in (-1, 1 << 30):
                case = attention_case(6, dtype, 4, 2, dim, 64, 64, [(70, 1), (30, 2)], poison=False)
                case["table"][0, 1] = value
                call_attention(ops, case)
                with pytest.raises(KernelError, match="outside the pool"):
                    ops.check_device_errors(torch.device("cuda:0"))
            case = attention_case(6, dtype, 4, 2, dim, 64, 64, [(70, 1), (30, 2)], poison=False)
            case["positions"][0] = 64 * case["table"].shape[1]
            case["table"] = case["table"].clamp(min=0)
            call_attention(ops, case)
            with pytest.raises(KernelError, match="beyond the block table"):
                ops.check_device_errors(torch.device("cuda:0"))
    ops.check_device_errors(torch.device("cuda:0"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
def test_attention_in_graphs_and_on_other_streams(ops, dtype):
    """Two captured calls, replayed in turn and at the same time as a plain call on another stream: each has its own workspace."""
    cases = [attention_case(7, dtype, 8, 2, 64, 64, 200, [(30, 1), (70, 1)]), attention_case(8, dtype, 8, 2, 64, 64, 130, [(30, 9), (70, 1), (1, 1)])]
    wants = [plain_attention(c) for c in cases]
    held, graphs = [], []
    for case in cases:
        call_attention(ops, case)   # builds and loads what a capture must not wait for
        c = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in case.items()}
        out = torch.full((c["qkv"].shape[0], 512), 7.0, dtype=dtype, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.shared_prefix_attention(c["qkv"], c["pages"], c["positions"], c["seq_starts"], c["table"], c["shared"], out, 8, 2, 64, 64)
        held.append((c, out))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(3):
        for (_, out) in held:
            out.fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            graphs[0].replay()
        with torch.cuda.stream(streams[1]):
            graphs[1].replay()
        with torch.cuda.stream(streams[2]):
            c = held[0][0]
            third = torch.full_like(held[0][1], 7.0)
            ops.shared_prefix_attention(c["qkv"], c["pages"], c["positions"], c["seq_starts"], c["table"], c["shared"], third, 8, 2, 64, 64)
        torch.cuda.synchronize()
        for (c, out), case, (want, off) in zip(held, cases, wants):
            compare_attention(out, case, want, off)
        assert torch.equal(third, held[0][1])
    # what the tensors hold may change between replays
    case = attention_case(9, dtype, 8, 2, 64, 64, 200, [(5, 1), (70, 1)])
    for name in ("qkv", "positions", "seq_starts"):
        held[0][0][name].copy_(case[name])
    held[0][0]["pages"][: case["pages"].shape[0]].copy_(case["pages"])
    held[0][0]["table"].copy_(case["table"])
    graphs[0].replay()
    compare_attention(held[0][1], case, *plain_attention(case))


def test_a_wait_of_the_prefix_kernel_that_gives_up_is_reported():
    """As in the other kernels with bounded waits: nobody reports by itself, all waits lie in front of the closing report, and tensor memory is given back behind it."""
    import re
    from pathlib import Path

    from tinyllama_inference_engine_b200 import ops

    source = (Path(ops.__file__).parent.parent / "csrc" / "attention_prefix_tc.cu").read_text()
    assert "if (*gave_up" not in source
    kernels = [part for part in re.split(r"(?=__global__ )", source)[1:] if "warp_wait(" in part]
    assert len(kernels) == 1
    for kernel in kernels:
        end = kernel.index("close_and_report(gave_up,")
        assert "_wait(&" not in kernel[end:] and kernel.index("tcgen05.dealloc", end) > end


def test_attention_refuses():
    from tinyllama_inference_engine_b200 import ops
    from tinyllama_inference_engine_b200.errors import KernelError

    good = dict(qkv=torch.zeros(3, 6 * 64), pages=torch.zeros(4, 2, 1, 16, 64), positions=torch.zeros(3, dtype=torch.int32), seq_starts=torch.zeros(3, dtype=torch.int32),
                block_table=torch.zeros(2, 2, dtype=torch.int32), shared=16, out=torch.zeros(3, 4 * 64), q_heads=4, kv_heads=1, head_dim=64, page_size=16)
    wrong = {
        "no CPU path": {}, "head sizes": dict(head_dim=60), "multiple of key/value heads": dict(kv_heads=3), "qkv must be": dict(qkv=torch.zeros(3, 255)),
        "out must be [rows": dict(out=torch.zeros(3, 255)), "of qkv's dtype": dict(out=torch.zeros(3, 256, dtype=torch.bfloat16)), "pages must be": dict(page_size=32),
        "fewer than 2^31 keys": dict(block_table=torch.zeros(1, dtype=torch.int32).expand(2, 1 << 27)),
        "16-byte boundary": dict(pages=torch.zeros(4 * 2 * 16 * 64 + 1)[1:].view(4, 2, 1, 16, 64)),
        "a block table": dict(seq_starts=torch.zeros(4, dtype=torch.int32)), "positions [rows]": dict(positions=torch.zeros(4, dtype=torch.int32)),
        "shared must be a whole number from 0 to the 32 keys": dict(shared=33), "got -1": dict(shared=-1), "got True": dict(shared=True), "scale must be": dict(scale=0.0),
        "got nan": dict(scale=float("nan")), "are int32": dict(positions=torch.zeros(3, dtype=torch.int64)), "contiguous rows": dict(qkv=torch.zeros(6 * 64, 3).t()),
    }
    for message, change in wrong.items():
        with pytest.raises(KernelError) as error:
            ops.shared_prefix_attention(**{**good, **change})
        assert message in str(error.value), (message, str(error.value))
    with pytest.raises(KernelError, match="float32 or bfloat16"):
        ops.shared_prefix_attention(**{**good, "qkv": good["qkv"].half(), "pages": good["pages"].half(), "out": good["out"].half()})


# --- choice of tokens -------------------------------------------------------------------------------------------------------------
def plain_choice(row, temperature, top_k, top_p, min_p, u):
    """The token in 64 bits, the kept ids, and whether the draw or a border lies within rounding of another answer (weights are off by 2^-22 at most)."""
    row = row.double().numpy()
    order = np.lexsort((np.arange(len(row)), -np.where(np.isnan(row), -np.inf, row), np.isnan(row)))
    largest = row[order[0]]
    if not temperature > 0 or not largest > -np.inf:
        return (0 if np.isnan(largest) else int(order[0])), order[:1], False
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(row == largest, 1.0, np.exp((row - largest) / max(temperature, 1e-30)))
    w = np.where(np.isnan(w), 0.0, w)[order]
    near = 0.0 if bool(((w == 0) | (w == 1)).all()) else 2.0 ** -22   # weights of 1 are exact, and so are their sums
    count = top_k if 0 < top_k < len(row) else len(row)
    close = False
    if top_p < 1:
        sums = np.cumsum(w[:count])
        by_p = int(np.searchsorted(sums, top_p * sums[-1])) + 1
        close |= bool((np.abs(sums - top_p * sums[-1]) < near * sums[-1]).any()) and top_p > 0
        count = min(count, max(1, by_p))
    if min_p > 0:
        close |= bool((np.abs(w[1:] - min_p) < near * min_p).any())
        count = min(count, max(1, int((w >= min_p).sum())))
    kept = np.sort(order[:count])
    rank = np.empty(len(row), dtype=np.int64)
    rank[order] = np.arange(len(row))
    sums = np.cumsum(w[rank[kept]])
    target = min(max(u, 0.0), 1.0) * sums[-1]
    close |= bool((np.abs(sums[:-1] - target) < near * sums[-1]).any())
    inside = np.nonzero(w[rank[kept]] > 0)[0]
    return int(kept[min(int(np.searchsorted(sums, target, side="right")), inside[-1])]), kept, close


def call_choice(ops, logits, temperature, top_k, top_p, min_p, u, rows=None, out=None):
    f = lambda x: torch.tensor(x, dtype=torch.float32, device="cuda")  # noqa: E731
    out = torch.full((logits.shape[0],), -7, dtype=torch.int32, device="cuda") if out is None else out
    ops.sample_filtered(logits.cuda(), f(temperature), torch.tensor(top_k, dtype=torch.int32, device="cuda"), f(top_p), f(min_p), f(u), out, rows)
    return out.cpu().tolist()


OPTIONS = [(1.0, 0, 1.0, 0.0), (0.7, 40, 0.95, 0.0), (0.0, 5, 0.5, 0.1), (1.3, 0, 0.9, 0.0), (0.9, 1, 1.0, 0.0), (1.0, 3, 1.0, 0.0), (0.8, 0, 1.0, 0.05),
           (1.0, 200, 0.6, 0.01), (5.0, 0, 0.99, 0.0), (0.05, 0, 0.999, 0.0), (1.0, 10 ** 9, 1.0, 1.0), (-1.0, 0, 1.0, 0.0), (2.0, 1500, 0.97, 0.0), (1.0, 0, 0.3, 0.9),
           (float("nan"), 7, 0.4, 0.0), (1.0, -3, 2.0, -1.0), (1.0, 0, 0.0, 0.0), (0.6, 0, 1.0, 1.5), (float("inf"), 9, 1.0, 0.0)]


def check_choices(ops, logits, options, uniforms, rows=None):
    got = call_choice(ops, logits, *[list(c) for c in zip(*options)], uniforms, rows)
    checked = 0
    for r, (option, u) in enumerate(zip(options, uniforms)):
        want, kept, close = plain_choice(logits[r], *[float(np.float32(x)) if i != 1 else x for i, x in enumerate(option)], float(np.float32(u)))
        if not close:
            assert got[r] == want, (r, option, u, got[r], want, len(kept))
            checked += 1
    assert checked >= len(options) * 3 // 4, "too many draws lie on a border for this test to say anything"


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 2, 31, 257, 1000, 4099, 32000, 50257, 128256, 262144])
@pytest.mark.parametrize("spread", [0.0, 0.3, 4.0, 40.0])
def test_choice_with_every_option(ops, vocab, spread):
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn(len(OPTIONS), vocab, generator=g) * spread
    check_choices(ops, logits, OPTIONS, torch.rand(len(OPTIONS), generator=g).tolist())


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [500, 32000, 128256])
def test_choice_with_many_equal_logits(ops, vocab):
    """Logits as 16-bit products leave them: few different numbers, so that borders fall among equals."""
    g = torch.Generator().manual_seed(vocab)
    logits = (torch.randn(len(OPTIONS), vocab, generator=g) * 3).bfloat16().float()
    check_choices(ops, logits, OPTIONS, torch.rand(len(OPTIONS), generator=g).tolist())
    check_choices(ops, logits.round(), OPTIONS, torch.rand(len(OPTIONS), generator=g).tolist())


@pytest.mark.gpu
def test_equal_weights_are_counted_to_the_token(ops):
    """All weights are 1: borders and draws are whole numbers and leave no room for rounding."""
    for vocab in (1000, 32000, 131072):
        logits = torch.zeros(1, vocab)
        for top_k, top_p, u in ((0, 0.5, 0.0), (0, 0.5, 1.0 - 2.0 ** -24), (vocab // 2, 0.25, 1.0 - 2.0 ** -24), (0, 1.0, 0.5), (7, 1.0, 1.0 - 2.0 ** -24), (0, 0.5, 0.25), (3, 0.34, 0.99)):
            kept = vocab if top_k == 0 else top_k
            kept = min(kept, math.ceil(float(np.float32(top_p)) * kept))
            assert call_choice(ops, logits, [1.0], [top_k], [top_p], [0.0], [u]) == [int(float(np.float32(u)) * kept)], (vocab, top_k, top_p, u)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40, 200])
@pytest.mark.parametrize("vocab", [2000, 32000, 128256])
def test_a_border_on_a_whole_number_of_equal_weights(ops, vocab, rows):
    """Some tokens weigh 1 and all others nothing: top_p of them ends exactly at a token, which what they weigh about cannot tell."""
    g = torch.Generator().manual_seed(vocab + rows)
    number = [int(n) for n in torch.randint(2, 180, (rows,), generator=g)]
    logits = torch.full((rows, vocab), -1e4)
    ids = [torch.randperm(vocab, generator=g)[:n].sort().values for n in number]
    for row, where in enumerate(ids):
        logits[row, where] = 3.0
    top_p = [float(np.float32(p)) for p in (0.5, 0.25, 0.75, 0.125, 0.9, 0.3)]
    u = torch.rand(rows, generator=g).tolist()
    want = []
    for row in range(rows):
        kept = max(1, math.ceil(top_p[row % 6] * number[row]))
        want.append(int(ids[row][int(float(np.float32(u[row])) * kept)]))
    assert call_choice(ops, logits, [0.8] * rows, [0] * rows, [top_p[row % 6] for row in range(rows)], [0.0] * rows, u) == want


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40, 200])
@pytest.mark.parametrize("vocab", [2000, 32000, 128256])
def test_a_number_that_falls_where_a_token_ends(ops, vocab, rows):
    """Without top-k, top-p and min-p, over equal weights: the number is where one token ends and the next begins, or just in front of it."""
    g = torch.Generator().manual_seed(vocab + rows)
    number = [2 ** int(n) for n in torch.randint(1, 11, (rows,), generator=g)]
    logits = torch.full((rows, vocab), -float("inf"))
    ids = [torch.randperm(vocab, generator=g)[:n].sort().values for n in number]
    place = [int(torch.randint(1, n, (1,), generator=g)) for n in number]
    for row, where in enumerate(ids):
        logits[row, where] = -2.0
    for before in (False, True):
        u = [float(np.nextafter(np.float32(k / n), np.float32(0))) if before else k / n for k, n in zip(place, number)]
        want = [int(where[k - before]) for where, k in zip(ids, place)]
        assert call_choice(ops, logits, [1.3] * rows, [0] * rows, [1.0] * rows, [0.0] * rows, u) == want


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 5, 2000, 32003, 128256])
def test_the_first_of_equal_largest_tokens(ops, vocab):
    g = torch.Generator().manual_seed(vocab)
    for rows in (1, 30, 200):
        logits = torch.randn(rows, vocab + 3, generator=g).round()[:, 1 : vocab + 1]   # (rows that do not start on 16 bytes)
        want = [int((row == row.max()).nonzero()[0]) for row in logits]
        assert call_choice(ops, logits, [0.0] * rows, [0] * rows, [1.0] * rows, [0.0] * rows, [0.5] * rows) == want
        assert call_choice(ops, logits, [1.0] * rows, [1] * rows, [1.0] * rows, [0.0] * rows, [0.5] * rows) == want


@pytest.mark.gpu
def test_logits_that_are_no_numbers(ops):
    inf, nan = float("inf"), float("nan")
    row = torch.tensor([nan, -inf, 1.0, nan, 2.0, -inf, 2.0, 0.0])
    logits = torch.stack([row, torch.full((8,), nan), torch.full((8,), -inf), torch.tensor([nan, nan, -inf, -inf, nan, nan, nan, nan]), torch.tensor([0.0, inf, 3.0, inf, nan, 1.0, -inf, 0.0]),
                          torch.tensor([0.0, -3.4e38, 3.4e38, 3.4e38, 0.0, 0.0, 0.0, 0.0]), torch.tensor([-0.0, 0.0, -0.0, -1.0, -1.0, -1.0, -1.0, -1.0])])
    for u in (0.0, 0.3, 0.6, 0.999):
        for option in ((1.0, 0, 1.0, 0.0), (1.0, 2, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.2), (1.0, 5, 0.99, 0.0)):
            got = call_choice(ops, logits, *[[x] * 7 for x in option], [u] * 7)
            for r in range(7):
                want, _, close = plain_choice(logits[r], *option, float(np.float32(u)))
                assert close or got[r] == want, (r, option, u)
    # masked vocabularies: the lowest number of a type, and a number of logits far below all others
    for low in (-inf, float(np.finfo(np.float32).min), -1e9):
        logits = torch.full((4, 5000), low)
        logits[:, 4000:4003] = torch.tensor([1.0, 1.5, 0.5])
        check_choices(ops, logits, [(1.0, 0, 1.0, 0.0), (1.0, 10, 0.9, 0.0), (0.5, 0, 0.7, 0.0), (1.0, 2, 1.0, 0.0)], [0.1, 0.9, 0.5, 0.99])


@pytest.mark.gpu
def test_numbers_outside_the_range_take_the_first_and_the_last(ops):
    logits = torch.zeros(6, 100)
    for column in range(90, 100):
        logits[:, column] = -float("inf")
    assert call_choice(ops, logits, [1.0] * 6, [0] * 6, [1.0] * 6, [0.0] * 6, [-1.0, float("nan"), 0.0, 1.0, 2.0, float("inf")]) == [0, 0, 0, 89, 89, 89]


@pytest.mark.gpu
def test_choice_for_some_rows_and_strides(ops):
    g = torch.Generator().manual_seed(1)
    wide = torch.randn(40, 1003, generator=g).cuda() * 3
    logits = wide[:, 1:1002]                               # rows start anywhere
    options = (OPTIONS * 3)[:40]
    columns = [list(c) for c in zip(*options)]
    u = torch.rand(40, generator=g).tolist()
    all_rows = call_choice(ops, logits, *columns, u)
    assert all_rows == call_choice(ops, logits.contiguous(), *columns, u)
    # some rows, in another order; numbers outside the logits are passed over
    rows = [39, -1, 0, 17, 40, 3, 1 << 30, -(1 << 31)]
    picked = [r if 0 <= r < 40 else 0 for r in rows]
    got = call_choice(ops, logits, *[[c[r] for r in picked] for c in columns], [u[r] for r in picked], torch.tensor(rows, dtype=torch.int32, device="cuda"))
    assert got == [all_rows[r] if r in (39, 0, 17, 3) else -7 for r in range(40)]
    # one row given to many
    same = wide[:1, :1000].expand(40, 1000)
    assert call_choice(ops, same, *columns, u) == call_choice(ops, same.contiguous(), *columns, u)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [3000, 32000, 128256])
def test_a_rows_token_does_not_depend_on_the_batch(ops, vocab):
    g = torch.Generator().manual_seed(2)
    logits = torch.randn(300, vocab, generator=g).cuda() * 2
    options = (OPTIONS * 20)[:300]
    columns = [list(c) for c in zip(*options)]
    u = torch.rand(300, generator=g).tolist()
    together = call_choice(ops, logits, *columns, u)
    for first, end in ((0, 1), (1, 5), (5, 25), (25, 100)):
        assert call_choice(ops, logits[first:end], *[c[first:end] for c in columns], u[first:end]) == together[first:end]


@pytest.mark.gpu
def test_choice_in_graphs_and_on_other_streams(ops):
    g = torch.Generator().manual_seed(3)
    f = lambda x: torch.tensor(x, dtype=torch.float32, device="cuda")  # noqa: E731
    columns = [list(c) for c in zip(*OPTIONS)]
    n = len(OPTIONS)
    sets = [(torch.randn(n, v, generator=g).cuda() * 3, f(columns[0]), torch.tensor(columns[1], dtype=torch.int32, device="cuda"), f(columns[2]), f(columns[3]),
             torch.rand(n, generator=g).cuda(), torch.zeros(n, dtype=torch.int32, device="cuda")) for v in (40000, 128256)]
    graphs, wants = [], []
    for s in sets:
        ops.sample_filtered(*s)
        wants.append(s[-1].clone())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.sample_filtered(*s)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for s in sets:
            s[-1].zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for s, want in zip(sets, wants):
            assert torch.equal(s[-1], want)


@pytest.mark.gpu
def test_uniform_numbers_of_draws(ops):
    seeds, counters = [0, 7, -1, (1 << 63) - 1, 123456789], [0, 3, 1 << 40, 5, 2]
    out = torch.empty(5, device="cuda")
    ops.uniforms(torch.tensor(seeds, dtype=torch.int64, device="cuda"), torch.tensor(counters, dtype=torch.int64, device="cuda"), out)
    assert out.tolist() == [ops.uniform_from(s, c) for s, c in zip(seeds, counters)]


def test_choice_refuses():
    from tinyllama_inference_engine_b200 import ops
    from tinyllama_inference_engine_b200.errors import KernelError

    good = dict(logits=torch.zeros(3, 50), temperature=torch.zeros(3), top_k=torch.zeros(3, dtype=torch.int32), top_p=torch.zeros(3), min_p=torch.zeros(3), uniforms=torch.zeros(3),
                out=torch.zeros(3, dtype=torch.int32))
    wrong = [("no CPU path", {}), ("32-bit logits", dict(logits=torch.zeros(3, 50).bfloat16())), ("32-bit logits", dict(min_p=torch.zeros(3).double())),
             ("int32", dict(top_k=torch.zeros(3, dtype=torch.int64))), ("int32", dict(out=torch.zeros(3, dtype=torch.int64))), ("int32", dict(rows=torch.zeros(3, dtype=torch.int64))),
             ("logits must be", dict(logits=torch.zeros(3, 0))), ("logits must be", dict(logits=torch.zeros(50))), ("logits must be", dict(logits=torch.zeros(50, 3).t())),
             ("logits must be", dict(logits=torch.zeros(1, 1).expand(3, (1 << 19) + 1))), ("one temperature", dict(top_p=torch.zeros(2))), ("one temperature", dict(out=torch.zeros(2, dtype=torch.int32))),
             ("one temperature", dict(rows=torch.zeros(2, dtype=torch.int32)))]
    for message, change in wrong:
        with pytest.raises(KernelError) as error:
            ops.sample_filtered(**{**good, **change})
        assert message in str(error.value), (message, str(error.value))
    with pytest.raises(KernelError, match="int64 seeds"):
        ops.uniforms(torch.zeros(3), torch.zeros(3, dtype=torch.int64), torch.zeros(3))
    with pytest.raises(KernelError, match="one number per seed"):
        ops.uniforms(torch.zeros(3, dtype=torch.int64), torch.zeros(3, dtype=torch.int64), torch.zeros(4))
