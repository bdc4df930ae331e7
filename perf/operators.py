"""Operators of a decode step that gives many answers to one prompt: attention over a prefix that the whole batch shares, and the
choice of tokens with temperature, top-k, top-p and min-p from given random numbers.

``shared_prefix_attention``  the step's query rows attend to their requests' cached keys up to their own positions; the first
``shared`` keys of every request are the same pages, as after one prompt that was run once.  Rows of one decoded token per request,
and portions of several rows (questions behind a system prompt).

``sample_filtered``  one token per row of 32-bit logits: the most probable tokens that top-k, top-p and min-p leave, drawn with a
uniform number that the caller gives.  Rows with temperature 0 are greedy.

Head counts and vocabularies are those of the models that ``bench.py`` runs.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

# query heads, key/value heads, head size, vocabulary
MODELS = {"tinyllama": (32, 4, 64, 32000), "llama2-7b": (32, 32, 128, 32000), "llama3-8b": (32, 8, 128, 128256)}


# --- the cases ----------------------------------------------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # A few answers to one short chat prompt, just begun: the smallest call, latency is all there is.
        _attention("four answers begun", "tinyllama", requests=4, shared=57, shortest=1, longest=40),
        # The benchmark's eight requests of 1,024 tokens, here eight answers to one prompt.
        _attention("eight answers", "tinyllama", requests=8, shared=1024, shortest=3, longest=64),
        # A full batch behind a system prompt of middling length, each with a dialogue of its own.
        _attention("full batch behind a system prompt", "tinyllama", requests=64, shared=700, shortest=90, longest=310),
        # A cache entry per head: the prefix is most of what there is to read.  The prompt ends inside a page.
        _attention("sixteen answers at 7B", "llama2-7b", requests=16, shared=2001, shortest=33, longest=500),
        # Readers of one long document, with larger pages.
        _attention("readers of a document at 8B", "llama3-8b", requests=48, shared=7001, shortest=100, longest=1100, page_size=128),
        # Many samples over a very long context: the largest call.
        _attention("many samples over a long context at 8B", "llama3-8b", requests=256, shared=24576, shortest=16, longest=256),
        # Questions of some hundred tokens run as one step behind a prompt that is in the cache.
        _attention("questions behind a prompt at 8B", "llama3-8b", requests=8, shared=4096, shortest=190, longest=256, rows=256),
        # The 32-bit path, as used to check a checkpoint's conversion.
        _attention("32-bit check", "tinyllama", dtype="float32", requests=4, shared=500, shortest=20, longest=100),
        # One user's answer, with the usual filters.
        _sampling("one answer", "tinyllama", rows=1, temperature=0.8, top_k=40, top_p=0.95, min_p=0.0),
        # A full batch over a long vocabulary, top-p alone: every probability counts.
        _sampling("full batch with top-p at 8B", "llama3-8b", rows=64, temperature=0.9, top_k=0, top_p=0.9, min_p=0.0),
        # A server's batch whose requests each ask for something else, some greedy, over a vocabulary with an added token.
        _sampling("requests of all kinds", "tinyllama", rows=24, added=1, mixed=True),
        # Many samples of one prompt with every filter on.
        _sampling("many samples at 8B", "llama3-8b", rows=256, temperature=0.7, top_k=50, top_p=0.95, min_p=0.02),
    ]


def _attention(name, model, *, dtype="bfloat16", requests, shared, shortest, longest, rows=1, page_size=64) -> dict:
    """``shortest`` to ``longest``: tokens of a request behind the shared ones, the step's rows (at most ``rows`` of them) included."""
    case = {"operator": "shared_prefix_attention", "model": model, "dtype": dtype, "requests": requests, "shared": shared, "shortest": shortest,
            "longest": longest, "rows": rows, "page_size": page_size}
    return {"name": name, **case} if name else case


def _sampling(name, model, *, rows, added=0, mixed=False, temperature=0.0, top_k=0, top_p=1.0, min_p=0.0) -> dict:
    case = {"operator": "sample_filtered", "model": model, "rows": rows, "added": added, "mixed": mixed, "temperature": temperature, "top_k": top_k,
            "top_p": top_p, "min_p": min_p}
    return {"name": name, **case} if name else case


def _log_int(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    """A case of the same ranges: either operator, any of the models, sizes spread over their logarithm, odd ones as likely as even ones."""
    most = {kind: max(work(c)["flops"] for c in listed() if c["operator"] == kind) for kind in ("shared_prefix_attention", "sample_filtered")}
    while True:
        model = rng.choice(list(MODELS))
        if rng.random() < 0.6:
            small = rng.random() < 0.12
            portion = rng.random() < 0.25
            requests = _log_int(rng, 1, 8 if small else 24 if portion else 256)
            longest = _log_int(rng, 1, 200 if small else 1100)
            case = _attention(None, model, dtype="float32" if small else "bfloat16", requests=requests, shared=_log_int(rng, 16, 1000 if small else 24576),
                              shortest=max(1, int(longest * rng.random())), longest=longest,
                              rows=_log_int(rng, 2, 300) if portion else 1, page_size=rng.choice([16, 32, 64, 64, 128]))
            if requests * longest > 100000:   # what a cache of this kind holds
                continue
        else:
            case = _sampling(None, model, rows=_log_int(rng, 1, 256), added=rng.choice([0, 0, rng.randint(1, 300)]), mixed=rng.random() < 0.3,
                             temperature=round(rng.uniform(0.4, 1.3), 2), top_k=rng.choice([0, _log_int(rng, 1, 200)]),
                             top_p=rng.choice([1.0, round(rng.uniform(0.5, 0.98), 2)]), min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.2), 3)]))
        if work(case)["flops"] <= most[case["operator"]]:
            return case


# --- what a program has in hand -------------------------------------------------------------------------------------------------
def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """Tokens that each request holds behind the shared ones, and how many of them are rows of this step."""
    n, low, high = case["requests"], case["shortest"], case["longest"]
    spread = [high if n == 1 else low + (high - low) * i // (n - 1) for i in range(n)]
    held = [spread[(i * 7 + 3) % n] for i in range(n)] if n % 7 else spread[::-1]
    return held, [min(case["rows"], h) for h in held]


def prepare(case: dict, seed: int) -> dict:
    return _prepare_attention(case, seed) if case["operator"] == "shared_prefix_attention" else _prepare_sampling(case, seed)


def _prepare_attention(case: dict, seed: int) -> dict:
    """The step's rows [q | k | v] with q rotated, a pool of pages in which every request's keys and values lie, and the block tables.
    A shared prefix that ends inside a page has that page copied for every request, which writes its own tokens behind it."""
    heads, kv_heads, dim, _ = MODELS[case["model"]]
    dtype = getattr(torch, case["dtype"])
    generator = torch.Generator(device="cuda").manual_seed(seed)
    held, rows = _lengths(case)
    shared, page_size, requests = case["shared"], case["page_size"], case["requests"]
    whole = shared // page_size                                       # pages that are the same for all
    own_pages = [-(-(shared + h) // page_size) - whole for h in held]
    total = whole + sum(own_pages)
    order = torch.randperm(total, generator=generator, device="cuda").int()
    width = whole + max(own_pages)
    table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    table[:, :whole] = order[:whole]
    at = whole
    for i, n in enumerate(own_pages):
        table[i, whole : whole + n] = order[at : at + n]
        at += n
    pages = torch.randn(total, 2, kv_heads, page_size, dim, generator=generator, device="cuda", dtype=torch.float32 if dtype == torch.float32 else dtype)
    if shared % page_size:
        boundary = table[:, whole].long()
        pages[boundary[1:], :, :, : shared % page_size] = pages[boundary[0], :, :, : shared % page_size].clone()
    tokens = sum(rows)
    qkv = torch.randn(tokens, (heads + 2 * kv_heads) * dim, generator=generator, device="cuda", dtype=torch.float32)
    qkv[:, : heads * dim] *= 2.0                                      # scores with a deviation of two: some keys count for more than others
    positions = [shared + h - r + i for h, r in zip(held, rows) for i in range(r)]
    starts = np.concatenate([[0], np.cumsum(rows)])
    return {"case": case, "qkv": qkv.to(dtype), "pages": pages, "table": table, "positions": torch.tensor(positions, dtype=torch.int32, device="cuda"),
            "seq_starts": torch.tensor(starts, dtype=torch.int32, device="cuda"), "out": torch.empty(tokens, heads * dim, dtype=dtype, device="cuda")}


_KINDS = [  # temperature, top_k, top_p, min_p of requests of all kinds
    (0.0, 0, 1.0, 0.0), (0.8, 40, 0.95, 0.0), (1.0, 0, 1.0, 0.0), (0.7, 0, 0.9, 0.0), (1.1, 0, 1.0, 0.1), (0.9, 5, 1.0, 0.0), (1.2, 200, 0.8, 0.05), (0.6, 1, 1.0, 0.0),
]


def _prepare_sampling(case: dict, seed: int) -> dict:
    """Logits as a trained head leaves them: a bell of unlikely tokens, and some hundred likelier ones whose logits fall off."""
    generator = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab = case["rows"], MODELS[case["model"]][3] + case["added"]
    logits = torch.randn(rows, vocab, generator=generator, device="cuda") * 1.8
    each = vocab // 300                                               # one likely token in every run of this many
    likely = torch.arange(300, device="cuda") * each + torch.randint(0, each, (rows, 300), generator=generator, device="cuda")
    logits.scatter_add_(1, likely, 6.0 + 8.0 * torch.rand(rows, 300, generator=generator, device="cuda") ** 3)
    kinds = [_KINDS[(i * 5 + seed) % len(_KINDS)] if case["mixed"] else (case["temperature"], case["top_k"], case["top_p"], case["min_p"]) for i in range(rows)]
    column = lambda i, dtype: torch.tensor([k[i] for k in kinds], dtype=dtype, device="cuda")  # noqa: E731
    return {"case": case, "logits": logits, "temperature": column(0, torch.float32), "top_k": column(1, torch.int32), "top_p": column(2, torch.float32),
            "min_p": column(3, torch.float32), "uniforms": torch.rand(rows, generator=generator, device="cuda"),
            "out": torch.empty(rows, dtype=torch.int32, device="cuda")}


# --- one pass -------------------------------------------------------------------------------------------------------------------
def run(state: dict):
    case = state["case"]
    if case["operator"] == "shared_prefix_attention":
        if not own:
            return _plain_attention(state)
        from tinyllama_inference_engine_b200 import ops

        heads, kv_heads, dim, _ = MODELS[case["model"]]
        ops.shared_prefix_attention(state["qkv"], state["pages"], state["positions"], state["seq_starts"], state["table"], case["shared"], state["out"], heads, kv_heads,
                                    dim, case["page_size"])
        return state["out"]
    if not own:
        return _plain_sampling(state)
    from tinyllama_inference_engine_b200 import ops

    ops.sample_filtered(state["logits"], state["temperature"], state["top_k"], state["top_p"], state["min_p"], state["uniforms"], state["out"])
    return state["out"]


def _plain_attention(state: dict) -> torch.Tensor:
    """Scores, softmax and weighted values in 32 bits: the prefix's keys once for all rows, each request's own behind them."""
    case = state["case"]
    heads, kv_heads, dim, _ = MODELS[case["model"]]
    group, shared, page_size = heads // kv_heads, case["shared"], case["page_size"]
    pages, table = state["pages"], state["table"].long()
    held, rows = _lengths(case)

    def gather(entry: int, first: int, end: int) -> torch.Tensor:   # keys and values [2, kv heads, tokens, dim] of positions first to end
        index = torch.arange(first, end, device="cuda")
        picked = pages[table[entry, index // page_size], :, :, index % page_size]       # [tokens, 2, kv heads, dim]
        return picked.permute(1, 2, 0, 3).float()

    q = state["qkv"][:, : heads * dim].float().view(-1, kv_heads, group, dim) * dim ** -0.5
    tokens = q.shape[0]
    prefix = gather(0, 0, shared)
    q_rows = q.permute(1, 0, 2, 3).reshape(kv_heads, tokens * group, dim)
    scores = q_rows @ prefix[0].transpose(1, 2)                                          # [kv heads, tokens * group, shared]
    top = scores.amax(2, keepdim=True)
    weights = torch.exp(scores - top)
    top, total, summed = (x.view(kv_heads, tokens, group, -1) for x in (top, weights.sum(2, keepdim=True), weights @ prefix[1]))
    del scores, weights
    out = torch.empty_like(q)
    at = 0
    for entry, (h, r) in enumerate(zip(held, rows)):
        mine = gather(entry, shared, shared + h)                                          # [2, kv heads, h, dim]
        q_mine = q[at : at + r].permute(1, 0, 2, 3)                                       # [kv heads, r, group, dim]
        own_scores = torch.einsum("krgd,kjd->krgj", q_mine, mine[0])
        if r > 1:
            later = torch.arange(h, device="cuda")[None, :] > torch.arange(h - r, h, device="cuda")[:, None]
            own_scores = torch.where(later[None, :, None, :], torch.full_like(own_scores, -math.inf), own_scores)
        t, n, s = top[:, at : at + r], total[:, at : at + r], summed[:, at : at + r]
        both = torch.maximum(t, own_scores.amax(3, keepdim=True))
        own_weights = torch.exp(own_scores - both)
        factor = torch.exp(t - both)
        o = (s * factor + torch.einsum("krgj,kjd->krgd", own_weights, mine[1])) / (n * factor + own_weights.sum(3, keepdim=True))
        out[at : at + r] = o.permute(1, 0, 2, 3)
        at += r
    return out.view(tokens, heads * dim).to(state["qkv"].dtype)


def _plain_sampling(state: dict) -> torch.Tensor:
    """In 64 bits: which token a sum's border falls on must not hang on a rounding."""
    logits = state["logits"].double()
    rows, vocab = logits.shape
    column = lambda x: x.double()[:, None]  # noqa: E731
    temperature, top_k, top_p, min_p, uniform = (column(state[k]) for k in ("temperature", "top_k", "top_p", "min_p", "uniforms"))
    ordered, ids = torch.sort(logits, dim=1, descending=True, stable=True)     # equal logits stay in order of ids
    greedy = temperature <= 0
    weights = torch.exp((ordered - ordered[:, :1]) / torch.where(greedy, torch.ones_like(temperature), temperature))
    place = torch.arange(vocab, device=logits.device)[None, :]
    in_top_k = place < torch.where(top_k > 0, top_k, torch.full_like(top_k, float(vocab)))
    running = torch.cumsum(torch.where(in_top_k, weights, torch.zeros_like(weights)), 1)
    before = torch.cat([torch.zeros_like(running[:, :1]), running[:, :-1]], 1)
    kept = in_top_k & ((before < top_p * running[:, -1:]) | (top_p >= 1)) & (weights >= min_p)
    by_id = torch.zeros_like(weights).scatter_(1, ids, torch.where(kept, weights, torch.zeros_like(weights)))
    sums = torch.cumsum(by_id, 1)
    drawn = (sums <= uniform * sums[:, -1:]).sum(1)
    return torch.where(greedy[:, 0], ids[:, 0], drawn).int()


# --- what a pass cannot do without ----------------------------------------------------------------------------------------------
def work(case: dict) -> dict:
    """Attention: queries, each key and value and the tables read once, the output written; 4 flops per query head, visible key and channel.
    Choice of tokens: logits and options read once; per token a difference, a product, an exponential, two comparisons and two sums."""
    if case["operator"] == "sample_filtered":
        rows, vocab = case["rows"], MODELS[case["model"]][3] + case["added"]
        return {"bytes": rows * (vocab * 4 + 24), "flops": 7 * rows * vocab}
    heads, kv_heads, dim, _ = MODELS[case["model"]]
    held, rows = _lengths(case)
    size = 4 if case["dtype"] == "float32" else 2
    tokens = sum(rows)
    visible = sum(r * (case["shared"] + h) - r * (r - 1) // 2 for h, r in zip(held, rows))
    table = -(-case["shared"] // case["page_size"]) + sum(-(-h // case["page_size"]) for h in held)
    return {"bytes": size * (2 * tokens * heads * dim + 2 * (case["shared"] + sum(held)) * kv_heads * dim) + 4 * (2 * tokens + table),
            "flops": 4 * heads * dim * visible}


# --- the definition in 64 bits --------------------------------------------------------------------------------------------------
def exact(case: dict, seed: int):
    state = prepare(case, seed)
    return _exact_attention(state) if case["operator"] == "shared_prefix_attention" else _exact_sampling(state)


def _exact_attention(state: dict) -> torch.Tensor:
    """Every request for itself, its whole context gathered page by page, one softmax over all of it."""
    case = state["case"]
    heads, kv_heads, dim, _ = MODELS[case["model"]]
    starts, positions = state["seq_starts"].tolist(), state["positions"].tolist()
    out = torch.empty(len(positions), heads, dim, dtype=torch.float64, device="cuda")
    for entry in range(len(starts) - 1):
        first, end = starts[entry], starts[entry + 1]
        length = positions[end - 1] + 1
        pages = state["table"][entry, : -(-length // case["page_size"])].long()
        context = state["pages"][pages].double().permute(1, 2, 0, 3, 4).reshape(2, kv_heads, -1, dim)[:, :, :length]
        keys, values = context[0], context[1]
        seen = torch.arange(length, device="cuda") <= torch.tensor(positions[first:end], device="cuda")[:, None]
        for h in range(heads):
            q = state["qkv"][first:end, h * dim : (h + 1) * dim].double()
            s = (q @ keys[h // (heads // kv_heads)].T) / math.sqrt(dim)
            p = torch.softmax(s.masked_fill(~seen, -math.inf), 1)
            out[first:end, h] = p @ values[h // (heads // kv_heads)]
    return out.view(len(positions), heads * dim)


def _exact_sampling(state: dict) -> np.ndarray:
    """Row by row with the kept tokens as a list."""
    logits = state["logits"].cpu().numpy().astype(np.float64)
    options = {k: state[k].cpu().numpy().astype(np.float64) for k in ("temperature", "top_p", "min_p", "uniforms")}
    tokens = np.empty(len(logits), dtype=np.int32)
    for r, row in enumerate(logits):
        order = np.argsort(-row, kind="stable")
        if options["temperature"][r] <= 0:
            tokens[r] = order[0]
            continue
        k = int(state["top_k"][r])
        order = order[:k] if k > 0 else order
        p = np.exp((row[order] - row[order[0]]) / options["temperature"][r])
        count = len(order)
        if options["top_p"][r] < 1:
            count = min(count, int(np.searchsorted(np.cumsum(p), options["top_p"][r] * p.sum())) + 1)
        count = min(count, int((p >= options["min_p"][r]).sum()))
        kept = np.sort(order[:count])
        mass = np.cumsum(np.exp((row[kept] - row[order[0]]) / options["temperature"][r]))
        tokens[r] = kept[min(int(np.searchsorted(mass, options["uniforms"][r] * mass[-1], side="right")), count - 1)]
    return tokens
