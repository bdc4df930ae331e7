"""Generation with top-k and min-p through the engine, and a decode loop of many answers to one prompt on the operators."""
from __future__ import annotations

import json

import numpy as np
import pytest
import torch

import plain_llama
import plain_ops
from test_answers_of_one_prompt import plain_choice
from tinyllama_inference_engine_b200 import EngineConfig
from tinyllama_inference_engine_b200.engine.api import Engine
from tinyllama_inference_engine_b200.engine.request import SamplingParams
from tinyllama_inference_engine_b200.errors import EngineError

MIXED = [dict(temperature=0.9, top_p=0.9), dict(temperature=0.8, top_k=7), dict(), dict(temperature=1.1, top_p=0.95, min_p=0.05), dict(temperature=1.0, top_k=3, top_p=0.8, min_p=0.1),
         dict(top_k=5, min_p=0.5)]


def _params(tokens: int) -> list[SamplingParams]:
    return [SamplingParams(max_tokens=tokens + 3 * i, seed=30 + i, **options) for i, options in enumerate(MIXED)]


def _prompts(vocab, lengths=(5, 21, 9, 14, 3, 8), seed=4):
    rng = np.random.default_rng(seed)
    return [[int(t) for t in rng.integers(0, vocab, size=n)] for n in lengths]


def _plain_generation(config, weights, prompt, params):
    """Token by token with the plain model, and whether some draw lay too near a border for 32-bit logits to tell."""
    tokens, generated, close = list(prompt), [], False
    for k in range(params.max_tokens):
        logits = plain_llama.forward(config, weights, tokens)[-1]
        u = plain_ops.uniform_from(params.seed, k)
        if params.filtered:
            token, _, near = plain_choice(logits, float(np.float32(params.temperature)), params.top_k, float(np.float32(params.top_p)), float(np.float32(params.min_p)), u)
            close |= near
        else:
            token = plain_llama.sample_top_p(logits.float(), params.temperature, params.top_p, u)
        generated.append(token)
        tokens.append(token)
    return generated, close


def _plain_sample_filtered(logits, temperature, top_k, top_p, min_p, uniforms, out, rows=None) -> None:
    for r in range(temperature.shape[0]):
        row = r if rows is None else int(rows[r])
        if 0 <= row < logits.shape[0]:
            out[row] = plain_choice(logits[row], float(temperature[r]), int(top_k[r]), float(top_p[r]), float(min_p[r]), float(uniforms[r]))[0]


def test_options_are_checked():
    assert not SamplingParams(top_k=5).filtered and SamplingParams(temperature=1.0, top_k=5).filtered and SamplingParams(temperature=1.0, min_p=0.1).filtered
    assert not SamplingParams(temperature=1.0, top_p=0.5).filtered
    for wrong in (dict(top_k=-1), dict(top_k=1.5), dict(top_k=True), dict(top_k=1 << 31), dict(min_p=-0.1), dict(min_p=1.1), dict(min_p=float("nan"))):
        with pytest.raises(EngineError):
            SamplingParams(**wrong)


def test_generation_with_filters_on_the_plain_functions(model_folders, monkeypatch):
    from tinyllama_inference_engine_b200 import ops

    plain_ops.install(monkeypatch)
    monkeypatch.setattr(ops, "sample_filtered", _plain_sample_filtered)
    config, weights = plain_llama.load_model(model_folders["a"])
    prompts, params = _prompts(config["vocab_size"]), _params(4)
    engine = Engine(model_folders["a"], EngineConfig(dtype="float32", page_size=16, max_cache_tokens=512, max_requests=6, max_batch_tokens=32, device="cpu"))
    got = [r.generated_tokens for r in engine.generate(prompts, params)]
    for prompt, p, tokens in zip(prompts, params, got):
        want, close = _plain_generation(config, weights, prompt, p)
        assert close or tokens == want, p


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [False, True])
def test_generation_with_filters(model_folders, graphs):
    config, weights = plain_llama.load_model(model_folders["b"])
    prompts, params = _prompts(config["vocab_size"]), _params(12)
    options = dict(page_size=16, max_cache_tokens=1024, max_requests=6, max_batch_tokens=64, use_cuda_graphs=graphs)
    engine = Engine(model_folders["b"], EngineConfig(dtype="float32", **options))
    together = [r.generated_tokens for r in engine.generate(prompts, params)]
    checked = 0
    for prompt, p, tokens in zip(prompts, params, together):
        assert len(tokens) == p.max_tokens
        want, close = _plain_generation(config, weights, prompt, p)
        if not close:
            assert tokens == want, p
            checked += 1
    assert checked >= 4
    # alone, and beside requests without filters: a request's tokens are its own
    for i in (1, 3, 4):
        assert engine.generate([prompts[i]], [params[i]])[0].generated_tokens == together[i]
    # a session's steps with and without filters are graphs of their own, taken up again in turn
    plain = [SamplingParams(max_tokens=14, temperature=0.9, top_p=0.9, seed=i) for i in range(6)]
    before = [r.generated_tokens for r in Engine(model_folders["b"], EngineConfig(dtype="float32", **options)).generate(prompts, plain)]
    for _ in range(2):
        assert [r.generated_tokens for r in engine.generate(prompts, plain)] == before
        assert [r.generated_tokens for r in engine.generate(prompts, params)] == together
    bf16 = Engine(model_folders["b"], EngineConfig(dtype="bfloat16", **options))
    assert all(0 <= t < config["vocab_size"] for r in bf16.generate(prompts, params) for t in r.generated_tokens)


@pytest.mark.gpu
def test_command_line_takes_the_filters(model_folders, capsys):
    from tinyllama_inference_engine_b200.cli import main

    line = ["generate", str(model_folders["a"]), "1,2,3", "8", "--dtype", "float32", "--temperature", "0.9", "--seed", "3"]
    runs = []
    for more in (["--top-k", "4", "--min-p", "0.05"], ["--top-k", "4", "--min-p", "0.05"], []):
        assert main(line + more) == 0
        runs.append(json.loads(capsys.readouterr().out.strip().splitlines()[-1])["generated_tokens"])
    config, weights = plain_llama.load_model(model_folders["a"])
    want, close = _plain_generation(config, weights, [1, 2, 3], SamplingParams(max_tokens=8, temperature=0.9, seed=3, top_k=4, min_p=0.05))
    assert runs[0] == runs[1] and (close or runs[0] == want)
    assert main(line + ["--min-p", "2"]) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("shared,answers", [(150, 5), (700, 40)])
def test_many_answers_to_one_prompt(dtype, shared, answers):
    """One layer's decode steps, captured once and replayed: the step's rows from the last tokens, keys and values stored, attention over the shared prompt, logits, a choice
    with every filter.  Every step's attention agrees with the kernel that shares nothing, every token with the plain choice from the step's own logits."""
    from tinyllama_inference_engine_b200 import ops

    heads, kv_heads, dim, page_size, vocab, steps = 8, 2, 64, 64, 2000, 6
    g = torch.Generator().manual_seed(answers)
    width = -(-(shared + steps) // page_size)
    whole = shared // page_size
    pages = (torch.randn(whole + answers * (width - whole), 2, kv_heads, page_size, dim, generator=g)).to(dtype).cuda()
    table = torch.empty(answers, width, dtype=torch.int32)
    table[:, :whole] = torch.arange(whole)
    table[:, whole:] = whole + torch.arange(answers * (width - whole)).view(answers, -1)
    if shared % page_size:   # every answer's own copy of the page that the prompt ends in
        for row in range(1, answers):
            pages[table[row, whole].item(), :, :, : shared % page_size] = pages[table[0, whole].item(), :, :, : shared % page_size]
    table = table.cuda()
    embedding = (torch.randn(vocab, (heads + 2 * kv_heads) * dim, generator=g)).to(dtype).cuda()
    head = torch.randn(vocab, heads * dim, generator=g).cuda() * 0.6
    inv_freq = (10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float32) / dim)).cuda()
    token_seq = torch.arange(answers, dtype=torch.int32, device="cuda")
    starts = torch.arange(answers + 1, dtype=torch.int32, device="cuda")
    positions = torch.full((answers,), shared, dtype=torch.int32, device="cuda")
    tokens = torch.randint(0, vocab, (answers,), generator=g).int().cuda()
    options = [torch.tensor(v, device="cuda").expand(answers).contiguous() for v in (0.9, 0.95, 0.01)]
    top_k = torch.full((answers,), 40, dtype=torch.int32, device="cuda")
    seeds, counters = torch.arange(answers, device="cuda"), torch.zeros(answers, dtype=torch.int64, device="cuda")
    uniforms = torch.empty(answers, device="cuda")
    out = torch.empty(answers, heads * dim, dtype=dtype, device="cuda")
    logits = torch.empty(answers, vocab, device="cuda")

    def step():
        qkv = embedding[tokens.long()]
        ops.rope_store(qkv, positions, token_seq, table, inv_freq, dim, pages, heads, kv_heads, dim, page_size)
        ops.shared_prefix_attention(qkv, pages, positions, starts, table, shared, out, heads, kv_heads, dim, page_size)
        torch.mm(out.float(), head.t(), out=logits)
        ops.uniforms(seeds, counters, uniforms)
        ops.sample_filtered(logits, options[0], top_k, options[1], options[2], uniforms, tokens)
        positions.add_(1)
        counters.add_(1)
        return qkv

    state = [t.clone() for t in (tokens, positions, counters, pages)]
    step()
    for t, kept in zip((tokens, positions, counters, pages), state):
        t.copy_(kept)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qkv = step()
    reach = float(pages.float().abs().max())
    for k in range(steps):
        graph.replay()
        whole_attention = torch.empty_like(out)
        ops.paged_attention(qkv, pages, positions - 1, token_seq, table, whole_attention, heads, kv_heads, dim, page_size)
        # each of the two may be off by what the tests of the kernels alone allow (weights and output rounded to 8 bits, or 32-bit sums of some 700 terms)
        bound = 2 * reach * (2 * 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24 * 2 * (shared + steps + 200))
        assert float((out.float() - whole_attention.float()).abs().max()) <= bound
        for row in range(answers):
            want, _, close = plain_choice(logits[row].cpu(), float(np.float32(0.9)), 40, float(np.float32(0.95)), float(np.float32(0.01)), ops.uniform_from(row, k))
            assert close or int(tokens[row]) == want
    assert positions.tolist() == [shared + steps] * answers
    ops.check_device_errors(torch.device("cuda:0"))
