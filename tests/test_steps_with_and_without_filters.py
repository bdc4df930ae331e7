"""Decode sessions that go from requests with top-k or min-p to requests without and back, and models whose vocabulary is too long for such requests."""
from __future__ import annotations

import numpy as np
import pytest

import plain_llama
import plain_ops
from test_answers_of_one_prompt import plain_choice
from test_filtered_generation import _params, _prompts
from tinyllama_inference_engine_b200 import EngineConfig
from tinyllama_inference_engine_b200.engine.api import Engine
from tinyllama_inference_engine_b200.engine.request import SamplingParams
from tinyllama_inference_engine_b200.errors import EngineError


@pytest.mark.gpu
def test_a_session_counts_the_kernels_of_the_steps_it_runs(model_folders):
    config, _ = plain_llama.load_model(model_folders["b"])
    prompts = _prompts(config["vocab_size"])[:4]
    kinds = {"plain": SamplingParams(max_tokens=8, temperature=0.9), "filtered": SamplingParams(max_tokens=8, temperature=0.9, top_k=5)}

    def engine():
        return Engine(model_folders["b"], EngineConfig(dtype="bfloat16", page_size=16, max_cache_tokens=512, max_requests=4, max_batch_tokens=64))

    def counts(e):
        session = e._sessions[4]
        return session.kernels_per_step, session.library_calls_per_step

    alone = {}
    for kind, params in kinds.items():
        e = engine()
        e.generate(prompts, params)
        alone[kind] = counts(e)
    assert alone["filtered"][0] == alone["plain"][0] + 2   # the numbers and the choice
    e = engine()
    for kind in ("plain", "filtered", "plain", "plain", "filtered", "plain"):
        e.generate(prompts, kinds[kind])
        assert counts(e) == alone[kind], kind


def test_filters_are_refused_where_the_vocabulary_is_too_long(model_folders, monkeypatch):
    """ops.sample_filtered takes vocabularies up to a limit: beyond it a request that needs it is refused when it is added, not in the middle of a step."""
    from tinyllama_inference_engine_b200 import ops

    plain_ops.install(monkeypatch)
    config, _ = plain_llama.load_model(model_folders["a"])
    engine = Engine(model_folders["a"], EngineConfig(dtype="float32", page_size=16, max_cache_tokens=512, max_requests=6, max_batch_tokens=32, device="cpu"))
    monkeypatch.setattr(ops, "SAMPLE_FILTERED_MAX_VOCAB", config["vocab_size"] - 1)
    for options in (dict(top_k=5), dict(min_p=0.1)):
        with pytest.raises(EngineError, match=f"{config['vocab_size']} tokens"):
            engine.add_request([1, 2, 3], SamplingParams(temperature=0.7, **options))
        engine.add_request([1, 2, 3], SamplingParams(**options))   # (greedy: these options say nothing)
    assert len(engine.requests) == 2
    monkeypatch.setattr(ops, "SAMPLE_FILTERED_MAX_VOCAB", config["vocab_size"])
    engine.add_request([1, 2, 3], SamplingParams(temperature=0.7, top_k=5))


@pytest.mark.gpu
def test_bfloat16_requests_get_the_choice_from_their_steps_logits(model_folders, monkeypatch):
    """Every token of a filtered request of a bfloat16 engine is the 64-bit choice from the logits that its step worked out."""
    from tinyllama_inference_engine_b200 import ops

    config, _ = plain_llama.load_model(model_folders["b"])
    prompts, params = _prompts(config["vocab_size"]), _params(6)
    engine = Engine(model_folders["b"], EngineConfig(dtype="bfloat16", page_size=16, max_cache_tokens=1024, max_requests=6, max_batch_tokens=64, use_cuda_graphs=False))
    chosen, choose = [], ops.sample_filtered

    def recorded(logits, temperature, top_k, top_p, min_p, uniforms, out, rows):
        choose(logits, temperature, top_k, top_p, min_p, uniforms, out, rows)
        chosen.append([t.clone() for t in (logits, temperature, top_k, top_p, min_p, uniforms, out, rows)])

    monkeypatch.setattr(ops, "sample_filtered", recorded)
    results = engine.generate(prompts, params)
    tokens, checked, token_of = 0, 0, {}
    for logits, temperature, top_k, top_p, min_p, uniforms, out, rows in chosen:
        for r, row in enumerate(rows.tolist()):
            if row < 0:   # (a request without filters)
                continue
            tokens += 1
            token_of[float(uniforms[r])] = int(out[row])
            want, _, close = plain_choice(logits[row].cpu(), float(temperature[r]), int(top_k[r]), float(top_p[r]), float(min_p[r]), float(uniforms[r]))
            if not close:
                assert int(out[row]) == want
                checked += 1
    assert tokens == sum(p.max_tokens for p in params if p.filtered) and checked >= tokens * 3 // 4
    for p, result in zip(params, results):
        assert len(result.generated_tokens) == p.max_tokens
        if p.filtered:   # draw k of a request is made with its k-th number
            assert [token_of[float(np.float32(ops.uniform_from(p.seed, k)))] for k in range(p.max_tokens)] == result.generated_tokens
