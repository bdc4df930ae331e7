"""The Python entry point: an engine that takes token ids and returns generated token ids.

The reference's Python side spawns its binaries and parses their JSON
(scripts/compare_logits.py:110-145); its request options live in the server
(app/server.cpp:601-613).  Here the engine is a Python object with the same option
names: ``Engine(model_dir).generate(prompts, SamplingParams(max_tokens=..., temperature=..., top_p=...))``.
"""
from __future__ import annotations

import itertools
import time
from dataclasses import dataclass, field
from pathlib import Path

from .. import ops
from ..config import EngineConfig
from ..errors import EngineError
from ..sampling import Sampler
from .batch import StepEntry
from .decode_session import DecodeSession
from .request import FINISHED, Request, SamplingParams
from .runner import ModelRunner
from .scheduler import Scheduler
from .timing import StepClock, StepTimings, nvtx_range


@dataclass
class TokenOutput:
    request_id: str
    token: int
    finished: bool
    finish_reason: str | None


@dataclass
class GenerationResult:
    request_id: str
    prompt_tokens: list[int]
    generated_tokens: list[int]
    finish_reason: str | None
    preemptions: int = 0


class Engine:
    def __init__(self, model_dir: str | Path, engine_config: EngineConfig | None = None, **options):
        if engine_config is None:
            engine_config = EngineConfig(**options)
        elif options:
            raise EngineError("give either an EngineConfig or keyword options, not both")
        self.config = engine_config
        self.runner = ModelRunner(model_dir, engine_config)
        self.model_config = self.runner.model_config
        self.scheduler = Scheduler(self.runner.cache, engine_config.max_batch_tokens, engine_config.max_requests, self.runner.spec.max_positions)
        self.sampler = Sampler(self.runner.device)
        self.requests: dict[str, Request] = {}
        self._sessions: dict[int, DecodeSession] = {}
        self._session_key: tuple | None = None   # requests whose next tokens the last step left on the device
        self._ahead: tuple | None = None         # (session, requests) of a decode step launched ahead of its step() call
        self._ids = itertools.count()
        self.generated_tokens = 0
        self.prompt_tokens = 0

    # --- requests ---------------------------------------------------------------------------
    def add_request(self, prompt_token_ids: list[int], params: SamplingParams | None = None, request_id: str | None = None) -> str:
        params = params or SamplingParams()
        request_id = request_id if request_id is not None else f"req-{next(self._ids)}"
        if request_id in self.requests and self.requests[request_id].state != FINISHED:
            raise EngineError(f"request id {request_id!r} is in use")
        vocab = self.runner.spec.vocab_size
        prompt = [int(t) for t in prompt_token_ids]
        for token in prompt:
            if not 0 <= token < vocab:
                raise EngineError(f"input token {token} is outside the model vocabulary", code="out_of_bounds")
        if params.filtered and vocab > ops.SAMPLE_FILTERED_MAX_VOCAB:
            raise EngineError(f"top_k and min_p are for vocabularies of at most {ops.SAMPLE_FILTERED_MAX_VOCAB} tokens, this model has {vocab} tokens")
        request = Request(request_id, prompt, params)
        self.scheduler.add(request)
        self.requests[request_id] = request
        return request_id

    def cancel(self, request_id: str) -> None:
        request = self.requests.get(request_id)
        if request is not None and request.state != FINISHED:
            self.scheduler.finish(request, "cancelled")

    def has_unfinished(self) -> bool:
        return self.scheduler.has_unfinished()

    # --- one step ---------------------------------------------------------------------------
    def step(self, timings: StepTimings | None = None) -> list[TokenOutput]:
        """Schedule, run one batch, sample; returns the tokens generated by this step.

        ``timings``: what the step cost is added to it (device time of the forward pass and of the copies, host wall time); a
        step that is timed is not launched ahead of its call."""
        if self._ahead is not None:
            return self._collect_ahead()
        portions = self.scheduler.schedule()
        if not portions:
            return []
        if self._can_use_session(portions):
            requests = [p.request for p in portions]
            with nvtx_range("decode"):
                clock = StepClock(self.runner.device, timings is not None)
                session = self._session_step(portions)
                clock.mark()
                tokens = session.read_tokens()
                clock.mark()
                clock.finish(timings, ("compute", "transfer"))
            if timings is None:
                self._launch_ahead(session, requests, tokens)
            return self._finish_step(portions, requests, tokens)
        self._session_key = None
        entries, sampling = [], []
        for portion in portions:
            request = portion.request
            tokens = request.next_tokens(portion.num_tokens)
            entries.append(StepEntry(request.request_id, tokens, [portion.num_tokens - 1] if portion.samples else []))
            if portion.samples:
                sampling.append(request)
        with nvtx_range("prefill" if any(p.num_tokens > 1 for p in portions) else "decode"):
            logits = self.runner.step(entries, timings)
        with nvtx_range("sampling"):
            clock = StepClock(self.runner.device, timings is not None and bool(sampling))
            tokens = self.sampler.select(logits, [r.params for r in sampling], [len(r.generated) for r in sampling]) if sampling else []
            clock.mark()
            if sampling and timings is not None:
                sampled = StepTimings()
                clock.finish(sampled, ("compute",))   # the choice of tokens and their way to the host
                timings.compute_ms += sampled.compute_ms
                timings.wall_ms += sampled.wall_ms
        return self._finish_step(portions, sampling, tokens)

    def _can_use_session(self, portions) -> bool:
        return (self.config.use_cuda_graphs and self.runner.device.type == "cuda" and self.runner.model.capturable
                and all(p.num_tokens == 1 and p.samples and p.request.computed > 0 for p in portions))   # live requests only: a one-token prompt is not

    def _session_step(self, portions) -> list[int]:
        """A step of single decoded tokens only: replay the decode graph of this many requests."""
        requests = [p.request for p in portions]
        key = tuple(r.request_id for r in requests)
        session = self._sessions.get(len(key))
        if session is None:
            session = self._sessions[len(key)] = DecodeSession(self.runner, len(key))
        tokens = [r.next_tokens(1)[0] for r in requests]   # the last generated token, or the only token of a one-token prompt
        if self._session_key == key:
            session.set_tokens(tokens)
        else:
            session.load(list(key), tokens, [r.params for r in requests], [len(r.generated) for r in requests])
        self._session_key = key
        session.step()
        return session

    # A run of pure decode steps is predictable: while nobody waits, nobody finishes and pages are there, the next step is
    # the same batch fed with the tokens just read.  It is launched right after those tokens reach the host, BEFORE the
    # bookkeeping of the step they belong to, so that bookkeeping and scheduling run under the GPU's next step instead
    # of between two steps.  Every step still takes its input ids from pinned host memory and returns its ids to the host.
    def _launch_ahead(self, session, requests, tokens) -> None:
        if self.scheduler.waiting or len(self.scheduler.running) != len(requests):
            return
        eos = getattr(self.model_config, "eos_token_id", None)
        for request, token in zip(requests, tokens):
            if len(request.generated) + 2 > request.params.max_tokens:   # finishes with this token or with the next one
                return
            if not request.params.ignore_eos and eos is not None and token == eos:
                return
        if not session.next_step_fits_its_pages():   # a page boundary: ask the cache (most steps stay inside the pages they have)
            cache = self.runner.cache
            if not cache.can_reserve([(r.request_id, cache.computed(r.request_id) + 1) for r in requests]):
                return   # out of pages: the scheduler decides who gives way
        session.set_tokens(tokens)
        session.step()
        self._ahead = (session, requests)

    def _collect_ahead(self) -> list[TokenOutput]:
        from .scheduler import ScheduledPortion

        session, requests = self._ahead
        self._ahead = None
        tokens = session.read_tokens()
        self.scheduler.steps += 1
        live = [(r, t) for r, t in zip(requests, tokens) if r.state != FINISHED]   # a request cancelled meanwhile drops out
        if len(live) == len(requests):
            self._launch_ahead(session, requests, tokens)
        else:
            self._session_key = None
        live_requests = [r for r, _ in live]
        return self._finish_step([ScheduledPortion(r, 1) for r in live_requests], live_requests, [t for _, t in live])

    def _finish_step(self, portions, sampling, tokens) -> list[TokenOutput]:
        outputs: list[TokenOutput] = []
        for portion in portions:
            self.prompt_tokens += portion.num_tokens if not portion.samples or portion.num_tokens > 1 else 0
            portion.request.computed += portion.num_tokens
        if sampling:
            eos = getattr(self.model_config, "eos_token_id", None)
            for request, token in zip(sampling, tokens):
                request.generated.append(token)
                self.generated_tokens += 1
                reason = None
                if len(request.generated) >= request.params.max_tokens:
                    reason = "length"
                elif not request.params.ignore_eos and eos is not None and token == eos:
                    reason = "stop"
                if reason:
                    self.scheduler.finish(request, reason)
                outputs.append(TokenOutput(request.request_id, token, reason is not None, reason))
        return outputs

    # --- whole generations --------------------------------------------------------------------
    def generate(self, prompts: list[list[int]], params: SamplingParams | list[SamplingParams] | None = None) -> list[GenerationResult]:
        """Generate for every prompt (lists of token ids); results in the order of the prompts."""
        if params is None or isinstance(params, SamplingParams):
            params = [params or SamplingParams()] * len(prompts)
        ids = [self.add_request(prompt, p) for prompt, p in zip(prompts, params)]
        while self.has_unfinished():
            self.step()
        results = []
        for request_id in ids:
            r = self.requests.pop(request_id)
            results.append(GenerationResult(request_id, r.prompt, r.generated, r.finish_reason, r.preemptions))
        return results

    def metrics(self) -> dict:
        """Counters in the manner of the reference's /metrics (app/server.cpp:216-231)."""
        return {
            "steps": self.runner.steps,
            "tokens_run": self.runner.tokens_run,
            "generated_tokens": self.generated_tokens,
            "preemptions": self.scheduler.preemptions,
            "waiting": len(self.scheduler.waiting),
            "running": len(self.scheduler.running),
            "cache": self.runner.cache.stats(),
        }


def generate(model_dir: str | Path, prompts: list[list[int]], max_tokens: int = 16, temperature: float = 0.0, top_p: float = 1.0,
             seed: int = 0, dtype: str = "bfloat16", **engine_options) -> list[list[int]]:
    """One call from a model folder and prompts (token ids) to generated token ids."""
    engine = Engine(model_dir, EngineConfig(dtype=dtype, **engine_options))
    results = engine.generate(prompts, SamplingParams(max_tokens=max_tokens, temperature=temperature, top_p=top_p, seed=seed))
    return [r.generated_tokens for r in results]
