"""The synchronous engine loop: plan a step, run it as one model call, sample on the device, read
the tokens, apply them, free what finished.

An entry point in the manner of the reference's ``ContinuousBatchEngine``
(src/mini_llm_runtime/engine.py:69-281): ``submit`` and ``step``, one device-to-host copy per step
(the chosen tokens), scheduler and cache rolled back when a step fails, a finished request's pages
free right after its results are applied, optional NVTX ranges under the reference's names.
Differences: one model call per step where the reference makes a prefill call and a decode call;
prompts may arrive in portions; requests may sample with a temperature; page admission is part of
the scheduler (its gate), so the constructor takes no admission controller; and a step of decoded
tokens sends the device nothing but the slots of its requests, because positions, last tokens and
sampling state live in the requests' slot records.  ``from_model_dir`` / ``from_model`` do the
assembly that the reference's runner script does by hand
(experiments/continuous_batch_engine_runner.py:227-278 there), and ``greedy_generate`` is the
single-request loop of src/mini_llm_runtime/generation.py:29-117.
"""

from __future__ import annotations

import contextlib
import time
from collections.abc import Callable, Collection, Sequence
from dataclasses import dataclass

import numpy as np
import torch

from .. import ops
from ..cache.allocator import OutOfPages
from ..cache.manager import CacheManager
from ..models.decoder import DecoderModel
from ..sampling import LogitRules, RequestLimits, SamplingParams
from .metrics import RequestMetricsCollector
from .scheduler import BatchingPolicy, CacheGate, Request, RequestScheduler, RequestStatus, StepOutcome, StepPlan, WorkKind
from .step import ModelRunner, StepEntry


@dataclass
class _TokensInFlight:
    """The tokens of a launched step on their way to the host: ``request_ids`` in row order, ``host``
    the pinned destination, ``event`` the end of the copy (None when nothing is asynchronous)."""

    request_ids: tuple[str, ...]
    host: torch.Tensor
    event: "torch.cuda.Event | None"

    def wait(self) -> dict[str, int]:
        if self.event is not None:
            self.event.synchronize()
        return dict(zip(self.request_ids, self.host[:len(self.request_ids)].tolist(), strict=True))


@dataclass(frozen=True)
class EngineStepResult:
    """One engine step: what was planned, what came out, and when (nanoseconds of the engine's clock)."""

    plan: StepPlan
    outcome: StepOutcome
    started_ns: int
    tokens_ready_ns: int
    completed_ns: int

    @property
    def freed(self):
        return self.outcome.freed


class ContinuousBatchEngine:
    def __init__(self, *, scheduler: RequestScheduler, runner: ModelRunner,
                 clock_ns: Callable[[], int] = time.perf_counter_ns,
                 metrics: RequestMetricsCollector | None = None, enable_nvtx: bool = False,
                 step_ahead: bool = False) -> None:
        gate = scheduler.gate
        if not isinstance(gate, CacheGate) or gate.cache is not runner.cache:
            raise ValueError("the scheduler's gate must be a CacheGate on the runner's cache manager")
        if enable_nvtx and runner.device.type != "cuda":
            raise ValueError("NVTX ranges need a CUDA engine")
        self.scheduler = scheduler
        self.runner = runner
        self._clock_ns = clock_ns
        self.metrics = metrics or RequestMetricsCollector()
        self.enable_nvtx = enable_nvtx
        # Stepping ahead: when a step decodes only, the same requests' next decode step is launched
        # right behind it, before the host has read the tokens: the device takes each request's input
        # from its slot record, where the sampling kernel has just stored it.  The host's work between
        # two steps then runs beside the GPU instead of idling it.  What step() returns does not
        # change; a request that ends on a stop token has computed one token too many, which is
        # dropped with its pages.
        self.step_ahead = step_ahead
        self._ahead: _TokensInFlight | None = None
        self._token_buffers: list[torch.Tensor] = []
        self._next_buffer = 0
        self._prefixes: dict[str, tuple[int, ...]] = {}      # tokens of the prefixes that requests may share, by name
        self._allowed: dict[str, np.ndarray] = {}      # grammars of requests that wait, until they own a slot

    # ------------------------------------------------------------------ assembly
    DEFAULT_MODEL_LEN = 32768

    @classmethod
    def from_model(cls, model: DecoderModel, *, block_size: int = 16, total_blocks: int | None = None,
                   max_running_requests: int = 8, max_batch_tokens: int = 2048,
                   max_mixed_prefill_tokens: int | None = None, max_model_len: int | None = None,
                   batching_policy: BatchingPolicy = BatchingPolicy.CONTINUOUS,
                   chunked_prefill: bool = True, enable_nvtx: bool = False,
                   step_ahead: bool = False, logit_rules: bool = False, max_prefixes: int = 0,
                   sampling_limits: bool = False, cache_dtype: str | None = None, cache_block: int = 1) -> "ContinuousBatchEngine":
        """``logit_rules``: requests may bring penalties, biases and grammars (``submit``, ``allow_tokens``); every step then applies them.
        ``max_prefixes``: how many prefixes the cache may hold for requests to share (``add_prefix``).  ``sampling_limits``: requests may
        limit what is drawn for them by top-k, top-p and min-p; every step then draws under the limits of its requests.
        ``cache_dtype="int8"``: the cache holds keys and values in 8 bits with a scale for each ``cache_block`` tokens and kv head (models
        whose layers all attend to such a cache).  With blocks of one token what is held for a token does not depend on how its
        prompt was cut nor on what follows it; larger blocks save up to four bytes per token and head."""
        if cache_dtype not in (None, "int8"):
            raise ValueError(f"unknown cache dtype {cache_dtype!r}; known: int8, or None for the model's own")
        # a model without a position limit of its own gets this engine's default
        max_model_len = min(max_model_len or min(model.spec.max_positions, cls.DEFAULT_MODEL_LEN),
                            model.spec.max_positions)
        if max_prefixes < 0:
            raise ValueError("max_prefixes must be >= 0")
        if total_blocks is None:
            total_blocks = (max_running_requests + max_prefixes) * -(-max_model_len // block_size)
        cache = CacheManager(model.cache_needs(), page_size=block_size, num_pages=total_blocks,
                             max_requests=max_running_requests + max_prefixes, max_tokens_per_request=max_model_len,
                             dtype=model.compute_dtype, device=model.device, max_step_tokens=max_batch_tokens,
                             quantized_block=None if cache_dtype is None else cache_block)
        scheduler = RequestScheduler(max_running_requests=max_running_requests, max_batch_tokens=max_batch_tokens,
                                     max_mixed_prefill_tokens=max_mixed_prefill_tokens, gate=CacheGate(cache),
                                     batching_policy=batching_policy, chunked_prefill=chunked_prefill)
        runner = ModelRunner(model, cache)
        if logit_rules:
            runner.rules = LogitRules(cache.max_requests, runner.vocab_size, model.device)
        if sampling_limits:
            runner.limits = RequestLimits(cache.max_requests, model.device)
        return cls(scheduler=scheduler, runner=runner, enable_nvtx=enable_nvtx, step_ahead=step_ahead)

    @classmethod
    def from_model_dir(cls, model_dir, *, dtype="bfloat16", device="cuda:0", **options) -> "ContinuousBatchEngine":
        from ..models.factory import load_model
        _, model = load_model(model_dir, dtype, device)
        return cls.from_model(model, **options)

    @property
    def manager(self) -> CacheManager:
        return self.runner.cache

    def _range(self, message: str):
        """An NVTX range around a phase of the step when tracing is on (names as in the reference:
        engine.py:158-168,191-195,233-236,251,257,267)."""
        return torch.cuda.nvtx.range(message) if self.enable_nvtx else contextlib.nullcontext()

    # ------------------------------------------------------------------ requests
    def submit(self, request_id: str, prompt_token_ids: Sequence[int], *, max_new_tokens: int,
               eos_token_ids: int | Collection[int] | None = None, temperature: float = 0.0,
               seed: int = 0, prefix: str | None = None, fork_of: str | None = None, **rules) -> Request:
        """``prefix``: a prefix of ``add_prefix`` that the prompt starts with; its whole pages are shared, not computed again.
        ``fork_of``: a request, waiting or running, whose prompt and output so far begin like the prompt; what its cache holds of them when the
        new request is admitted is taken from there (whole pages held by both, the last one copied), or from another fork of it if it has ended,
        and computed if there is none.
        ``rules``: ``repetition_penalty``, ``presence_penalty``, ``frequency_penalty``, ``logit_bias`` of ``SamplingParams`` (an engine
        made with ``logit_rules=True``), and its ``top_k``, ``top_p``, ``min_p`` (an engine made with ``sampling_limits=True``)."""
        arrival_ns = self._clock_ns()
        request = self.scheduler.submit(request_id, prompt_token_ids, **self._checked(
            request_id, prompt_token_ids, max_new_tokens, eos_token_ids, temperature, seed, prefix, fork_of, rules))
        self.metrics.register_request(request_id, arrival_ns)
        return request

    def _checked(self, request_id, prompt_token_ids, max_new_tokens, eos_token_ids, temperature, seed, prefix, fork_of, rules) -> dict:
        """What the scheduler is told of a request that the engine can run; an error for another."""
        vocab = self.runner.vocab_size
        outside = [t for t in prompt_token_ids if not isinstance(t, int) or isinstance(t, bool) or not 0 <= t < vocab]
        if outside:
            raise ValueError(f"prompt token ids must be integers in [0, {vocab}); got {outside[:5]}")
        longest = len(prompt_token_ids) + max_new_tokens - 1
        if longest > self.manager.max_tokens_per_request:
            raise ValueError(f"prompt + max_new_tokens - 1 = {longest} exceeds the engine's limit of "
                             f"{self.manager.max_tokens_per_request} tokens per request")
        sampling = SamplingParams(temperature, seed, **rules)
        if self.runner.rules is not None:
            self.runner.rules.check(sampling)
        elif sampling.has_rules:
            raise ValueError("rules on logits need an engine made with logit_rules=True")
        if sampling.has_limits and self.runner.limits is None:
            raise ValueError("limits on what is drawn need an engine made with sampling_limits=True")
        if any(request_id == self._holder(name) for name in self._prefixes):
            raise ValueError(f"{request_id!r} is the name under which the cache holds a prefix")
        common = self._common_tokens(request_id, fork_of, prefix, prompt_token_ids)
        holder, shared = self._shared_by(prefix, prompt_token_ids)
        if self._prefixes and not self.manager.can_be_admitted(longest, None if holder is None else (holder, shared)):
            raise ValueError(self.manager.why_not_admitted(request_id, longest, shared // self.manager.page_size))
        return {"max_new_tokens": max_new_tokens, "eos_token_ids": eos_token_ids, "sampling": sampling, "prefix": holder, "shared": shared,
                "fork": None if not common else (fork_of, common)}

    # ------------------------------------------------------------------ forks
    def _common_tokens(self, request_id: str, fork_of: str | None, prefix: str | None, prompt: Sequence[int]) -> int:
        """How many of the prompt's tokens, less one, are the first of the other request."""
        if fork_of is None:
            return 0
        if prefix is not None:
            raise ValueError("a fork shares the prefix of the request it starts with; prefix and fork_of exclude one another")
        if not self.manager.can_share_pages:
            raise ValueError("requests fork in models whose layers keep every key, without windows or states")
        if fork_of == request_id:
            raise ValueError(f"request {request_id!r} cannot fork from itself")
        other = self.scheduler.get_request(fork_of)
        known = (*other.prompt, *other.output)
        common = 0
        for mine, theirs in zip(prompt[:len(prompt) - 1], known):
            if mine != theirs:
                break
            common += 1
        return common

    def resize_cache(self, total_blocks: int | Sequence[int]) -> None:
        """Pools of another size for the cache, between steps: memory given back to others, or more room.  What requests hold moves along;
        decode steps are captured anew."""
        manager = self.manager
        counts = manager.can_resize(total_blocks)
        for request_id in self.scheduler.waiting_request_ids:
            request = self.scheduler.get_request(request_id)
            named = None if request.prefix is None else (request.prefix, request.shared)
            if not manager.can_be_admitted(request.lifetime_tokens, named, pools=counts):      # beside the prefixes' pages
                raise OutOfPages(f"the waiting request {request_id!r} could never be admitted to pools of {counts} pages")
        self.runner.forget_captured_steps()
        manager.resize(counts)

    # ------------------------------------------------------------------ shared prefixes
    @staticmethod
    def _holder(name: str) -> str:
        return f"prefix {name}"

    @torch.inference_mode()
    def add_prefix(self, name: str, token_ids: Sequence[int]) -> int:
        """Compute a prefix that requests may start with (a system prompt, a document) and keep its pages until ``drop_prefix``; to be
        called between steps.  Returns how many of its tokens are shared: those on whole pages."""
        tokens = tuple(int(t) for t in token_ids)
        page = self.manager.page_size
        if not self.manager.can_share_pages:
            raise ValueError("pages are shared by models whose layers keep every key, without windows or states")
        if name in self._prefixes:
            raise ValueError(f"prefix {name!r} exists already")
        if self._holder(name) in (*self.scheduler.waiting_request_ids, *self.scheduler.running_request_ids):
            raise ValueError(f"a request is called {self._holder(name)!r}, as the cache would call prefix {name!r}")
        if len(tokens) < page:
            raise ValueError(f"a prefix of {len(tokens)} tokens fills no page of {page}")
        if any(not 0 <= t < self.runner.vocab_size for t in tokens):
            raise ValueError(f"prefix token ids must lie in [0, {self.runner.vocab_size})")
        shared = len(tokens) // page * page
        holder = self._holder(name)
        if self.manager.slots.free_count <= self.scheduler.max_running_requests - len(self.scheduler.running_request_ids):
            raise ValueError(f"the engine was made for {self.manager.max_requests - self.scheduler.max_running_requests} prefixes")
        for request_id in self.scheduler.waiting_request_ids:
            request = self.scheduler.get_request(request_id)
            named = None if request.prefix is None else (request.prefix, request.shared)
            if (self.manager.can_be_admitted(request.lifetime_tokens, named)
                    and not self.manager.can_be_admitted(request.lifetime_tokens, named, beside=shared)):
                raise OutOfPages(f"beside the {shared // page} pages of prefix {name!r} the waiting request {request_id!r} could never be admitted")
        beside_others = not self.manager.can_ever_hold(shared) or self.manager.can_be_admitted(shared)
        if not beside_others or self.manager.create_request(holder, lifetime_tokens=shared, lasting=True) is None:
            raise OutOfPages(f"no room for the {shared // page} pages of prefix {name!r}")
        try:
            portion = self.scheduler.max_batch_tokens
            for start in range(0, shared, portion):
                self.runner.step([StepEntry(holder, tokens[start:min(shared, start + portion)])])
            if self.manager.slot_state.is_cuda:
                torch.cuda.synchronize(self.manager.slot_state.device)
            try:
                self.runner.check_device()
            except ops.KernelError:
                self._give_up_after_device_error(())
                raise
        except BaseException:
            self.manager.release(holder)
            raise
        self._prefixes[name] = tokens
        return shared

    def drop_prefix(self, name: str) -> None:
        """Give a prefix's pages back; every request that shares them must have ended."""
        if name not in self._prefixes:
            raise KeyError(f"no prefix {name!r}")
        holder = self._holder(name)
        users = [rid for rid in (*self.scheduler.waiting_request_ids, *self.scheduler.running_request_ids)
                 if self.scheduler.get_request(rid).prefix == holder]
        if users:
            raise RuntimeError(f"prefix {name!r} is shared by requests {users[:5]}")
        self.manager.release(holder)
        del self._prefixes[name]

    def _shared_by(self, name: str | None, prompt: Sequence[int]) -> tuple[str | None, int]:
        """The cached request that holds the prefix and the tokens the prompt shares with it: whole pages, and fewer than the prompt's."""
        if name is None:
            return None, 0
        if name not in self._prefixes:
            raise ValueError(f"no prefix {name!r}; known: {sorted(self._prefixes)}")
        tokens, page = self._prefixes[name], self.manager.page_size
        if tuple(prompt[:len(tokens)]) != tokens[:len(prompt)]:
            raise ValueError(f"the prompt does not start with the tokens of prefix {name!r}")
        shared = min(len(tokens), len(prompt) - 1) // page * page
        return (self._holder(name), shared) if shared else (None, 0)

    def allow_tokens(self, request_id: str, tokens: "Collection[int] | None") -> None:
        """The tokens that the request may choose from its next step on (None: all), as a grammar finds them after each token.  A
        request that allows nothing chooses token 0."""
        if self.runner.rules is None:
            raise ValueError("allowed tokens need an engine made with logit_rules=True")
        if self.step_ahead:
            raise ValueError("an engine that steps ahead chooses a request's next token before its grammar can follow the last one")
        request = self.scheduler.get_request(request_id)
        if request.status is RequestStatus.FINISHED:
            raise ValueError(f"request {request_id!r} has finished")
        words = self.runner.rules.words_of(tokens)
        held = self.manager.requests.get(request_id)
        if held is None:
            self._allowed[request_id] = words
        else:
            self._allowed.pop(request_id, None)
            self.runner.rules.allow(held.slot, words)

    def _admit_rules(self, request_id: str) -> None:
        """The request owns a slot now: its rules go there.  (A step that fails gives the slot back, and its request is admitted
        once more: a grammar named while it waited is kept until the request has a token.)"""
        request, slot = self.scheduler.get_request(request_id), self.manager.get(request_id).slot
        self.runner.rules.admit(slot, request.sampling, request.prompt)
        if request_id in self._allowed:
            self.runner.rules.allow(slot, self._allowed[request_id])

    # ------------------------------------------------------------------ one step
    @torch.inference_mode()
    def step(self) -> EngineStepResult | None:
        """Plan and run one step; None when nothing can run."""
        started_ns = self._clock_ns()
        with self._range("scheduler.schedule_step"):
            plan = self.scheduler.schedule_step()
        if plan is None:
            return None
        with self._range(f"engine.step:{plan.index}:prefill={len(plan.prefill_request_ids)}:"
                         f"decode={len(plan.decode_request_ids)}"):
            return self._run(plan, started_ns)

    def _run(self, plan: StepPlan, started_ns: int) -> EngineStepResult:
        ahead, self._ahead = self._ahead, None
        covered = set(ahead.request_ids) if ahead is not None else set()
        try:
            self.metrics.require_registered(tuple(item.request_id for item in plan.items))
            # Decodes whose step is already on the GPU take their token from it; the rest is launched now.
            entries, emitting = [], []
            for item in plan.items:
                if item.kind is WorkKind.DECODE and item.request_id in covered:
                    continue
                tokens = item.tokens
                if item.kind is not WorkKind.DECODE and len(tokens) > 16:
                    request = self.scheduler.get_request(item.request_id)     # a prompt portion: starts at the cursor
                    tokens = request.prompt_span(request.cursor, len(tokens))
                entries.append(StepEntry(item.request_id, tokens, [len(tokens) - 1] if item.emits else []))
                if item.admitted and self.runner.rules is not None:
                    self._admit_rules(item.request_id)
                if item.admitted and self.runner.limits is not None:
                    self.runner.limits.admit(self.manager.get(item.request_id).slot, self.scheduler.get_request(item.request_id).sampling)
                if item.admitted:
                    self.metrics.record_prefill_started(item.request_id, self._clock_ns())
                if item.emits:
                    emitting.append(item.request_id)
            launched = None
            if entries:
                with self._range(f"model.step:tokens={sum(len(e.tokens) for e in entries)}"):
                    # a step of decodes takes its inputs from the slot records (the tokens sampled last)
                    decodes_only = all(item.kind is WorkKind.DECODE for item in plan.items)
                    _, tokens = self.runner.step(entries, sample=True, borrow=True, feed=decodes_only)
                if emitting:
                    launched = self._start_token_copy(tuple(emitting), tokens)
        except Exception:
            with self._range("engine.rollback"):
                self.scheduler.abort_step()      # the requests it admitted give slot and pages back
            self._ahead = ahead                  # its decodes are done and stay valid for the retried step
            raise

        if self.step_ahead:
            self._launch_ahead(plan, ahead, launched)

        with self._range("token.d2h_sync"):
            generated: dict[str, int] = {}
            for source in (ahead, launched):
                if source is not None:
                    generated.update(source.wait())
            try:
                self.runner.check_device()
            except ops.KernelError:
                self._give_up_after_device_error([item.request_id for item in plan.items])
                raise
            generated = {rid: generated[rid] for rid in plan.emitting_request_ids}   # drops rows of ended requests
        tokens_ready_ns = self._clock_ns()
        with self._range("scheduler.apply_and_release"):
            outcome = self.scheduler.apply_step_results(generated)
        for request_id in generated if self._allowed else ():
            self._allowed.pop(request_id, None)
        completed_ns = self._clock_ns()
        self.metrics.record_tokens(outcome.emitted_tokens, tokens_ready_ns)
        self.metrics.record_completed(outcome.finished_request_ids, completed_ns)
        return EngineStepResult(plan, outcome, started_ns, tokens_ready_ns, completed_ns)

    def _give_up_after_device_error(self, request_ids: Sequence[str]) -> None:
        """A kernel reported that a bounded wait ran out: nothing computed since the last check can
        be trusted, and the cache already holds those steps' keys and values.  The requests of the
        step (and of the step launched ahead of it) end with ``FinishReason.ERROR`` and give their
        pages back; waiting requests and the engine itself stay usable."""
        with self._range("engine.rollback"):
            touched = list(request_ids)
            if self._ahead is not None:
                touched += [rid for rid in self._ahead.request_ids if rid not in touched]
                self._ahead.wait()
                self._ahead = None
            failed = self.scheduler.fail_requests(touched)
            for request_id in failed:
                self._allowed.pop(request_id, None)
            self.metrics.record_completed(failed, self._clock_ns())

    def _start_token_copy(self, request_ids: tuple[str, ...], tokens: torch.Tensor) -> _TokensInFlight:
        """Begin the device-to-host copy of a step's tokens; the caller waits on the event."""
        if tokens.device.type != "cuda":
            return _TokensInFlight(request_ids, tokens.to(torch.int32), None)
        if not self._token_buffers:
            size = max(64, self.scheduler.max_running_requests)
            self._token_buffers = [torch.empty(size, dtype=torch.int32, pin_memory=True) for _ in range(4)]
        host = self._token_buffers[self._next_buffer]
        self._next_buffer = (self._next_buffer + 1) % len(self._token_buffers)
        if host.numel() < tokens.numel():
            host = torch.empty(tokens.numel(), dtype=torch.int32, pin_memory=True)
        host[:tokens.numel()].copy_(tokens, non_blocking=True)
        event = torch.cuda.Event()
        event.record()
        return _TokensInFlight(request_ids, host, event)

    def _launch_ahead(self, plan: StepPlan, ahead: _TokensInFlight | None, launched: _TokensInFlight | None) -> None:
        """Launch the next decode step of this plan's requests behind the current one, if the
        current one decodes only, was launched (or had been launched ahead) as one step in the plan's
        order, and none of its requests reaches its token limit with this step."""
        if not plan.items or not plan.decode_only:
            return
        request_ids = tuple(item.request_id for item in plan.items)
        current = ahead if launched is None else (launched if ahead is None else None)
        if current is None or current.request_ids != request_ids:
            return
        requests = [self.scheduler.get_request(rid) for rid in request_ids]
        if any(len(request.output) + 1 >= request.max_new_tokens for request in requests):
            return
        entries = [StepEntry(rid, [0], [0]) for rid in request_ids]
        try:
            with self._range(f"model.step_ahead:tokens={len(entries)}"):
                _, tokens = self.runner.step(entries, sample=True, borrow=True, feed=True)
        except Exception:
            return          # nothing was launched and the cache is as before: go on step by step
        self._ahead = self._start_token_copy(request_ids, tokens)

    # ------------------------------------------------------------------ conveniences
    def run(self) -> list[EngineStepResult]:
        """Step until every submitted request has finished."""
        results = []
        while self.scheduler.has_unfinished_requests:
            result = self.step()
            if result is None:
                raise RuntimeError("requests are waiting but nothing can be scheduled")
            results.append(result)
        return results

    def generate(self, prompts: Sequence[Sequence[int]], *, max_new_tokens: int,
                 eos_token_ids: int | Collection[int] | None = None, temperature: float = 0.0,
                 seed: int = 0, answers: int = 1, **rules) -> list[list[int]]:
        """Token ids in, generated token ids out, for a list of prompts (host lists both ways); ``rules`` as for ``submit``.  ``answers``:
        so many outputs for each prompt, one behind the other, each drawn with a seed of its own.  A prompt is computed once where one of its
        answers still runs when another begins (not with one running request, one new token or no room), in models whose requests can fork."""
        if isinstance(answers, bool) or not isinstance(answers, int) or answers <= 0:
            raise ValueError("answers must be a positive integer")
        if answers > 1:
            return self._generate_answers(prompts, answers, max_new_tokens=max_new_tokens, eos_token_ids=eos_token_ids, temperature=temperature,
                                          seed=seed, **rules)
        scheduler = self.scheduler
        first = (len(scheduler.finished_request_ids) + len(scheduler.running_request_ids)
                 + len(scheduler.waiting_request_ids))
        ids = [f"generate-{first + i}" for i in range(len(prompts))]
        for i, (request_id, prompt) in enumerate(zip(ids, prompts)):
            self.submit(request_id, list(prompt), max_new_tokens=max_new_tokens,
                        eos_token_ids=eos_token_ids, temperature=temperature, seed=seed + i, **rules)
        self.run()
        return [list(scheduler.get_request(request_id).generated_token_ids) for request_id in ids]


    def _check_answers(self, prompts, ids, *, max_new_tokens, eos_token_ids=None, temperature=0.0, prefix=None, **rules) -> None:
        for prompt, names in zip(prompts, ids):
            self.scheduler.check(names[0], list(prompt), **self._checked(names[0], list(prompt), max_new_tokens, eos_token_ids, temperature, 0, prefix,
                                                                         None, rules))

    def _generate_answers(self, prompts, answers: int, *, seed: int, **options) -> list[list[int]]:
        scheduler = self.scheduler
        first = len(scheduler.finished_request_ids) + len(scheduler.running_request_ids) + len(scheduler.waiting_request_ids)
        ids = [[f"generate-{first + i}-{j}" for j in range(answers)] for i in range(len(prompts))]
        self._check_answers(prompts, ids, **options)          # before the first one runs
        forks = self.manager.can_share_pages
        # a fork has its first answer's prefix; by itself it needs room for all of its pages
        alone = {name: value for name, value in options.items() if name != "prefix"}
        fits = [forks and self.manager.can_be_admitted(len(prompt) + options["max_new_tokens"] - 1) for prompt in prompts]
        to_begin, leading = list(reversed(range(len(prompts)))), []
        while to_begin or leading or scheduler.has_unfinished_requests:
            # the other answers follow as soon as the first one's prompt is in the cache (or its request has ended)
            for i in list(leading):
                request = scheduler.get_request(ids[i][0])
                if request.output or request.status is RequestStatus.FINISHED or not forks:
                    leading.remove(i)
                    for j in range(1, answers):
                        if fits[i]:
                            self.submit(ids[i][j], list(prompts[i]), seed=seed + i * answers + j, fork_of=ids[i][0], **alone)
                        else:
                            self.submit(ids[i][j], list(prompts[i]), seed=seed + i * answers + j, **options)
            # the next prompt as soon as the requests that run and those still to follow leave a place, so that a prompt's answers run together
            while to_begin and (not forks or len(scheduler.waiting_request_ids) + len(scheduler.running_request_ids)
                                + len(leading) * (answers - 1) < scheduler.max_running_requests):
                i = to_begin.pop()
                self.submit(ids[i][0], list(prompts[i]), seed=seed + i * answers, **options)
                leading.append(i)
            if scheduler.has_unfinished_requests and self.step() is None:
                raise RuntimeError("requests are waiting but nothing can be scheduled")
        return [list(scheduler.get_request(request_id).generated_token_ids) for group in ids for request_id in group]


@dataclass(frozen=True)
class GreedyGenerationOutput:
    generated_token_ids: list[int]
    stopped_by_eos: bool
    prefill_tokens: int
    decode_steps: int
    cache_length: int
    step_logits: tuple[torch.Tensor, ...] | None = None


@torch.inference_mode()
def greedy_generate(runner: ModelRunner, input_ids: Sequence[int], *, max_new_tokens: int,
                    eos_token_ids: int | Collection[int] | None = None,
                    return_step_logits: bool = False, request_id: str = "greedy") -> GreedyGenerationOutput:
    """One prompt, one prefill step, then one-token steps (reference: generation.py:29-117).  EOS
    is tested before the token would be fed back; N tokens need N-1 decode steps and leave
    prompt + N - 1 tokens in the cache, which is given back at the end."""
    prompt = [int(t) for t in input_ids]
    if not prompt:
        raise ValueError("greedy_generate needs a non-empty prompt")
    if max_new_tokens <= 0:
        raise ValueError("max_new_tokens must be > 0")
    if eos_token_ids is None:
        eos = frozenset()
    else:
        eos = frozenset([eos_token_ids] if isinstance(eos_token_ids, int) else [int(t) for t in eos_token_ids])
    invalid = sorted(t for t in eos if not 0 <= t < runner.vocab_size)
    if invalid:
        raise ValueError(f"EOS token ids outside the vocabulary: {invalid}")
    if len(prompt) + max_new_tokens - 1 > min(runner.max_positions, runner.cache.max_tokens_per_request):
        raise ValueError("prompt_length + max_new_tokens - 1 exceeds the model's or the cache's limit")
    runner.cache.create_request(request_id)
    generated: list[int] = []
    captured: list[torch.Tensor] = []
    stopped = False
    decode_steps = 0
    try:
        logits = runner.step([StepEntry(request_id, prompt, [len(prompt) - 1])])
        for index in range(max_new_tokens):
            if return_step_logits:
                captured.append(logits[0].clone())
            token = int(torch.argmax(logits[0]))     # the host waits for the step here
            runner.check_device()
            generated.append(token)
            stopped = token in eos
            if stopped or index == max_new_tokens - 1:
                break
            logits = runner.step([StepEntry(request_id, [token], [0])])
            decode_steps += 1
        cache_length = runner.cache.get(request_id).committed
    finally:
        runner.cache.release(request_id)
    return GreedyGenerationOutput(generated, stopped, len(prompt), decode_steps, cache_length,
                                  tuple(captured) if return_step_logits else None)
