"""The Python entry point: token ids in, token ids out.

`Engine.generate` plays the reference's `generate_kv` (src/model.br:2280-2306: chunked prefill,
then sample, stop on an end token, else feed the token back), for many requests at once: the
scheduler builds each step's batch, the runner computes logits, the device sampler picks tokens.
"""
from __future__ import annotations

import copy
import itertools
import time
from typing import Dict, List, Optional, Sequence

import torch

from ..cache import CacheError
from ..config import EngineOptions
from ..models.loading import load_model, load_random_model
from ..sampling.params import SamplingParams
from ..sampling.sampler import Sampler
from .runner import ModelRunner, OutOfPages, StepEntry, TreeEntry
from .scheduler import RUNNING, WAITING, Request, Scheduler


class Engine:
    def __init__(self, model_dir: str, options: Optional[EngineOptions] = None, **overrides):
        """Loads the model folder (config.json chooses the model class) onto the device.
        `overrides` set fields of `EngineOptions` (dtype, ctx_size, max_tokens, ...)."""
        if options is None:
            options = EngineOptions(**overrides)
        elif overrides:
            raise TypeError("give either options or keyword overrides, not both")
        if not torch.cuda.is_available():
            raise RuntimeError("no CUDA device: this engine runs on an sm_100a GPU only (there is no CPU path)")
        self.options = options
        if isinstance(model_dir, tuple):
            self.config, self.model = model_dir          # (configuration, model already on the device)
        else:
            self.config, self.model = load_model(model_dir, options.dtype, options.device)
        max_pos = getattr(self.config, "max_position_embeddings", None)
        if max_pos is not None and options.ctx_size > max_pos:
            raise ValueError(f"ctx_size {options.ctx_size} exceeds the model's max_position_embeddings {max_pos}")
        self.runner = ModelRunner(self.model, options)
        self.scheduler = Scheduler(self.runner.cache, options)
        self.sampler = Sampler(options.device)
        if options.draft_tokens and not self.runner.takes_trees:
            raise ValueError("draft_tokens: this model's mixers keep state of their own beside pages, or attend in a way of their own; "
                             "drafted tokens could not be taken back")
        self._ids = itertools.count()
        self._inflight = None                 # (scheduled step, PendingDecode): launched, tokens not read yet
        self.stats_time = {"engine_steps": 0, "step_seconds": 0.0}

    @classmethod
    def from_model(cls, config, model, options: EngineOptions) -> "Engine":
        """An engine around a model that is already built and loaded on the device."""
        return cls((config, model), options)

    @classmethod
    def from_random(cls, config, seed: int, options: Optional[EngineOptions] = None, std: float = 0.02,
                    weight_dtype=None) -> "Engine":
        """An engine around a model with seeded random weights, made on the device without a file (the same
        tensors as `write_random_model` writes for this configuration, seed and standard deviation)."""
        options = options if options is not None else EngineOptions()
        return cls(load_random_model(config, seed, options.dtype, options.device, std, weight_dtype), options)

    # ---- requests ----------------------------------------------------------------------------------
    def add_request(self, prompt: Sequence[int], params: Optional[SamplingParams] = None, request_id=None) -> Request:
        if params is None:
            params = SamplingParams()
        if not params.eos_token_ids and not params.ignore_eos:
            params.eos_token_ids = tuple(getattr(self.config, "eos_token_ids", ()))
        for t in prompt:
            if not 0 <= int(t) < self.runner.vocab_size:
                raise ValueError(f"token id {t} is outside the vocabulary (0..{self.runner.vocab_size - 1})")
        rid = request_id if request_id is not None else next(self._ids)
        return self.scheduler.add(rid, prompt, params)

    def step(self) -> List[Request]:
        """One scheduler step. Returns the requests that finished in it.

        While the running requests only decode, the step after this one is launched before this one's tokens are
        read (`EngineOptions.lookahead`): the device feeds the sampled tokens back itself, the host reads them one
        step behind, and the GPU does not wait for the host between steps. A request that ends with an end token
        has then already got a row in the step after; that row's result is dropped (the reference's loop,
        src/model.br:2293-2304, feeds no token after the end token either: nothing of the row is kept).

        When a step fails, requests whose tokens are in the cache already end with the reason "error"; the others, those of a step of drafted
        trees among them, are as they were before it."""
        done = self._step()
        early, self.scheduler.unreported = self.scheduler.unreported, []
        return early + done

    def _step(self) -> List[Request]:
        t0 = time.perf_counter()
        if self._inflight is None:
            sched = self.scheduler.schedule()
            if sched is None:
                return []
            # the third item is the request itself: its token history is only put together if a penalty asks for it
            rows = [(r.params, r.rng, r) for r, s in zip(sched.requests, sched.samples) if s]
            said = self._drafted_step(sched, rows) if self.options.draft_tokens else None
            if said is not None:
                self.stats_time["engine_steps"] += 1
                self.stats_time["step_seconds"] += time.perf_counter() - t0
                return self.scheduler.apply_drafted(sched, said)
            pending = self.runner.launch_decode(sched.entries, rows) if self.options.lookahead and not self.options.draft_tokens else None
            if pending is None:
                try:
                    sampled = self.runner.step_and_sample(sched.entries, rows, self.sampler)
                    return self._finish_step(sched, sampled, t0)
                except BaseException:
                    self._abort_rows(r for r in sched.requests if self._is_ahead(r))
                    raise
            self._inflight = (sched, pending)
        sched, pending = self._inflight
        ahead = self.scheduler.lookahead(sched)
        nxt = None
        if ahead is not None:
            rows = [(r.params, r.rng, r) for r in ahead.requests]
            p2 = self.runner.launch_decode(ahead.entries, rows, from_device=True)
            if p2 is not None:
                nxt = (ahead, p2)
        try:
            sampled = self.runner.collect_decode(pending)
            done = self._finish_step(sched, sampled, t0)
        except BaseException:
            # The step in flight failed (a kernel gave up on a bounded wait, the read of its tokens failed). The step
            # ahead has already been launched: it has taken cache positions and random numbers for every row. Nothing of
            # either step can be kept: forget both and end their requests, so that the scheduler and the cache agree
            # again before the error reaches the caller.
            self._inflight = None
            self._abort_rows(sched.requests + (nxt[0].requests if nxt is not None else []))
            raise
        if nxt is not None and not any(r.state == RUNNING for r in nxt[0].requests):
            nxt = None                            # every row of the step ahead has ended: nobody reads it
        self._inflight = nxt
        return done

    def _drafted_step(self, sched, rows):
        """A step that only decodes, with drafted tokens; None when it is another kind of step, nothing is drafted, or the cache has
        no pages for the drafts (then nothing has been done)."""
        trees = self.scheduler.draft(sched)
        if trees is None:
            return None
        try:
            return self.runner.step_tree([TreeEntry(e.request_id, *tree) for e, tree in zip(sched.entries, trees)], rows)
        except OutOfPages:
            return None

    def fork(self, request, params: Optional[SamplingParams] = None, request_id=None) -> Request:
        """A second running request that goes on from where `request` (a `Request` that runs, its prompt computed) is, with parameters
        and a generator of its own. The pages of what both have in common are shared."""
        self.scheduler.unreported += self.drain()
        if request.state != RUNNING or request.remaining != 1:
            raise ValueError(f"request {request.request_id!r} cannot be forked: it has ended, or its prompt is not computed yet")
        return self._fork(request, params if params is not None else copy.copy(request.params), request_id, request.num_computed,
                          len(request.output))

    def _fork(self, request, params, request_id, n_keep: int, n_output: int) -> Request:
        if not params.eos_token_ids and not params.ignore_eos:
            params.eos_token_ids = tuple(getattr(self.config, "eos_token_ids", ()))
        source = self.runner.cache.get(request.request_id)
        new = self.scheduler.fork(request, request_id if request_id is not None else next(self._ids), params, n_keep, n_output)
        self.runner.storage.copy_slot(source.slot, self.runner.cache.get(new.request_id).slot)
        return new

    def _is_ahead(self, request) -> bool:
        """Whether the cache holds tokens of the request that its record does not know of: of a step that failed once they were committed."""
        held = self.runner.cache.find(request.request_id)
        return held is not None and held.num_tokens != request.num_computed

    def _abort_rows(self, requests) -> None:
        seen = set()
        for r in requests:
            if r.request_id in seen:
                continue
            seen.add(r.request_id)
            self.scheduler.abort(r.request_id, "error")

    def drain(self) -> List[Request]:
        """Reads the step that was launched ahead, if there is one, so that the host's view is complete.
        Returns the requests that finished in it."""
        if self._inflight is None:
            return []
        (sched, pending), self._inflight = self._inflight, None
        try:
            return self._finish_step(sched, self.runner.collect_decode(pending), time.perf_counter())
        except BaseException:
            self._abort_rows(sched.requests)              # its tokens are committed: as in `step`
            raise

    def _finish_step(self, sched, sampled, t0) -> List[Request]:
        self.runner.check_kernels()
        self.stats_time["engine_steps"] += 1
        self.stats_time["step_seconds"] += time.perf_counter() - t0
        return self.scheduler.apply(sched, sampled)

    def run_until_done(self) -> None:
        while self.scheduler.has_work():
            before = self.scheduler.progress()
            self.step()
            after = self.scheduler.progress()
            if before == after and not self.scheduler.running:
                raise RuntimeError("the scheduler made no progress with requests still waiting")

    def generate(self, prompts: Sequence[Sequence[int]], n_predict: int = 40, temperature: float = 0.0,
                 seed: int = 0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0,
                 repeat_penalty: float = 1.0, repeat_last_n: int = 64,
                 eos_token_ids: Optional[Sequence[int]] = None, ignore_eos: bool = False, n: int = 1) -> List[List[int]]:
        """Generated token ids for each prompt (lists of token ids), in the prompts' order. Request i
        draws from a generator seeded with `seed + i`, so a batch and the same prompts one by one
        give the same tokens. `n` > 1: as many answers to each prompt, one behind the other (answer k of prompt i is request
        i * n + k); where the model keeps nothing but pages a prompt is computed once and its answers share its pages."""
        if n < 1:
            raise ValueError(f"n must be positive, got {n}")
        reqs, waiting = [], []
        for i, prompt in enumerate(prompts):
            answers = []
            for k in range(n):
                params = SamplingParams(n_predict=n_predict, temperature=temperature, seed=seed + i * n + k, top_k=top_k,
                                        top_p=top_p, min_p=min_p, repeat_penalty=repeat_penalty,
                                        repeat_last_n=repeat_last_n,
                                        eos_token_ids=tuple(eos_token_ids) if eos_token_ids is not None else (),
                                        ignore_eos=ignore_eos)
                if k and len(prompt) > 1 and not self.runner.cache.state_groups:
                    waiting.append((answers[0], prompt, params, i * n + k))
                    answers.append(None)
                else:
                    answers.append(self.add_request(prompt, params))
            reqs += answers
        while waiting:
            # a source whose prompt is computed is forked in front of the prompt's last token, which each answer runs itself: its logits
            # are what the first tokens are drawn from. One that has ended or waits again by then, or for want of a slot: another request.
            left = []
            for source, prompt, params, at in waiting:
                if source.state == WAITING and not source.output or source.state == RUNNING and source.num_computed < len(prompt):
                    left.append((source, prompt, params, at))
                elif source.state == RUNNING and self.runner.cache.has_free_slot() and params.n_predict != 0:
                    try:
                        reqs[at] = self._fork(source, params, None, len(prompt) - 1, 0)
                    except CacheError:                # a window has passed the prompt's end: its pages are gone
                        reqs[at] = self.add_request(prompt, params)
                else:
                    reqs[at] = self.add_request(prompt, params)
            waiting = left
            if waiting and not self.step() and not self.scheduler.running:
                # nothing runs and the sources cannot start: wait with them
                for _, prompt, params, at in waiting:
                    reqs[at] = self.add_request(prompt, params)
                break
        self.run_until_done()
        return [list(r.output) for r in reqs]

    def stats(self) -> dict:
        s = dict(self.runner.cache.stats())
        s.update(drafted_tokens=self.runner.drafted, accepted_tokens=self.runner.accepted)
        s.update(steps=self.runner.steps, tokens_run=self.runner.tokens_run,
                 preemptions=self.scheduler.num_preemptions, **self.stats_time)
        return s


def generate(model_dir: str, prompts: Sequence[Sequence[int]], n_predict: int = 40, temperature: float = 0.0,
             seed: int = 0, dtype: str = "bfloat16", ctx_size: int = 4096, **sampling) -> List[List[int]]:
    """One call from a model folder and prompts (token ids) to generated token ids."""
    eng = Engine(model_dir, dtype=dtype, ctx_size=ctx_size, max_num_seqs=max(1, min(64, len(prompts))))
    return eng.generate(prompts, n_predict=n_predict, temperature=temperature, seed=seed, **sampling)
