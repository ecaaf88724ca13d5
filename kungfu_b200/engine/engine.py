"""The engine a user drives: requests in (token ids), tokens out.

`Engine` wraps a model, a cache manager, the step runner, the scheduler and the sampler.  The reference's
counterpart is a `Session` under a `Scheduler` (crates/kf-engine/src/session.rs:84-103,
crates/kf-serve/src/engine.rs:375-430); its `generate` command is `Engine.generate` here
(crates/kungfu/src/main.rs:611-645: seed 42, greedy at temperature 0).
"""
from __future__ import annotations

import time
from collections import deque
from dataclasses import dataclass
from typing import Hashable, Sequence

import numpy as np
import torch

from .. import events as _events
from .. import ops
from ..cache.manager import CacheError, OutOfPages
from ..sampling.sampler import STATE_WORDS, Sampling, pack_state
from ..sampling.scores import MAX_ALTERNATIVES, ScoreRows, TokenScore, check_alternatives
from .scheduler import Request, Scheduler
from .step import Runner, StepEntry


def emit_event(name: str, **fields) -> None:
    """One structured line on stderr, `kungfu event=<name> k=v ...` (reference: crates/kf-core/src/event.rs:31-44)."""
    was, _events.enabled = _events.enabled, True
    try:
        _events.emit(name, **fields)
    finally:
        _events.enabled = was


@dataclass
class Beam:
    """One answer of a beam search."""
    tokens: list
    logprob: float                     # the sum of its tokens' log probabilities
    finish_reason: str                 # eos, length or context


class Engine:
    def __init__(self, model_dir: str | None = None, *, config=None, seed: int = 0, dtype="bfloat16", device="cuda:0",
                 ctx: int | str = 4096, batch: int = 512, parallel: int = 8, page_size: int | None = None,
                 max_tokens_in_cache: int | None = None, events: bool = False, runner: Runner | None = None,
                 cuda_graphs: bool = True, pipeline: bool = True):
        """`model_dir`: folder with config.json and model.safetensors; or `config` (typed configuration, dictionary
        or config.json path) with `seed` for random weights.  `ctx`: context length per request ('auto' = the
        model's trained length); `batch`: most tokens one step runs; `parallel`: most live requests.
        `max_tokens_in_cache`: size of a cache group's pool in tokens (default: parallel * ctx; a windowed group never
        gets more than parallel * (window + batch + page), and all pools are cut to fit the memory left after the weights).
        `pipeline`: decode steps are launched before the tokens of the step before them have been read (tokens are
        drawn on the device and stay there as the next step's input), so `step()` returns a step's tokens one call
        later and the GPU does not wait for the host between steps."""
        from .. import api
        self.events = events
        if runner is not None:
            self.runner = runner
            self.cfg = None
        else:
            self.device = api.require_cuda(device)
            ops.library()
            t0 = time.time()
            if model_dir is not None:
                self.cfg, model = api.load_model(model_dir, dtype=dtype, device=self.device)
            elif config is not None:
                self.cfg, model = api.random_model(config, seed, dtype=dtype, device=self.device)
            else:
                raise ValueError("Engine needs a model folder or a configuration")
            trained = getattr(self.cfg, "max_position_embeddings", None)      # None: the architecture names no trained length
            if trained is None:
                n_ctx = 8192 if (ctx == "auto" or not ctx) else int(ctx)
            else:
                n_ctx = trained if ctx == "auto" else min(int(ctx), trained) if ctx else trained
            page = page_size or api.DEFAULT_PAGE_SIZE
            if events:
                _events.enabled = True
            pool = f"cuda{self.device.index or 0}"
            _events.alloc(pool, "weights", model.weight_bytes())
            # what the cache may take: the memory that is free now, less a reserve for the step's own buffers
            # (activations of `batch` rows, logits of the wanted rows, split sums) and the allocator's slack
            free, total = torch.cuda.mem_get_info(self.device)
            budget = max(0, int(free) - max(2 << 30, int(total) // 16))
            self.runner = api.make_runner(self.cfg, model, dtype=dtype, device=self.device, page_size=page,
                                          max_tokens=max_tokens_in_cache, max_requests=parallel, max_context=n_ctx,
                                          cuda_graphs=cuda_graphs, batch=batch, budget_bytes=budget)
            plan = self.runner.cache.plan
            _events.emit("plan", **plan.fields())
            _events.alloc(pool, "cache", plan.paged_bytes)
            if plan.fixed_bytes:
                _events.alloc(pool, "state", plan.fixed_bytes)
            _events.emit("ready", model=self.cfg.architecture, dtype=str(api.parse_dtype(dtype)).split(".")[-1],
                         weight_bytes=model.weight_bytes(), cache_bytes_per_token=self.runner.cache.bytes_per_token(),
                         pool_pages=",".join(str(g.pages) for g in plan.groups), ctx=n_ctx,
                         load_s=f"{time.time() - t0:.2f}")
        self.scheduler = Scheduler(self.runner.cache, max_batch_tokens=batch, max_requests=parallel,
                                   pad_decode_rows=bool(getattr(self.runner, "cuda_graphs", False)))
        self._next_id = 0
        self.requests: dict[Hashable, Request] = {}
        self._t_start: dict = {}
        # what the device needs to draw a request's tokens (rules, generator, recent tokens), one block per state slot
        self._states = torch.zeros((self.runner.cache.max_requests, STATE_WORDS), dtype=torch.int32, device=self.runner.device)
        self.pipeline = bool(pipeline)
        self._inflight = None                  # (requests and their output places, picked ids on the device, fetch, fetch of scores)
        self._held: list[tuple] = []           # events that a call other than `step()` had to read: the next `step()` returns them

    # ---- requests ---------------------------------------------------------------------------------------
    def add_request(self, ids: Sequence[int], sampling: Sampling | None = None, *, max_tokens: int = 64,
                    eos: Sequence[int] | None = None, ignore_eos: bool = False, seed: int = 42,
                    request_id: Hashable | None = None, logprobs: int | None = None) -> Hashable:
        """Queue a prompt.  `logprobs`: score every token that is produced (its log probability, rank and entropy under the logits as
        the model gives them, with that many alternatives, 0 to 64): `requests[id].scores` then holds one `TokenScore` per token of
        `requests[id].output` as far as their values have arrived."""
        if logprobs is not None:
            logprobs = check_alternatives(logprobs, self.runner.vocab)
        if request_id is None:
            request_id = self._next_id
            self._next_id += 1
        if request_id in self.requests and self.requests[request_id].status != "finished":
            raise ValueError(f"request id {request_id!r} is in use")
        vocab = self.runner.vocab
        for t in ids:
            if not (0 <= int(t) < vocab):
                raise ValueError(f"token id {t} is outside the vocabulary of {vocab}")
        if eos is None:
            eos = tuple(getattr(self.cfg, "eos_token_id", ()) or ()) if self.cfg is not None else ()
        req = Request(request_id, list(ids), sampling or Sampling(temperature=0.0), max_tokens=max_tokens,
                      eos=tuple(eos), ignore_eos=ignore_eos, seed=seed, logprobs=logprobs)
        self.requests[request_id] = req
        self._t_start[request_id] = time.time()
        self.scheduler.add(req)
        return request_id

    def cancel(self, request_id: Hashable) -> list[tuple]:
        """End a request now.  Returns the events of the step that was in flight (tokens of every request, this one
        included, and finish reasons that only that step's tokens reveal) followed by (request_id, None, 'cancelled')
        if the request had not ended by itself; a caller that streams from `step()` must handle them like `step()`'s."""
        events = self.flush()
        req = self.requests[request_id]
        if req.status != "finished":
            self.scheduler.finish(req, "cancelled")
            events.append((request_id, None, "cancelled"))
            if self.events:
                self._request_event(req)
        return events

    @property
    def idle(self) -> bool:
        return self.scheduler.idle and self._inflight is None and not self._held

    # ---- tokens that a launched step has not delivered yet ---------------------------------------------------
    def flush(self) -> list[tuple]:
        """Wait for the step in flight, if any, and return its events, after those that other calls have held back."""
        events, self._held = self._held, []
        return events + self._collect() if self._inflight is not None else events

    def _collect(self, flight=None) -> list[tuple]:
        """Read the tokens of a launched step, put them where their placeholders stand and see which of them end a
        request by their value."""
        if flight is None:
            flight, self._inflight = self._inflight, None
        items, _picked, fetch, fetch_scores = flight
        events = []
        tokens = fetch()
        scores = fetch_scores(tokens) if fetch_scores is not None else None
        for i, ((r, at), tok) in enumerate(zip(items, tokens)):
            if at >= len(r.output):                      # produced after the token that ended the request: dropped
                continue
            r.output[at] = int(tok)
            if scores is not None:
                self._keep_score(r, at, scores[i])
            reason = None
            if not r.ignore_eos and int(tok) in r.eos:
                del r.output[at + 1:]                    # the placeholder of a step launched since
                if r.status != "finished":
                    self.scheduler.finish(r, "eos")
                else:
                    r.finish_reason = "eos"
                reason = "eos"
            elif r.status == "finished" and at == len(r.output) - 1:
                reason = r.finish_reason
            events.append((r.id, int(tok), reason))
            if reason is not None and self.events:
                self._request_event(r)
        return events

    def _tokens_needed_first(self) -> bool:
        """True if the coming plan must not be made on counts alone: a request may be admitted or preempted (its
        tokens are then read back as a prompt), which needs every token's value."""
        sched = self.scheduler
        if sched.waiting:
            return True
        running = len(sched.running)
        return any(g.pool.n_free < running for g in self.runner.cache.groups)

    # ---- one step -----------------------------------------------------------------------------------------
    def step(self) -> list[tuple]:
        """Plan and run one step.  Returns (request id, token, finish reason or None) for every token produced,
        and (request id, None, reason) for requests that ended without one (no_fit).  With `pipeline`, the tokens of
        a greedy decode step are returned by the next call (or by `flush()`); a request that one of them ends by its
        value (an end-of-sequence id) has then already run one more step, whose token is dropped."""
        events, self._held = self._held, []
        if self._inflight is not None and self._tokens_needed_first():
            events += self._collect()
        n_fin = len(self.scheduler.finished)
        plan = self.scheduler.schedule()
        events += [(r.id, None, r.finish_reason) for r in self.scheduler.finished[n_fin:]]
        wanting = [p for p in plan if p.wants_logits]
        # a step of one token per request: its tokens can stay on the device for the step after it
        decode_only = self.pipeline and bool(wanting) and len(wanting) == len(plan) and all(p.n == 1 for p in plan)
        feedback = None
        if self._inflight is not None:
            if decode_only and [id(p.request) for p in plan] == [id(r) for r, _ in self._inflight[0]]:
                feedback = self._inflight[1]
            else:                                        # another step than the one in flight was counted on
                events += self._collect()
                plan = [p for p in plan if p.request.status != "finished"]    # ended by a token that was in flight
                wanting = [p for p in plan if p.wants_logits]
        if not plan:
            return events
        entries = []
        for p in plan:
            toks = p.request.slice(p.start, p.n)
            entries.append(StepEntry(p.request.id, toks, [p.n - 1] if p.wants_logits else []))
        if wanting:                                      # tokens are drawn in the step's own pass, on the device
            self._upload_sampler_states(wanting)
            whole = any(p.request.sampling.needs_whole_ranking for p in wanting)
            logits, picked = self.runner.step(entries, sample=(self._states, whole), feedback=feedback)
        else:
            logits, picked = self.runner.step(entries), None
        for p in plan:
            self.scheduler.advance(p)
        if decode_only and picked is not None:
            fetch = self.runner.fetch_async(picked, len(wanting))
            fetch_scores = self._start_scores(logits, picked, wanting, range(len(wanting)))
            items = []
            for p in wanting:
                self.scheduler.on_token_pending(p.request)
                items.append((p.request, len(p.request.output) - 1))
            before, self._inflight = self._inflight, (items, picked, fetch, fetch_scores)
            if before is not None:                       # the step before this one: its tokens are read while this one runs
                events += self._collect(before)
            return events
        if wanting:
            fetch_scores = self._start_scores(logits, picked, wanting, self.runner.last_logit_index)
            drawn = picked.cpu().tolist()
            tokens = [drawn[i] for i in self.runner.last_logit_index]
            scores = fetch_scores(tokens) if fetch_scores is not None else None
            for i, (p, tok) in enumerate(zip(wanting, tokens)):
                at = len(p.request.output)
                reason = self.scheduler.on_token(p.request, tok)
                if scores is not None:
                    self._keep_score(p.request, at, scores[i])
                events.append((p.request.id, tok, reason))
                if reason is not None and self.events:
                    self._request_event(p.request)
        return events

    def _start_scores(self, logits, picked, wanting, index):
        """Score the drawn tokens of a step on the device, if any of its requests asked for it, and start the results' way to the host.
        Returns None, or a function from the wanted rows' tokens to their scores; `index`: the row of each."""
        asked = [p.request.logprobs for p in wanting]
        if all(a is None for a in asked):
            return None
        top = max(a for a in asked if a is not None)
        rows = self.runner.score_rows(logits, picked, top)
        fetch, n, index = self.runner.fetch_scores(rows), rows.rows, list(index)

        def scores(tokens):
            by_row, keep = [0] * n, [0] * n
            for i, tok, a in zip(index, tokens, asked):
                by_row[i], keep[i] = tok, a or 0
            every = ScoreRows.parse(fetch(), n, top, by_row, keep)
            return [every[i] if a is not None else None for i, a in zip(index, asked)]
        return scores

    @staticmethod
    def _keep_score(r: Request, at: int, score: TokenScore | None) -> None:
        del r.scores[at:]
        if score is not None:
            r.scores += [None] * (at - len(r.scores)) + [score]

    def _upload_sampler_states(self, wanting) -> None:
        """Write the sampler state of every request that is about to draw its first token since it was (re)admitted:
        its rules, its generator advanced past the draws it has already made, and the tokens it has produced."""
        for p in wanting:
            r = p.request
            if r.sampler_epoch == r.n_preempted:
                continue
            st = pack_state(r.sampling, r.seed, recent=r.output)
            if r.sampling.temperature > 0.0 and r.output:        # after a preemption: one draw per token so far
                x = max(int(r.seed), 1) & ((1 << 64) - 1)
                for _ in r.output:
                    x ^= (x << 13) & ((1 << 64) - 1)
                    x ^= x >> 7
                    x ^= (x << 17) & ((1 << 64) - 1)
                st[0:2] = np.array([x & 0xFFFFFFFF, x >> 32], dtype=np.uint32).view(np.int32)
            slot = self.runner.cache.state_slot(r.id)
            self._states[slot].copy_(torch.from_numpy(st))
            r.sampler_epoch = r.n_preempted

    def _request_event(self, r: Request) -> None:
        dt = max(time.time() - self._t_start.get(r.id, time.time()), 1e-9)
        emit_event("request", id=r.id, prompt_tokens=len(r.prompt), completion_tokens=len(r.output),
                   finish=r.finish_reason, preempted=r.n_preempted, seconds=f"{dt:.3f}")

    # ---- whole generations --------------------------------------------------------------------------------------
    def generate(self, prompts: Sequence[Sequence[int]], sampling: Sampling | None = None, *, max_tokens: int = 64,
                 eos: Sequence[int] | None = None, ignore_eos: bool = False, seed: int = 42) -> list[list[int]]:
        """Token ids in, generated token ids out, one list per prompt (host lists both ways)."""
        ids = [self.add_request(p, sampling, max_tokens=max_tokens, eos=eos, ignore_eos=ignore_eos, seed=seed + i)
               for i, p in enumerate(prompts)]
        self.run_to_end(ids)
        return [list(self.requests[i].output) for i in ids]

    def run_to_end(self, ids: Sequence[Hashable]) -> None:
        """Step until these requests are finished and nothing is in flight; raises what a kernel has recorded on the device."""
        while any(self.requests[i].status != "finished" for i in ids) or self._inflight is not None:
            before = sum(len(self.requests[i].output) for i in ids)
            ev = self.step()
            if not ev and before == sum(len(self.requests[i].output) for i in ids) and self.idle:
                break
        if self.runner.device.type == "cuda":
            ops.raise_on_device_error(self.runner.device)

    # ---- scoring, forks, beams -----------------------------------------------------------------------------------
    def score(self, prompts: Sequence[Sequence[int]], *, top: int = 0) -> list[list[TokenScore]]:
        """For every prompt, one `TokenScore` for each of its tokens but the first: how likely it was after those before it, and how
        many alternatives `top` asks for (0 to 64; without any, the logits are never stored and no ranks come back).  Prompts run
        in portions of up to `batch` tokens, several prompts in a step, beside whatever the cache holds of running requests.  Raises
        CacheError or OutOfPages if those leave no state slot or no pages."""
        prompts = [[int(t) for t in p] for p in prompts]
        top = check_alternatives(top, self.runner.vocab)
        cache, vocab = self.runner.cache, self.runner.vocab
        for p in prompts:
            if any(not (0 <= t < vocab) for t in p):
                raise ValueError(f"a token id is outside the vocabulary of {vocab}")
            if len(p) > cache.max_context:
                raise ValueError(f"a prompt of {len(p)} tokens is longer than the context of {cache.max_context}")
        self._held = self.flush()
        out: list[list] = [[] for _ in prompts]
        waiting = deque(i for i, p in enumerate(prompts) if len(p) > 1)
        fed: dict[int, int] = {}                          # live prompt -> tokens of it that have run
        key = object()                                    # no request of anyone else's has this id
        try:
            while waiting or fed:
                room, entries, targets = self.scheduler.max_batch_tokens, [], []
                for i in list(fed) + list(waiting):
                    if room <= 0:
                        break
                    at = fed.get(i, 0)
                    n = min(room, len(prompts[i]) - 1 - at)   # the last token predicts nothing that is asked for
                    if i not in fed:
                        if cache.n_live >= cache.max_requests or (fed and not self._room_for_prompt(prompts, fed, key, len(prompts[i]) - 1)):
                            break
                        waiting.popleft()
                        cache.add_request((key, i))
                        fed[i] = 0
                    while n > 0 and not self._pages_for(entries, (key, i), n):
                        n //= 2
                    if n == 0:
                        break
                    entries.append(StepEntry((key, i), prompts[i][at:at + n], list(range(n))))
                    targets.append(prompts[i][at + 1:at + n + 1])
                    room -= n
                if not entries:
                    if not fed and cache.n_live >= cache.max_requests:
                        raise CacheError(f"no state slot is free for a prompt to score ({cache.n_live} live requests)")
                    raise OutOfPages("no page is free for the prompts to score")
                rows = self.runner.score(entries, targets, top)
                flat = [t for ts in targets for t in ts]
                scores = iter(ScoreRows.parse(self.runner.fetch_scores(rows)(), len(flat), top, flat))
                for e in entries:
                    i = e.request[1]
                    out[i] += [next(scores) for _ in e.tokens]
                    fed[i] += len(e.tokens)
                    if fed[i] == len(prompts[i]) - 1:
                        cache.release(e.request)
                        del fed[i]
        finally:
            for i in fed:
                cache.release((key, i))
        if self.runner.device.type == "cuda":
            ops.raise_on_device_error(self.runner.device)
        return out

    def _room_for_prompt(self, prompts, fed, key, n: int) -> bool:
        """Whether another prompt of `n` tokens fits beside all that the prompts already begun still need: so that none is left half fed."""
        cache = self.runner.cache
        need = [-(-n // cache.page_size)] * len(cache.groups)
        for i, at in fed.items():
            need = [a + b for a, b in zip(need, cache.pages_needed((key, i), len(prompts[i]) - 1 - at))]
        return all(a <= b for a, b in zip(need, cache.free_pages()))

    def _pages_for(self, entries, request, n: int) -> bool:
        """Whether the pools cover `n` more tokens of `request` beside what `entries` will take."""
        cache = self.runner.cache
        need = cache.pages_needed(request, n)
        for e in entries:
            need = [a + b for a, b in zip(need, cache.pages_needed(e.request, len(e.tokens)))]
        return all(a <= b for a, b in zip(need, cache.free_pages()))

    def fork(self, request_id: Hashable, *, new_id: Hashable | None = None, seed: int | None = None, sampling: Sampling | None = None,
             max_tokens: int | None = None, logprobs: int | str | None = "inherit") -> Hashable:
        """Another request that goes on from where `request_id` stands (which must be producing tokens): the same prompt, the same output so
        far, the same cached context, of which only the last page and the recurrent states are copied.  It draws by its own
        generator (`seed`, default one more than the parent's: forks of one parent that are to differ need seeds of their own), and by other
        rules and lengths if given.  `logprobs`: as of `add_request` (None: no scores); by default the parent's.  Raises OutOfPages or
        CacheError if the cache has no page or state slot for it."""
        self._held = self.flush()
        parent = self.requests[request_id]
        if not parent.decoding:
            raise ValueError(f"request {request_id!r} is {parent.status} and not producing tokens")
        limit = parent.max_tokens if max_tokens is None else int(max_tokens)
        if limit <= len(parent.output):
            raise ValueError(f"max_tokens {limit} is not above the {len(parent.output)} tokens already produced")
        if logprobs == "inherit":
            logprobs = parent.logprobs
        if logprobs is not None:
            logprobs = check_alternatives(logprobs, self.runner.vocab)
        if new_id is None:
            new_id = self._next_id
            self._next_id += 1
        if new_id in self.requests and self.requests[new_id].status != "finished":
            raise ValueError(f"request id {new_id!r} is in use")
        req = Request(new_id, list(parent.prompt), sampling or parent.sampling, max_tokens=limit, eos=parent.eos,
                      ignore_eos=parent.ignore_eos, seed=parent.seed + 1 if seed is None else seed,
                      logprobs=logprobs)
        req.output, req.n_cached = list(parent.output), parent.n_cached
        req.scores = [] if logprobs is None else list(parent.scores)
        self.runner.cache.fork(request_id, new_id)
        self.scheduler.adopt(req)
        self.requests[new_id] = req
        self._t_start[new_id] = time.time()
        return new_id

    def beam_search(self, prompt: Sequence[int], *, beams: int = 4, max_tokens: int = 64, eos: Sequence[int] | None = None,
                    ignore_eos: bool = False, length_penalty: float = 0.0) -> list[Beam]:
        """The `beams` best answers found by a search that keeps that many open ones, best first.  An answer's value is the sum of its
        tokens' log probabilities over length ** length_penalty.  Every step asks each open answer for its 2 * beams best next tokens, or
        for as many as leave `beams` of them beside every id of `eos`, but no more than 64; the cache of an answer that goes on in several ways
        is forked, that of a dropped one freed.  At most 32 beams, and no more than the cache has free state slots."""
        prompt = [int(t) for t in prompt]
        cache, vocab = self.runner.cache, self.runner.vocab
        if not prompt or any(not (0 <= t < vocab) for t in prompt):
            raise ValueError(f"a prompt is one or more token ids of the vocabulary of {vocab}")
        if len(prompt) >= cache.max_context:
            raise ValueError(f"a prompt of {len(prompt)} tokens leaves nothing of the context of {cache.max_context}")
        if not 1 <= beams <= 32 or max_tokens < 1:
            raise ValueError(f"{beams} beams of {max_tokens} tokens: 1 to 32 beams of at least one token")
        self._held = self.flush()
        if beams > cache.max_requests - cache.n_live:
            raise CacheError(f"{beams} beams, but {cache.max_requests - cache.n_live} free state slots")
        if eos is None:
            eos = tuple(getattr(self.cfg, "eos_token_id", ()) or ()) if self.cfg is not None else ()
        eos = set() if ignore_eos else set(eos)
        top = min(max(2 * beams, beams + len(eos)), MAX_ALTERNATIVES, vocab)

        def value(logprob, n):
            return logprob / n ** length_penalty

        key, names = object(), 0                          # ids of the open answers' caches: (key, number)
        live = [((key, 0), [], 0.0)]                      # (cache, tokens, log probability)
        done: list[Beam] = []
        cache.add_request((key, 0))
        try:
            logits = None
            for a in range(0, len(prompt), self.scheduler.max_batch_tokens):
                part = prompt[a:a + self.scheduler.max_batch_tokens]
                logits = self.runner.step([StepEntry((key, 0), part, [len(part) - 1] if a + len(part) == len(prompt) else [])])
            for n in range(1, max_tokens + 1):
                ids, lps = self._beam_candidates(logits, top)
                found = sorted(((-value(lp + float(lps[b, k]), n), b, k) for b, (_c, _t, lp) in enumerate(live) for k in range(top)
                                if float(lps[b, k]) > float("-inf")), key=lambda c: c)
                last = n == max_tokens or len(prompt) + n >= cache.max_context
                nxt = []                                  # (parent, token, log probability) of the answers that stay open
                for place, (_v, b, k) in enumerate(found):
                    token, total = int(ids[b, k]), live[b][2] + float(lps[b, k])
                    if token in eos:
                        if place < beams:
                            done.append(Beam(live[b][1] + [token], total, "eos"))
                    elif last:
                        done.append(Beam(live[b][1] + [token], total, "length" if n == max_tokens else "context"))
                        nxt.append(None)
                    else:
                        nxt.append((b, token, total))
                    if len(nxt) == beams:
                        break
                done = sorted(done, key=lambda d: -value(d.logprob, len(d.tokens)))[:beams]
                if last or not nxt:
                    break
                # no open answer can still beat the ones that are done: log probabilities only fall
                if length_penalty == 0.0 and len(done) == beams and max(t for _b, _k, t in nxt) <= done[-1].logprob:
                    break
                children: dict = {}
                for i, (b, _token, _total) in enumerate(nxt):
                    children.setdefault(b, []).append(i)
                for b, (c, _t, _lp) in enumerate(live):
                    if b not in children:
                        cache.release(c)
                held, forks = [None] * len(nxt), []
                for b, kids in children.items():
                    held[kids[0]] = live[b][0]
                    for i in kids[1:]:
                        names += 1
                        held[i] = (key, names)
                        forks.append((live[b][0], held[i]))
                live = [(c, live[b][1] + [token], total) for c, (b, token, total) in zip(held, nxt)]
                if forks:
                    cache.fork_all(forks)
                logits = self.runner.step([StepEntry(c, [t[-1]], [0]) for c, t, _lp in live])
        finally:
            for i in range(names + 1):
                if (key, i) in cache:
                    cache.release((key, i))
        if self.runner.device.type == "cuda":
            ops.raise_on_device_error(self.runner.device)
        return done

    def _beam_candidates(self, logits, top: int):
        """The `top` best next tokens of every open answer and their log probabilities, on the host."""
        n = logits.shape[0]
        words = self.runner._score_buffers.get("beam_candidates", (2 * n * top,), torch.int32)
        ids, lps = words[:n * top].view(n, top), words[n * top:2 * n * top].view(torch.float32).view(n, top)
        ops.token_logprobs(logits, None, None, out_top_ids=ids, out_top_logprobs=lps)
        host = words[:2 * n * top].cpu().numpy()
        return host[:n * top].reshape(n, top), host[n * top:].view(np.float32).reshape(n, top)

    def warm_up(self) -> None:
        """Run a few tokens of 1, 2, 4, ... up to `parallel` one-token requests, greedy and with a temperature, so that the
        decode steps of every batch bucket are captured as CUDA graphs before the first real request (a layout's first step
        is launched kernel by kernel and its second is captured; from the third on it is one replay).  Optional; call it
        when the engine is idle."""
        if not self.idle:
            raise RuntimeError("warm_up() wants an idle engine")
        limit = self.runner.cache.max_requests
        n = 1
        while True:
            for s in (Sampling(temperature=0.0), Sampling(temperature=0.8)):
                self.generate([[1 % self.runner.vocab]] * n, s, max_tokens=4, ignore_eos=True)
            if n >= limit:
                break
            n = min(2 * n, limit)

    def finish_reason(self, request_id: Hashable) -> str | None:
        return self.requests[request_id].finish_reason
