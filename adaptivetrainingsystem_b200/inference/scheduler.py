"""Continuous batching: a fixed pool of cache rows, requests of any length admitted and retired between decode steps.

The rows live in a :class:`SequencePool` (one cache of ``max_batch`` rows and one captured decode step over it).  Every call of
:meth:`ContinuousBatcher.step`

1. admits waiting requests into free rows and prefills them straight into the row (a one-row view of the pool's cache), either the
   whole prompt at once or, with ``prefill_chunk``, at most that many prompt tokens per step, so that a long prompt does not hold up the
   rows that are decoding; the first token is sampled from the logits of the prompt's last position;
2. replays the decode graph once for all rows (each row at its own length; rows that are free or still in their prompt come out
   unchanged and their output is ignored), samples one token per row in one launch;
3. retires rows that produced a stop token or their token budget and frees their slots.

With ``page_size`` the rows live in a :class:`PagedPool` instead: a request takes pages for its own prompt and budget rather than a row of
``max_len``, and the portions that a step admits run as one packed batch.  A request may bring sampling numbers of its own
(:meth:`ContinuousBatcher.submit`); the step's tokens of such requests are drawn by ``ops.sample_rows`` in one launch, those of the others in
another, from random numbers of their own: what one kind draws does not depend on the other.

The reference's own generator serves one sequence at a time and re-runs the context for every token (``Chat.py:355-465``); its
vendored serving engine keeps a slot table per batch (``colossalai/inference/kv_cache/kvcache_manager.py:11-106`` allocator,
``kv_cache/batch_infer_state.py:13-118`` per-batch lengths and start locations), which is the bookkeeping done here on rows.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from .. import ops
from .engine import GenerationEngine, SamplingParams, sample_next
from .pool import PagedPool, SequencePool

MAX_PACKED = 8192   # prompt tokens that run as one packed batch


@dataclass
class Request:
    rid: int
    prompt: torch.Tensor                      # [Lp] token ids (host or device)
    max_new_tokens: int
    tokens: List[int] = field(default_factory=list)
    slot: int = -1
    prefilled: int = 0                        # prompt tokens the row already holds
    done: bool = False
    params: Optional[SamplingParams] = None   # sampling numbers of its own


class ContinuousBatcher:
    def __init__(self, engine: GenerationEngine, max_batch: int = 64, max_len: int = 2048, params: Optional[SamplingParams] = None,
                 prefill_chunk: Optional[int] = None, page_size: Optional[int] = None, pages: Optional[int] = None):
        """``page_size``: rows share ``pages`` pages of so many tokens (by default as many as ``max_batch`` rows of ``max_len`` take)."""
        self.engine, self.model = engine, engine.model
        self.params = params or SamplingParams.from_mode("greedy")
        self.max_batch, self.max_len = max_batch, max_len
        self.prefill_chunk = prefill_chunk
        self.device = next(self.model.parameters()).device
        if getattr(self.model, "_ep_comm", None) is not None:
            # admission prefills one request on one rank, which the expert-parallel exchange (a collective of all ranks) cannot serve
            raise RuntimeError("continuous batching runs on one GPU (or on replicas): the model must not be expert-parallel")
        self.paged = page_size is not None
        self.pool = PagedPool(self.model, max_batch, max_len, pages, page_size) if self.paged else SequencePool(self.model, max_batch, max_len)
        self.cache, self.slots = self.pool.cache, self.pool.slots
        self.history = torch.zeros(max_batch, self.params.repetition_window, dtype=torch.long, device=self.device)
        self.by_slot: Dict[int, Request] = {}          # rows that decode
        self.prefilling: List[Request] = []            # rows still in their prompt, oldest first
        self.waiting: List[Request] = []
        self.finished: Dict[int, Request] = {}
        self._next_id = 0
        self._stop = set(int(t) for t in (self.params.stop_token_ids or ()))
        self._own = 0                                  # requests under way that bring sampling numbers of their own
        self._numbers: Optional[Dict[str, torch.Tensor]] = None   # per row, once such a request has come
        self._brings: Optional[torch.Tensor] = None    # rows of such requests
        self.steps = 0
        self.generator, self.own_generator = (torch.Generator(device=self.device).manual_seed(self.params.seed) if self.params.seed is not None else None for _ in range(2))

    # -- requests --------------------------------------------------------------------------------------------------
    def submit(self, prompt: Sequence[int], max_new_tokens: Optional[int] = None, params: Optional[SamplingParams] = None) -> int:
        """``params``: sampling numbers, stop tokens and token budget of this request (its ``repetition_window`` and seed are the batcher's)."""
        ids = torch.as_tensor(prompt, dtype=torch.long).flatten()
        budget = int(max_new_tokens if max_new_tokens is not None else (params or self.params).max_new_tokens)
        if self.paged and self.pool.cache.pool.pages_for(ids.numel() + budget) > self.pool.pages:
            raise ValueError(f"prompt of {ids.numel()} tokens + {budget} new tokens does not fit {self.pool.pages} pages")
        if ids.numel() < 1 or ids.numel() + budget > self.max_len:
            raise ValueError(f"prompt of {ids.numel()} tokens + {budget} new tokens does not fit rows of {self.max_len}")
        r = Request(self._next_id, ids, budget, params=params)
        self._next_id += 1
        self.waiting.append(r)
        return r.rid

    @property
    def pending(self) -> int:
        return len(self.waiting) + len(self.prefilling) + len(self.by_slot)

    # -- sampling ----------------------------------------------------------------------------------------------------
    _FIELDS: Tuple[Tuple[str, torch.dtype], ...] = (("temperature", torch.float32), ("top_k", torch.int32), ("top_p", torch.float32), ("min_p", torch.float32),
                                                    ("repetition_penalty", torch.float32))

    _NOT_ASKED = SamplingParams.from_mode("greedy")   # of rows without numbers of their own: the least work

    def _set_numbers(self, slot: int, params: Optional[SamplingParams]) -> None:
        if self._numbers is None:
            if params is None:
                return
            self._numbers = {n: torch.full((self.max_batch,), getattr(self._NOT_ASKED, n), dtype=t, device=self.device) for n, t in self._FIELDS}
            self._brings = torch.zeros(self.max_batch, dtype=torch.bool, device=self.device)
        self._brings[slot] = params is not None
        for n, t in self._FIELDS:
            v = getattr(params or self._NOT_ASKED, n)
            self._numbers[n][slot] = v if t.is_floating_point else min(max(v, 0), torch.iinfo(t).max)   # (0, and more than there are: all tokens)

    def _sample(self, logits: torch.Tensor, rows: slice, own: int, others: int) -> torch.Tensor:
        """Tokens of ``rows``, of which ``own`` bring numbers of their own and ``others`` do not (the rest is not asked).  Either kind is drawn as though the
        other were not there: with its own sampler, from a generator of its own."""
        history = self.history[rows]
        tokens = sample_next(logits, self.params, history, self.generator) if others else None
        if not own:
            return tokens
        n = {k: v[rows] for k, v in self._numbers.items()}
        uniform = torch.rand(logits.shape[0], device=self.device, generator=self.own_generator)
        mine = ops.sample_rows(logits, uniform, n["temperature"], n["top_k"], n["top_p"], n["min_p"], n["repetition_penalty"], history)
        return mine if tokens is None else torch.where(self._brings[rows], mine, tokens)

    # -- one scheduling step ---------------------------------------------------------------------------------------
    @torch.no_grad()
    def _admit(self) -> None:
        budget = self.prefill_chunk or (1 << 62)       # prompt tokens this step may still run
        while budget > 0:
            if self.paged:
                used = self._admit_packed(min(budget, MAX_PACKED))
                if not used:
                    return
                budget -= used
                continue
            if not self.prefilling:
                if not (self.waiting and self.pool.available):
                    return
                r = self.waiting.pop(0)
                r.slot = self.pool.open()
                self.prefilling.append(r)
            r = self.prefilling[0]
            n = min(budget, r.prompt.numel() - r.prefilled)
            budget -= n
            part = r.prompt[r.prefilled:r.prefilled + n]
            r.prefilled += n
            done = r.prefilled == r.prompt.numel()
            logits = self.pool.extend(r.slot, part, active=done)
            if done:
                self.prefilling.pop(0)
                self._first_token(r, logits)

    def _admit_packed(self, room: int) -> int:
        """The next portions of prompts, oldest first, up to ``room`` tokens in one packed batch -> tokens that were run."""
        taken: List[Tuple[Request, torch.Tensor]] = []
        left = room
        while left > 0:
            r = self.prefilling[len(taken)] if len(taken) < len(self.prefilling) else None
            if r is None:
                # (requests wait for their turn: a later one that is shorter does not overtake)
                if not (self.waiting and self.pool.fits(self.waiting[0].prompt.numel() + self.waiting[0].max_new_tokens)):
                    break
                r = self.waiting.pop(0)
                r.slot = self.pool.open(r.prompt.numel() + r.max_new_tokens)
                self.prefilling.append(r)
            n = min(left, r.prompt.numel() - r.prefilled)
            taken.append((r, r.prompt[r.prefilled:r.prefilled + n]))
            left -= n
        if not taken:
            return 0
        logits = self.pool.extend_many([(r.slot, part) for r, part in taken])
        for i, (r, part) in enumerate(taken):
            r.prefilled += part.numel()
            if r.prefilled == r.prompt.numel():
                self.prefilling.remove(r)
                self._first_token(r, logits[i:i + 1])
        return room - left

    def _first_token(self, r: Request, logits: torch.Tensor) -> None:
        slot, ids, w = r.slot, r.prompt.to(self.device), self.history.shape[1]
        n = ids.numel()
        self.history[slot].fill_(int(r.prompt[0]))     # left padding of a short prompt repeats its first token
        self.history[slot, -min(n, w):] = ids[-min(n, w):]
        self._own += r.params is not None
        self._set_numbers(slot, r.params)
        first = self._sample(logits, slice(slot, slot + 1), r.params is not None, r.params is None)
        self.pool.last[slot:slot + 1] = first
        self.history[slot] = torch.roll(self.history[slot], -1)
        self.history[slot, -1:] = first
        self.by_slot[slot] = r
        self._accept(slot, int(first))

    def _accept(self, slot: int, token: int) -> None:
        """Host-side bookkeeping of one generated token (the device-side state was updated for all rows at once)."""
        r = self.by_slot[slot]
        r.tokens.append(token)
        own = r.params and r.params.stop_token_ids
        stop = self._stop if r.params is None else () if own is None else own
        if token in stop or len(r.tokens) >= r.max_new_tokens:
            self._retire(slot)

    def _retire(self, slot: int) -> None:
        r = self.by_slot.pop(slot)
        r.done = True
        self._own -= r.params is not None
        self.finished[r.rid] = r
        self.pool.close(slot)

    @torch.no_grad()
    def step(self) -> int:
        """Admit, decode one token for every live row, retire.  Returns the number of live rows that were decoded."""
        self._admit()
        live = sorted(self.by_slot)
        if not live:
            return 0
        logits = self.pool.decode(live)
        nxt_dev = self._sample(logits, slice(None), self._own, len(live) - self._own)
        self.pool.last.copy_(nxt_dev)
        self.history = torch.roll(self.history, -1, dims=1)
        self.history[:, -1] = nxt_dev
        nxt = nxt_dev.tolist()                       # the one device-to-host read of the step
        for slot in live:
            self._accept(slot, int(nxt[slot]))
        self.steps += 1
        return len(live)

    def run(self, prompts: Sequence[Sequence[int]], max_new_tokens: Optional[int] = None) -> List[List[int]]:
        """Serve all prompts; returns the generated ids in the order of ``prompts``."""
        rids = [self.submit(p, max_new_tokens) for p in prompts]
        while self.pending:
            self.step()
        return [self.finished.pop(r).tokens for r in rids]
