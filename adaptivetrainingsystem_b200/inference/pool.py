"""A pool of cache rows that sequences come to and leave one by one.

One cache of ``rows`` rows, a free list, and one decode step over all rows -- captured into a CUDA graph on a GPU.  A sequence opens a
row, is extended by portions of any size (written straight into the row through a one-row view of the cache), decodes one token at a
time together with the other rows, and closes the row again.  Rows that do not take part in a decode step come out of it unchanged.
``ContinuousBatcher`` schedules requests on such a pool; ``TraceRunner`` replays recorded steps on one.

:class:`PagedPool` is the same over a paged cache: rows take pages as they grow, and portions of several sequences run as one packed batch.
"""
from __future__ import annotations

from typing import Dict, Optional, Sequence, Tuple

import torch


from ..ops.gemm import chained_launches
from .engine import GraphDecoder, KVSlotManager


class SequencePool:
    def __init__(self, model, rows: int, max_len: int, use_graph: Optional[bool] = None):
        self.model, self.rows, self.max_len = model, rows, max_len
        p = next(model.parameters())
        self.device = p.device
        self.cache = model.make_cache(rows, max_len)
        self.slots = KVSlotManager(rows)
        self.lengths: Dict[int, int] = {}                 # open rows -> tokens they hold
        self.use_graph = (self.device.type == "cuda") if use_graph is None else use_graph
        if not self.use_graph and not getattr(model, "eager_row_decode", False):
            raise RuntimeError("decoding rows of different lengths replays a CUDA graph of the decode step: a CUDA device is required")
        self._decoder: Optional[GraphDecoder] = None
        self.last = torch.zeros(rows, dtype=torch.long, device=self.device)
        if self.use_graph:
            self.decoder()
        else:
            self.cache.enable_device_lengths()
        self.cache.device_lengths.zero_()
        self.cache.device_positions.zero_()
        self.cache.device_active.zero_()

    @torch.no_grad()
    def decoder(self) -> GraphDecoder:
        if self._decoder is None:
            self._decoder = GraphDecoder(self.model, self.cache)   # captured once; rows come and go underneath it
        return self._decoder

    # -- rows -----------------------------------------------------------------------------------------------------
    @property
    def available(self) -> int:
        return self.slots.available

    def open(self) -> int:
        slot = self.slots.alloc(1)
        if slot is None:
            raise RuntimeError(f"all {self.rows} rows of the pool are taken")
        self.lengths[int(slot[0])] = 0
        return int(slot[0])

    def close(self, slot: int) -> None:
        del self.lengths[slot]
        self.cache.set_row(slot, 0, False)
        self.slots.free(torch.tensor([slot]))

    # -- tokens ---------------------------------------------------------------------------------------------------
    @torch.no_grad()
    def extend(self, slot: int, ids: Sequence[int], logits_at: Optional[Sequence[int]] = None, active: bool = False) -> Optional[torch.Tensor]:
        """Runs the next portion of a sequence -> logits [1, V] of its last token, or [n, V] of the places ``logits_at`` of the portion
        (``None`` when that is empty).  ``active``: the row takes part in decode steps from now on."""
        ids = torch.as_tensor(ids, dtype=torch.long).flatten()
        n = self.lengths[slot]
        view = self.cache.row(slot)
        view.length = n
        at = [ids.numel() - 1] if logits_at is None else list(logits_at)
        logits = self.model(ids.to(self.device).view(1, -1), cache=view, logits_at=at or [0], return_aux_loss=False)
        self.lengths[slot] = n + ids.numel()
        self.cache.set_row(slot, self.lengths[slot], active)
        return logits[0] if at else None

    @torch.no_grad()
    def decode(self, slots: Sequence[int]) -> torch.Tensor:
        """One decode step: every row of ``slots`` feeds its token in ``last`` -> logits [rows, V] (rows outside ``slots`` are
        meaningless; a static buffer that the next step overwrites).  ``cache.device_active`` must mark exactly these rows."""
        for s in slots:
            if self.lengths[s] + 1 > self.max_len:
                raise RuntimeError(f"cache overflow: {self.lengths[s]}+1 > {self.max_len}")
        if self.use_graph:
            d = self.decoder()
            d.tokens.copy_(self.last.view(-1, 1))
            d.graph.replay()
            logits = d.logits
        else:
            logits = self.model(self.last.view(-1, 1), cache=self.cache, last_token_only=True, return_aux_loss=False)[:, -1]
            self.cache.device_advance()
        for s in slots:
            self.lengths[s] += 1
        return logits



class PagedPool:
    """Rows over ``pages`` pages of ``page_size`` tokens (by default as many as all rows at ``max_len`` need; fewer serve more rows than would fit).
    A row is opened for a number of tokens; these pages are set aside on the host, so that no row that is under way runs out of them, and taken on
    the device only as the row grows."""

    def __init__(self, model, rows: int, max_len: int, pages: Optional[int] = None, page_size: int = 64, use_graph: Optional[bool] = None):
        self.model, self.rows, self.max_len = model, rows, max_len
        if not hasattr(model, "make_paged_cache"):
            raise ValueError(f"{type(model).__name__} has no paged cache")
        self.device = next(model.parameters()).device
        self.pages = pages if pages is not None else rows * -(-max_len // page_size)
        self.cache = model.make_paged_cache(rows, max_len, self.pages, page_size)
        self.slots = KVSlotManager(rows)
        self.lengths: Dict[int, int] = {}                 # open rows -> tokens they hold
        self.reserved: Dict[int, int] = {}                # open rows -> pages set aside for them
        self.use_graph = (self.device.type == "cuda") if use_graph is None else use_graph
        self.last = torch.zeros(rows, dtype=torch.long, device=self.device)
        self.fresh = torch.zeros(rows, dtype=torch.int32, device=self.device)   # new tokens of the next decode step
        self._live: Tuple[int, ...] = ()
        self._graph = None

    # -- rows -----------------------------------------------------------------------------------------------------
    @property
    def available(self) -> int:
        return self.slots.available

    @property
    def pages_left(self) -> int:
        return self.pages - sum(self.reserved.values())

    def fits(self, tokens: int) -> bool:
        """Whether a row for ``tokens`` tokens can be opened now."""
        return self.available > 0 and tokens <= self.max_len and self.cache.pool.pages_for(tokens) <= self.pages_left

    def open(self, tokens: Optional[int] = None) -> int:
        tokens = self.max_len if tokens is None else tokens
        if not self.fits(tokens):
            raise RuntimeError(f"no row for {tokens} tokens: {self.available} of {self.rows} rows and {self.pages_left} of {self.pages} pages are free")
        slot = int(self.slots.alloc(1)[0])
        self.lengths[slot] = 0
        self.reserved[slot] = self.cache.pool.pages_for(tokens)
        return slot

    def close(self, slot: int) -> None:
        if self.lengths[slot]:
            fresh = torch.zeros(self.rows, dtype=torch.int32)
            fresh[slot] = -1
            self.cache.plan(fresh.to(self.device), 0)
        del self.lengths[slot], self.reserved[slot]
        self.slots.free(torch.tensor([slot]))

    def _check_room(self, more: Dict[int, int]) -> None:
        for slot, n in more.items():
            if self.lengths[slot] + n > self.max_len:
                raise RuntimeError(f"cache overflow: {self.lengths[slot]}+{n} > {self.max_len}")
            if self.cache.pool.pages_for(self.lengths[slot] + n) > self.reserved[slot]:
                raise RuntimeError(f"row {slot} was opened for {self.reserved[slot]} pages and holds {self.lengths[slot]} tokens: no room for {n} more")

    def _grow(self, more: Dict[int, int]) -> None:
        """The step has been planned on the device: rows hold these tokens more."""
        for slot, n in more.items():
            self.lengths[slot] += n

    # -- tokens ---------------------------------------------------------------------------------------------------
    @torch.no_grad()
    def extend_many(self, portions: Sequence[Tuple[int, Sequence[int]]]) -> torch.Tensor:
        """Runs the next portions ``(row, token ids)`` of different rows as one packed batch -> logits [portions, V] of each one's last token."""
        ids = {slot: torch.as_tensor(part, dtype=torch.long).flatten() for slot, part in portions}
        if len(ids) != len(portions) or not portions or any(t.numel() == 0 for t in ids.values()):
            raise ValueError("portions of at least one token, of different rows, are needed")
        more = {slot: part.numel() for slot, part in ids.items()}
        self._check_room(more)
        order = sorted(ids)                                # rows lie in the packed batch in their own order
        fresh = torch.zeros(self.rows, dtype=torch.int32)
        fresh[order] = torch.tensor([ids[s].numel() for s in order], dtype=torch.int32)
        ends = fresh[order].cumsum(0) - 1
        packed = torch.cat([ids[s] for s in order]).to(self.device)
        self.cache.plan(fresh.to(self.device), packed.numel(), max_new=int(fresh.max()), max_len=max(self.lengths[s] + more[s] for s in order))
        self._grow(more)
        at = dict(zip(order, ends.tolist()))
        return self.model(packed.view(1, -1), cache=self.cache, logits_at=[at[slot] for slot, _ in portions], return_aux_loss=False)[0]

    def extend(self, slot: int, ids: Sequence[int]) -> torch.Tensor:
        """Runs the next portion of a sequence -> logits [1, V] of its last token."""
        return self.extend_many([(slot, ids)])

    def _decode(self, slots: Sequence[int] = ()) -> torch.Tensor:
        plan = self.cache.plan(self.fresh, self.rows, single=True)
        self._grow({s: 1 for s in slots})
        place = plan.starts[:-1].long()                    # of a row's token in the packed batch
        packed = torch.zeros(self.rows + 1, dtype=torch.long, device=self.device).scatter_(0, torch.where(self.fresh > 0, place, self.rows), self.last)[:-1]
        # (several ranks: their barriers keep launches in order)
        alone = not (torch.distributed.is_available() and torch.distributed.is_initialized() and torch.distributed.get_world_size() > 1)
        with chained_launches(alone and self.use_graph and self.device.type == "cuda"):
            logits = self.model(packed.view(-1, 1), cache=self.cache, last_token_only=True, return_aux_loss=False)[:, -1]
        return logits.index_select(0, place.clamp(max=self.rows - 1))

    def _capture(self) -> None:
        self.fresh.zero_()                                 # warm-up steps in which no row has a token change nothing
        self._live = ()
        side = torch.cuda.Stream(device=self.device)
        side.wait_stream(torch.cuda.current_stream(self.device))
        with torch.cuda.stream(side), torch.no_grad():
            for _ in range(2):
                self._decode()
        torch.cuda.current_stream(self.device).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph), torch.no_grad():
            self._logits = self._decode()
            self._plan = self.cache.step                   # (the graph writes it again whenever it is replayed)
        self._graph = graph                                # (only a whole one)

    @torch.no_grad()
    def decode(self, slots: Sequence[int]) -> torch.Tensor:
        """One decode step: every row of ``slots`` feeds its token in ``last`` -> logits [rows, V] (rows outside ``slots`` are meaningless; a static
        buffer that the next step overwrites)."""
        if len(set(slots)) != len(slots):
            raise ValueError("every row decodes one token of a step")
        self._check_room({s: 1 for s in slots})
        if self.use_graph and self._graph is None:
            self._capture()
        if self._live != tuple(slots):
            live = torch.zeros(self.rows, dtype=torch.int32)
            live[list(slots)] = 1
            self.fresh.copy_(live)
            self._live = tuple(slots)
        if not self.use_graph:
            return self._decode(slots)
        self._graph.replay()
        self._grow({s: 1 for s in slots})
        return self._logits
