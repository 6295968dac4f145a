"""What a decoder keeps per sequence between steps.

:class:`SequenceCache` is the part every model shares: the fill level, its device-side copy for decode steps that are replayed from a
CUDA graph, and row views for schedulers that admit sequences one by one into a pool.  ``KVCache`` (``transformer.py``) holds keys and
values of every position in a row per sequence, :class:`PagedKVCache` the same in pages that rows share out among themselves;
:class:`LayerStateCache` holds whatever its layers declare -- rings of the last tokens, recurrent states,
convolution inputs -- one entry per layer *run*, so a layer that is run several times per token has a state for each run.
"""
from __future__ import annotations

from typing import Dict, List, Optional

import torch

from .. import ops


class SequenceCache:
    """``length`` (host) is the number of tokens every row holds during a portion of a prompt; decode steps read the device-side
    ``device_lengths`` / ``device_positions`` (int32 [batch]).  Rows whose ``device_active`` entry is 0 are computed by a replayed decode
    step but must come out of it unchanged."""

    def __init__(self, batch: int, max_len: int, device):
        self.batch, self.max_len, self.device = batch, max_len, torch.device(device)
        self.length = 0
        self.device_lengths: Optional[torch.Tensor] = None
        self.device_positions: Optional[torch.Tensor] = None
        self.device_active: Optional[torch.Tensor] = None
        self._device_counters: Optional[torch.Tensor] = None   # lengths and positions side by side: one launch moves both on

    def enable_device_lengths(self) -> None:
        self._device_counters = torch.full((2, self.batch), self.length, dtype=torch.int32, device=self.device)
        self.device_lengths, self.device_positions = self._device_counters
        self.device_active = torch.ones(self.batch, dtype=torch.int32, device=self.device)

    def device_advance(self) -> None:
        """One decoded token of every active row: called inside the captured step."""
        rows = (self.device_lengths, self.device_positions)
        if self._device_counters is not None and [t.data_ptr() for t in rows] == [t.data_ptr() for t in self._device_counters]:
            self._device_counters += self.device_active
        else:   # (tensors of the caller's in their place)
            for t in rows:
                t += self.device_active

    def set_row(self, row: int, length: int, active: bool) -> None:
        self.device_lengths[row] = length
        self.device_positions[row] = length
        self.device_active[row] = int(active)

    def advance(self, n: int) -> None:
        self.length += n

    def reset(self) -> None:
        self.length = 0

    def row(self, i: int) -> "SequenceCache":
        """Row ``i`` as an empty cache of batch 1 whose writes land in this cache."""
        raise NotImplementedError


class LayerStateCache(SequenceCache):
    """``states[r]``: named tensors ``[batch, ...]`` of layer run ``r``.  A sequence at position 0 starts from nothing whatever its row
    still holds, so a row can be handed to the next sequence without being cleared."""

    def __init__(self, batch: int, max_len: int, device, states: List[Dict[str, torch.Tensor]]):
        super().__init__(batch, max_len, device)
        self.states = states

    def row(self, i: int) -> "LayerStateCache":
        return LayerStateCache(1, self.max_len, self.device, [{k: t[i:i + 1] for k, t in s.items()} for s in self.states])


class PagedKVCache(SequenceCache):
    """Keys and values of ``batch`` rows in ``pages`` pages of ``page_size`` tokens, per layer ``[pages, page_size, Hkv, D]`` (``ops.PagePool``).  A row
    takes pages as it grows, so memory follows the tokens that rows hold, not the longest that they might.

    A step of the model is planned first (:meth:`plan`): it runs the new tokens of all rows packed one row after the other, portions of prompts
    ``[1, T]`` or, with ``single``, at most one token per row ``[rows, 1]`` (the form that is captured in a CUDA graph)."""

    def __init__(self, num_layers: int, batch: int, max_len: int, pages: int, page_size: int, n_kv: int, head_dim: int, dtype, device):
        super().__init__(batch, -(-max_len // max(page_size, 1)) * page_size, device)   # a row may fill its last page: rotary tables reach that far
        self.pool = ops.PagePool(batch, max_len, pages, page_size, device)
        self.k = [torch.zeros(pages, page_size, n_kv, head_dim, dtype=dtype, device=device) for _ in range(num_layers)]
        self.v = [torch.zeros(pages, page_size, n_kv, head_dim, dtype=dtype, device=device) for _ in range(num_layers)]
        self.step: Optional[ops.PagePlan] = None

    def plan(self, fresh: torch.Tensor, tokens: int, max_new: Optional[int] = None, max_len: Optional[int] = None, single: bool = False) -> "ops.PagePlan":
        """``fresh`` int32 [batch]: new tokens of every row (-1: the row is closed), ``tokens`` of them in all at most."""
        self.step = ops.page_plan(self.pool, fresh, tokens, max_new=1 if single else max_new, max_len=max_len)
        # a step of single tokens reads positions from the device, like a replayed step over contiguous rows
        self.device_lengths, self.device_positions = (self.step.lengths, self.step.positions) if single else (None, None)
        return self.step

    def reset(self) -> None:
        fresh = torch.full((self.batch,), -1, dtype=torch.int32, device=self.device)
        self.plan(fresh, 0)

    def advance(self, n: int) -> None:
        pass   # the plan moves the rows on

    def device_advance(self) -> None:
        pass

    def attend(self, layer: int, qkv: torch.Tensor, n_q: int, n_kv: int, d: int, cos: Optional[torch.Tensor], sin: Optional[torch.Tensor]) -> torch.Tensor:
        """qkv [..., (n_q + 2 n_kv) d], the step's packed projection, rotated already where ``cos`` is ``None`` -> [..., n_q * d]."""
        if cos is not None and qkv.is_cuda and d % 16:   # (heads that the kernel does not rotate)
            qkv, cos, sin = ops.rope_packed(qkv, cos, sin, n_q, n_kv, d, positions=self.step.positions.view(qkv.shape[:-1])), None, None
        q = ops.paged_append(qkv.reshape(-1, qkv.shape[-1]), cos, sin, self.step, self.k[layer], self.v[layer], n_q, n_kv, d)
        return ops.paged_attention(q, self.k[layer], self.v[layer], self.step).reshape(*qkv.shape[:-1], n_q * d)
