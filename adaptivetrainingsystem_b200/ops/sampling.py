"""Next tokens of a batch whose rows have sampling numbers of their own (``csrc/sample_rows.cu``).

:func:`serving.sample_tokens` serves a batch with one set of numbers and keeps all tokens that tie at a cut; here every request of a batch
brings its own, there is min-p, ties are broken (lower index first), and the answer is that of a 64-bit evaluation, so that given random
numbers name the same tokens whatever the batch they are drawn in.  The order of the rules is the reference's (repetition penalty, temperature,
top-k, top-p, draw: reference ``Chat.py:391-425``) with min-p behind top-p.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _lib
from .paged import _fn, _need, _on, _p, _stream

MAX_ROWS, MAX_VOCAB = 65535, 1 << 20
PerRow = Union[int, float, torch.Tensor]


def _numbers(value: PerRow, dtype: torch.dtype):
    """-> (tensor [B] or None, number)."""
    if not isinstance(value, torch.Tensor):
        return None, min(max(int(value), 0), MAX_VOCAB) if dtype == torch.int32 else float(value)
    if dtype == torch.int32 and value.dtype != dtype:
        value = value.clamp(0, MAX_VOCAB)   # (64-bit numbers keep their meaning)
    return (value if value.dtype == dtype and value.is_contiguous() else value.to(dtype).contiguous()), 0


def sample_rows(logits: torch.Tensor, uniform: torch.Tensor, temperature: PerRow = 1.0, top_k: PerRow = 0, top_p: PerRow = 1.0, min_p: PerRow = 0.0,
                repetition_penalty: PerRow = 1.0, history: Optional[torch.Tensor] = None) -> torch.Tensor:
    """logits [B, V] (bfloat16 or float32), ``uniform`` [B] in [0, 1) -> token ids [B] int64.  Every sampling number is one for all rows or a tensor [B].

    ``history`` [B, n] int64: scores of these tokens are divided by the row's ``repetition_penalty`` where positive and multiplied elsewhere, once
    however often a token is listed; ids outside the vocabulary (-1 as padding) are ignored.  ``temperature`` <= 0: the largest score, lowest index
    among equals.  Otherwise, with the tokens in order of their scores (lowest index first among equals): the first ``top_k`` (0: all); of
    these, the ones with at most ``top_p`` of their mass before them; of these, the ones with at least ``min_p`` of the first one's mass; and
    of what is kept, in index order, the token at which the cumulative mass exceeds ``uniform`` times the total.  NaN counts as -infinity; a row
    of nothing but -infinity gives its first token."""
    _need(logits.dim() == 2 and logits.shape[1] >= 1 and logits.shape[1] <= MAX_VOCAB, f"logits: [rows, vocabulary], at most {MAX_VOCAB} wide")
    B, V = logits.shape
    _need(B <= MAX_ROWS, "at most 65535 rows")
    _need(isinstance(uniform, torch.Tensor) and uniform.shape == (B,) and uniform.device == logits.device, "uniform: one number per row on the logits' device")
    if history is not None:
        _need(history.dim() == 2 and history.shape[0] == B and history.dtype == torch.int64 and history.device == logits.device,
              "history: int64 [rows, n] on the logits' device")
    for name, v in (("temperature", temperature), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p), ("repetition_penalty", repetition_penalty)):
        if isinstance(v, torch.Tensor) and (v.shape != (B,) or v.device != logits.device):
            raise ValueError(f"{name}: a number, or one per row on the logits' device")
    if not logits.is_cuda:
        return sample_rows_reference(logits, uniform, temperature, top_k, top_p, min_p, repetition_penalty, history)
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{logits.dtype}: sample_rows takes bfloat16 and float32")
    out = torch.empty(B, dtype=torch.int64, device=logits.device)
    if B == 0:
        return out
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    if history is not None and history.shape[1] and history.stride(1) != 1:
        history = history.contiguous()
    t, t1 = _numbers(temperature, torch.float32)
    k, k1 = _numbers(top_k, torch.int32)
    tp, tp1 = _numbers(top_p, torch.float32)
    mp, mp1 = _numbers(min_p, torch.float32)
    rp, rp1 = _numbers(repetition_penalty, torch.float32)
    u, _ = _numbers(uniform, torch.float32)
    n = 0 if history is None else history.shape[1]
    with _on(logits.device):
        _lib.check(_fn("ats_sample_rows")(_p(logits), int(logits.dtype == torch.float32), logits.stride(0), B, V, _p(u), _p(t), t1, _p(k), k1, _p(tp), tp1, _p(mp), mp1, _p(rp), rp1,
                     _p(history) if n else 0, n, history.stride(0) if n else 0, _p(out), _stream(logits.device)), "ats_sample_rows")
    return out


def sample_rows_reference(logits: torch.Tensor, uniform: torch.Tensor, temperature: PerRow = 1.0, top_k: PerRow = 0, top_p: PerRow = 1.0, min_p: PerRow = 0.0,
                          repetition_penalty: PerRow = 1.0, history: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The definition, with a sort and 64-bit masses."""
    B, V = logits.shape

    def column(v, dtype):
        v = v if isinstance(v, torch.Tensor) else torch.full((B,), v, device=logits.device)
        return v.to(dtype)[:, None]
    x = logits.float()
    if history is not None and history.numel():
        # (a column more for the ids that are ignored)
        ids = torch.where((history >= 0) & (history < V), history, V)
        seen = torch.zeros(B, V + 1, dtype=torch.bool, device=x.device).scatter_(1, ids, True)[:, :V]
        pen = column(repetition_penalty, torch.float32)
        x = torch.where(seen & (pen != 1), torch.where(x > 0, x / pen, x * pen), x)
    x = torch.where(torch.isnan(x), float("-inf"), x)
    t = column(temperature, torch.float32)
    first = x.argmax(-1)
    top = x.gather(1, first[:, None]).double()
    greedy = ~(t > 0) | torch.isinf(top) & (top < 0)
    order = x.argsort(dim=-1, descending=True, stable=True)
    gap = torch.where(x.double() == top, 0.0, x.double() - top)
    w = torch.where(torch.isinf(gap), gap, gap / torch.where(greedy, 1.0, t.double())).exp().gather(1, order)
    k = column(top_k, torch.int64)
    w = torch.where(torch.arange(V, device=x.device)[None] < torch.where(k > 0, k, V), w, 0.0)
    before = w.cumsum(-1) - w
    p = column(top_p, torch.float32).double()
    keep = ((before <= p.clamp(min=0) * w.sum(-1, keepdim=True)) | (p >= 1)) & (w >= column(min_p, torch.float32).double().clamp(max=1))
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    cdf = kept.cumsum(-1)
    pick = (cdf <= uniform.double().clamp(min=0)[:, None] * cdf[:, -1:]).sum(-1)
    last = V - 1 - (kept > 0).to(torch.int8).flip(-1).argmax(-1)      # a number of 1 or more takes the last token that is kept
    return torch.where(greedy[:, 0], first, torch.minimum(pick, last))
