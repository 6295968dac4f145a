"""Paged key / value cache: page tables kept on the GPU, the write of new tokens into their pages, and attention over them
(``csrc/paged.cu``).

A pool of pages holds the keys and values of many sequences ("rows"): token ``i`` of row ``r`` lies in slot
``tables[r, i // page_size] * page_size + i % page_size`` of ``[pages, page_size, n_kv, d]`` tensors, one pair per layer; free pages are a
stack.  A step feeds every row some new tokens (none, one, or a portion of a prompt), packed one row after the other:

* :func:`page_plan` takes the pages that the step needs, and says where each new token goes;
* :func:`paged_append` rotates queries and keys and writes keys and values to their slots;
* :func:`paged_attention` lets every new token attend to its row's tokens up to itself.

Nothing of a step depends on lengths that the host would have to read, so a step of single tokens can be captured in a CUDA graph and
replayed while rows come and go.  Tensors on the CPU run the PyTorch definitions below, which are also the oracles of the kernel tests.
The reference has no cache (it runs the whole context again for every token, reference ``Chat.py:379-452``); its vendored serving engine keeps
whole rows per request (``colossalai/inference/kv_cache/kvcache_manager.py:11-106``).
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import math
from typing import Optional

import torch

from . import _lib

_vp, _ci, _cll, _cf = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float
MAX_ROWS, MAX_TOKENS, MAX_SLOTS = 4096, 1 << 18, (1 << 31) - 257
_REFUSED = {1: "a row gets more tokens than its table or the packed batch holds", 2: "not enough free pages", 3: "the stack of free pages is inconsistent"}


_SIGNATURES = {
    "ats_page_plan": [_vp] * 10 + [_ci] * 6 + [_vp],
    "ats_paged_append": [_vp, _cll, _vp, _vp, _ci, _vp, _vp, _vp, _vp, _vp, _ci, _ci, _ci, _ci, _cll, _ci, _vp, _vp],
    "ats_paged_attn_any": [_vp, _cll, _vp, _vp, _vp, _vp, _vp, _vp, _cll] + [_ci] * 8 + [_cf, _ci, _ci, _ci, _vp, _vp, _vp],
    "ats_paged_any_splits": [_ci, _ci, _ci, _cll],
    "ats_paged_decode": [_vp, _cll, _vp, _vp, _vp, _vp, _vp, _vp, _cll] + [_ci] * 8 + [_cll, _ci, _ci, _cf, _ci, _ci, _vp, _vp, _vp],
    "ats_paged_decode_scratch": [_ci, _ci, _ci, _cll, _ci],
    "ats_paged_portion": [_vp, _cll, _vp, _vp, _vp, _vp, _vp, _vp, _cll] + [_ci] * 9 + [_cf, _ci, _vp, _vp, _vp],
    "ats_paged_portion_scratch": [_ci],
    "ats_sample_rows": [_vp, _ci, _cll, _ci, _ci, _vp, _vp, _cf, _vp, _ci, _vp, _cf, _vp, _cf, _vp, _cf, _vp, _ci, _cll, _vp, _vp],
}
_fns = {}


def _fn(name: str):
    f = _fns.get(name)
    if f is None:
        f = getattr(_lib.cuda_lib(), name)
        f.restype, f.argtypes = _cll if name.endswith(("_scratch", "_splits")) else _ci, _SIGNATURES[name]
        _fns[name] = f
    return f


@functools.lru_cache(maxsize=1024)
def _scratch(name: str, *sizes: int) -> int:
    return _fn(name)(*sizes)


def _p(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


_here = contextlib.nullcontext()


def _on(device: torch.device):
    """Launches go to the tensors' device, whichever is current."""
    return _here if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _ints(t: torch.Tensor, name: str, shape, device) -> None:
    if not (isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.shape == shape and t.is_contiguous() and t.device == device):
        raise ValueError(f"{name}: a contiguous int32 tensor {list(shape)} on {device} is needed")


class PagePool:
    """Page tables of ``rows`` rows of up to ``max_len`` tokens (and what their last page holds beyond) over ``pages`` pages of ``page_size`` tokens (a power of two).  ``tables``
    [rows, max_len / page_size], ``lengths`` [rows] (tokens a row holds) and the stack ``free`` live on the device; ``state`` holds the number of free
    pages and the refusal code of the last committed step.  Steps of one pool follow one another: plan them on one stream, or order the streams."""

    def __init__(self, rows: int, max_len: int, pages: int, page_size: int = 64, device="cuda"):
        _need(page_size >= 1 and page_size & (page_size - 1) == 0, f"page_size {page_size}: a power of two is needed")
        _need(1 <= rows <= MAX_ROWS, f"{rows} rows: 1 to {MAX_ROWS} are possible")
        width = -(-max_len // page_size)
        _need(max_len >= 1 and pages >= 1 and pages * page_size <= MAX_SLOTS and rows * width < 1 << 31 and width * page_size <= MAX_SLOTS,
              "pages and rows: at least one page and one token, and slots below 2^31 - 256")
        self.rows, self.pages, self.page_size, self.width = rows, pages, page_size, width
        self.max_len = max_len
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.device = device
        i32 = dict(dtype=torch.int32, device=device)
        self.tables = torch.zeros(rows, width, **i32)
        self.lengths = torch.zeros(rows, **i32)
        self.free = torch.arange(pages - 1, -1, -1, **i32)   # page 0 is handed out first
        self.state = torch.tensor([pages, 0, 0, 0], **i32)

    def pages_for(self, tokens: int) -> int:
        return -(-tokens // self.page_size)

    def check(self) -> None:
        """Raises if the last committed step was refused (reads the device)."""
        code = int(self.state[1])
        if code:
            raise RuntimeError(f"the step was refused: {_REFUSED.get(code, code)}")


class PagePlan:
    """What the operators of one step read:

    * ``starts`` int32 [rows + 1]: row r's new tokens are packed at starts[r] .. starts[r + 1];
    * ``slots``, ``positions`` int32 [tokens] (slot -1: no row's token);
    * ``lengths`` int32 [rows]: tokens of the row, the new ones among them;
    * ``tables`` int32 [rows, width], ``page_size``;
    * ``max_new`` / ``max_len``: the longest portion and the longest row of the step as far as the host knows them (upper bounds that choose kernels and
      grids; by default the packed batch and the tables' width);
    * ``info`` int32 [2]: free pages after the step, refusal code."""

    def __init__(self, starts: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor, lengths: torch.Tensor, tables: torch.Tensor, page_size: int,
                 max_new: Optional[int] = None, max_len: Optional[int] = None, info: Optional[torch.Tensor] = None):
        # (_good: the tokens and the device that the tensors have been checked for)
        self.__dict__.update(starts=starts, slots=slots, positions=positions, lengths=lengths, tables=tables, page_size=page_size, max_new=max_new, max_len=max_len,
                             info=info, _good=None)

    def __setattr__(self, name, value):
        self.__dict__[name] = value
        self.__dict__["_good"] = None

    @property
    def count(self) -> torch.Tensor:
        """int32 [1]: free pages after the step."""
        return self.info[:1]

    def check(self) -> None:
        """Raises if the step was refused (reads the device)."""
        code = int(self.info[1])
        if code:
            raise RuntimeError(f"the step was refused: {_REFUSED.get(code, code)}")


# ----------------------------------------------------------------------------------------------------------
# page tables and slots
# ----------------------------------------------------------------------------------------------------------
def page_plan(pool: PagePool, fresh: torch.Tensor, tokens: int, commit: bool = True, max_new: Optional[int] = None, max_len: Optional[int] = None) -> PagePlan:
    """Plans a step.  ``fresh`` int32 [rows]: new tokens of every row; 0: the row sits out; -1: the row is closed, its pages go back.
    ``tokens``: rows of the packed batch, at least as many as there are new tokens (slots behind them are -1).

    Closed rows push their pages onto the stack in row order, then rows take from its top in row order.  With ``commit`` the pool moves on in
    the same launch; without, its tables hold the step's pages but lengths and free pages stay, so the step can be planned again (or another
    one instead).  A step that does not fit is refused as a whole: no row has tokens in it, nothing changes, and :meth:`PagePlan.check`
    (without ``commit``) or :meth:`PagePool.check` raises."""
    if not 0 <= tokens <= MAX_TOKENS:
        raise ValueError(f"{tokens} tokens in a step: at most {MAX_TOKENS}")
    _ints(fresh, "fresh", (pool.rows,), pool.device)
    i32 = dict(dtype=torch.int32, device=pool.device)
    R = pool.rows
    # one allocation: starts, slots, positions, free pages and refusal, lengths
    sizes = (R + 1, tokens, tokens, 2, 0 if commit else R)
    buf = torch.empty(sum(sizes), **i32)
    starts, slots, positions, info, lengths = buf.split_with_sizes(sizes)
    if commit:
        lengths = pool.lengths
    plan = PagePlan(starts, slots, positions, lengths, pool.tables, pool.page_size, max_new, max_len, info)
    if not pool.device.type == "cuda":
        _page_plan_reference(pool, fresh, plan, commit)
        return plan
    at = buf.data_ptr()
    with _on(pool.device):
        _lib.check(_fn("ats_page_plan")(
            _p(pool.lengths), _p(fresh), _p(pool.tables), _p(pool.free), _p(pool.state), at, at + 4 * (R + 1), at + 4 * (R + 1 + tokens), _p(lengths), at + 4 * (R + 1 + 2 * tokens), R,
            pool.width, pool.pages, pool.page_size, tokens, int(commit), _stream(pool.device)), "ats_page_plan")
    return plan


def _page_plan_reference(pool: PagePool, fresh: torch.Tensor, plan: PagePlan, commit: bool) -> None:
    ps, room, T = pool.page_size, pool.width * pool.page_size, plan.slots.numel()
    old, new, n = pool.lengths.tolist(), fresh.tolist(), int(pool.state[0])
    plan.slots.fill_(-1)
    plan.positions.zero_()
    plan.starts.zero_()
    bad = any(o < 0 or o > room or f < -1 or o + max(f, 0) > room for o, f in zip(old, new)) or sum(max(f, 0) for f in new) > T
    refused, stack = int(bad), pool.free[:max(n, 0)].tolist()
    if not refused:
        for r, f in enumerate(new):
            if f < 0:
                stack += pool.tables[r, :-(-old[r] // ps)].tolist()
        need = sum(-(-(o + f) // ps) - -(-o // ps) for o, f in zip(old, new) if f >= 0)
        refused = 2 if need > len(stack) else 3 if n < 0 or len(stack) > pool.pages else 0
    after = list(old)
    if not refused:
        at = 0
        for r, (o, f) in enumerate(zip(old, new)):
            plan.starts[r] = at
            if f < 0:
                after[r] = 0
                continue
            for j in range(-(-o // ps), -(-(o + f) // ps)):
                pool.tables[r, j] = stack.pop()
            for i in range(f):
                pos = o + i
                page = int(pool.tables[r, pos // ps])
                plan.positions[at + i] = pos
                plan.slots[at + i] = page * ps + pos % ps if 0 <= page < pool.pages else -1
            at += f
            after[r] = o + f
        plan.starts[pool.rows] = at
        if len(stack) > n:
            pool.free[n:len(stack)] = torch.tensor(stack[n:], dtype=torch.int32)
        n = len(stack)
    plan.lengths.copy_(torch.tensor(after, dtype=torch.int32))
    plan.info.copy_(torch.tensor([n, refused], dtype=torch.int32))
    if commit:
        pool.state[0], pool.state[1] = n, refused


# ----------------------------------------------------------------------------------------------------------
# writing new tokens
# ----------------------------------------------------------------------------------------------------------
def _check_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, plan: PagePlan, like: torch.Tensor):
    if not (k_pages.dim() == 4 and k_pages.shape == v_pages.shape and k_pages.is_contiguous() and v_pages.is_contiguous() and k_pages.shape[1] == plan.page_size):
        raise ValueError("k_pages, v_pages: contiguous [pages, page_size, n_kv, d] tensors of the plan's page size are needed")
    device = like.device
    if not (k_pages.dtype == v_pages.dtype == like.dtype and k_pages.device == v_pages.device == device):
        raise ValueError("pages and tokens: one type, one device")
    pages, ps, n_kv, d = k_pages.shape
    if not (pages and n_kv and d):
        raise ValueError("pages without tokens, heads or columns")
    if torch.is_grad_enabled() and (like.requires_grad or k_pages.requires_grad or v_pages.requires_grad):
        raise RuntimeError("the paged operators have no backward pass: call them under torch.no_grad(), or with tensors that ask for no gradient")
    if (k_pages.data_ptr() | v_pages.data_ptr()) % 16:
        raise ValueError("k_pages, v_pages: they have to begin at a multiple of 16 bytes")
    if pages * ps > MAX_SLOTS:
        raise ValueError("slots have to stay below 2^31 - 256")
    if plan._good != (like.shape[0], device):
        _check_plan(plan, like.shape[0], device)
    return pages, ps, n_kv, d


def _check_plan(plan: PagePlan, T: int, device: torch.device) -> None:
    R, width = plan.tables.shape
    if width * plan.page_size > MAX_SLOTS or not 1 <= R <= MAX_ROWS:
        raise ValueError("a table reaches below 2^31 - 256 tokens and has up to 4096 rows")
    _ints(plan.tables, "plan.tables", (R, width), device)
    _ints(plan.lengths, "plan.lengths", (R,), device)
    _ints(plan.starts, "plan.starts", (R + 1,), device)
    _ints(plan.slots, "plan.slots", (T,), device)
    _ints(plan.positions, "plan.positions", (T,), device)
    plan.__dict__["_good"] = (T, device)


def _kernel_type(t: torch.Tensor, d: int) -> None:
    if t.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{t.dtype}: the paged kernels take bfloat16 and float32")
    if not 8 <= d <= 256 or d % 8:
        raise ValueError(f"heads of {d}: multiples of 8 up to 256")


def _rows_of(t: torch.Tensor) -> torch.Tensor:
    """A [T, heads, d] (or [T, width]) tensor as its kernel takes it: rows of contiguous heads, one behind the other, that start at multiples of 16 bytes.
    Any other one is copied."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t
        inner = t.stride(-1) == 1 and (t.dim() == 2 or t.shape[1] == 1 or t.stride(1) == t.shape[2])
        if inner and (t.shape[0] == 1 or t.stride(0) % 8 == 0 and t.stride(0) >= t.numel() // t.shape[0]):
            return t
    return t.clone(memory_format=torch.contiguous_format)   # (contiguous() would give back one that only starts off 16 bytes)


def paged_append(qkv: torch.Tensor, cos: Optional[torch.Tensor], sin: Optional[torch.Tensor], plan: PagePlan, k_pages: torch.Tensor, v_pages: torch.Tensor, n_q: int,
                 n_kv: int, d: int) -> torch.Tensor:
    """qkv [T, (n_q + 2 n_kv) d], the packed projection of a step's new tokens -> queries [T, n_q, d]; keys and values go to ``plan.slots``
    of ``k_pages`` / ``v_pages`` [pages, page_size, n_kv, d] (slot -1: nowhere).  Queries and keys are rotated at ``plan.positions`` with the
    tables ``cos`` / ``sin`` [max position, d / 2] fp32 (halves of a head, d a multiple of 16); with ``cos`` = ``None`` they are rotated already and the
    queries are a view of ``qkv``.  No two tokens of a step have the same slot (a plan's never have).  A slot outside the pages or a position behind the
    tables is reported by ``ops.check_status``, and nothing of that token is written.  For serving: tensors that
    ask for a gradient are refused."""
    T = qkv.shape[0]
    if qkv.dim() != 2 or qkv.shape[1] != (n_q + 2 * n_kv) * d:
        raise ValueError(f"qkv: [tokens, {(n_q + 2 * n_kv) * d}] is needed")
    pages, ps, hk, dk = _check_pages(k_pages, v_pages, plan, qkv)
    if (hk, dk) != (n_kv, d):
        raise ValueError(f"pages hold {hk} heads of {dk}, the projection {n_kv} of {d}")
    if cos is not None:
        _need(sin is not None and cos.shape == sin.shape and cos.dim() == 2 and cos.shape[1] == d // 2 and cos.dtype == sin.dtype == torch.float32
              and cos.is_contiguous() and sin.is_contiguous() and cos.device == sin.device == qkv.device and (d % 16 == 0 or not qkv.is_cuda and d % 2 == 0),
              "cos, sin: contiguous float32 tables [positions, d / 2] on the projection's device, d a multiple of 16")
        _need((cos.data_ptr() | sin.data_ptr()) % 16 == 0, "cos, sin: they have to begin at a multiple of 16 bytes")
    if not qkv.is_cuda:
        return _paged_append_reference(qkv, cos, sin, plan, k_pages, v_pages, n_q, n_kv, d)
    _kernel_type(qkv, d)
    src = _rows_of(qkv)
    q = torch.empty(T, n_q, d, dtype=qkv.dtype, device=qkv.device) if cos is not None else src[:, :n_q * d].unflatten(1, (n_q, d))
    if T == 0:
        return q
    device = qkv.device
    with _on(device):
        _lib.check(_fn("ats_paged_append")(
            _p(src), src.stride(0) if T > 1 else src.shape[1], _p(cos), _p(sin), 0 if cos is None else cos.shape[0], _p(plan.positions), _p(plan.slots), _p(q), _p(k_pages),
            _p(v_pages), T, n_q, n_kv, d, pages * ps, int(qkv.dtype == torch.float32), _p(_lib.status_tensor(device)), _stream(device)),
            "ats_paged_append")
    return q


def _paged_append_reference(qkv, cos, sin, plan, k_pages, v_pages, n_q, n_kv, d):
    T = qkv.shape[0]
    qk, v = qkv[:, :(n_q + n_kv) * d].reshape(T, n_q + n_kv, d), qkv[:, (n_q + n_kv) * d:].reshape(T, n_kv, d)
    if cos is not None:
        pos = plan.positions.long()
        if T and int(pos.max()) >= cos.shape[0]:
            raise ValueError(f"position {int(pos.max())} lies behind the rotary tables ({cos.shape[0]})")
        c, s = cos[pos][:, None], sin[pos][:, None]
        a, b = qk.float().chunk(2, -1)
        qk = torch.cat([a * c - b * s, b * c + a * s], -1).to(qkv.dtype)
    live = plan.slots >= 0
    slots = plan.slots[live].long()
    k_pages.view(-1, n_kv, d)[slots] = qk[live, n_q:]
    v_pages.view(-1, n_kv, d)[slots] = v[live]
    return qk[:, :n_q]


# ----------------------------------------------------------------------------------------------------------
# attention
# ----------------------------------------------------------------------------------------------------------
def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, plan: PagePlan, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """q [T, n_q, d], a step's queries (rotated; rows may be views of a wider projection) -> [T, n_q, d].  Token i of a row's new tokens attends to the
    row's tokens up to itself, in the pages of ``plan.tables``; its keys and values are there already.  ``scale`` (default 1 / sqrt(d)) times the scores.
    Tokens behind the last row come out as zeros, or keep what ``out`` holds where it is given (``q`` itself may be: answers replace their queries).  Heads of up to 256 dimensions (multiples of 8).
    A table entry outside the pool is reported by ``ops.check_status`` and nothing is read there (what its row gets has no meaning).  bf16: scores, statistics and sums in fp32, probabilities rounded to
    bf16 for their product with the values; fp32 in true 32-bit.  For serving: tensors that ask for a gradient are refused."""
    if q.dim() != 3:
        raise ValueError("q: [tokens, heads, d] is needed")
    pages, ps, n_kv, d = _check_pages(k_pages, v_pages, plan, q)
    T, n_q, d_q = q.shape
    if d_q != d or n_q < n_kv or n_q % n_kv:
        raise ValueError(f"{n_q} query heads of {d_q} over {n_kv} key heads of {d}")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    _need(scale > 0 and math.isfinite(scale), "scale: a positive number")
    if out is not None:
        _need(out.shape == q.shape and out.dtype == q.dtype and out.device == q.device and (T == 0 or _rows_of(out) is out) and (T < 2 or out.stride(0) >= n_q * d),
              "out: like q, rows of contiguous heads that start at multiples of 16 bytes and do not overlap")
    if not q.is_cuda:
        return _paged_attention_reference(q, k_pages, v_pages, plan, scale, out)
    _kernel_type(q, d)
    keep_tail = out is not None
    if out is None:
        out = torch.empty(T, n_q, d, dtype=q.dtype, device=q.device)
    if T == 0:
        return out
    q = _rows_of(q)
    ldq, ldo = (q.stride(0), out.stride(0)) if T > 1 else (n_q * d, n_q * d)
    R, width = plan.tables.shape
    rep, new, keys = n_q // n_kv, min(plan.max_new or T, T), min(plan.max_len or width * ps, width * ps)
    device = q.device
    status, stream = _p(_lib.status_tensor(device)), _stream(device)
    head = (_p(q), ldq, _p(k_pages), _p(v_pages), _p(plan.starts), _p(plan.lengths), _p(plan.tables), _p(out), ldo, T, R, n_q, n_kv, d, width, pages, ps)
    with _on(device):
        if q.dtype != torch.bfloat16 or d not in (64, 128) or ps < 8 or rep > 128 or (width * ps // 16 + 1) * R * n_kv >= 1 << 32:
            splits = _scratch("ats_paged_any_splits", T, n_q, n_kv, max(keys, 1))
            part = torch.empty(splits * T * n_q * (d + 2), dtype=torch.float32, device=device) if splits > 1 else None
            _lib.check(_fn("ats_paged_attn_any")(*head, scale, int(keep_tail), int(q.dtype == torch.float32), splits, _p(part), status, stream), "ats_paged_attn_any")
            return out
        # Rows of a few query rows (new tokens times heads of a group) are a stream of the cache, longer portions a matter of the tensor cores.  A batch may
        # hold both, and which is which the kernels find in the plan; the host only knows when there can be none of one kind.
        limit = 0 if rep > 16 else 8 if new * rep <= 8 or rep <= 8 < 16 < new * rep else 16
        portions = new * rep > limit
        if portions:
            scratch = torch.empty(_scratch("ats_paged_portion_scratch", d), dtype=torch.uint8, device=device)
            _lib.check(_fn("ats_paged_portion")(*head, limit, scale, int(not keep_tail), _p(scratch), status, stream), "ats_paged_portion")
        if limit:
            scratch = torch.empty(_scratch("ats_paged_decode_scratch", R, n_kv, d, keys, limit), dtype=torch.uint8, device=device)
            _lib.check(_fn("ats_paged_decode")(*head, keys, T if portions else new, limit, scale, int(not keep_tail and not portions), int(portions), _p(scratch), status, stream), "ats_paged_decode")
    return out


def _paged_attention_reference(q, k_pages, v_pages, plan, scale, out):
    T, n_q, d = q.shape
    n_kv, ps = k_pages.shape[2], plan.page_size
    if out is None:
        out = torch.zeros_like(q, memory_format=torch.contiguous_format)
    starts, lengths = plan.starts.tolist(), plan.lengths.tolist()
    rep = n_q // n_kv
    for r, total in enumerate(lengths):
        a, b = starts[r], starts[r + 1]
        if a == b:
            continue
        table = plan.tables[r, :-(-total // ps)].long()
        k = k_pages[table].reshape(-1, n_kv, d)[:total].float().repeat_interleave(rep, 1)
        v = v_pages[table].reshape(-1, n_kv, d)[:total].float().repeat_interleave(rep, 1)
        s = torch.einsum("qhd,khd->hqk", q[a:b].float() * scale, k)
        seen = torch.arange(total, device=q.device)[None] <= torch.arange(total - (b - a), total, device=q.device)[:, None]
        out[a:b] = torch.einsum("hqk,khd->qhd", torch.softmax(s.masked_fill(~seen, float("-inf")), -1), v).to(q.dtype)
    return out
