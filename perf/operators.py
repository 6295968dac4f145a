"""Cases for the operators that serve sequences from a paged key / value cache.

* ``plan``: page tables and the slots of a step's new tokens from the rows' lengths (``ops.page_plan``);
* ``append``: rotary embedding of queries and keys, keys and values into their pages (``ops.paged_append``);
* ``attend``: causal grouped-query attention of the new tokens over the pages, single tokens, portions of prompts or both in one batch
  (``ops.paged_attention``);
* ``sample``: the next token of every row from given random numbers, each row with its own sampling numbers (``ops.sample_rows``).

Head counts and widths are those of the ``dense_1b`` and ``mixtral_8x7b`` presets (32 / 4 heads of 64, 32 / 8 of 128), sampling numbers
those of the generation modes.  A case describes its rows by ranges; the lengths themselves come from the case alone (a fixed generator),
so that the work of a case does not change with the seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False

ROPE_THETA = 10000.0


def listed():
    return [
        # the step of a decoding batch: every row gets one token, now and then a page
        dict(name="plan_decode", kind="plan", rows=64, old_min=200, old_max=2000, new_min=1, new_max=1, closed=0.0, page=64),
        # a batcher that retires, admits and decodes at once: portions of prompts beside single tokens
        dict(name="plan_mixed", kind="plan", rows=500, old_min=0, old_max=4000, new_min=1, new_max=65, closed=0.1, page=16),
        # one token of each of 64 sequences
        dict(name="append_decode", kind="append", rows=64, old_min=200, old_max=2000, new_min=1, new_max=1, page=64, heads=32, kv_heads=4, dim=64),
        # prompts of several requests in one packed batch
        dict(name="append_prompts", kind="append", rows=9, old_min=0, old_max=0, new_min=500, new_max=1400, page=32, heads=32, kv_heads=8, dim=128),
        # interactive generation, one sequence: latency
        dict(name="attend_one", kind="attend", rows=1, old_min=511, old_max=511, new_min=1, new_max=1, page=64, heads=32, kv_heads=4, dim=64),
        # a serving batch on the 64-wide heads
        dict(name="attend_decode", kind="attend", rows=64, old_min=200, old_max=2000, new_min=1, new_max=1, page=64, heads=32, kv_heads=4, dim=64),
        # few long conversations on the 128-wide heads, four tokens proposed for each
        dict(name="attend_drafts", kind="attend", rows=8, old_min=5000, old_max=31000, new_min=4, new_max=4, page=16, heads=32, kv_heads=8, dim=128),
        # prompts of several requests in one packed batch, no row a multiple of any tile
        dict(name="attend_prompts", kind="attend", rows=6, old_min=0, old_max=0, new_min=300, new_max=2500, page=32, heads=32, kv_heads=8, dim=128),
        # the next portion of a long prompt beside rows that decode
        dict(name="attend_portion", kind="attend", rows=33, old_min=300, old_max=3000, new_min=1, new_max=1, page=64, heads=32, kv_heads=8, dim=128, portion=1000, before=15000),
        # a few requests of a small vocabulary
        dict(name="sample_few", kind="sample", rows=4, vocab=32000, dtype="bf16", truncated=True),
        # a serving batch whose requests all truncate, odd vocabulary
        dict(name="sample_batch", kind="sample", rows=64, vocab=100003, dtype="fp32", truncated=True),
        # a large batch; some rows cut by top-p alone, some not at all
        dict(name="sample_large", kind="sample", rows=256, vocab=131072, dtype="bf16", truncated=False),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["plan", "append", "attend", "attend", "attend", "sample", "sample"])
    page = rng.choice([16, 32, 64, 128])
    if kind == "plan":
        top = log(1, 64)
        return dict(kind=kind, rows=log(1, 500), old_min=0, old_max=log(1, 4000), new_min=rng.choice([0, 1]), new_max=top, closed=rng.choice([0.0, 0.1, 0.3]), page=page)
    heads, kv_heads, dim = rng.choice([(32, 4, 64), (32, 8, 128), (16, 4, 64), (16, 2, 128), (12, 4, 128), (16, 16, 64)])
    shape = dict(page=page, heads=heads, kv_heads=kv_heads, dim=dim)
    if kind == "append":
        if rng.random() < 0.5:
            return dict(kind=kind, rows=log(1, 256), old_min=0, old_max=log(1, 4000), new_min=1, new_max=1, **shape)
        rows = log(1, 16)
        return dict(kind=kind, rows=rows, old_min=0, old_max=log(1, 2000), new_min=1, new_max=max(1, log(8, 8000) // rows), **shape)
    if kind == "attend":
        form = rng.choice(["decode", "drafts", "prompts", "portion"])
        if form == "decode":
            rows = log(1, 128)
            return dict(kind=kind, rows=rows, old_min=0, old_max=log(30, min(60000, 150000 // rows)), new_min=1, new_max=1, **shape)
        if form == "drafts":
            rows = log(1, 32)
            return dict(kind=kind, rows=rows, old_min=0, old_max=log(30, min(30000, 150000 // rows)), new_min=1, new_max=rng.randint(2, 8), **shape)
        if form == "prompts":
            rows = log(1, 12)
            return dict(kind=kind, rows=rows, old_min=0, old_max=rng.choice([0, log(10, 2000)]), new_min=1, new_max=max(2, log(20, 7000) // rows), **shape)
        return dict(kind=kind, rows=log(1, 32), old_min=0, old_max=log(30, 3000), new_min=1, new_max=1, portion=log(20, 1000), before=log(100, 15000), **shape)
    return dict(kind=kind, rows=log(1, 256), vocab=rng.choice([32000, 50257, log(2000, 131072)]), dtype=rng.choice(["bf16", "fp32"]),
                truncated=rng.random() < 0.5)


def _lengths(case):
    """(tokens held, tokens to come) of every row; -1 closes a row."""
    g = random.Random(str(sorted((k, str(v)) for k, v in case.items() if k != "name")))
    old = [g.randint(case["old_min"], case["old_max"]) for _ in range(case["rows"])]
    new = [g.randint(case["new_min"], case["new_max"]) for _ in range(case["rows"])]
    if case.get("closed"):
        new = [-1 if g.random() < case["closed"] else n for n in new]
    if case.get("portion"):
        old[0], new[0] = case["before"], case["portion"]
    return old, new


def _pages_of(tokens, page):
    return (tokens + page - 1) // page


# ------------------------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    if case["kind"] == "sample":
        return _prepare_sample(case, seed, dev, g)
    old, new = _lengths(case)
    page, R = case["page"], case["rows"]
    held = [_pages_of(o, page) for o in old]
    after = [_pages_of(o + max(n, 0), page) for o, n in zip(old, new)]
    pages = sum(after) + R + 8
    width = max(after) + 1
    # pages handed out in no order, as in a pool that has served for a while
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    if case["kind"] == "plan":
        tables = torch.zeros(R, width, dtype=torch.int32, device=dev)
        at = 0
        for r, n in enumerate(held):
            tables[r, :n] = order[at:at + n]
            at += n
        free = torch.zeros(pages, dtype=torch.int32, device=dev)
        free[:pages - at] = order[at:]
        st = dict(case=case, old=torch.tensor(old, dtype=torch.int32, device=dev), new=torch.tensor(new, dtype=torch.int32, device=dev), tables=tables, free=free,
                  count=pages - at, page=page, tokens=sum(max(n, 0) for n in new))
        if own:
            from adaptivetrainingsystem_b200 import ops
            pool = ops.PagePool(R, width * page, pages, page, device=dev)
            pool.tables.copy_(tables)
            pool.free.copy_(free)
            pool.lengths.copy_(st["old"])
            pool.state[0] = st["count"]
            st["pool"] = pool
        return st
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    T = sum(new)
    tables = torch.zeros(R, width, dtype=torch.int32, device=dev)
    slots, positions, at = [], [], 0
    for r in range(R):
        tables[r, :after[r]] = order[at:at + after[r]]
        at += after[r]
        pos = torch.arange(old[r], old[r] + new[r], device=dev)
        positions.append(pos)
        slots.append(tables[r].long()[pos // page] * page + pos % page)
    starts = torch.tensor([sum(new[:r]) for r in range(R + 1)], dtype=torch.int32, device=dev)
    lengths = torch.tensor([o + n for o, n in zip(old, new)], dtype=torch.int32, device=dev)
    st = dict(case=case, old=old, new=new, tables=tables, starts=starts, lengths=lengths, slots=torch.cat(slots).to(torch.int32),
              positions=torch.cat(positions).to(torch.int32), pages=pages)
    st["k"] = torch.randn(pages, page, hk, d, generator=g, device=dev).bfloat16()
    st["v"] = torch.randn(pages, page, hk, d, generator=g, device=dev).bfloat16()
    if case["kind"] == "append":
        st["qkv"] = torch.randn(T, (hq + 2 * hk) * d, generator=g, device=dev).bfloat16()
        angle = torch.arange(max(o + n for o, n in zip(old, new)) + 1, device=dev).double()[:, None] * ROPE_THETA ** (
            -torch.arange(0, d, 2, device=dev).double() / d)
        st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
    else:
        # normed queries and keys: scores of a few units, as trained heads have them
        st["q"] = (1.5 * torch.randn(T, hq, d, generator=g, device=dev)).bfloat16()
    if own:
        from adaptivetrainingsystem_b200 import ops
        st["plan"] = ops.PagePlan(starts=starts, slots=st["slots"], positions=st["positions"], lengths=lengths, tables=tables, page_size=page,
                                  max_new=max(new), max_len=max(o + n for o, n in zip(old, new)))
    return st


def _prepare_sample(case, seed, dev, g):
    R, V = case["rows"], case["vocab"]
    x = 2.2 * torch.randn(R, V, generator=g, device=dev)
    # a handful of likely tokens per row, from very sure to undecided
    likely = torch.randint(0, V, (R, 24), generator=g, device=dev)
    x.scatter_add_(1, likely, 4.0 + 8.0 * torch.rand(R, 24, generator=g, device=dev) * torch.rand(R, 1, generator=g, device=dev))
    rng = random.Random(seed)
    modes = [(0.8, 50, 0.9, 0.0, 1.1), (1.0, 100, 0.95, 0.0, 1.05), (0.3, 20, 0.7, 0.0, 1.2), (0.0, 0, 1.0, 0.0, 1.0), (1.2, 0, 1.0, 0.05, 1.0), (0.5, 40, 0.8, 0.02, 1.15)]
    if not case["truncated"]:
        modes += [(0.7, 0, 0.9, 0.0, 1.0), (1.0, 0, 0.98, 0.0, 1.1), (1.0, 0, 1.0, 0.0, 1.0), (0.9, 1000, 0.95, 0.0, 1.0)]
    rows = [modes[rng.randrange(len(modes))] for _ in range(R)]
    col = lambda i, t: torch.tensor([r[i] for r in rows], dtype=t, device=dev)  # noqa: E731
    return dict(case=case, logits=x.bfloat16() if case["dtype"] == "bf16" else x, uniform=torch.rand(R, generator=g, device=dev), temperature=col(0, torch.float32),
                top_k=col(1, torch.int32), top_p=col(2, torch.float32), min_p=col(3, torch.float32), penalty=col(4, torch.float32),
                history=torch.randint(0, V, (R, 50), generator=g, device=dev))


# ------------------------------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------------------------------
def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        from adaptivetrainingsystem_b200 import ops
        if kind == "plan":
            p = ops.page_plan(st["pool"], st["new"], st["tokens"], commit=False)
            return dict(starts=p.starts, slots=p.slots, positions=p.positions, lengths=p.lengths, tables=p.tables, free=st["pool"].free, count=p.count)
        if kind == "append":
            q = ops.paged_append(st["qkv"], st["cos"], st["sin"], st["plan"], st["k"], st["v"], case["heads"], case["kv_heads"], case["dim"])
            return dict(q=q, k=st["k"], v=st["v"])
        if kind == "attend":
            return ops.paged_attention(st["q"], st["k"], st["v"], st["plan"])
        return ops.sample_rows(st["logits"], st["uniform"], st["temperature"], st["top_k"], st["top_p"], st["min_p"], st["penalty"], st["history"])
    if kind == "plan":
        return _plan(st)
    if kind == "append":
        return _append(st)
    if kind == "attend":
        return _attend(st)
    return _sample(st["logits"], st)


def _plan(st):
    old, page, T = st["old"].long(), st["page"], st["tokens"]
    new = st["new"].long()
    dev = old.device
    add = new.clamp(min=0)
    starts = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), add.cumsum(0)])
    held = (old + page - 1) // page
    need = torch.where(new < 0, torch.zeros_like(held), (old + add + page - 1) // page - held)
    freed = torch.where(new < 0, held, torch.zeros_like(held))
    tables, free = st["tables"].clone(), st["free"].clone()
    n = st["count"]
    col = torch.arange(tables.shape[1], device=dev)[None]
    stack = torch.cat([free[:n], tables[col < freed[:, None]]])          # row by row, page by page
    grow = (col >= held[:, None]) & (col < (held + need)[:, None])
    taken = grow.sum()
    tables[grow] = stack.flip(0)[:grow.sum()]
    count = stack.numel() - taken
    at = torch.arange(free.numel(), device=dev)
    free = torch.where((at >= n) & (at < count), torch.cat([stack, free])[:free.numel()], free)
    row = torch.repeat_interleave(torch.arange(old.numel(), device=dev), add, output_size=T)
    pos = old[row] + torch.arange(T, device=dev) - starts[row]
    slots = tables.long()[row, pos // page] * page + pos % page
    i32 = torch.int32
    return dict(starts=starts.to(i32), slots=slots.to(i32), positions=pos.to(i32), lengths=torch.where(new < 0, 0, old + add).to(i32), tables=tables, free=free,
                count=count.to(i32).reshape(1))


def _append(st):
    case = st["case"]
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    qkv, T = st["qkv"], st["qkv"].shape[0]
    qk = qkv[:, :(hq + hk) * d].view(T, hq + hk, d).float()
    pos = st["positions"].long()
    c, s = st["cos"][pos][:, None], st["sin"][pos][:, None]
    u, w = qk[..., :d // 2], qk[..., d // 2:]
    qk = torch.cat([u * c - w * s, w * c + u * s], -1).to(qkv.dtype)
    slots = st["slots"].long()
    st["k"].view(-1, hk, d)[slots] = qk[:, hq:]
    st["v"].view(-1, hk, d)[slots] = qkv[:, (hq + hk) * d:].view(T, hk, d)
    return dict(q=qk[:, :hq].contiguous(), k=st["k"], v=st["v"])


def _attend(st):
    case = st["case"]
    hk, d, page = case["kv_heads"], case["dim"], case["page"]
    rep = case["heads"] // hk
    out, at = [], 0
    for r, (o, n) in enumerate(zip(st["old"], st["new"])):
        total = o + n
        table = st["tables"][r, :_pages_of(total, page)].long()
        q = st["q"][at:at + n].float().view(n, hk, rep, d) / math.sqrt(d)
        seen = torch.arange(total, device=q.device)[None] <= torch.arange(o, total, device=q.device)[:, None]
        heads = []
        for h in range(hk):   # one key head at a time: the scores of all of them need not fit
            k = st["k"][table, :, h].reshape(-1, d)[:total].float()
            v = st["v"][table, :, h].reshape(-1, d)[:total].float()
            s = (q[:, h].reshape(n * rep, d) @ k.t()).view(n, rep, total).masked_fill(~seen[:, None], float("-inf"))
            p = (s - s.amax(-1, keepdim=True)).exp()
            heads.append((p.view(n * rep, total) @ v).view(n, rep, d) / p.sum(-1, keepdim=True))
        out.append(torch.stack(heads, 1).reshape(n, hk * rep, d).to(st["q"].dtype))
        at += n
    return torch.cat(out)


def _sample(logits, st):
    """64 bits from the scores on: a random number may lie next to a border."""
    R, V = logits.shape
    x = logits.float()
    seen = torch.zeros(R, V, dtype=torch.bool, device=x.device).scatter_(1, st["history"], True)
    pen = st["penalty"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / pen, x * pen), x)
    greedy = x.argmax(-1)
    t = torch.where(st["temperature"] > 0, st["temperature"], torch.ones_like(st["temperature"])).double()[:, None]
    top = x.amax(-1, keepdim=True).double()
    order = x.argsort(dim=-1, descending=True, stable=True)
    e = ((x.double() - top) / t).exp()
    se = e.gather(1, order)
    k = torch.where(st["top_k"] > 0, st["top_k"], V)[:, None]
    se = torch.where(torch.arange(V, device=x.device)[None] < k, se, 0.0)
    before = se.cumsum(-1) - se
    keep = (before <= st["top_p"].double()[:, None] * se.sum(-1, keepdim=True)) & (se >= st["min_p"].double()[:, None])
    e = torch.zeros_like(e).scatter_(1, order, torch.where(keep, se, 0.0))
    cdf = e.cumsum(-1)
    pick = (cdf <= st["uniform"].double()[:, None] * cdf[:, -1:]).sum(-1)
    return torch.where(st["temperature"] > 0, pick, greedy)


# ------------------------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "sample":
        R, V = case["rows"], case["vocab"]
        return {"bytes": R * V * (2 if case["dtype"] == "bf16" else 4) + R * (50 * 8 + 24 + 8), "flops": 4 * R * V}
    old, new = _lengths(case)
    page, R = case["page"], case["rows"]
    T = sum(max(n, 0) for n in new)
    if case["kind"] == "plan":
        touched = sum(_pages_of(o + n, page) - o // page for o, n in zip(old, new) if n > 0) + sum(_pages_of(o, page) for o, n in zip(old, new) if n < 0)
        return {"bytes": 16 * R + 8 * T + 8 * touched, "flops": 4 * T}
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "append":
        return {"bytes": T * (hq + 2 * hk) * d * 4 + T * (4 * d + 8), "flops": 3 * T * (hq + hk) * d}
    pairs = sum(n * o + n * (n + 1) // 2 for o, n in zip(old, new))
    return {"bytes": 4 * T * hq * d + 4 * sum(o + n for o, n in zip(old, new)) * hk * d, "flops": 4 * d * hq * pairs}


# ------------------------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    kind = case["kind"]
    if kind == "plan":
        return None   # whole numbers only
    st = prepare(case, seed)
    if kind == "sample":
        return _exact_sample(st)
    hq, hk, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    if kind == "append":
        T = st["qkv"].shape[0]
        parts = st["qkv"].double().view(T, hq + 2 * hk, d)
        z = torch.complex(parts[:, :hq + hk, :d // 2], parts[:, :hq + hk, d // 2:])
        turn = torch.complex(st["cos"].double(), st["sin"].double())[st["positions"].long()]
        z = z * turn[:, None]
        qk = torch.cat([z.real, z.imag], -1)
        k, v = st["k"].double().flatten(0, 1), st["v"].double().flatten(0, 1)
        k[st["slots"].long()] = qk[:, hq:]
        v[st["slots"].long()] = parts[:, hq + hk:]
        return dict(q=qk[:, :hq], k=k.view(st["k"].shape), v=v.view(st["v"].shape))
    rows, first = [], 0
    for r, n in enumerate(st["new"]):
        total = st["old"][r] + n
        at = torch.arange(total, device=st["q"].device)
        where = st["tables"][r].long()[at // page] * page + at % page
        k, v = st["k"].flatten(0, 1)[where].double(), st["v"].flatten(0, 1)[where].double()      # [total, hk, d]
        o = torch.empty(n, hq, d, dtype=torch.float64, device=k.device)
        for i in range(0, n, 512):
            m = min(512, n - i)
            upto = st["old"][r] + i + m
            future = at[None, :upto] > (st["old"][r] + i + torch.arange(m, device=k.device))[:, None]
            for h in range(hq):
                s = st["q"][first + i:first + i + m, h].double() @ k[:upto, h // (hq // hk)].T * d ** -0.5
                s[future] = -math.inf
                o[i:i + m, h] = torch.softmax(s, -1) @ v[:upto, h // (hq // hk)]
        rows.append(o)
        first += n
    return torch.cat(rows)


def _exact_sample(st):
    """Row by row: the tokens in order of their scores, cut one rule after the other."""
    out = []
    for r in range(st["logits"].shape[0]):
        x = st["logits"][r].float()
        t, k, p, low, pen = (float(st[n][r]) for n in ("temperature", "top_k", "top_p", "min_p", "penalty"))
        ids = st["history"][r].unique()
        x[ids] = torch.where(x[ids] > 0, x[ids] / st["penalty"][r], x[ids] * st["penalty"][r])
        if t <= 0:
            out.append(x.argmax())
            continue
        value, token = torch.sort(x.double(), descending=True, stable=True)
        if k > 0:
            value, token = value[:int(k)], token[:int(k)]
        mass = torch.exp((value - value[0]) / t)
        ahead = torch.cumsum(mass, 0) - mass
        mass = mass[(ahead <= p * mass.sum()) & (mass >= low)]   # (both rules hold for a leading run)
        token, back = token[:mass.numel()].sort()
        cdf = torch.cumsum(mass[back], 0)
        out.append(token[torch.searchsorted(cdf, st["uniform"][r].double() * cdf[-1], right=True)])
    return torch.stack(out)
