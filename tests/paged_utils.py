"""Plain 64-bit forms that the tests of the paged operators compare with, and the plans they run on."""
import torch

from adaptivetrainingsystem_b200 import ops


def make_plan(old, new, page, device, extra_pages=3, tail=0, seed=0, width=None):
    """A step over rows holding ``old`` tokens that get ``new`` ones, on pages in random order; ``tail`` packed rows belong to no row.
    -> (plan, number of pages)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-(o + n) // page) for o, n in zip(old, new)]
    pages = sum(need) + extra_pages
    order = torch.randperm(pages, generator=g)
    width = width or max(max(need), 1)
    tables = torch.full((len(old), width), 2 ** 31 - 1, dtype=torch.int32)   # entries that no token needs are never followed
    at, slots, positions, starts = 0, [], [], [0]
    for r, (o, n) in enumerate(zip(old, new)):
        tables[r, :need[r]] = order[at:at + need[r]].int()
        at += need[r]
        for p in range(o, o + n):
            positions.append(p)
            slots.append(int(tables[r, p // page]) * page + p % page)
        starts.append(starts[-1] + n)
    i32 = dict(dtype=torch.int32, device=device)
    return ops.PagePlan(torch.tensor(starts, **i32), torch.tensor(slots + [-1] * tail, **i32), torch.tensor(positions + [0] * tail, **i32),
                        torch.tensor([o + n for o, n in zip(old, new)], **i32), tables.to(device), page), pages


def rows_of_pages(pages, plan, r):
    """The tokens of row r, [tokens, n_kv, d]."""
    n, ps = int(plan.lengths[r]), plan.page_size
    table = plan.tables[r, :-(-n // ps)].long()
    return pages[table].flatten(0, 1)[:n]


def attend64(q, k_pages, v_pages, plan, scale):
    """-> (outputs, the same with |v|) in 64 bits; rows of the batch that belong to no row are zero."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mass = torch.zeros_like(out)
    starts = plan.starts.tolist()
    rep = q.shape[1] // k_pages.shape[2]
    for r in range(len(starts) - 1):
        a, b = starts[r], starts[r + 1]
        if a == b:
            continue
        k = rows_of_pages(k_pages, plan, r).double().repeat_interleave(rep, 1)
        v = rows_of_pages(v_pages, plan, r).double().repeat_interleave(rep, 1)
        n = k.shape[0]
        s = torch.einsum("qhd,khd->hqk", q[a:b].double() * scale, k)
        hidden = torch.arange(n, device=q.device)[None] > torch.arange(n - (b - a), n, device=q.device)[:, None]
        p = torch.softmax(s.masked_fill(hidden, float("-inf")), -1)
        out[a:b] = torch.einsum("hqk,khd->qhd", p, v)
        mass[a:b] = torch.einsum("hqk,khd->qhd", p, v.abs())
    return out, mass


def sample64(logits, u, temperature, top_k, top_p, min_p, penalty, history):
    """One row at a time, the rules as they are written down."""
    out = []
    for r in range(logits.shape[0]):
        x = logits[r].float()
        ids = history[r][(history[r] >= 0) & (history[r] < x.numel())].unique() if history is not None else torch.zeros(0, dtype=torch.long)
        if penalty[r] != 1:
            x[ids] = torch.where(x[ids] > 0, x[ids] / penalty[r].to(x.device), x[ids] * penalty[r].to(x.device))
        x = torch.where(torch.isnan(x), float("-inf"), x)
        if not temperature[r] > 0 or bool((x == float("-inf")).all()):
            out.append(int((x == x.max()).nonzero()[0]))
            continue
        value, token = torch.sort(x.double(), descending=True, stable=True)
        if top_k[r] > 0:
            value, token = value[:int(top_k[r])], token[:int(top_k[r])]
        gap = torch.where(value == value[0], 0.0, value - value[0])
        mass = torch.where(torch.isinf(gap), gap, gap / float(temperature[r])).exp()      # (an infinite gap is one at an infinite temperature too)
        ahead = mass.cumsum(0) - mass
        keep = (ahead <= max(float(top_p[r]), 0.0) * mass.sum()) & (mass >= min(float(min_p[r]), 1.0))
        mass, token = mass[keep], token[keep]
        token, back = token.sort()
        cdf = mass[back].cumsum(0)
        pick = int((cdf <= max(float(u[r]), 0.0) * cdf[-1]).sum())
        live = (mass[back] > 0).nonzero()[-1]
        out.append(int(token[min(pick, int(live))]))
    return torch.tensor(out)
