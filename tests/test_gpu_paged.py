"""The paged cache's kernels against 64-bit forms of the same operators."""
import math
import random

import pytest
import torch

from adaptivetrainingsystem_b200 import ops
from paged_utils import attend64, make_plan, sample64

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ plan
def _pools(rows, max_len, pages, page):
    return [ops.PagePool(rows, max_len, pages, page, device=d) for d in ("cpu", "cuda")]


def _same(a, b, plan_a, plan_b):
    for name in ("starts", "slots", "positions", "lengths", "info"):
        assert torch.equal(getattr(plan_a, name), getattr(plan_b, name).cpu()), name
    n = int(a.state[0])
    assert torch.equal(a.free[:n], b.free[:n].cpu()) and torch.equal(a.lengths, b.lengths.cpu()) and a.state[:2].tolist() == b.state[:2].tolist()
    for r in range(a.rows):
        j = a.pages_for(int(a.lengths[r]))
        assert torch.equal(a.tables[r, :j], b.tables[r, :j].cpu())


@pytest.mark.parametrize("rows,max_len,page,longest", [(1, 40, 1, 3), (7, 200, 16, 40), (300, 500, 64, 90), (513, 64, 8, 9)])
def test_plan_equals_its_definition(rows, max_len, page, longest):
    g = random.Random(rows)
    a, b = _pools(rows, max_len, rows * -(-max_len // page) * 3 // 4 + 2, page)
    for step in range(8):
        lengths = a.lengths.tolist()
        fresh = [-1 if n and g.random() < 0.2 else min(g.choice([0, 1, g.randint(1, longest)]), max_len - n) for n in lengths]
        T = sum(max(f, 0) for f in fresh) + g.choice([0, 0, 5])
        f = torch.tensor(fresh, dtype=torch.int32)
        commit = step % 3 != 2
        _same(a, b, ops.page_plan(a, f, T, commit=commit), ops.page_plan(b, f.cuda(), T, commit=commit))


def test_plan_many_rows_long_batch_and_refusals():
    a, b = _pools(4096, 4096, 9000, 64)
    f = torch.randint(0, 100, (4096,), generator=torch.Generator().manual_seed(1)).int()
    _same(a, b, ops.page_plan(a, f, 1 << 18), ops.page_plan(b, f.cuda(), 1 << 18))
    a, b = _pools(3, 32, 5, 8)
    for fresh, T in (((17, 8, 0), 25), ((8, 1, 1), 10), ((16, 0, 0), 16), ((1, 1, 0), 1), ((-2, 0, 0), 4), ((0, 0, 0), 0), ((-1, 1, 8), 9), ((-1, -1, -1), 0), ((2 ** 31 - 1, 2 ** 31 - 1, 1), 3)):
        f = torch.tensor(fresh, dtype=torch.int32)
        for commit in (False, True):
            _same(a, b, ops.page_plan(a, f, T, commit=commit), ops.page_plan(b, f.cuda(), T, commit=commit))


def test_plan_replayed_from_a_graph():
    a, b = _pools(6, 100, 40, 4)
    fresh = torch.zeros(6, dtype=torch.int32, device="cuda")
    ops.page_plan(b, fresh, 6)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = ops.page_plan(b, fresh, 6)
    g = random.Random(0)
    for _ in range(50):
        f = [-1 if n and g.random() < 0.05 else int(n < 100 and g.random() < 0.8) for n in a.lengths.tolist()]
        fresh.copy_(torch.tensor(f))
        graph.replay()
        _same(a, b, ops.page_plan(a, torch.tensor(f, dtype=torch.int32), 6), plan)


# ------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n_q,n_kv,d,page,strided", [(32, 4, 64, 64, False), (4, 4, 128, 16, True), (6, 2, 96, 8, False), (3, 1, 16, 1, True), (8, 1, 256, 32, False)])
def test_append(dtype, n_q, n_kv, d, page, strided):
    old, new = [0, 70, 3, 1000, 12], [5, 1, 0, 17, 2]
    plan, pages = make_plan(old, new, page, "cuda", tail=3)
    g = torch.Generator(device="cuda").manual_seed(d)
    T, width = plan.slots.numel(), (n_q + 2 * n_kv) * d
    qkv = torch.randn(T, width + 24, generator=g, device="cuda").to(dtype)[:, 8:width + 8] if strided else torch.randn(T, width, generator=g, device="cuda").to(dtype)
    k, v = (torch.randn(pages, page, n_kv, d, generator=g, device="cuda").to(dtype) for _ in range(2))
    cos, sin = ops.rope_tables(1100, d, 10000.0, device="cuda")
    k0, v0 = k.clone(), v.clone()
    parts = qkv.double().view(T, n_q + 2 * n_kv, d)
    c, s = (t[plan.positions.long()].double()[:, None] for t in (cos, sin))
    x, y = parts[:, :n_q + n_kv].chunk(2, -1)
    turned = torch.cat([x * c - y * s, y * c + x * s], -1)
    # three fp32 roundings on either product, then the one to the type
    bound = 4 * 2.0 ** -24 * torch.cat([(x * c).abs() + (y * s).abs(), (y * c).abs() + (x * s).abs()], -1) + torch.finfo(dtype).eps / 2 * turned.abs()
    q = ops.paged_append(qkv, cos, sin, plan, k, v, n_q, n_kv, d)
    assert ((q.double() - turned[:, :n_q]).abs() <= bound[:, :n_q]).all()
    slots = plan.slots[:-3].long()
    got = k.view(-1, n_kv, d)[slots].double()
    assert ((got - turned[:-3, n_q:]).abs() <= bound[:-3, n_q:]).all()
    assert torch.equal(v.view(-1, n_kv, d)[slots], qkv.view(T, -1, d)[:-3, n_q + n_kv:])
    rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    rest[slots] = False
    assert torch.equal(k.view(-1, n_kv, d)[rest], k0.view(-1, n_kv, d)[rest]) and torch.equal(v.view(-1, n_kv, d)[rest], v0.view(-1, n_kv, d)[rest])
    # rotated already: keys and values as they are
    q = ops.paged_append(qkv, None, None, plan, k, v, n_q, n_kv, d)
    assert torch.equal(q, qkv.view(T, -1, d)[:, :n_q]) and torch.equal(k.view(-1, n_kv, d)[slots], qkv.view(T, -1, d)[:-3, n_q:n_q + n_kv])


def test_append_reports_positions_behind_the_tables():
    plan, pages = make_plan([30], [4], 16, "cuda")
    k = torch.zeros(pages, 16, 1, 16, device="cuda")
    cos, sin = ops.rope_tables(32, 16, 10000.0, device="cuda")
    ops.paged_append(torch.ones(4, 48, device="cuda"), cos, sin, plan, k, k.clone(), 1, 1, 16)
    with pytest.raises(ops.KernelError, match="bad argument"):
        ops.check_status()
    assert int((k != 0).any(-1).sum()) == 2


# ------------------------------------------------------------------------------------------------ attention
def _attention_bound(dtype, ref, mass, n, d):
    """bf16: probabilities rounded for the second product (half a step of their weighted values; their sum is taken before) and the output rounded
    once; the approximate exponential and fp32 sums stay below half of the first.  fp32: products of d terms in front of the exponential (scores
    of up to 32, so 32 d of relative error at most, d / 8 as it grows with the root), sums of n."""
    if dtype == torch.bfloat16:
        return 1.5 * 2.0 ** -8 * mass + 2.0 ** -8 * ref.abs() + 1e-6
    return 2.0 ** -24 * (32 * math.sqrt(d) + math.sqrt(n) + 64) * mass + 1e-7


def _attend_case(old, new, page, n_q, n_kv, d, dtype, tail=0, seed=0, hints=True, strided=False, scale=None):
    plan, pages = make_plan(old, new, page, "cuda", tail=tail, seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed + d)
    k, v = (torch.randn(pages, page, n_kv, d, generator=g, device="cuda").to(dtype) for _ in range(2))
    used = torch.zeros(pages * page, dtype=torch.bool)
    for r, n in enumerate(plan.lengths.tolist()):
        at = torch.arange(n)
        used[plan.tables[r].cpu().long()[at // page] * page + at % page] = True
    for t in (k, v):   # what other rows or earlier generations left in the pages is never used
        t.view(-1, n_kv, d)[~used.cuda()] = float("nan")
    T = sum(new) + tail
    q = torch.randn(T, n_q * d + (16 if strided else 0), generator=g, device="cuda").to(dtype)
    q = (q[:, 8:8 + n_q * d] if strided else q).unflatten(1, (n_q, d))
    if hints:
        plan.max_new, plan.max_len = max(new), max(o + n for o, n in zip(old, new))
    s = 1 / math.sqrt(d) if scale is None else scale
    ref, mass = attend64(q, k, v, plan, s)
    out = ops.paged_attention(q, k, v, plan, scale=scale)
    bound = _attention_bound(dtype, ref, mass, max(o + n for o, n in zip(old, new)), d)
    err = (out.double() - ref).abs()
    assert bool((err <= bound).all()), (float((err / bound).max()), (err > bound).nonzero()[:4].tolist())
    kept = torch.full_like(out, 7.0)
    ops.paged_attention(q, k, v, plan, scale=scale, out=kept)
    assert torch.equal(kept[:sum(new)], out[:sum(new)]) and (kept[sum(new):] == 7).all() and (out[sum(new):] == 0).all()


HEADS = [(8, 8, 64), (8, 4, 64), (12, 4, 128), (32, 4, 64), (32, 8, 128), (16, 1, 128), (5, 1, 64), (14, 2, 128), (20, 1, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n_q,n_kv,d", HEADS + [(4, 2, 96), (2, 2, 8), (6, 2, 256), (3, 1, 40)])
@pytest.mark.parametrize("page", [1, 16, 128])
def test_attention_single_tokens(n_q, n_kv, d, page, dtype):
    _attend_case([0, 1, 15, 16, 31, 63, 64, 127, 300, 5], [1, 1, 1, 1, 1, 1, 1, 1, 1, 0], page, n_q, n_kv, d, dtype, tail=2, strided=True)


@pytest.mark.parametrize("n_q,n_kv,d", HEADS)
@pytest.mark.parametrize("page", [8, 16, 32, 64, 256])
@pytest.mark.parametrize("hints", [True, False])
def test_attention_a_few_tokens(n_q, n_kv, d, page, hints):
    _attend_case([0, 7, 30, 100, 126, 500], [2, 3, 0, 4, 5, 2], page, n_q, n_kv, d, torch.bfloat16, tail=1, hints=hints)


@pytest.mark.parametrize("n_q,n_kv,d", HEADS)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_attention_portions_beside_single_tokens(n_q, n_kv, d, page):
    _attend_case([0, 200, 0, 129, 77, 1000, 0], [300, 1, 129, 64, 0, 33, 1], page, n_q, n_kv, d, torch.bfloat16, tail=5, strided=True)


@pytest.mark.parametrize("n_q,n_kv,d", [(32, 4, 64), (8, 2, 128), (4, 4, 128)])
def test_attention_long_rows(n_q, n_kv, d):
    """Rows whose keys are split, and a portion at the end of a long cache."""
    _attend_case([20000, 3, 9000], [1, 1, 1], 64, n_q, n_kv, d, torch.bfloat16)
    _attend_case([20000], [3], 16, n_q, n_kv, d, torch.bfloat16)
    _attend_case([9000, 40], [70, 1], 32, n_q, n_kv, d, torch.bfloat16)
    _attend_case([9000, 40], [70, 1], 32, n_q, n_kv, d, torch.bfloat16, hints=False)


@pytest.mark.parametrize("old,new", [([0], [1]), ([0], [128]), ([0], [129]), ([127], [1]), ([128], [1]), ([0, 0], [0, 1]), ([511], [513])])
@pytest.mark.parametrize("n_q,n_kv,d", [(32, 4, 64), (6, 2, 128)])
def test_attention_borders(old, new, n_q, n_kv, d):
    _attend_case(old, new, 64, n_q, n_kv, d, torch.bfloat16, scale=0.3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n_q,n_kv,d", [(32, 4, 64), (6, 2, 128), (8, 8, 128), (16, 1, 64)])
@pytest.mark.parametrize("old,new,odd", [([100, 9], [4, 1], [102, 3]), ([0, 0], [2, 2], [1, 0]), ([0, 300], [400, 200], [130, 333]), ([0, 50], [129, 64], [128, 51]), ([700], [300], [900])])
def test_attention_values_that_are_not_finite_reach_no_token_before_their_own(old, new, odd, n_q, n_kv, d, dtype):
    """Row r's token odd[r] holds an infinity in one column of its first head and nothing but NaN in its last head, and the keys behind it are NaN."""
    plan, pages = make_plan(old, new, 16, "cuda")
    g = torch.Generator(device="cuda").manual_seed(d)
    k, v = (torch.randn(pages, 16, n_kv, d, generator=g, device="cuda").to(dtype) for _ in range(2))
    q = torch.randn(sum(new), n_q, d, generator=g, device="cuda").to(dtype)
    plan.max_new, plan.max_len = max(new), max(o + n for o, n in zip(old, new))
    ref, mass = attend64(q, k, v, plan, 1 / math.sqrt(d))
    at = [int(plan.tables[r, t // 16]) * 16 + t % 16 for r, t in enumerate(odd)]
    late = [[int(plan.tables[r, t // 16]) * 16 + t % 16 for t in range(odd[r] + 1, old[r] + new[r])] for r in range(len(old))]
    kept = k.clone()
    v.view(-1, n_kv, d)[at, 0, 5] = float("inf")
    v.view(-1, n_kv, d)[at, n_kv - 1] = float("nan")
    for rows in late:
        k.view(-1, n_kv, d)[rows] = float("nan")
    out = ops.paged_attention(q, k, v, plan)
    bound = _attention_bound(dtype, ref, mass, plan.max_len, d)
    rep = n_q // n_kv
    for r, (o, n) in enumerate(zip(old, new)):
        a = int(plan.starts[r])
        for i in range(n):
            err = (out[a + i].double() - ref[a + i]).abs()
            if o + i < odd[r]:
                assert bool((err <= bound[a + i]).all()), (r, i)
            elif o + i > odd[r] and odd[r] + 1 < o + n:
                assert out[a + i].isnan().all(), (r, i)      # a key that is NaN
            else:
                first, last = out[a + i, :rep], out[a + i, (n_kv - 1) * rep:]
                assert last.isnan().all()
                if n_kv > 1:
                    assert (first[:, 5] == float("inf")).all()
                    cols = [c for c in range(d) if c != 5]
                    assert bool((err[:rep][:, cols] <= bound[a + i, :rep][:, cols]).all())
    assert not torch.equal(k, kept) or all(len(x) == 0 for x in late)


def test_attention_fp32_portion():
    _attend_case([0, 50], [90, 33], 16, 6, 2, 128, torch.float32, tail=3)


def test_attention_of_an_empty_step():
    plan, pages = make_plan([5, 0], [0, 0], 16, "cuda", tail=4)
    k = torch.randn(pages, 16, 2, 64, device="cuda").bfloat16()
    q = torch.randn(4, 8, 64, device="cuda").bfloat16()
    assert (ops.paged_attention(q, k, k, plan) == 0).all()
    empty = ops.PagePlan(plan.starts, plan.slots[:0], plan.positions[:0], plan.lengths, plan.tables, 16)
    assert ops.paged_attention(q[:0], k, k, empty).shape == (0, 8, 64)


@pytest.mark.parametrize("new,d", [(1, 64), (3, 128), (200, 128)])
def test_attention_reports_pages_that_do_not_exist(new, d):
    """A table entry outside the pool is found by the kernels' own checks: nothing is read there."""
    plan, pages = make_plan([100], [new], 16, "cuda")
    plan.max_new, plan.max_len = new, 100 + new
    k = torch.randn(pages, 16, 2, d, device="cuda").bfloat16()
    q = torch.randn(new, 8, d, device="cuda").bfloat16()
    for bad in (pages, -1, 2 ** 31 - 1, -2 ** 31):
        plan.tables[0, 3] = bad
        ops.paged_attention(q, k, k, plan)
        with pytest.raises(ops.KernelError, match="bad argument"):
            ops.check_status()


def test_attention_step_in_a_graph_on_another_stream():
    """Plan, append and attention of single tokens, captured once and replayed while rows grow."""
    n_q, n_kv, d, page = 8, 2, 64, 16
    pool = ops.PagePool(3, 64, 12, page)
    k, v = (torch.zeros(12, page, n_kv, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cos, sin = ops.rope_tables(64, d, 10000.0, device="cuda")
    fresh = torch.zeros(3, dtype=torch.int32, device="cuda")
    qkv = torch.zeros(3, (n_q + 2 * n_kv) * d, dtype=torch.bfloat16, device="cuda")

    def step():
        plan = ops.page_plan(pool, fresh, 3, max_new=1)
        return ops.paged_attention(ops.paged_append(qkv, cos, sin, plan, k, v, n_q, n_kv, d), k, v, plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step()
    history = [[], [], []]
    g = torch.Generator(device="cuda").manual_seed(0)
    with torch.cuda.stream(side):
        for i in range(40):
            live = [1, int(i % 3 == 0), int(i > 20)]
            qkv.copy_(torch.randn(qkv.shape, generator=g, device="cuda"))
            fresh.copy_(torch.tensor(live))
            graph.replay()
            at = 0
            for r in range(3):
                if not live[r]:
                    continue
                x = ops.rope_packed(qkv[None, at:at + 1].contiguous(), cos, sin, n_q, n_kv, d, pos_offset=len(history[r]))[0, 0].view(-1, d)
                history[r].append(x[n_q:].double())
                kk, vv = torch.stack([h[:n_kv] for h in history[r]]), torch.stack([h[n_kv:] for h in history[r]])
                s = torch.einsum("hd,khd->hk", x[:n_q].double(), kk.repeat_interleave(n_q // n_kv, 1)) / math.sqrt(d)
                p = torch.softmax(s, -1)
                vv = vv.repeat_interleave(n_q // n_kv, 1)
                ref, mass = torch.einsum("hk,khd->hd", p, vv), torch.einsum("hk,khd->hd", p, vv.abs())
                assert ((out[at].double() - ref).abs() <= _attention_bound(torch.bfloat16, ref, mass, 40, d)).all()
                at += 1
            assert (out[at:] == 0).all()
    torch.cuda.current_stream().wait_stream(side)


def test_attention_rows_that_share_pages_and_repeat():
    """Two rows may name the same pages; the same call gives the same bits."""
    plan, pages = make_plan([700, 700], [1, 1], 64, "cuda")
    plan.tables[1] = plan.tables[0]
    k, v = (torch.randn(pages, 64, 4, 64, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(1, 32, 64, device="cuda").bfloat16().expand(2, -1, -1)
    a = ops.paged_attention(q, k, v, plan)
    assert torch.equal(a[0], a[1]) and torch.equal(a, ops.paged_attention(q, k, v, plan))


# ------------------------------------------------------------------------------------------------ sampling
def _sample_case(B, V, dtype, seed, numbers=None, scores=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = 2.5 * torch.randn(B, V, generator=g, device="cuda") if scores is None else scores
    x = x.to(dtype)
    u = torch.rand(B, generator=g, device="cuda")
    pick = lambda vals, t: torch.tensor([vals[i % len(vals)] for i in range(B)], dtype=t, device="cuda")  # noqa: E731
    t, k, p, low, pen = numbers or (pick([0.8, 1.0, 0.3, 2.0, 0.0, 1e-3, 50.0], torch.float32), pick([0, 50, 1, V, 3, 2000], torch.int32),
                                    pick([1.0, 0.9, 0.5, 0.0, 0.999], torch.float32), pick([0.0, 0.05, 1.0, 0.0], torch.float32), pick([1.0, 1.3, 0.8], torch.float32))
    hist = torch.randint(-1, V + 2, (B, 30), generator=g, device="cuda")
    got = ops.sample_rows(x, u, t, k, p, low, pen, hist)
    want = sample64(x.cpu(), u.cpu(), t.cpu(), k.cpu(), p.cpu(), low.cpu(), pen.cpu(), hist.cpu())
    assert torch.equal(got.cpu(), want), (got.cpu() != want).nonzero().flatten().tolist()
    return x, u, (t, k, p, low, pen), hist, got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (420, 33), (70, 1000), (210, 5003), (41, 32000), (9, 131072), (150, 50257)])
def test_sample_rows(B, V, dtype):
    _sample_case(B, V, dtype, seed=V + B)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sample_rows_shapes_of_scores(dtype):
    """All equal, two values, sorted both ways, one certain token, a wide range, zeros of both signs, infinities and NaN."""
    V = 20011
    ramp = torch.linspace(-30, 30, V, device="cuda")
    rows = [torch.zeros(V, device="cuda"), (torch.arange(V, device="cuda") % 2).float(), ramp, ramp.flip(0), torch.where(ramp == ramp[777], 60.0, 0.0), 1e4 * ramp,
            torch.where(torch.arange(V, device="cuda") % 2 == 0, 0.0, -0.0), torch.where(ramp > 3, float("nan"), ramp), torch.where(ramp > 3, float("-inf"), ramp),
            torch.where((ramp > 3) & (ramp < 3.2), float("inf"), ramp), torch.full((V,), float("-inf"), device="cuda"), torch.full((V,), float("nan"), device="cuda"),
            1e-30 * ramp, torch.full((V,), torch.finfo(torch.float32).min, device="cuda")]
    for seed in range(3):
        _sample_case(len(rows) * 5, V, dtype, seed, scores=torch.stack(rows).repeat_interleave(5, 0))


def test_sample_rows_numbers_strides_and_repeats():
    x, u, (t, k, p, low, pen), hist, got = _sample_case(64, 3001, torch.float32, 5)
    wide = torch.zeros(64, 6002, device="cuda")
    wide[:, ::2] = x
    assert torch.equal(ops.sample_rows(wide[:, ::2], u, t, k, p, low, pen, hist), got)
    odd = torch.zeros(64, 3008, device="cuda")[:, 3:3004]
    odd.copy_(x)
    assert torch.equal(ops.sample_rows(odd, u, t, k, p, low, pen, hist), got)
    order = torch.randperm(64, device="cuda")   # a row's token does not depend on the batch around it
    assert torch.equal(ops.sample_rows(x[order], u[order], t[order], k[order], p[order], low[order], pen[order], hist[order]), got[order])
    for i in (1, 10, 30):
        assert int(ops.sample_rows(x[i:i + 1], u[i:i + 1], float(t[i]), int(k[i]), float(p[i]), float(low[i]), float(pen[i]), hist[i:i + 1])[0]) == int(got[i])
    assert torch.equal(ops.sample_rows(x, u, 0.0), x.argmax(-1)) and ops.sample_rows(x[:0], u[:0]).shape == (0,)
    edge = torch.tensor([0.0, 1.0, 2.0, -1.0], device="cuda")
    a = ops.sample_rows(x[:4], edge, 1.0, 10)
    top = x[:4].topk(10).indices.sort().values
    assert a.tolist() == [int(top[0, 0]), int(top[1, -1]), int(top[2, -1]), int(top[3, 0])]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sample_rows_extreme_numbers(dtype):
    """Temperatures from next to nothing to infinite, cuts of every size, infinite scores, tokens named in the history over and over."""
    g = torch.Generator(device="cuda").manual_seed(9)
    temps = [1e-38, 1e-8, 1e-4, 0.02, 1.0, 300.0, 1e9, 1e30, float("inf"), float("nan"), -1.0]
    B, V = 8 * len(temps), 30011
    x = (3 * torch.randn(B, V, generator=g, device="cuda")).to(dtype)
    x[::7, 50:60] = float("inf")
    x[1::7, ::2] = float("-inf")
    x[2::7, 1::2] = float("nan")
    x[3::7] += 1000
    pick = lambda vals, t: torch.tensor([vals[i % len(vals)] for i in range(B)], dtype=t, device="cuda")  # noqa: E731
    numbers = (pick(temps, torch.float32), pick([0, 0, 7, 1024, 1025, 30010, -5, 300], torch.int32), pick([1.0, 0.6, 2.0, -1.0, 0.9999], torch.float32),
               pick([0.0, 1e-3, 2.0, -1.0, 0.3, 1e-30], torch.float32), pick([1.0, 1.5], torch.float32))
    _sample_case(B, V, dtype, 11, numbers=numbers, scores=x)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [270001, 1000003, 1 << 20])
def test_sample_rows_large_vocabularies(V, dtype):
    """Slices that stay in shared memory and such that do not fit; the last token of the largest vocabulary can be drawn."""
    _sample_case(10, V, dtype, seed=V)
    x = torch.zeros(2, V, device="cuda", dtype=dtype)
    x[:, -1] = 60.0
    u = torch.tensor([0.0, 0.999], device="cuda")
    for k in (0, 1, 40):
        assert ops.sample_rows(x, u, 1.0, k, 0.9).tolist() == [V - 1, V - 1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,scale", [(3000, 0.02), (3000, 1.0), (50257, 0.3), (50257, 2.0), (131072, 1.0), (131072, 4.0), (300001, 0.7)])
def test_sample_rows_undecided(V, scale, dtype):
    """Cuts that lie among hundreds or thousands of tokens of about equal mass: the bracket's list short, long and overflowing, with min-p beside it and without."""
    B = 40
    g = torch.Generator(device="cuda").manual_seed(V)
    x = scale * torch.randn(B, V, generator=g, device="cuda")
    pick = lambda vals, t: torch.tensor([vals[i % len(vals)] for i in range(B)], dtype=t, device="cuda")  # noqa: E731
    numbers = (pick([1.0, 0.7, 1.3], torch.float32), pick([0, 0, 0, 400, 1000], torch.int32), pick([0.9, 0.5, 0.98, 0.999], torch.float32),
               pick([0.0, 0.0, 1e-4, 0.0, 0.02], torch.float32), pick([1.0, 1.2], torch.float32))
    _sample_case(B, V, dtype, V, numbers=numbers, scores=x)


def test_sample_rows_draws_by_mass():
    """20,000 evenly spaced numbers over ten tokens: every token is named as often as its probability says, but for one at either border."""
    n = 20000
    x = torch.linspace(0, 3, 10, device="cuda").expand(n, 10).contiguous()
    u = (torch.arange(n, device="cuda") + 0.5) / n
    f = torch.bincount(ops.sample_rows(x, u), minlength=10).double() / n
    p = torch.softmax(x[0].double(), 0)
    assert ((f - p).abs() <= 2 / n).all()


@pytest.mark.parametrize("old,new", [([200, 5, 63], [1, 1, 1]), ([0, 100, 40], [150, 1, 20]), ([6000], [1])])
@pytest.mark.parametrize("n_q,n_kv,d", [(8, 2, 64), (4, 4, 128), (6, 2, 96)])
def test_attention_replaces_its_queries(old, new, n_q, n_kv, d):
    """``out`` may be ``q``: the same numbers, and rows of the batch that belong to no row keep what they hold."""
    plan, pages = make_plan(old, new, 16, "cuda", tail=2)
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn(pages, 16, n_kv, d, generator=g, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(sum(new) + 2, n_q, d, generator=g, device="cuda").bfloat16()
    want = ops.paged_attention(q, k, v, plan)
    tail = q[-2:].clone()
    assert ops.paged_attention(q, k, v, plan, out=q) is q
    assert torch.equal(q[:-2], want[:-2]) and torch.equal(q[-2:], tail)


def test_sample_rows_takes_any_top_k_on_the_gpu():
    logits = torch.randn(3, 4000, generator=torch.Generator().manual_seed(0)).cuda()
    u = torch.tensor([0.2, 0.6, 0.95], device="cuda")
    everything = ops.sample_rows(logits, u)
    for k in (4000, 1 << 31, 1 << 40, -5, torch.tensor([1 << 40, -(1 << 40), 0], device="cuda")):
        assert torch.equal(ops.sample_rows(logits, u, top_k=k), everything)


@pytest.mark.parametrize("hints", [True, False])
@pytest.mark.parametrize("n_q,n_kv,d,page,dtype", [(8, 2, 96, 64, torch.bfloat16), (4, 4, 64, 16, torch.float32), (6, 1, 256, 4, torch.float32), (3, 3, 8, 1, torch.bfloat16)])
def test_attention_general_form_of_long_rows(n_q, n_kv, d, page, dtype, hints):
    """Rows whose keys several thread blocks share, beside rows shorter than one block's share, tokens of no row and a row without new tokens."""
    _attend_case([9000, 0, 130, 2047, 50], [1, 1, 2, 1, 0], page, n_q, n_kv, d, dtype, tail=2, hints=hints)
    _attend_case([20011], [1], page, n_q, n_kv, d, dtype, hints=hints, strided=True)


def _off(t, elements=1):
    """``t``'s values, contiguous, that many elements behind a multiple of sixteen bytes."""
    room = torch.empty(t.numel() + 16, dtype=t.dtype, device=t.device)
    start = (-room.data_ptr() % 16) // t.element_size() + elements
    return room[start:start + t.numel()].view(t.shape).copy_(t)


@pytest.mark.parametrize("n_q,n_kv,d,dtype", [(8, 2, 64, torch.bfloat16), (4, 4, 128, torch.bfloat16), (6, 2, 96, torch.bfloat16), (4, 2, 64, torch.float32)])
@pytest.mark.parametrize("old,new", [([200, 5, 63], [1, 1, 1]), ([40], [1]), ([0, 100, 40], [150, 1, 20])])
def test_operands_that_start_off_16_bytes_or_lie_on_one_another(old, new, n_q, n_kv, d, dtype):
    """The bits of the same operands in rows of their own that start at whole 16 bytes."""
    plan, pages = make_plan(old, new, 16, "cuda", tail=2)
    g = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randn(pages, 16, n_kv, d, generator=g, device="cuda").to(dtype) for _ in range(2))
    T, width = sum(new) + 2, (n_q + 2 * n_kv) * d
    q, qkv = torch.randn(T, n_q, d, generator=g, device="cuda").to(dtype), torch.randn(T, width, generator=g, device="cuda").to(dtype)
    want = ops.paged_attention(q, k, v, plan)
    for odd in (_off(q), _off(q, 3), torch.cat([q.flatten(1), q[:, 0]], 1).as_strided((T, n_q, d), ((n_q + 1) * d, d, 1))):
        assert torch.equal(ops.paged_attention(odd, k, v, plan), want)
    same = q[:1].expand(T, -1, -1)
    assert torch.equal(ops.paged_attention(same, k, v, plan), ops.paged_attention(same.contiguous(), k, v, plan))
    with pytest.raises(ValueError, match="16 bytes"):
        ops.paged_attention(q, k, v, plan, out=_off(q))
    for cos, sin in ((None, None), ops.rope_tables(600, d, 10000.0, device="cuda")):
        a, b = (k.clone(), v.clone()), (k.clone(), v.clone())
        x, y = ops.paged_append(qkv, cos, sin, plan, *a, n_q, n_kv, d), ops.paged_append(_off(qkv), cos, sin, plan, *b, n_q, n_kv, d)
        assert torch.equal(x, y) and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("d", [64, 128])
def test_attention_short_portions_behind_values_that_are_not_finite(d):
    """Every fourteenth row is two tiles of tokens whose values hold an infinity each, which its second tile adds one by one; the portions between them have
    one tile, so that a CTA's other warps run ahead of that one's.  Rows beside them stay as they are."""
    new = [256 if r % 14 == 0 else 17 + r % 5 for r in range(2100)]
    plan, pages = make_plan([0] * len(new), new, 16, "cuda")
    plan.max_new = plan.max_len = 256
    g = torch.Generator(device="cuda").manual_seed(d)
    k, v = (torch.randn(pages, 16, 1, d, generator=g, device="cuda").bfloat16() for _ in range(2))
    T = sum(new)
    q = torch.randn(T, 1, d, generator=g, device="cuda").bfloat16()
    ref, mass = attend64(q, k, v, plan, 1 / math.sqrt(d))
    inf = torch.zeros(T, d, dtype=torch.bool, device="cuda")
    tokens = torch.arange(256, device="cuda")
    for r in range(0, len(new), 14):
        v.view(-1, d)[plan.slots[int(plan.starts[r]) + tokens].long(), tokens % d] = float("inf")
        inf[int(plan.starts[r]) + tokens] = torch.arange(d, device="cuda")[None] <= tokens[:, None]   # token i sees the values of 0 to i
    bound = _attention_bound(torch.bfloat16, ref, mass, 256, d)
    first = ops.paged_attention(q, k, v, plan)
    for out in (first, ops.paged_attention(q, k, v, plan)):
        assert torch.equal(out[:, 0] == float("inf"), inf)
        assert bool(((out.double() - ref).abs() <= bound)[:, 0][~inf].all())
        assert torch.equal(out, first)
    ops.check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n_q,n_kv,d", [(8, 2, 64), (4, 4, 128), (6, 2, 96)])
@pytest.mark.parametrize("old,new", [([700, 0, 130], [1, 1, 2]), ([700, 0, 130], [300, 150, 40]), ([9000], [20])])
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("size", [1e4, 1e11, 4e30, 1e37])
def test_attention_scores_of_any_size(size, sign, old, new, n_q, n_kv, d, dtype):
    """Two scores, the smaller one further below than any probability reaches, and minus infinity: an even share of the values at the larger one's keys."""
    plan, pages = make_plan(old, new, 16, "cuda")
    g = torch.Generator(device="cuda").manual_seed(d)
    v = torch.randn(pages, 16, n_kv, d, generator=g, device="cuda").to(dtype)
    k = torch.zeros(pages, 16, n_kv, d, device="cuda", dtype=dtype)
    root = 2.0 ** round(math.log2(size) / 2)
    near, far = (1.7109375, 2.5) if sign < 0 else (2.5, 1.7109375)          # (in all their digits: products with the scale are rounded)
    low = torch.rand(pages, 16, n_kv, generator=g, device="cuda") < 0.5
    for r in range(len(old)):   # every row's first key has the larger score: every token sees one
        low[int(plan.tables[r, 0]), 0] = False
    k[..., 3] = sign * root * torch.where(low, far, near)
    gone = torch.rand(low.shape, generator=g, device="cuda") < 0.1
    k[..., 3] = torch.where(gone & low, float("-inf"), k[..., 3])
    q = torch.zeros(sum(new), n_q, d, device="cuda", dtype=dtype)
    q[..., 3] = 1.6640625 * root
    ref, mass = attend64(q, k, v, plan, 1.1)
    out = ops.paged_attention(q, k, v, plan, scale=1.1)
    assert ref.isfinite().all() and bool(((out.double() - ref).abs() <= _attention_bound(dtype, ref, mass, max(o + n for o, n in zip(old, new)), d)).all())


def test_sample_rows_from_two_threads():
    """Threads that sample vocabularies of different sizes at the same time do not get in each other's way (the entry point itself, so that they meet in it)."""
    import threading
    from adaptivetrainingsystem_b200.ops import paged
    sizes, wrong = (33, 131072), []
    x = [torch.randn(2, V, generator=torch.Generator().manual_seed(V)).bfloat16().cuda() for V in sizes]
    u = torch.tensor([0.3, 0.8], device="cuda")
    want = [ops.sample_rows(t, u, 1.0, 40) for t in x]
    out = [torch.zeros_like(t) for t in want]
    streams = [torch.cuda.Stream() for _ in sizes]
    torch.cuda.synchronize()
    entry = paged._fn("ats_sample_rows")

    def work(i):
        args = (x[i].data_ptr(), 0, sizes[i], 2, sizes[i], u.data_ptr(), 0, 1.0, 0, 40, 0, 1.0, 0, 0.0, 0, 1.0, 0, 0, 0, out[i].data_ptr(), streams[i].cuda_stream)
        wrong.extend(code for code in (entry(*args) for _ in range(30000)) if code)
    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong, (len(wrong), wrong[0])
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.parametrize("old,new", [([100, 50], [1, 1]), ([0, 40], [200, 60])])
def test_first_call_of_a_thread_may_be_a_captured_one(old, new):
    import threading
    plan, pages = make_plan(old, new, 16, "cuda")
    plan.max_new = max(new)
    k, v = (torch.randn(pages, 16, 2, 64, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(sum(new), 8, 64, device="cuda").bfloat16()
    want, got = ops.paged_attention(q, k, v, plan), []
    torch.cuda.synchronize()

    def work():
        try:
            stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
            with torch.cuda.stream(stream):
                with torch.cuda.graph(graph, stream=stream):
                    out = ops.paged_attention(q, k, v, plan)
                graph.replay()
            torch.cuda.synchronize()
            got.append(out)
        except Exception as e:
            got.append(e)
    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    assert isinstance(got[0], torch.Tensor), got[0]
    assert torch.equal(got[0], want)
