"""Paged cache operators on the CPU: the definitions, the life of a pool, refusals."""
import math
import random

import pytest
import torch

from adaptivetrainingsystem_b200 import ops
from paged_utils import attend64, make_plan, rows_of_pages, sample64


def _random_step(g, pool, lengths, tokens_left=60):
    fresh = []
    for n in lengths:
        kind = g.random()
        f = -1 if kind < 0.15 and n else 0 if kind < 0.4 else 1 if kind < 0.8 else g.randint(1, 12)
        if f > 0 and (f > tokens_left or n + f > pool.width * pool.page_size):
            f = 0
        tokens_left -= max(f, 0)
        fresh.append(f)
    return fresh


@pytest.mark.parametrize("page", [1, 4, 16])
def test_plan_life_of_a_pool(page):
    """However rows come, grow and go: no page belongs to two, and slots hold what was written to them."""
    g = random.Random(page)
    pool = ops.PagePool(5, 48, 5 * -(-48 // page), page, device="cpu")
    lengths, content = [0] * 5, {}
    memory = torch.full((pool.pages * page,), -1)
    for step in range(60):
        fresh = _random_step(g, pool, lengths)
        T = sum(max(f, 0) for f in fresh)
        plan = ops.page_plan(pool, torch.tensor(fresh, dtype=torch.int32), T + 2)
        pool.check()
        at = 0
        for r, f in enumerate(fresh):
            assert int(plan.starts[r]) == at
            for i in range(max(f, 0)):
                assert int(plan.positions[at + i]) == lengths[r] + i
                memory[int(plan.slots[at + i])] = 1000 * step + at + i
                content[r, lengths[r] + i] = 1000 * step + at + i
            at += max(f, 0)
            lengths[r] = 0 if f < 0 else lengths[r] + f
        assert plan.slots[T:].tolist() == [-1, -1] and int(plan.starts[-1]) == T and pool.lengths.tolist() == lengths
        used = [int(pool.tables[r, j]) for r in range(5) for j in range(pool.pages_for(lengths[r]))]
        free = pool.free[:int(pool.state[0])].tolist()
        assert sorted(used + free) == list(range(pool.pages))
        for r, n in enumerate(lengths):
            assert [int(memory[int(pool.tables[r, i // page]) * page + i % page]) for i in range(n)] == [content[r, i] for i in range(n)]


def test_plan_refuses_a_step_as_a_whole():
    pool = ops.PagePool(3, 32, 5, 8, device="cpu")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    ops.page_plan(pool, i32(17, 8, 0), 25)
    before = (pool.tables.clone(), pool.lengths.clone(), pool.free.clone(), int(pool.state[0]))
    for fresh, tokens, why in ((i32(8, 1, 1), 10, "free pages"), (i32(16, 0, 0), 16, "table"), (i32(1, 1, 0), 1, "packed batch"), (i32(-2, 0, 0), 4, "table")):
        plan = ops.page_plan(pool, fresh, tokens, commit=False)
        with pytest.raises(RuntimeError, match=why):
            plan.check()
        assert plan.slots.tolist() == [-1] * tokens and plan.starts.tolist() == [0] * 4 and torch.equal(plan.lengths, before[1])
        ops.page_plan(pool, fresh, tokens)
        with pytest.raises(RuntimeError, match=why):
            pool.check()
        assert torch.equal(pool.tables, before[0]) and torch.equal(pool.lengths, before[1]) and torch.equal(pool.free, before[2]) and int(pool.state[0]) == before[3]
    ops.page_plan(pool, i32(-1, 1, 8), 9)   # a row closed in the same step gives its pages back first
    pool.check()
    assert pool.lengths.tolist() == [0, 9, 8] and int(pool.state[0]) == 2


def test_plan_without_commit_can_be_repeated():
    pool = ops.PagePool(2, 32, 8, 4, device="cpu")
    fresh = torch.tensor([5, 2], dtype=torch.int32)
    a = ops.page_plan(pool, fresh, 7, commit=False)
    b = ops.page_plan(pool, fresh, 7, commit=False)
    assert torch.equal(a.slots, b.slots) and a.lengths.tolist() == [5, 2] and pool.lengths.tolist() == [0, 0] and int(a.count) == 5 and int(pool.state[0]) == 8


def test_append_and_attention_definitions():
    old, new, page, n_q, n_kv, d = [0, 5, 3, 7], [4, 1, 0, 6], 4, 6, 2, 16
    plan, pages = make_plan(old, new, page, "cpu", tail=2)
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(pages, page, n_kv, d, generator=g) for _ in range(2))
    T = plan.slots.numel()
    qkv = torch.randn(T, (n_q + 2 * n_kv) * d, generator=g)
    cos, sin = ops.rope_tables(32, d, 10000.0)
    q = ops.paged_append(qkv, cos, sin, plan, k, v, n_q, n_kv, d)
    want = ops.rope_reference(qkv[:, :(n_q + n_kv) * d].view(T, 1, n_q + n_kv, d), cos, sin, plan.positions.long()[:, None])[:, 0]
    assert torch.allclose(q, want[:, :n_q], atol=1e-6)
    for i in range(T - 2):
        s = int(plan.slots[i])
        assert torch.allclose(k.view(-1, n_kv, d)[s], want[i, n_q:], atol=1e-6) and torch.equal(v.view(-1, n_kv, d)[s], qkv[i, (n_q + n_kv) * d:].view(n_kv, d))
    out = ops.paged_attention(q, k, v, plan)
    ref, mass = attend64(q, k, v, plan, 1 / math.sqrt(d))
    assert ((out.double() - ref).abs() <= 1e-5 * mass + 1e-7).all() and (out[T - 2:] == 0).all()
    # and the dense attention of the framework over the same tokens
    for r, (a, b) in enumerate(zip(plan.starts.tolist(), plan.starts.tolist()[1:])):
        if b > a:
            dense = ops.attention(q[None, a:b], rows_of_pages(k, plan, r)[None], rows_of_pages(v, plan, r)[None], causal=True, q_offset=old[r])
            assert torch.allclose(out[a:b], dense[0], atol=1e-5)


def test_refusals():
    plan, pages = make_plan([3], [2], 4, "cpu")
    k = torch.zeros(pages, 4, 2, 16)
    q = torch.zeros(2, 4, 16)
    with pytest.raises(ValueError, match="power of two"):
        ops.PagePool(2, 16, 4, 12, device="cpu")
    with pytest.raises(ValueError, match="rows"):
        ops.PagePool(5000, 16, 4, 16, device="cpu")
    with pytest.raises(ValueError, match="2\\^31"):
        ops.PagePool(2, 16, 1 << 26, 64, device="cpu")
    pool = ops.PagePool(2, 16, 4, 4, device="cpu")
    with pytest.raises(ValueError, match="fresh"):
        ops.page_plan(pool, torch.zeros(3, dtype=torch.int32), 4)
    with pytest.raises(ValueError, match="fresh"):
        ops.page_plan(pool, torch.zeros(2, dtype=torch.int64), 4)
    with pytest.raises(ValueError, match="tokens"):
        ops.page_plan(pool, torch.zeros(2, dtype=torch.int32), (1 << 18) + 1)
    with pytest.raises(ValueError, match="page size"):
        ops.paged_attention(q, k.view(pages * 2, 2, 2, 16), k.view(pages * 2, 2, 2, 16), plan)
    with pytest.raises(ValueError, match="one type"):
        ops.paged_attention(q.bfloat16(), k, k, plan)
    with pytest.raises(ValueError, match="query heads"):
        ops.paged_attention(q[:, :3], k, k, plan)
    with pytest.raises(ValueError, match="plan.slots"):
        ops.paged_attention(q[:1], k, k, plan)
    with pytest.raises(ValueError, match="scale"):
        ops.paged_attention(q, k, k, plan, scale=0.0)
    with pytest.raises(ValueError, match="out"):
        ops.paged_attention(q, k, k, plan, out=torch.zeros(2, 4, 16, dtype=torch.float64))
    with pytest.raises(ValueError, match="qkv"):
        ops.paged_append(torch.zeros(2, 100), None, None, plan, k, k, 4, 2, 16)
    with pytest.raises(ValueError, match="rotary tables"):
        ops.paged_append(torch.zeros(2, 128), *ops.rope_tables(4, 16, 10000.0), plan, k, k, 4, 2, 16)
    with pytest.raises(ValueError, match="uniform"):
        ops.sample_rows(torch.zeros(2, 8), torch.zeros(3))
    with pytest.raises(ValueError, match="top_k"):
        ops.sample_rows(torch.zeros(2, 8), torch.zeros(2), top_k=torch.ones(3))
    with pytest.raises(ValueError, match="history"):
        ops.sample_rows(torch.zeros(2, 8), torch.zeros(2), history=torch.zeros(2, 3, dtype=torch.int32))


def test_sample_rows_definition():
    g = torch.Generator().manual_seed(3)
    B, V = 40, 57
    logits = (3 * torch.randn(B, V, generator=g)).bfloat16().float().round()     # many ties
    logits[5, 3:9], logits[6], logits[7, 11], logits[8, 4] = float("nan"), float("-inf"), float("inf"), float("-inf")
    u = torch.rand(B, generator=g)
    u[:4] = torch.tensor([0.0, 1.0, 1.5, 0.999999])
    t = torch.tensor([0.7, 1.0, 2.5, 0.0])[torch.arange(B) % 4]
    k = torch.tensor([0, 1, 5, 57, 100])[torch.arange(B) % 5].int()
    p = torch.tensor([1.0, 0.9, 0.5, 0.0, 0.99, 1.0, 0.3])[torch.arange(B) % 7]
    low = torch.tensor([0.0, 0.1, 1.0])[torch.arange(B) % 3]
    pen = torch.tensor([1.0, 1.3])[torch.arange(B) % 2]
    hist = torch.randint(-1, V + 3, (B, 9), generator=g)
    got = ops.sample_rows(logits, u, t, k, p, low, pen, hist)
    assert torch.equal(got, sample64(logits, u, t, k, p, low, pen, hist))


def test_refusals_of_memory_that_the_kernels_cannot_take():
    plan, pages = make_plan([3], [2], 4, "cpu")
    n = pages * 4 * 2 * 16
    k, odd = torch.zeros(pages, 4, 2, 16), torch.zeros(n + 1)[1:].view(pages, 4, 2, 16)   # four bytes behind a multiple of sixteen
    q = torch.zeros(2, 4, 16)
    for a, b in ((k, odd), (odd, k)):
        with pytest.raises(ValueError, match="16 bytes"):
            ops.paged_attention(q, a, b, plan)
        with pytest.raises(ValueError, match="16 bytes"):
            ops.paged_append(torch.zeros(2, 128), None, None, plan, a, b, 4, 2, 16)
    cos, sin = ops.rope_tables(32, 16, 10000.0)
    late = torch.zeros(sin.numel() + 1)[1:].view_as(sin)
    with pytest.raises(ValueError, match="cos, sin"):
        ops.paged_append(torch.zeros(2, 128), cos, late, plan, k, k.clone(), 4, 2, 16)
    for out in (torch.zeros(1, 4, 16).expand(2, 4, 16), torch.zeros(3 * 64).as_strided((2, 4, 16), (32, 16, 1))):   # tokens whose answers lie on one another
        with pytest.raises(ValueError, match="out"):
            ops.paged_attention(q, k, k, plan, out=out)
    with pytest.raises(ValueError, match="without"):
        ops.paged_attention(torch.zeros(2, 0, 16), k[:, :, :0], k[:, :, :0], plan)


def test_sample_rows_takes_any_top_k():
    logits = torch.randn(3, 40, generator=torch.Generator().manual_seed(0))
    u = torch.tensor([0.2, 0.6, 0.95])
    everything = ops.sample_rows(logits, u)
    for k in (40, 1 << 31, 1 << 40, -5, torch.tensor([1 << 40, -(1 << 40), 0])):
        assert torch.equal(ops.sample_rows(logits, u, top_k=k), everything)


def _off(t, elements=1):
    """``t``'s values, contiguous, that many elements behind a multiple of sixteen bytes."""
    room = torch.empty(t.numel() + 16, dtype=t.dtype, device=t.device)
    start = (-room.data_ptr() % 16) // t.element_size() + elements
    return room[start:start + t.numel()].view(t.shape).copy_(t)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_operands_that_start_off_16_bytes_are_copied(dtype):
    from adaptivetrainingsystem_b200.ops.paged import _rows_of
    wide = torch.randn(6, 5 * 64 + 8).to(dtype)
    cases = [_off(torch.randn(4, 8, 64).to(dtype)), _off(torch.randn(4, 320).to(dtype), 2), wide[:1, 1:321], wide[:, 1:321], wide[:, 8:328][:, :320].unflatten(1, (5, 64))[..., ::2],
             wide[:1, :320].expand(4, 320), torch.randn(9 * 64).to(dtype).as_strided((4, 5, 64), (64, 64, 1)), wide[0, :320].view(1, 5, 64).expand(3, 5, 64)]
    for t in cases:
        got = _rows_of(t)
        assert got is not t and got.data_ptr() % 16 == 0 and got.is_contiguous() and torch.equal(got, t)
    for t in (wide, wide[:, 8:328], wide[:, 8:328].unflatten(1, (5, 64)), wide[:1, 8:328], wide[3:4].view(1, 41, 8)):   # nothing to copy
        assert _rows_of(t) is t
    plan, pages = make_plan([3], [2], 4, "cpu")
    k = torch.zeros(pages, 4, 2, 16, dtype=dtype)
    q = torch.zeros(2, 4, 16, dtype=dtype)
    with pytest.raises(ValueError, match="16 bytes"):
        ops.paged_attention(q, k, k, plan, out=_off(q))


def test_entry_points_refuse_operands_off_16_bytes():
    """Before they look at what the operands point to."""
    import ctypes
    import os
    from adaptivetrainingsystem_b200.ops import _lib, paged
    if not os.path.exists(_lib.CUDA_LIB):
        pytest.skip("the CUDA library has not been built")
    lib = ctypes.CDLL(_lib.CUDA_LIB)

    def call(name, *args):
        f = getattr(lib, name)
        f.restype, f.argtypes = ctypes.c_int, paged._SIGNATURES[name]
        return f(*args)
    at = 1 << 20
    for bad in range(6):   # queries and projections, pages, outputs, tables, scratch
        q, k, v, out, cos, scratch = (at + (2 if i == bad else 0) for i in range(6))
        attend = (q, 256, k, v, at, at, at, out, 256, 3, 1, 4, 2, 64, 4, 8, 16)
        if bad < 5:
            assert bad == 4 or call("ats_paged_portion", *attend, 8, 1.0, 0, at, at, None) == 1003
            assert call("ats_paged_append", q, 512, cos, at, 64, at, at, out, k, v, 3, 4, 2, 64, 128, 0, at, None) == 1003
        if bad != 4:
            assert call("ats_paged_decode", *attend, 64, 1, 8, 1.0, 0, 0, scratch, at, None) == 1003
        if bad in (1, 2):
            assert call("ats_paged_attn_any", *attend, 1.0, 0, 0, 1, None, at, None) == 1003


def test_warps_of_the_portion_kernel_give_up_a_wait_together():
    """Roles of whole warps go on with instructions that all lanes take part in: where a wait runs out, none of them may go on alone.  (One lane issues products.)"""
    import pathlib
    import adaptivetrainingsystem_b200
    text = (pathlib.Path(adaptivetrainingsystem_b200.__file__).parents[1] / "csrc" / "paged_attention_tcgen05.cu").read_text()
    kernel = text[text.index("paged_portion_kernel("):text.index("paged_portion_join_kernel")]
    roles = kernel.split("  // ------------------------------------------------------------------")
    assert len(roles) == 5
    for role in roles[1:]:
        assert ("mbar_wait_bounded" in role) == role.lstrip("- ").startswith("MMA issuer"), role[:80]
    for told in kernel.split("next_piece(n_pieces);")[2:]:
        assert told.lstrip().startswith("if (!__all_sync(0xffffffffu, told != nullptr)) break;")


def test_operators_refuse_tensors_that_ask_for_gradients():
    plan, pages = make_plan([3], [2], 4, "cpu")
    k, v = torch.zeros(pages, 4, 2, 16), torch.zeros(pages, 4, 2, 16)
    q, qkv = torch.zeros(2, 4, 16), torch.zeros(2, 128)
    for bad in (q, k, v):
        bad.requires_grad_(True)
        with pytest.raises(RuntimeError, match="backward"):
            ops.paged_attention(q, k, v, plan)
        if bad is not q:
            with pytest.raises(RuntimeError, match="backward"):
                ops.paged_append(qkv, None, None, plan, k, v, 4, 2, 16)
        with torch.no_grad():
            assert not ops.paged_attention(q, k, v, plan).requires_grad
        bad.requires_grad_(False)
    qkv.requires_grad_(True)
    with pytest.raises(RuntimeError, match="backward"):
        ops.paged_append(qkv, None, None, plan, k, v, 4, 2, 16)
    assert not k.requires_grad
