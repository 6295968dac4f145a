"""Rows over a paged cache: the pool and the batcher on it (CPU; on a GPU in test_gpu_paged_pool.py)."""
import pytest
import torch

from adaptivetrainingsystem_b200.config import ModelConfig
from adaptivetrainingsystem_b200.inference import ContinuousBatcher, GenerationEngine, PagedPool, SamplingParams, sample_next
from adaptivetrainingsystem_b200.models import DeepSeekTransformer


def _model(moe=False, **kw):
    torch.manual_seed(0)
    cfg = ModelConfig(vocab_size=97, hidden_size=32, num_layers=2, num_heads=4, num_kv_heads=2, intermediate_size=64, seq_length=64, use_moe=moe, num_experts=4,
                      moe_top_k=2, capacity_factor=4.0, routing_noise_std=0.0, **kw)
    model = DeepSeekTransformer(cfg).eval()
    with torch.no_grad():
        model.lm_head.mul_(8.0)
    return model


@pytest.mark.parametrize("moe", [False, True])
@torch.no_grad()
def test_rows_equal_sequences_of_their_own(moe):
    """Portions packed with other rows' and single tokens beside other rows give the logits of the whole sequence on its own."""
    model = _model(moe)
    pool = PagedPool(model, 4, 40, pages=14, page_size=8, use_graph=False)
    g = torch.Generator().manual_seed(1)
    seqs = [torch.randint(0, 97, (n,), generator=g) for n in (20, 33, 9)]
    rows = [pool.open(n) for n in (20, 33, 9)]
    fed = [7, 16, 1]
    logits = pool.extend_many([(rows[i], seqs[i][:fed[i]]) for i in (2, 0, 1)])      # in any order
    got = {i: logits[j] for j, i in enumerate((2, 0, 1))}
    for step in range(12):
        for i, s in enumerate(seqs):
            want = model(s[None, :fed[i]], return_aux_loss=False)[0, -1]
            assert torch.allclose(got[i], want, atol=2e-4), (step, i)
        live = [i for i in range(3) if fed[i] < seqs[i].numel() and (i + step) % 3]
        if step == 5:                                                             # a portion in the middle
            live = []
            if fed[1] + 6 <= 33:
                got[1] = pool.extend(rows[1], seqs[1][fed[1]:fed[1] + 6])[0]
                fed[1] += 6
        if not live:
            continue
        for i in live:
            pool.last[rows[i]] = seqs[i][fed[i]]
            fed[i] += 1
        out = pool.decode(sorted(rows[i] for i in live))
        for i in live:
            got[i] = out[rows[i]]
    pool.cache.pool.check()
    for r in rows:
        pool.close(r)
    assert pool.pages_left == 14 and int(pool.cache.pool.state[0]) == 14 and pool.available == 4


def test_pool_refusals():
    model = _model()
    pool = PagedPool(model, 2, 32, pages=5, page_size=8, use_graph=False)
    a = pool.open(17)
    assert pool.pages_left == 2 and pool.fits(16) and not pool.fits(17)
    with pytest.raises(RuntimeError, match="pages are free"):
        pool.open(17)
    with pytest.raises(RuntimeError, match="no room"):
        pool.extend(a, torch.zeros(25, dtype=torch.long))
    b = pool.open(2)
    pool.extend_many([(a, [1] * 17), (b, [1])])
    with pytest.raises(RuntimeError, match="no room"):
        pool.extend_many([(b, [1]), (a, [1] * 9)])
    assert pool.lengths == {a: 17, b: 1}      # nothing of a refused step has happened
    with pytest.raises(ValueError, match="one token"):
        pool.decode([b, b])
    pool.close(b)
    with pytest.raises(ValueError, match="different rows"):
        pool.extend_many([(a, [1]), (a, [2])])
    with pytest.raises(ValueError, match="at least one token"):
        pool.extend_many([(a, [])])
    pool.cache.reset()
    assert pool.cache.pool.lengths.tolist() == [0, 0] and int(pool.cache.pool.state[0]) == 5
    with pytest.raises(ValueError, match="power of two"):
        PagedPool(model, 2, 32, page_size=12)
    with pytest.raises(ValueError, match="Mixture-of-Depths"):
        PagedPool(_model(use_mod=True), 2, 32)
    with pytest.raises(ValueError, match="plan"):
        model(torch.zeros(1, 2, dtype=torch.long), attention_mask=torch.ones(1, 2), cache=pool.cache)


@pytest.mark.parametrize("chunk", [None, 5])
def test_batcher_serves_more_rows_than_whole_rows_would_fit(chunk, monkeypatch):
    """Greedy requests over pages against each one on its own; pages for a third of the rows at full length."""
    model = _model()
    eng = GenerationEngine(model)
    monkeypatch.setattr(PagedPool, "_capture", lambda self: setattr(self, "use_graph", False))
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 97, (n,), generator=g).tolist() for n in (5, 17, 3, 11, 8, 2, 14)]
    budgets = [6, 4, 9, 5, 7, 3, 6]
    batcher = ContinuousBatcher(eng, max_batch=6, max_len=40, params=SamplingParams.from_mode("greedy"), prefill_chunk=chunk, page_size=4, pages=20)
    rids = [batcher.submit(p, b) for p, b in zip(prompts, budgets)]
    peak = 0
    while batcher.pending:
        peak = max(peak, batcher.step())
    for p, b, r in zip(prompts, budgets, rids):
        want = eng.generate(torch.tensor([p]), SamplingParams.from_mode("greedy", max_new_tokens=b), use_graph=False)["tokens"][0].tolist()
        assert batcher.finished[r].tokens == want
    assert peak >= 3 and batcher.pool.pages_left == 20 and int(batcher.cache.pool.state[0]) == 20
    with pytest.raises(ValueError, match="pages"):
        ContinuousBatcher(eng, max_batch=2, max_len=40, page_size=4, pages=5).submit([1] * 20, 8)


def test_requests_with_sampling_numbers_of_their_own():
    model = _model()
    eng = GenerationEngine(model)
    batcher = ContinuousBatcher(eng, max_batch=4, max_len=40, params=SamplingParams.from_mode("greedy", seed=3), page_size=8)
    batcher.pool.use_graph = False
    greedy = batcher.submit([1, 2, 3], 8)
    sure = batcher.submit([1, 2, 3], params=SamplingParams(temperature=2.0, top_k=1, repetition_penalty=1.0, max_new_tokens=8))
    tiny = batcher.submit([1, 2, 3], params=SamplingParams(temperature=2.0, top_k=0, top_p=1.0, min_p=1.0, repetition_penalty=1.0, max_new_tokens=8))
    wild = batcher.submit([1, 2, 3], params=SamplingParams(temperature=50.0, top_k=0, top_p=1.0, repetition_penalty=1.0, max_new_tokens=8))
    first = eng.generate(torch.tensor([[1, 2, 3]]), SamplingParams.from_mode("greedy", max_new_tokens=8), use_graph=False)["tokens"][0].tolist()
    stops = batcher.submit([1, 2, 3], params=SamplingParams.from_mode("greedy", stop_token_ids=(first[2],), max_new_tokens=8))
    while batcher.pending:
        batcher.step()
    done = {n: batcher.finished[r].tokens for n, r in (("greedy", greedy), ("sure", sure), ("tiny", tiny), ("wild", wild), ("stops", stops))}
    assert done["greedy"] == done["sure"] == done["tiny"] == first and done["wild"] != first and done["stops"] == first[:first.index(first[2]) + 1]
    assert batcher._own == 0


def test_min_p_in_sampling_params():
    x = torch.tensor([[0.0, 5.0, 4.0, -3.0]]).expand(200, -1)
    kept = sample_next(x, SamplingParams(temperature=1.0, top_k=0, top_p=1.0, repetition_penalty=1.0, min_p=0.2)).unique().tolist()
    assert kept == [1, 2]


@torch.no_grad()
def test_rows_whose_length_is_no_multiple_of_a_page():
    """A pool's rows end at ``max_len``; a cache that is planned by hand may fill the last page, and positions reach as far."""
    model = _model()
    pool = PagedPool(model, 2, 70, page_size=16, use_graph=False)
    ids = torch.randint(0, 97, (80,), generator=torch.Generator().manual_seed(3))
    row = pool.open(70)
    pool.extend(row, ids[:69])
    pool.last[row] = ids[69]
    pool.decode([row])
    with pytest.raises(RuntimeError, match="overflow"):
        pool.decode([row])
    with pytest.raises(RuntimeError, match="overflow"):
        pool.extend(row, ids[:1])
    assert pool.lengths[row] == 70
    cache = model.make_paged_cache(2, 70, 10, 16)
    assert cache.max_len == 80
    cache.plan(torch.tensor([0, 80], dtype=torch.int32), 80)
    got = model(ids[None], cache=cache, return_aux_loss=False)[0]
    want = model(ids[None], return_aux_loss=False)[0]
    assert torch.allclose(got, want, atol=2e-4)


def test_steps_that_do_not_come_to_be_planned_leave_the_rows_as_they_were(monkeypatch):
    model = _model()
    pool = PagedPool(model, 2, 300000, pages=5000, page_size=64, use_graph=False)
    row, other = pool.open(270000), pool.open(100)
    pool.extend(other, [1, 2, 3])
    with pytest.raises(ValueError, match="tokens in a step"):
        pool.extend(row, torch.zeros((1 << 18) + 1, dtype=torch.long))
    assert pool.lengths == {row: 0, other: 3}
    plan = type(pool.cache).plan

    def fail(self, *args, **kw):
        raise RuntimeError("out of memory")
    monkeypatch.setattr(type(pool.cache), "plan", fail)
    with pytest.raises(RuntimeError, match="memory"):
        pool.decode([other])
    assert pool.lengths == {row: 0, other: 3}
    # a batcher goes on where it was
    monkeypatch.setattr(PagedPool, "_capture", lambda self: setattr(self, "use_graph", False))
    eng = GenerationEngine(model)
    batcher = ContinuousBatcher(eng, max_batch=2, max_len=40, params=SamplingParams.from_mode("greedy"), page_size=4)
    rid = batcher.submit([5, 6, 7, 8, 9], 6)
    with pytest.raises(RuntimeError, match="memory"):
        batcher.step()
    monkeypatch.setattr(type(pool.cache), "plan", plan)
    while batcher.pending:
        batcher.step()
    want = eng.generate(torch.tensor([[5, 6, 7, 8, 9]]), SamplingParams.from_mode("greedy", max_new_tokens=6), use_graph=False)["tokens"][0].tolist()
    assert batcher.finished[rid].tokens == want


def test_neighbours_do_not_choose_how_a_request_is_drawn():
    """Requests without sampling numbers of their own draw the same tokens whether or not ones with numbers are served beside them, and the other way round."""
    eng = GenerationEngine(_model())
    loud = SamplingParams(temperature=6.0, top_k=0, top_p=1.0, repetition_penalty=1.0, max_new_tokens=12, seed=5)
    own = SamplingParams(temperature=4.0, top_k=60, top_p=0.95, repetition_penalty=1.0, max_new_tokens=12)

    def serve(kinds):
        batcher = ContinuousBatcher(eng, max_batch=3, max_len=40, params=loud, page_size=8)
        batcher.pool.use_graph = False
        rids = [batcher.submit([3, 1, 4, 1, 5], 12 if kind else 1, params=own if kind == "own" else None) for kind in kinds]   # (None: gone after its first token)
        while batcher.pending:
            batcher.step()
        return [batcher.finished[r].tokens for r in rids]
    both = serve(["plain", "own"])
    assert both[0] == serve(["plain"])[0] and len(set(both[0])) > 3
    assert both[1] == serve([None, "own"])[1] and len(set(both[1])) > 3


@torch.no_grad()
def test_rows_of_either_kind_are_drawn_by_their_own_sampler():
    eng = GenerationEngine(_model())
    params = SamplingParams(temperature=1.0, top_k=5, top_p=1.0, repetition_penalty=1.0, seed=2)
    batcher = ContinuousBatcher(eng, max_batch=6, max_len=16, params=params, page_size=8)
    logits = torch.zeros(6, 97)     # nothing but ties: the samplers' rules for them differ
    for slot in (1, 4):
        batcher._set_numbers(slot, SamplingParams(temperature=1.0, top_k=5, top_p=1.0, repetition_penalty=1.0))
    assert batcher._brings.tolist() == [False, True, False, False, True, False]
    state = batcher.generator.get_state()
    alone = batcher._sample(logits, slice(None), 0, 6)
    batcher.generator.set_state(state)
    mixed = batcher._sample(logits, slice(None), 2, 4)
    others = [0, 2, 3, 5]
    assert torch.equal(mixed[others], alone[others]) and (mixed[[1, 4]] < 5).all()
    batcher._set_numbers(4, None)
    assert batcher._brings.tolist() == [False, True, False, False, False, False]


def test_a_request_may_say_that_it_has_no_stop_tokens():
    eng = GenerationEngine(_model())
    batcher = ContinuousBatcher(eng, max_batch=2, max_len=40, params=SamplingParams.from_mode("greedy", stop_token_ids=None), page_size=8)
    batcher.pool.use_graph = False
    rids = [batcher.submit([1, 2, 3], 5), batcher.submit([1, 2, 3], params=SamplingParams.from_mode("greedy", stop_token_ids=None, max_new_tokens=5))]
    while batcher.pending:
        batcher.step()
    first, second = (batcher.finished[r].tokens for r in rids)
    assert first == second and len(first) == 5


@torch.no_grad()
def test_experts_drop_no_token_of_a_packed_batch():
    """An expert's room is counted per batch: prompts that fit it one by one would not together, and a request's logits would depend on its neighbours."""
    torch.manual_seed(0)
    cfg = ModelConfig(vocab_size=97, hidden_size=32, num_layers=2, num_heads=4, num_kv_heads=2, intermediate_size=64, seq_length=128, use_moe=True, num_experts=4,
                      moe_top_k=2, capacity_factor=0.25, routing_noise_std=0.0)
    model = DeepSeekTransformer(cfg).eval()
    g = torch.Generator().manual_seed(1)
    seqs = [torch.randint(0, 97, (100,), generator=g) for _ in range(6)]
    pool = PagedPool(model, 200, 128, pages=250, page_size=16, use_graph=False)
    rows = [pool.open(102) for _ in seqs]
    packed = pool.extend_many(list(zip(rows, seqs)))
    for s, got in zip(seqs, packed):
        assert torch.allclose(got, model(s[None], return_aux_loss=False)[0, -1], atol=2e-4)
    pool.last[rows] = torch.tensor([5] * 6)
    out = pool.decode(rows)          # 200 rows, 194 of them empty
    for r, s in zip(rows, seqs):
        assert torch.allclose(out[r], model(torch.cat([s, torch.tensor([5])])[None], return_aux_loss=False)[0, -1], atol=2e-4)


def test_a_request_may_ask_for_any_top_k():
    eng = GenerationEngine(_model())
    batcher = ContinuousBatcher(eng, max_batch=2, max_len=40, params=SamplingParams.from_mode("greedy", seed=1), page_size=8)
    batcher.pool.use_graph = False
    rids = [batcher.submit([1, 2, 3], params=SamplingParams(temperature=2.0, top_k=k, max_new_tokens=4)) for k in (1 << 40, -(1 << 40))]
    while batcher.pending:
        batcher.step()
    assert all(len(batcher.finished[r].tokens) == 4 for r in rids)
