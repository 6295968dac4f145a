"""The paged pool and the batcher on it, with the decode step replayed from a CUDA graph."""
import pytest
import torch

from adaptivetrainingsystem_b200.config import ModelConfig
from adaptivetrainingsystem_b200.inference import ContinuousBatcher, GenerationEngine, PagedPool, SamplingParams
from adaptivetrainingsystem_b200.models import DeepSeekTransformer

pytestmark = pytest.mark.gpu


def _model(moe=False, dtype=torch.bfloat16, heads=4, kv=2, hidden=256):
    torch.manual_seed(4)
    cfg = ModelConfig(vocab_size=512, hidden_size=hidden, num_layers=2, num_heads=heads, num_kv_heads=kv, intermediate_size=512, seq_length=256, use_moe=moe,
                      num_experts=4, moe_top_k=2, capacity_factor=4.0, routing_noise_std=0.0)
    model = DeepSeekTransformer(cfg).to("cuda", dtype).eval()
    with torch.no_grad():      # sharpen the next-token distribution so that greedy decoding has no near-ties
        model.lm_head.mul_(8.0)
    return model


@pytest.mark.parametrize("moe", [False, True])
@pytest.mark.parametrize("chunk", [None, 13])
def test_batcher_over_pages_matches_one_by_one_generation(moe, chunk):
    """More requests than rows, more rows than the pages would hold at full length."""
    eng = GenerationEngine(_model(moe))
    g = torch.Generator().manual_seed(1)
    lengths, budgets = [5, 17, 33, 8, 64, 21, 3, 40, 12], [12, 6, 9, 15, 4, 10, 14, 5, 8]
    prompts = [torch.randint(0, 512, (n,), generator=g) for n in lengths]
    batcher = ContinuousBatcher(eng, max_batch=6, max_len=128, params=SamplingParams.from_mode("greedy", max_new_tokens=16), prefill_chunk=chunk, page_size=16, pages=18)
    rids = [batcher.submit(p, b) for p, b in zip(prompts, budgets)]
    while batcher.pending:
        batcher.step()
    batcher.cache.pool.check()
    assert batcher.slots.available == 6 and batcher.pool.pages_left == 18 and int(batcher.cache.pool.state[0]) == 18
    same = 0
    for p, b, r in zip(prompts, budgets, rids):
        ref = eng.generate(p.view(1, -1).cuda(), SamplingParams.from_mode("greedy", max_new_tokens=b), use_graph=True)["tokens"][0].tolist()
        got = batcher.finished[r].tokens
        assert len(got) == b
        same += got == ref
        if not moe:
            assert got == ref, (len(p), ref, got)
    assert same >= 7, same         # a routing near-tie may flip a token of a MoE sequence; most must agree exactly


@pytest.mark.parametrize("heads,kv,hidden,dtype", [(4, 2, 256, torch.bfloat16), (4, 1, 512, torch.bfloat16), (4, 4, 96, torch.bfloat16), (4, 2, 256, torch.float32)])
@torch.no_grad()
def test_rows_equal_sequences_of_their_own(heads, kv, hidden, dtype):
    """Logits of packed portions and of replayed single-token steps against the whole sequence on its own, in 64 bits."""
    model = _model(dtype=dtype, heads=heads, kv=kv, hidden=hidden)
    plain = DeepSeekTransformer(model.config).double().eval()
    plain.load_state_dict({k: v.double() for k, v in model.state_dict().items()})
    pool = PagedPool(model, 4, 64, page_size=8)
    g = torch.Generator().manual_seed(3)
    seqs = [torch.randint(0, 512, (n,), generator=g) for n in (20, 50, 30)]
    rows, fed = [pool.open(n) for n in (20, 50, 30)], [1, 37, 12]
    got = list(pool.extend_many([(r, s[:n]) for r, s, n in zip(rows, seqs, fed)]).float())
    scale = float(plain(seqs[1][None], return_aux_loss=False).abs().max())
    # two layers of roundings: a few steps of the type of the largest logit (each layer adds four, the sum of their squares under the root)
    bound = 16 * torch.finfo(dtype).eps * scale if dtype == torch.bfloat16 else 1e-3 * scale
    for step in range(9):
        for i, s in enumerate(seqs):
            want = plain(s[None, :fed[i]], return_aux_loss=False)[0, -1]
            assert float((got[i].double().cpu() - want).abs().max()) <= bound, (step, i)
        live = [i for i in range(3) if (i + step) % 3]
        for i in live:
            pool.last[rows[i]] = int(seqs[i][fed[i]])
            fed[i] += 1
        out = pool.decode([rows[i] for i in live])
        for i in live:
            got[i] = out[rows[i]].float().clone()   # (the next step overwrites the buffer)
    pool.cache.pool.check()


def test_two_pools_of_one_model_replay_side_by_side():
    """Two captured steps on two streams share no memory of theirs."""
    model = _model()
    eng = GenerationEngine(model)
    prompts = [[7, 8, 9], [100, 3], [50] * 20, [11, 12]]
    alone = [ContinuousBatcher(eng, max_batch=4, max_len=64, page_size=16).run(prompts, 12) for _ in range(1)][0]
    batchers = [ContinuousBatcher(eng, max_batch=4, max_len=64, page_size=16) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    rids = []
    for b, s in zip(batchers, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            rids.append([b.submit(p, 12) for p in prompts])
    while any(b.pending for b in batchers):
        for b, s in zip(batchers, streams):
            with torch.cuda.stream(s):
                b.step()
    torch.cuda.synchronize()
    for b, r in zip(batchers, rids):
        assert [b.finished[i].tokens for i in r] == alone


def test_requests_with_numbers_of_their_own():
    model = _model()
    eng = GenerationEngine(model)
    batcher = ContinuousBatcher(eng, max_batch=4, max_len=64, params=SamplingParams.from_mode("greedy", seed=1), page_size=16)
    ids = [1, 2, 3]
    greedy = batcher.submit(ids, 10)
    sure = batcher.submit(ids, params=SamplingParams(temperature=3.0, top_k=1, repetition_penalty=1.0, max_new_tokens=10))
    tiny = batcher.submit(ids, params=SamplingParams(temperature=3.0, top_k=0, top_p=1.0, min_p=1.0, repetition_penalty=1.0, max_new_tokens=10))
    wild = batcher.submit(ids, params=SamplingParams(temperature=80.0, top_k=0, top_p=1.0, repetition_penalty=1.0, max_new_tokens=10))
    while batcher.pending:
        batcher.step()
    want = eng.generate(torch.tensor([ids], device="cuda"), SamplingParams.from_mode("greedy", max_new_tokens=10))["tokens"][0].tolist()
    assert batcher.finished[greedy].tokens == batcher.finished[sure].tokens == batcher.finished[tiny].tokens == want
    assert batcher.finished[wild].tokens != want


@torch.no_grad()
def test_rows_of_either_kind_are_drawn_by_their_own_sampler():
    """Rows without numbers of their own draw what they draw alone, beside rows with numbers, which draw what ``ops.sample_rows`` draws for all of them."""
    params = SamplingParams(temperature=1.0, top_k=20, top_p=0.9, repetition_penalty=1.1, seed=2)
    batcher = ContinuousBatcher(GenerationEngine(_model()), max_batch=8, max_len=64, params=params, page_size=16)
    logits = (2 * torch.randn(8, 512, device="cuda")).round().bfloat16()     # ties, for which the samplers have different rules
    for slot in (0, 3, 4):
        batcher._set_numbers(slot, SamplingParams(temperature=2.0, top_k=100, top_p=1.0, min_p=0.01, repetition_penalty=1.0))
    states = [g.get_state() for g in (batcher.generator, batcher.own_generator)]

    def draw(*counts):
        for g, s in zip((batcher.generator, batcher.own_generator), states):
            g.set_state(s)
        return batcher._sample(logits, slice(None), *counts)
    plain, own, mixed = draw(0, 8), draw(3, 0), draw(3, 5)
    rows = torch.tensor([True, False, False, True, True, False, False, False], device="cuda")
    assert torch.equal(mixed, torch.where(rows, own, plain)) and not torch.equal(own, plain)
    assert batcher.own_generator.get_state().equal(states[1]) is False


@torch.no_grad()
def test_a_capture_that_fails_is_made_again(monkeypatch):
    model = _model()
    pool, plain = PagedPool(model, 2, 64, page_size=16), PagedPool(model, 2, 64, page_size=16, use_graph=False)
    for p in (pool, plain):
        p.extend(p.open(40), [5, 6, 7])
        p.last[0] = 9
    decode, calls = PagedPool._decode, []

    def fail(self, *args):
        calls.append(1)
        if len(calls) == 3:
            raise RuntimeError("out of memory")
        return decode(self, *args)
    monkeypatch.setattr(PagedPool, "_decode", fail)
    with pytest.raises(RuntimeError, match="memory"):
        pool.decode([0])
    assert pool.lengths == {0: 3} and pool.cache.pool.lengths.tolist() == [3, 0]
    monkeypatch.undo()
    assert torch.equal(pool.decode([0])[0], plain.decode([0])[0]) and pool.lengths == {0: 4}
