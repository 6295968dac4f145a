"""Continuous batching over whole rows and over pages: requests of mixed lengths served to the end.

    python benchmarks/bench_serving.py [--layers 8] [--requests 160] [--rows 64] [--max-len 2048] [--pages 896]

The dense 1B shape with random weights, greedy.  Wall-clock from the first request's submission to the last one's end, the decode graphs captured before."""
import argparse
import os
import random
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from adaptivetrainingsystem_b200 import ops  # noqa: E402
from adaptivetrainingsystem_b200.config import ConfigPresets  # noqa: E402
from adaptivetrainingsystem_b200.inference import ContinuousBatcher, GenerationEngine, SamplingParams  # noqa: E402
from adaptivetrainingsystem_b200.models import DeepSeekTransformer  # noqa: E402


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--layers", type=int, default=8)
    ap.add_argument("--requests", type=int, default=160)
    ap.add_argument("--rows", type=int, default=64)
    ap.add_argument("--max-len", type=int, default=2048)
    ap.add_argument("--pages", type=int, default=896, help="pages of 64 tokens of the smaller pool")
    a = ap.parse_args()
    cfg = ConfigPresets.get("dense_1b", gradient_checkpointing=False, num_layers=a.layers).to_model_config()
    cfg.seq_length = max(cfg.seq_length, a.max_len)
    torch.manual_seed(0)
    with torch.device("cuda"):
        torch.set_default_dtype(torch.bfloat16)
        model = DeepSeekTransformer(cfg)
        torch.set_default_dtype(torch.float32)
    engine = GenerationEngine(model.eval())
    g = random.Random(0)
    prompts = [[g.randrange(cfg.vocab_size) for _ in range(g.randint(50, a.max_len * 3 // 4 - 36))] for _ in range(a.requests)]
    budgets = [g.randint(32, 256) for _ in prompts]
    for options in ({}, {"page_size": 64}, {"page_size": 64, "pages": a.pages}, {"prefill_chunk": 1024}, {"page_size": 64, "prefill_chunk": 1024}):
        batcher = ContinuousBatcher(engine, max_batch=a.rows, max_len=a.max_len, params=SamplingParams.from_mode("greedy"), **options)
        batcher.run(prompts[:8], 8)
        torch.cuda.synchronize()
        start = time.perf_counter()
        for p, n in zip(prompts, budgets):
            batcher.submit(p, n)
        while batcher.pending:
            batcher.step()
        torch.cuda.synchronize()
        seconds = time.perf_counter() - start
        held = sum(t.numel() * t.element_size() for t in batcher.cache.k + batcher.cache.v)
        print(f"{options}: {seconds:.2f} s, {sum(budgets) / seconds:,.0f} new tokens/s, cache {held / 1e9:.2f} GB", flush=True)
        del batcher
    ops.check_status()


if __name__ == "__main__":
    main()
