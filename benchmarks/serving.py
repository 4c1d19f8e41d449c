#!/usr/bin/env python
"""Ragged batch generation on one GPU: ``Gemma.generate_batch`` over the paged cache (prompts packed,
decoding in a CUDA graph) against ``Gemma.generate`` one prompt at a time over the dense cache.

    python benchmarks/serving.py                                   # 12-layer model, 32 prompts
    python benchmarks/serving.py --prompts 8 --new 64 --heads 16 --kv-heads 4 --embed 2048 --hidden 8192 --layers 24

Random weights and prompts (bf16 autocast); prompt lengths are spread evenly over 1 .. ``--longest``. Times are
wall clock around whole calls that return their tokens, after one warm-up call.
"""

from __future__ import annotations

import argparse
import json
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from mint_b200.models.gemma import Gemma, GemmaConfig  # noqa: E402


def timed(fn) -> float:  # noqa: ANN001
    fn()
    torch.cuda.synchronize()
    t = time.perf_counter()
    fn()
    torch.cuda.synchronize()
    return time.perf_counter() - t


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--prompts", type=int, default=32)
    p.add_argument("--longest", type=int, default=1024)
    p.add_argument("--new", type=int, default=128)
    p.add_argument("--embed", type=int, default=768)
    p.add_argument("--hidden", type=int, default=3072)
    p.add_argument("--layers", type=int, default=12)
    p.add_argument("--heads", type=int, default=6)
    p.add_argument("--kv-heads", type=int, default=6)
    p.add_argument("--seq", type=int, default=2048)
    p.add_argument("--single", type=int, default=4, help="prompts timed one at a time")
    a = p.parse_args()
    torch.manual_seed(0)
    cfg = GemmaConfig(embed_dim=a.embed, hidden_dim=a.hidden, seq_length=a.seq, vocab_size=65536, n_layers=a.layers,
                      n_heads=a.heads, n_kv_heads=a.kv_heads, head_dim=128, init_std=0.02)
    model = Gemma(cfg).cuda().eval()
    lens = [1 + (a.longest - 1) * i // max(1, a.prompts - 1) for i in range(a.prompts)]
    prompts = [torch.randint(0, 65536, (n,)) for n in lens]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        batch = timed(lambda: model.generate_batch(prompts, a.new, temperature=0, max_batch=a.prompts))
        eager = timed(lambda: model.generate_batch(prompts, a.new, temperature=0, max_batch=a.prompts, cuda_graph=False))
        some = prompts[:: max(1, a.prompts // a.single)][: a.single]
        single = timed(lambda: [model.generate(q[None].cuda(), a.new, temperature=0, use_cache=True) for q in some])
    print(json.dumps({
        "prompts": a.prompts, "new_tokens": a.new, "longest_prompt": a.longest,
        "batch_tok_s": a.prompts * a.new / batch, "batch_no_graph_tok_s": a.prompts * a.new / eager,
        "one_at_a_time_tok_s": len(some) * a.new / single, "ms_per_step": batch / a.new * 1e3,
    }))


if __name__ == "__main__":
    main()
