"""Ragged batch generation on the GPU: bf16 kernels, paged cache, decoding in a CUDA graph.

Logits of the paged path and of a full forward differ by bf16 rounding: about ten roundings (2^-8 each, of
independent sign) per layer and path, below 5 % of the largest logit for the two layers here."""

import pytest
import torch

from mint_b200.kvcache.paged import PagedKVCache
from mint_b200.models.gemma import Gemma, GemmaConfig
from mint_b200.ops import _ext

pytestmark = pytest.mark.gpu


def _model(**over):
    torch.manual_seed(0)
    cfg = dict(embed_dim=256, hidden_dim=512, seq_length=512, vocab_size=1000, n_layers=2, n_heads=4, n_kv_heads=2,
               head_dim=128, init_std=0.05)
    return Gemma(GemmaConfig(**{**cfg, **over})).cuda().eval()


def _prompts(*lens):
    g = torch.Generator().manual_seed(1)
    return [torch.randint(0, 1000, (n,), generator=g) for n in lens]


@pytest.mark.parametrize("over", [{}, {"n_kv_heads": 4}, {"pos_embedding": "alibi"}, {"head_dim": 64, "n_kv_heads": 1},
                                  {"pos_embedding": "nope", "attention_pattern": "L"}])
def test_tokens_are_the_models_own(over):
    model = _model(**over)
    prompts = _prompts(1, 200, 33, 7, 129, 64, 300)
    _ext.reset_fallbacks()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = model.generate_batch(prompts, 40, temperature=0, max_batch=4)
        counts = _ext.fallback_counts()
        again = model.generate_batch(prompts, 40, temperature=0, max_batch=4, cuda_graph=False)
        for p, g, a in zip(prompts, got, again):
            assert len(g) == len(p) + 40 and torch.equal(g[: len(p)].cpu(), p) and torch.equal(g, a)
            with torch.no_grad():
                logits = model(g[None, :-1])[0, len(p) - 1 :].float()
            short = logits.max(-1).values - logits.gather(-1, g[len(p) :, None])[:, 0]
            assert float(short.max()) <= 0.05 * float(logits.abs().max())
    if over.get("head_dim", 128) == 128:  # prompts of other head sizes run the dense attention's PyTorch code
        assert not counts, counts
    _ext.check_device_status()


def test_sampling_and_reuse_of_a_cache():
    model = _model()
    cache = PagedKVCache(2, 64, 16, 2, 128, max_batch=3, max_seq_len=256, dtype=torch.bfloat16, device="cuda")
    prompts = _prompts(5, 70, 20, 11)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        first = model.generate_batch(prompts, 12, temperature=0, cache=cache)
        torch.manual_seed(1)
        drawn = model.generate_batch(prompts, 12, temperature=0.8, top_k=20, top_p=0.9, cache=cache)
        second = model.generate_batch(prompts, 12, temperature=0, cache=cache)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    assert all(len(d) == len(f) for d, f in zip(drawn, first))
    assert cache.n_free_pages == 64 and int(cache.free_head) == 0
    _ext.check_device_status()
