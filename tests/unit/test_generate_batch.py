"""Paged cache bookkeeping and ragged batch generation against one-at-a-time generation (CPU)."""

import pytest
import torch

from mint_b200.kvcache.paged import PagedKVCache
from mint_b200.models.gemma import Gemma, GemmaConfig

CFG = dict(embed_dim=64, hidden_dim=128, seq_length=48, vocab_size=100, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=16)


def _model(**over):
    torch.manual_seed(3)
    model = Gemma(GemmaConfig(**{**CFG, **over})).eval()
    with torch.no_grad():
        for p in model.parameters():
            p.normal_(0, 0.1)
    return model


def _prompts(*lens):
    g = torch.Generator().manual_seed(1)
    return [torch.randint(0, 100, (n,), generator=g) for n in lens]


@pytest.mark.parametrize("pos", ["rope", "linear_rope", "nope", "alibi"])
@pytest.mark.parametrize("max_batch", [1, 2, 8])
def test_matches_single_generation(pos, max_batch):
    model = _model(pos_embedding=pos)
    prompts = _prompts(1, 9, 17, 8, 30)
    got = model.generate_batch(prompts, 7, temperature=0, max_batch=max_batch, page_size=8)
    for p, g in zip(prompts, got):
        assert torch.equal(g, model.generate(p[None], 7, temperature=0, use_cache=True)[0])


def test_eos_sequence_limit_and_lists():
    model = _model()
    prompts = _prompts(5, 44, 48)
    free = [model.generate(p[None], 10, temperature=0, use_cache=True)[0] for p in prompts]
    got = model.generate_batch([p.tolist() for p in prompts], 10, temperature=0)
    assert all(torch.equal(a, b) for a, b in zip(got, free))
    eos = int(free[0][7])  # the third new token of the first prompt
    got = model.generate_batch(prompts, 10, temperature=0, eos_token_id=eos)
    for g, f, p in zip(got, free, prompts):
        new = f[len(p) :].tolist()
        stop = new.index(eos) + 1 if eos in new else len(new)
        assert torch.equal(g, f[: len(p) + stop])
    assert [len(o) for o in model.generate_batch(prompts, 0)] == [5, 44, 48]


def test_small_shared_cache_queues_prompts():
    model = _model()
    prompts = _prompts(9, 12, 3, 20)
    cache = PagedKVCache(2, 5, 8, 2, 16, max_batch=3, max_seq_len=32)
    got = model.generate_batch(prompts, 6, temperature=0, cache=cache)
    assert cache.n_free_pages == 5 and cache.lens == [0, 0, 0] and sorted(cache.free_pages.tolist()) == list(range(5))
    for p, g in zip(prompts, got):
        assert torch.equal(g, model.generate(p[None], 6, temperature=0, use_cache=True)[0])
    with pytest.raises(ValueError, match="too small"):
        model.generate_batch(_prompts(40), 8, cache=PagedKVCache(2, 5, 8, 2, 16, max_batch=1, max_seq_len=48))


def test_follow_up_prompts_use_the_cached_ones():
    """A second turn: more tokens for a request that has some, next to a new request."""
    model = _model()
    a, b = _prompts(13, 6)
    cache = PagedKVCache(2, 8, 8, 2, 16, max_batch=2, max_seq_len=32)
    with torch.no_grad():
        step = cache.plan([7])
        model(a[None, :7], kv_caches=step.layers)
        step = cache.plan([6, 6], n_tokens=14)
        out = model(torch.cat([a[7:], b, b[:2]])[None], kv_caches=step.layers)[0]
        torch.testing.assert_close(out[:6], model(a[None])[0, 7:], rtol=1e-4, atol=1e-4)
        torch.testing.assert_close(out[6:12], model(b[None])[0], rtol=1e-4, atol=1e-4)


def test_cache_refusals_leave_it_unchanged():
    cache = PagedKVCache(1, 3, 8, 2, 16, max_batch=2, max_seq_len=24)
    cache.plan([9])
    before = (cache.lens[:], cache.n_free_pages, cache.block_tables.clone(), int(cache.free_head))
    for bad, match in (([0, 9], "pages needed"), ([16], "max_seq_len"), ([1, 1, 1], "at most 2"), ([-1], "non-negative")):
        with pytest.raises(ValueError, match=match):
            cache.plan(bad)
    with pytest.raises(ValueError, match="n_tokens"):
        cache.plan([2], n_tokens=1)
    assert before[:2] == (cache.lens, cache.n_free_pages) and torch.equal(before[2], cache.block_tables)
    cache.release([0])
    assert cache.n_free_pages == 3 and int(cache.free_head) == 0 and sorted(cache.free_pages.tolist()) == [0, 1, 2]
    cache.plan([24])
    cache.reset()
    assert cache.n_free_pages == 3 and cache.lens == [0, 0]
    for kw in ({"page_size": 12}, {"n_pages": 0}):
        with pytest.raises(ValueError):
            PagedKVCache(**{"n_layers": 1, "n_pages": 2, **kw})


def test_model_refusals():
    with pytest.raises(ValueError, match="positions"):
        _model(pos_embedding="sinusoidal").generate_batch(_prompts(4), 2)
    model = _model()
    for bad in ([[]], [torch.zeros(49, dtype=torch.int64)]):
        with pytest.raises(ValueError, match="1 to 48"):
            model.generate_batch(bad, 2)
    step = PagedKVCache(2, 4, 8, 2, 16, max_batch=2, max_seq_len=16).plan([4, 4])
    with pytest.raises(ValueError, match="one row"), torch.no_grad():
        model(torch.zeros(2, 4, dtype=torch.int64), kv_caches=step.layers)


def test_tensor_parallel_models_are_refused():
    from mint_b200.parallel.tp import TPInfo

    model = _model()
    tp = TPInfo(**{"group": None, "rank": 0, "size": 2, "sp": False})
    model.tp = tp
    with pytest.raises(ValueError, match="tensor parallel"):
        model.generate_batch(_prompts(4), 2)
    model.tp = None
    model.blocks[0].gqa.tp = tp
    step = PagedKVCache(2, 4, 8, 2, 16, max_batch=1, max_seq_len=16).plan([4])
    with pytest.raises(ValueError, match="tensor parallel"), torch.no_grad():
        model(torch.zeros(1, 4, dtype=torch.int64), kv_caches=step.layers)
