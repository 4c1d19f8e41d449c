"""A generate_batch call that is left by an error gives its rows and pages back (CPU)."""

import pytest
import torch

from mint_b200.kvcache.paged import PagedKVCache
from mint_b200.models import gemma
from mint_b200.models.gemma import Gemma, GemmaConfig

CFG = dict(embed_dim=64, hidden_dim=128, seq_length=48, vocab_size=100, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=16)


def _prompts(*lens):
    g = torch.Generator().manual_seed(1)
    return [torch.randint(0, 100, (n,), generator=g) for n in lens]


class Stop(Exception):
    pass


@pytest.fixture()
def model():
    torch.manual_seed(3)
    return Gemma(GemmaConfig(**CFG)).eval()


def _fail_at(monkeypatch, owner, name, call):
    calls = [0]
    real = getattr(owner, name)

    def wrapped(*a, **k):
        calls[0] += 1
        if calls[0] == call:
            raise Stop
        return real(*a, **k)

    monkeypatch.setattr(owner, name, wrapped)


@pytest.mark.parametrize("owner,name", [
    (gemma, "_sample"), (PagedKVCache, "plan_on_device"), (PagedKVCache, "advance"), (Gemma, "forward"),
])
@pytest.mark.parametrize("call", [1, 2, 3, 5])
def test_an_error_leaves_the_cache_as_it_was(model, monkeypatch, owner, name, call):
    prompts = _prompts(9, 12, 3, 20)
    cache = PagedKVCache(2, 7, 8, 2, 16, max_batch=3, max_seq_len=32)
    kept = _prompts(10)[0]  # a request of the caller's own
    with torch.no_grad():
        step = cache.plan([0, 10])
        model(kept[None], kv_caches=step.layers)
    lens, free = cache.lens[:], cache.n_free_pages
    want = model.generate_batch(prompts, 6, temperature=0, cache=cache)
    with monkeypatch.context() as m:
        _fail_at(m, owner, name, call)
        with pytest.raises(Stop):
            model.generate_batch(prompts, 6, temperature=0, cache=cache)
    assert cache.lens == lens == cache.seq_lens.tolist() and cache.n_free_pages == free
    used = cache.block_tables[1, :2].tolist()
    head = int(cache.free_head)
    assert cache.n_pages - head == free and sorted(cache.free_pages[head:].tolist() + used) == list(range(7))
    got = model.generate_batch(prompts, 6, temperature=0, cache=cache)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():  # the caller's request goes on
        step = cache.plan([0, 1])
        out = model(torch.tensor([[7]]), kv_caches=step.layers)[0]
        full = model(torch.cat([kept, torch.tensor([7])])[None])[0, -1:]
    torch.testing.assert_close(out, full, rtol=1e-4, atol=1e-4)
