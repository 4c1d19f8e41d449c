"""generate_batch does not return tokens that a kernel reported an error about."""

import pytest
import torch

from mint_b200.kvcache.paged import PagedKVCache
from mint_b200.models import gemma
from mint_b200.models.gemma import Gemma, GemmaConfig
from mint_b200.ops import _ext, paged_plan

pytestmark = pytest.mark.gpu


def test_a_reported_error_is_raised(monkeypatch):
    torch.manual_seed(0)
    cfg = GemmaConfig(embed_dim=256, hidden_dim=512, seq_length=128, vocab_size=1000, n_layers=2, n_heads=4, n_kv_heads=2,
                      head_dim=128, init_std=0.05)
    model = Gemma(cfg).cuda().eval()
    cache = PagedKVCache(2, 16, 16, 2, 128, max_batch=2, max_seq_len=64, dtype=torch.bfloat16, device="cuda")
    prompts = [torch.randint(0, 1000, (n,)) for n in (3, 20)]
    real = gemma._sample
    i32 = {"dtype": torch.int32, "device": "cuda"}

    def sample(*args):  # a plan with one page too few, next to a step: refused by the kernel's checks and recorded
        paged_plan(torch.zeros(1, **i32), torch.ones(1, **i32), torch.zeros(1, 1, **i32), torch.zeros(1, **i32),
                   torch.ones(1, **i32), page_size=16, n_tokens=1)
        return real(*args)

    with torch.autocast("cuda", dtype=torch.bfloat16):
        want = model.generate_batch(prompts, 5, temperature=0, cache=cache)
        monkeypatch.setattr(gemma, "_sample", sample)
        with pytest.raises(_ext.DeviceStatusError, match="bad kernel argument"):
            model.generate_batch(prompts, 5, temperature=0, cache=cache)
        monkeypatch.undo()
        assert cache.n_free_pages == 16
        assert all(torch.equal(a, b) for a, b in zip(want, model.generate_batch(prompts, 5, temperature=0, cache=cache)))
    _ext.check_device_status()
