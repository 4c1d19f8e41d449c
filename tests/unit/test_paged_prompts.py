"""Which attention the prompts of new requests run (CPU)."""

import importlib

import pytest
import torch

from mint_b200.kvcache.paged import PagedKVCache
from mint_b200.models.gemma import Gemma, GemmaConfig

dense_ops = importlib.import_module("mint_b200.ops.attention")  # the package has a function of that name


@pytest.mark.parametrize("pattern", ["SL", "L"])
def test_prompts_attend_one_by_one_without_a_kernel(pattern, monkeypatch):
    """No mask over all packed tokens: its size would grow with the square of everything that was admitted."""
    torch.manual_seed(3)
    model = Gemma(GemmaConfig(embed_dim=64, hidden_dim=128, seq_length=48, vocab_size=100, n_layers=2, n_heads=4,
                              n_kv_heads=2, head_dim=16, attention_pattern=pattern)).eval()
    lens = [9, 0, 17, 1, 30]
    prompts = [torch.randint(0, 100, (n,)) for n in lens]
    sizes = []
    real = dense_ops.build_mask

    def build_mask(q_len, k_len, *args, **kw):
        sizes.append((q_len, k_len))
        return real(q_len, k_len, *args, **kw)

    cache = PagedKVCache(2, 12, 8, 2, 16, max_batch=5, max_seq_len=48)
    with torch.no_grad():
        step = cache.plan(lens, n_tokens=sum(lens) + 3)
        packed = torch.cat([*prompts, torch.zeros(3, dtype=torch.int64)])
        with monkeypatch.context() as m:
            m.setattr(dense_ops, "build_mask", build_mask)
            out = model(packed[None], kv_caches=step.layers)[0]
        assert sizes == [(n, n) for n in lens if n] * 2
        end = 0
        for p in prompts:
            if len(p):
                torch.testing.assert_close(out[end : end + len(p)], model(p[None])[0], rtol=1e-4, atol=1e-4)
            end += len(p)


@pytest.mark.parametrize("dtype,head_dim,switch,want", [
    (torch.bfloat16, 128, "0", True), (torch.bfloat16, 64, "0", False), (torch.float16, 128, "0", False),
    (torch.float32, 128, "0", False), (torch.bfloat16, 128, "1", False),
])
def test_what_the_dense_kernel_takes(dtype, head_dim, switch, want, monkeypatch):
    monkeypatch.setenv("MINT_DISABLE_KERNELS", switch)
    assert dense_ops.has_kernel(dtype, head_dim) == want


@pytest.mark.parametrize("kw", [{"start_pos": 3}, {"doc_ids": torch.zeros(1, 4, dtype=torch.int32)},
                                {"attn_mask": torch.ones(1, 1, 4, 4, dtype=torch.bool)}])
def test_positions_masks_and_documents_next_to_a_step_are_refused(kw):
    model = Gemma(GemmaConfig(embed_dim=64, hidden_dim=128, seq_length=48, vocab_size=100, n_layers=2, n_heads=4,
                              n_kv_heads=2, head_dim=16)).eval()
    step = PagedKVCache(2, 4, 8, 2, 16, max_batch=1, max_seq_len=16).plan([4])
    with torch.no_grad(), pytest.raises(ValueError, match="positions and requests"):
        model(torch.zeros(1, 4, dtype=torch.int64), kv_caches=step.layers, **kw)
