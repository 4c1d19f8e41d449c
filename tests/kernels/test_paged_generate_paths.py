"""generate_batch on the GPU for head sizes without paged or dense kernels, and with the kernels switched off."""

import pytest
import torch

from mint_b200.models.gemma import Gemma, GemmaConfig
from mint_b200.ops import _ext

pytestmark = pytest.mark.gpu


def _model(**over):
    torch.manual_seed(0)
    cfg = dict(embed_dim=256, hidden_dim=512, seq_length=256, vocab_size=1000, n_layers=2, n_heads=4, n_kv_heads=2,
               head_dim=128, init_std=0.05)
    return Gemma(GemmaConfig(**{**cfg, **over})).cuda().eval()


def _prompts(*lens):
    g = torch.Generator().manual_seed(1)
    return [torch.randint(0, 1000, (n,), generator=g) for n in lens]


def _check_tokens(model, prompts, got, new, share):
    """Each token is the model's own choice, up to ``share`` of the largest logit."""
    for p, g in zip(prompts, got):
        assert len(g) == len(p) + new and torch.equal(g[: len(p)].cpu(), p)
        with torch.no_grad():
            logits = model(g[None, :-1])[0, len(p) - 1 :].float()
        short = logits.max(-1).values - logits.gather(-1, g[len(p) :, None])[:, 0]
        assert float(short.max()) <= share * float(logits.abs().max())


@pytest.mark.parametrize("over", [{}, {"head_dim": 32}, {"pos_embedding": "alibi"}])
def test_kernels_switched_off(over, monkeypatch):
    """fp32 (2^-24 a rounding; 10-bit tf32 products where torch uses them, 2^-10 each) is within 1 % of the largest
    logit, bf16 (ten roundings per layer and path) within 5 %."""
    monkeypatch.setenv("MINT_DISABLE_KERNELS", "1")
    model, prompts = _model(**over), _prompts(1, 40, 7, 65)
    _check_tokens(model, prompts, model.generate_batch(prompts, 6, temperature=0, max_batch=3), 6, 0.01)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = model.generate_batch(prompts, 6, temperature=0, max_batch=3)
        _check_tokens(model, prompts, got, 6, 0.05)


@pytest.mark.filterwarnings("ignore::RuntimeWarning")
def test_bf16_heads_without_a_paged_kernel():
    model, prompts = _model(head_dim=32), _prompts(1, 40, 7, 65)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = model.generate_batch(prompts, 6, temperature=0, max_batch=3)
        _check_tokens(model, prompts, got, 6, 0.05)


@pytest.mark.parametrize("head_dim", [64, 256])
@pytest.mark.parametrize("pattern", ["SL", "L"])
def test_prompts_of_other_head_sizes_run_kernels(head_dim, pattern):
    model, prompts = _model(head_dim=head_dim, attention_pattern=pattern), _prompts(1, 200, 33, 7, 129)
    _ext.reset_fallbacks()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = model.generate_batch(prompts, 10, temperature=0, max_batch=4)
        assert not _ext.fallback_counts()
        _check_tokens(model, prompts, got, 10, 0.05)
    _ext.check_device_status()
