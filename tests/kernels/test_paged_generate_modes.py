"""generate_batch on the GPU under inference mode."""

import pytest
import torch

from mint_b200.models.gemma import Gemma, GemmaConfig
from mint_b200.ops import _ext

pytestmark = pytest.mark.gpu


def _model():
    torch.manual_seed(0)
    cfg = GemmaConfig(embed_dim=256, hidden_dim=512, seq_length=256, vocab_size=1000, n_layers=2, n_heads=4, n_kv_heads=2,
                      head_dim=128, init_std=0.05)
    return Gemma(cfg).cuda().eval()


PROMPTS = [torch.randint(0, 1000, (n,), generator=torch.Generator().manual_seed(n)) for n in (1, 40, 7, 65)]


def test_inference_mode_changes_nothing():
    model = _model()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        want = model.generate_batch(PROMPTS, 12, temperature=0)
        with torch.inference_mode():
            got = model.generate_batch(PROMPTS, 12, temperature=0)
        again = model.generate_batch(PROMPTS, 12, temperature=0)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, again))
    _ext.check_device_status()
