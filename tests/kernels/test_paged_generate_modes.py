"""generate_batch on the GPU under inference mode and with adapters."""

import pytest
import torch

from mint_b200.models.gemma import Gemma, GemmaConfig
from mint_b200.ops import _ext
from mint_b200.sft.peft.lora import LoRA
from mint_b200.sft.peft.qlora import QLoRA

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


@pytest.mark.parametrize("adapter", [LoRA, QLoRA])
def test_models_with_adapters(adapter):
    model = _model()
    adapter.apply(model)
    model.cuda().eval()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = model.generate_batch(PROMPTS, 12, temperature=0)
        want = model.generate_batch(PROMPTS, 12, temperature=0, cuda_graph=False)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    _ext.check_device_status()
