"""generate_batch for a model that is not on the current device."""

import pytest
import torch

from mint_b200.models.gemma import Gemma, GemmaConfig

pytestmark = pytest.mark.gpu


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_model_on_another_device_than_the_current_one():
    torch.manual_seed(0)
    cfg = GemmaConfig(embed_dim=256, hidden_dim=512, seq_length=256, vocab_size=1000, n_layers=2, n_heads=4, n_kv_heads=2,
                      head_dim=128, init_std=0.05)
    model = Gemma(cfg).to("cuda:1").eval()
    prompts = [torch.randint(0, 1000, (n,)) for n in (3, 50, 17)]
    with torch.cuda.device(0):
        torch.cuda.graph(torch.cuda.CUDAGraph())  # makes the default capture stream, on device 0
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = model.generate_batch(prompts, 12, temperature=0)
        want = model.generate_batch(prompts, 12, temperature=0, cuda_graph=False)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
