"""The NF4 levels are copied to a device once and stay usable outside inference mode."""

import torch

from mint_b200.sft.peft.qlora import NF4_LEVELS, _levels, nf4_dequantize, nf4_quantize


def test_levels_are_kept_per_device():
    dev = torch.device("cpu")
    with torch.inference_mode():
        first = _levels(dev)
    assert first is _levels(dev) and not first.is_inference() and torch.equal(first, NF4_LEVELS)
    w = NF4_LEVELS.repeat(4, 4) * 0.5
    torch.testing.assert_close(nf4_dequantize(nf4_quantize(w)), w, rtol=0.0, atol=1e-6)
