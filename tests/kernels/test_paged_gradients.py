"""The paged operators refuse every operand that would need a gradient, and take it under no_grad."""

import pytest
import torch

from mint_b200.ops import paged_attention, qk_norm_rope_paged


def _attend(dev, dtype):
    i32 = {"dtype": torch.int32, "device": dev}
    f = {"dtype": dtype, "device": dev}
    return paged_attention, {"q": torch.randn(2, 4, 64, **f), "k_pages": torch.randn(3, 2, 8, 64, **f),
                             "v_pages": torch.randn(3, 2, 8, 64, **f), "block_tables": torch.zeros(2, 2, **i32),
                             "positions": torch.tensor([1, 2], **i32), "alibi_slopes": torch.rand(4, device=dev)}


def _append(dev, dtype):
    i32 = {"dtype": torch.int32, "device": dev}
    f = {"dtype": dtype, "device": dev}
    return qk_norm_rope_paged, {"qkv": torch.randn(2, 3 * 64, **f), "n_q": 1, "n_kv": 1, "head_dim": 64,
                                "q_scale": torch.zeros(64, device=dev), "k_scale": torch.zeros(64, device=dev),
                                "cos": torch.ones(4, 32, device=dev), "sin": torch.zeros(4, 32, device=dev),
                                "positions": torch.arange(2, **i32), "slots": torch.arange(2, **i32),
                                "k_pages": torch.randn(3, 1, 8, 64, **f), "v_pages": torch.randn(3, 1, 8, 64, **f)}


CASES = [(_attend, n) for n in ("q", "k_pages", "v_pages", "alibi_slopes")] + [
    (_append, n) for n in ("qkv", "q_scale", "k_scale", "cos", "sin", "k_pages", "v_pages")]


def _check(make, name, dev, dtype):
    op, args = make(dev, dtype)
    args[name].requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        op(**args)
    with torch.no_grad():
        op(**args)


@pytest.mark.parametrize("make,name", CASES)
def test_cpu(make, name):
    _check(make, name, "cpu", torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("make,name", CASES)
def test_cuda(make, name):
    _check(make, name, "cuda", torch.bfloat16)
