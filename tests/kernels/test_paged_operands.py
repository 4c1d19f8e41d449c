"""Operands of the paged operators that are easy to get half right."""

import pytest
import torch

from mint_b200.ops import paged_attention, qk_norm_rope_paged


def _append(dev, dtype, **over):
    i32 = {"dtype": torch.int32, "device": dev}
    f = {"dtype": dtype, "device": dev}
    args = {"qkv": torch.randn(1, 3 * 64, **f), "n_q": 1, "n_kv": 1, "head_dim": 64,
            "q_scale": torch.zeros(64, device=dev), "k_scale": torch.zeros(64, device=dev),
            "cos": torch.ones(4, 32, device=dev), "sin": torch.zeros(4, 32, device=dev),
            "positions": torch.arange(1, **i32), "slots": torch.arange(1, **i32),
            "k_pages": torch.randn(3, 1, 8, 64, **f), "v_pages": torch.randn(3, 1, 8, 64, **f)}
    return qk_norm_rope_paged(**{**args, **over})


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("missing", ["cos", "sin"])
def test_half_a_rotation_is_refused(dev, missing):
    """cos without sin, or sin without cos, which was taken for no rotation."""
    with pytest.raises(ValueError, match="both cos and sin"):
        _append(dev, torch.bfloat16, **{missing: None})


@pytest.mark.gpu
def test_one_token_may_have_any_row_stride():
    wide = torch.randn(1, 3 * 64 + 3, device="cuda", dtype=torch.bfloat16)
    row = wide[:, : 3 * 64]
    assert row.stride(0) % 8
    assert torch.equal(_append("cuda", torch.bfloat16, qkv=row), _append("cuda", torch.bfloat16, qkv=row.contiguous()))


def test_positions_beyond_the_table_are_refused():
    """They were answered with the keys that the table does have."""
    i32 = {"dtype": torch.int32}
    pool = torch.randn(3, 2, 8, 16)
    q = torch.randn(2, 4, 16)
    table = torch.tensor([[0, 1], [2, 0]], **i32)
    assert paged_attention(q, pool, pool, table, torch.tensor([15, -1], **i32))[0].any()
    with pytest.raises(ValueError, match="beyond block_tables"):
        paged_attention(q, pool, pool, table, torch.tensor([16, 3], **i32))
