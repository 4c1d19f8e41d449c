"""Operands that the append kernel's 16-byte loads could not read are refused before any launch."""

import pytest
import torch

from mint_b200.ops import _ext, qk_norm_rope_paged

pytestmark = pytest.mark.gpu


def _args(dim=128, n=3):
    i32 = {"dtype": torch.int32, "device": "cuda"}
    bf16 = {"dtype": torch.bfloat16, "device": "cuda"}
    f32 = {"dtype": torch.float32, "device": "cuda"}
    return {
        "qkv": torch.randn(n, 3 * dim, **bf16), "n_q": 1, "n_kv": 1, "head_dim": dim,
        "q_scale": torch.zeros(dim, **f32), "k_scale": torch.zeros(dim, **f32),
        "cos": torch.ones(8, dim // 2, **f32), "sin": torch.zeros(8, dim // 2, **f32),
        "positions": torch.arange(n, **i32), "slots": torch.arange(n, **i32),
        "k_pages": torch.zeros(2, 1, 16, dim, **bf16), "v_pages": torch.zeros(2, 1, 16, dim, **bf16),
    }


def _shifted(t, by):
    """The same values, contiguous, ``by`` elements into a larger buffer."""
    flat = torch.zeros(t.numel() + by, dtype=t.dtype, device=t.device)
    out = flat[by:].view(t.shape)
    out.copy_(t)
    assert out.is_contiguous()
    return out


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("name", ["q_scale", "k_scale", "cos", "sin"])
@pytest.mark.parametrize("by", [1, 2, 3])
def test_misaligned_scales_and_tables_are_refused(dim, name, by):
    args = _args(dim)
    args[name] = _shifted(args[name], by)
    before = _ext.require().launch_count()
    with pytest.raises(RuntimeError, match=f"{name} must be 16-byte aligned"):
        qk_norm_rope_paged(**args)
    assert _ext.require().launch_count() == before


def test_a_view_on_a_16_byte_boundary_is_taken():
    args = _args()
    want = qk_norm_rope_paged(**args)
    for name in ("q_scale", "k_scale", "cos", "sin"):
        args[name] = _shifted(args[name], 4)
    assert torch.equal(qk_norm_rope_paged(**args), want)
    _ext.check_device_status()


def test_empty_rotation_tables_are_refused():
    args = _args()
    args["cos"], args["sin"] = args["cos"][:0], args["sin"][:0]
    before = _ext.require().launch_count()
    with pytest.raises(RuntimeError, match="one position at least"):
        qk_norm_rope_paged(**args)
    assert _ext.require().launch_count() == before
