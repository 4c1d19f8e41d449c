"""Paged attention at the ends of its ranges: fp16 weights far below the largest, infinite values.

Tolerances. As for ordinary inputs (tests/kernels/test_paged.py): one rounding to the output type (half of its eps
times |out|; half of the smallest subnormal, 2^-25, where an fp16 output is subnormal) and 2^-11 of sum p|v|. The
scores here are single products of fp16 numbers and exact, at most 18 below the largest: exp(-18) is above 2^-26."""

import math

import pytest
import torch

from mint_b200.ops import _ext, paged_attention

pytestmark = pytest.mark.gpu

U = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16)}
HEADS = [(4, 4), (8, 2), (8, 1), (12, 1)]  # groups of 1 and 4 (one block, twice), 8, 12 (two blocks)


@pytest.fixture(autouse=True)
def _clean_status():
    _ext.reset_fallbacks()
    yield
    assert not _ext.fallback_counts()
    _ext.check_device_status()


def _call(q, k, v, scale, page=16):
    """q [N, Hq, D] at the last of n keys k, v [n, Hkv, D], pages in reverse order."""
    n, hkv, d = k.shape
    count = -(-n // page)
    pools = []
    for t in (k, v):
        full = torch.full((count * page, hkv, d), float("nan"), dtype=t.dtype)
        full[:n] = t
        pools.append(full.view(count, page, hkv, d).transpose(1, 2).flip(0).contiguous().cuda())
    i32 = {"dtype": torch.int32, "device": "cuda"}
    table = torch.arange(count - 1, -1, -1, **i32)[None]
    rows = torch.zeros(q.shape[0], **i32)
    return paged_attention(q.cuda(), *pools, table, torch.full_like(rows, n - 1), rows, scale=scale).cpu()


def _oracle(q, k, v, scale):
    g = q.shape[1] // k.shape[1]
    kk, vv = k.double().repeat_interleave(g, 1), v.double().repeat_interleave(g, 1)
    p = torch.softmax(torch.einsum("nhd,khd->nhk", q.double(), kk) * scale, -1)
    return torch.einsum("nhk,khd->nhd", p, vv), torch.einsum("nhk,khd->nhd", p, vv.abs())


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", HEADS)
@pytest.mark.parametrize("below", [12, 15, 17.5])
def test_fp16_weights_far_below_the_largest(dim, hq, hkv, below):
    """A few keys take nearly all the weight and have zero values, as attention sinks have: what is left of the
    output is the sum over the many others."""
    g = torch.Generator().manual_seed(dim + hq)
    n = 3000
    k, v = torch.zeros(n, hkv, dim), torch.rand(n, hkv, dim, generator=g) + 0.5
    k[:, :, 0] = -below + 0.5 * torch.rand(n, hkv, generator=g) - 0.25
    k[::16, :, 0], v[::16] = 0.0, 0.0
    k, v = k.half(), v.half()
    q = torch.zeros(2, hq, dim).half()
    q[:, :, 0] = 1.0
    got = _call(q, k, v, 1.0).double()
    want, mag = _oracle(q, k, v, 1.0)
    tol = U[torch.float16] * want.abs() + 2.0**-25 + 2.0**-11 * mag
    worst = ((got - want).abs() / mag).max().item()
    assert bool(((got - want).abs() <= tol).all()), f"off by {worst:.3g} of sum p|v|"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv", HEADS)
@pytest.mark.parametrize("n,at", [(1, 0), (64, 3), (200, 199), (1500, 700)])
def test_infinite_values_stay_infinite(dtype, hq, hkv, n, at):
    """An infinite value that a query sees makes its column infinite and no other."""
    g = torch.Generator().manual_seed(n)
    dim = 128
    k, v = (torch.randn(n, hkv, dim, generator=g).to(dtype) for _ in range(2))
    q = torch.randn(1, hq, dim, generator=g).to(dtype)
    want, mag = _oracle(q, k, v, dim**-0.5)
    v[at, :, 5], v[at, :, 64] = math.inf, -math.inf
    got = _call(q, k, v, dim**-0.5).double()
    assert bool((got[..., 5] == math.inf).all()) and bool((got[..., 64] == -math.inf).all())
    rest = [c for c in range(dim) if c not in (5, 64)]
    err = (got - want).abs()[..., rest]
    assert bool((err <= U[dtype] * want.abs()[..., rest] + 2.0**-11 * mag[..., rest] + 1e-7).all())
