"""Paged-cache operators on CPU tensors: the reference forms against dense attention, and refusals."""

import math

import pytest
import torch

from mint_b200.ops import attention, paged_attention, paged_plan, qk_norm_rope, qk_norm_rope_paged, rope_cos_sin


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("window,alibi", [(-1, False), (5, False), (-1, True), (0, True)])
def test_plan_append_attend_match_dense_decoding(window, alibi):
    torch.manual_seed(0)
    lens, page, hq, hkv, d = [7, 19, 1], 8, 4, 2, 16
    tables = torch.full((3, 4), -1, dtype=torch.int32)
    free = torch.randperm(9).to(torch.int32)
    p = paged_plan(_i32(0, 0, 0), _i32(*lens), tables, free, _i32(0), page_size=page, n_tokens=sum(lens) + 2)
    assert p.ends.tolist() == [7, 26, 27] and p.seq_lens.tolist() == lens and int(p.free_head) == 5
    cos, sin = rope_cos_sin(32, d, 10000.0)
    qs, ks = 0.1 * torch.randn(d), 0.1 * torch.randn(d)
    x = torch.randn(sum(lens) + 2, (hq + 2 * hkv) * d)
    kp, vp = torch.full((9, hkv, page, d), float("nan")), torch.full((9, hkv, page, d), float("nan"))
    slopes = torch.rand(hq) if alibi else None
    q, k, v = qk_norm_rope_paged(x, hq, hkv, d, qs, ks, cos, sin, p.positions, p.slots, kp, vp, return_kv=True)
    out = paged_attention(q, kp, vp, tables, p.positions, p.rows, window_left=window, alibi_slopes=slopes)
    assert not out[sum(lens) :].any() and not q[sum(lens) :].any()
    at = 0
    for n in lens:
        dq, dk, dv = qk_norm_rope(x[None, at : at + n], hq, hkv, d, qs, ks, cos, sin)
        bias = None
        if alibi:
            i = torch.arange(n)
            bias = slopes[None, :, None, None] * (i[None, :] - i[:, None]).float()
        want = attention(dq, dk, dv, causal=True, window_left=window, bias=bias)[0]
        torch.testing.assert_close(out[at : at + n], want, rtol=1e-5, atol=1e-5)
        at += n


def test_plan_grows_requests_page_by_page():
    tables = torch.full((2, 3), -1, dtype=torch.int32)
    free, head, seq = torch.arange(6, dtype=torch.int32), _i32(0), _i32(0, 0)
    want = []
    for _ in range(20):
        p = paged_plan(seq, _i32(1, 1), tables, free, head, page_size=8, n_tokens=2)
        head, seq = p.free_head, p.seq_lens
        want.append(p.slots.tolist())
    assert int(head) == 6 and sorted(s for r in want for s in r) == sorted(
        t * 8 + i for b in range(2) for j, t in enumerate(tables[b].tolist()) for i in range(8 if j < 2 else 4))
    with pytest.raises(ValueError, match="pages needed"):
        paged_plan(seq, _i32(5, 0), tables, free, head, page_size=8, n_tokens=5)


def test_refusals():
    tables, seq = torch.zeros(2, 2, dtype=torch.int32), _i32(3, 4)
    free = torch.arange(4, dtype=torch.int32)
    for bad in (4, 12, 0, 2048):
        with pytest.raises(ValueError, match="page size"):
            paged_plan(seq, seq, tables, free, _i32(0), page_size=bad, n_tokens=7)
    with pytest.raises(ValueError, match="negative"):
        paged_plan(seq, _i32(-1, 0), tables, free, _i32(0), page_size=8, n_tokens=7)
    with pytest.raises(ValueError, match="n_tokens"):
        paged_plan(seq, _i32(1, 1), tables, free, _i32(0), page_size=8, n_tokens=1)
    with pytest.raises(ValueError, match="block_tables"):
        paged_plan(seq, _i32(14, 0), tables, free, _i32(0), page_size=8, n_tokens=14)
    kp = torch.zeros(3, 2, 8, 16)
    q = torch.randn(2, 4, 16)
    with pytest.raises(ValueError, match="fit"):
        paged_attention(torch.randn(2, 3, 16), kp, kp, tables, seq)
    with pytest.raises(ValueError, match="one row per query"):
        paged_attention(torch.randn(3, 4, 16), kp, kp, tables, _i32(1, 2, 3))
    with pytest.raises(ValueError, match="pages are"):
        paged_attention(q.bfloat16(), kp, kp, tables, seq)
    with pytest.raises(ValueError, match="beyond the pool"):
        paged_attention(q, kp, kp, tables + 3, seq)
    with pytest.raises(RuntimeError, match="no gradient"):
        paged_attention(q.clone().requires_grad_(), kp, kp, tables, seq)
    x = torch.randn(2, 8 * 16)
    one = torch.zeros(16)
    with pytest.raises(ValueError, match="qkv must be"):
        qk_norm_rope_paged(x, 4, 1, 16, one, one, None, None, seq, seq, kp, kp)
    with pytest.raises(ValueError, match="rotation table"):
        qk_norm_rope_paged(x, 4, 2, 16, one, one, torch.ones(4, 8), torch.ones(4, 8), seq, seq, kp, kp)
    with pytest.raises(ValueError, match="slot beyond"):
        qk_norm_rope_paged(x, 4, 2, 16, one, one, None, None, seq, seq + 21, kp, kp)
    with pytest.raises(RuntimeError, match="no gradient"):
        qk_norm_rope_paged(x.clone().requires_grad_(), 4, 2, 16, one, one, None, None, seq, seq, kp, kp)


def test_default_scale():
    kp = torch.randn(1, 1, 8, 16)
    q = torch.randn(1, 1, 16)
    a = paged_attention(q, kp, kp, torch.zeros(1, 1, dtype=torch.int32), _i32(5))
    b = paged_attention(q, kp, kp, torch.zeros(1, 1, dtype=torch.int32), _i32(5), scale=1 / math.sqrt(16))
    assert torch.equal(a, b)
