"""Paged key-value cache operators for serving ragged batches.

A cache layer is two pools ``k_pages`` and ``v_pages`` of shape ``[pages, Hkv, page_size, D]`` (any
strides with a contiguous last dimension: a ``[pages, page_size, Hkv, D]`` pool is passed as
``pool.transpose(1, 2)``). ``page_size`` is a power of two from 8 to 1024. Request ``b``'s key ``j``
lives on line ``j % page_size`` of page ``block_tables[b, j // page_size]``; *slot*
``page * page_size + line`` names that place.

A step packs the new tokens of all requests into one row of ``n_tokens`` tokens:

* :func:`paged_plan` hands out pages and returns each token's position, slot and request,
* :func:`qk_norm_rope_paged` normalizes and rotates q and k and stores k and v into the slots,
* :func:`paged_attention` lets every token attend to its request's keys.

A position of ``-1`` marks a padding token (nothing is stored for it, its outputs are zero), so the
shapes of a decoding step stay fixed while requests come and go. The operators are for inference: they
raise when a gradient would be needed. CUDA tensors run the kernels in
``mint_b200/csrc/paged_cache.cu`` and ``mint_b200/csrc/paged_attention.cu``; the reference has a dense
cache of equal lengths only (mint/kvcache/base.py:4-65).
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from mint_b200.ops import _ext
from mint_b200.ops.norm import _rms_ref
from mint_b200.ops.rope import _rotate_ref

_HEAD_DIMS = (64, 128, 256)
_KERNEL_DTYPES = (torch.bfloat16, torch.float16)


class PagedPlan(NamedTuple):
    """One step's packed tokens (all int32): token ``i`` has position ``positions[i]`` in request
    ``rows[i]`` and is stored in ``slots[i]``; the tokens of request ``b`` end before ``ends[b]``."""

    positions: torch.Tensor
    slots: torch.Tensor
    rows: torch.Tensor
    ends: torch.Tensor
    seq_lens: torch.Tensor
    free_head: torch.Tensor


def has_kernels(dtype: torch.dtype, head_dim: int) -> bool:
    """Whether append and attention of CUDA tensors run kernels, which never wait for the host, or PyTorch code."""
    return _ext.kernels_enabled() and dtype in _KERNEL_DTYPES and head_dim in _HEAD_DIMS


def _inference_only(op: str, *tensors: torch.Tensor | None) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"mint_b200: {op} has no gradient; call it under torch.no_grad()")


def check_page_size(page_size: int) -> None:
    if page_size < 8 or page_size > 1024 or page_size & (page_size - 1):
        raise ValueError(f"the page size must be a power of two from 8 to 1024, got {page_size}")


def _plan_ref(seq_lens, new_lens, block_tables, free_pages, free_head, page_size, n_tokens):  # noqa: ANN001, ANN202
    seq, new = seq_lens.long(), new_lens.long()
    if bool((seq < 0).any()) or bool((new < 0).any()):
        raise ValueError("paged_plan: negative length")
    have = (seq + page_size - 1) // page_size
    total = (seq + new + page_size - 1) // page_size
    need = total - have
    head, n_need, n_new = int(free_head), int(need.sum()), int(new.sum())
    if head < 0 or head + n_need > free_pages.numel():
        raise ValueError(f"paged_plan: {n_need} pages needed, {free_pages.numel() - head} free")
    if n_new > n_tokens:
        raise ValueError(f"paged_plan: {n_new} new tokens do not fit n_tokens={n_tokens}")
    if seq.numel() and int(total.max()) > block_tables.shape[1]:
        raise ValueError(f"paged_plan: a request needs {int(total.max())} pages, block_tables has {block_tables.shape[1]}")
    rows = torch.repeat_interleave(torch.arange(seq.numel(), device=seq.device), new)
    ends = torch.cumsum(new, 0)
    fresh = torch.repeat_interleave(torch.arange(seq.numel(), device=seq.device), need)
    k = torch.arange(n_need, device=seq.device)
    col = have[fresh] + k - (torch.cumsum(need, 0) - need)[fresh]
    block_tables[fresh, col] = free_pages[head : head + n_need]
    pos = seq[rows] + torch.arange(n_new, device=seq.device) - (ends - new)[rows]
    slots = block_tables[rows, pos // page_size].long() * page_size + pos % page_size
    out = torch.full((3, n_tokens), -1, dtype=torch.int32, device=seq.device)
    out[:, :n_new] = torch.stack([pos, slots, rows]).to(torch.int32)
    return PagedPlan(out[0], out[1], out[2], ends.to(torch.int32), (seq + new).to(torch.int32),
                     (free_head + n_need).to(torch.int32))


def paged_plan(
    seq_lens: torch.Tensor,
    new_lens: torch.Tensor,
    block_tables: torch.Tensor,
    free_pages: torch.Tensor,
    free_head: torch.Tensor,
    *,
    page_size: int,
    n_tokens: int,
) -> PagedPlan:
    """Plan one step in which request ``b`` grows from ``seq_lens[b]`` by ``new_lens[b]`` tokens.

    Requests that need more pages get them, in request order, from ``free_pages[free_head:]``; the new
    entries are written into ``block_tables`` ([B, W], in place), nothing else is changed. All tensors
    are int32. ``n_tokens`` is the packed length, at least ``new_lens.sum()``: tokens beyond the sum are
    padding (position, slot and row -1). Calling it again with the same arguments gives the same result.

    CUDA: one kernel, no host synchronization. What cannot be placed (no page left, a request longer than
    its table row, more new tokens than ``n_tokens``) gets slot -1 and "bad kernel argument" in the
    device status word; CPU tensors raise ValueError."""
    if _ext.use_cuda_kernels(seq_lens):
        return PagedPlan(*_ext.require().paged_plan(seq_lens, new_lens, block_tables, free_pages, free_head,
                                                    page_size, n_tokens))
    check_page_size(page_size)
    return _plan_ref(seq_lens, new_lens, block_tables, free_pages, free_head, page_size, n_tokens)


def _append_ref(qkv, n_q, n_kv, head_dim, q_scale, k_scale, cos, sin, positions, slots, k_pages, v_pages, eps):  # noqa: ANN001, ANN202
    n, page_size = qkv.shape[0], k_pages.shape[2]
    x = qkv.view(n, n_q + 2 * n_kv, head_dim)
    q = _rms_ref(x[:, :n_q], q_scale, eps, None)
    k = _rms_ref(x[:, n_q : n_q + n_kv], k_scale, eps, None)
    pos = positions.long()
    live = pos >= 0
    if cos is not None:
        if bool((pos >= cos.shape[0]).any()):
            raise ValueError(f"qk_norm_rope_paged: position {int(pos.max())} is beyond the rotation table ({cos.shape[0]})")
        c, s = cos[pos.clamp(min=0)][:, None, :], sin[pos.clamp(min=0)][:, None, :]
        q, k = _rotate_ref(q, c, s), _rotate_ref(k, c, s)
    drop = ~live[:, None, None]
    q = q.masked_fill(drop, 0).to(qkv.dtype)
    k = k.masked_fill(drop, 0).to(qkv.dtype)
    v = x[:, n_q + n_kv :].masked_fill(drop, 0)
    slot = slots.long()
    if bool((slot >= k_pages.shape[0] * page_size).any()):
        raise ValueError("qk_norm_rope_paged: slot beyond the pool")
    keep = live & (slot >= 0)
    at = slot[keep]
    k_pages[at // page_size, :, at % page_size] = k[keep].to(k_pages.dtype)
    v_pages[at // page_size, :, at % page_size] = v[keep].to(v_pages.dtype)
    return q, k, v


def qk_norm_rope_paged(
    qkv: torch.Tensor,
    n_q: int,
    n_kv: int,
    head_dim: int,
    q_scale: torch.Tensor,
    k_scale: torch.Tensor,
    cos: torch.Tensor | None,
    sin: torch.Tensor | None,
    positions: torch.Tensor,
    slots: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    eps: float = 1e-6,
    *,
    return_kv: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """QK-RMSNorm and rotation of the packed projection ``qkv`` ([N, (n_q + 2 n_kv) D]) at per-token
    positions; k and v go straight into their slots of ``k_pages`` / ``v_pages``. Returns
    ``q`` [N, n_q, D], with ``return_kv`` also k and v as [N, n_kv, D].

    ``cos`` / ``sin`` are fp32 ``[positions, D / 2]`` tables (half-split rotation), or None for no
    rotation. Norm and rotation are computed in fp32 and rounded once. A token with slot -1 is not
    stored; one whose position or slot is out of range is not stored either and is reported in the
    device status word (CPU tensors raise ValueError)."""
    if (cos is None) != (sin is None):
        raise ValueError("qk_norm_rope_paged: rotation needs both cos and sin")
    if _ext.use_cuda_kernels(qkv):
        if qkv.dtype in _KERNEL_DTYPES and head_dim in _HEAD_DIMS:
            if q_scale.dtype != torch.float32 or k_scale.dtype != torch.float32:
                q_scale, k_scale = q_scale.float(), k_scale.float()
            out = _ext.require().qk_norm_rope_paged(qkv, n_q, n_kv, head_dim, q_scale, k_scale, cos, sin, positions, slots,
                                                    k_pages, v_pages, eps, return_kv)
            return tuple(out) if return_kv else out[0]
        _ext.fallback("qk_norm_rope_paged", "dtype / head_dim without a kernel")
    _inference_only("qk_norm_rope_paged", qkv, q_scale, k_scale, cos, sin, k_pages, v_pages)
    if qkv.dim() != 2 or qkv.shape[1] != (n_q + 2 * n_kv) * head_dim:
        raise ValueError(f"qkv must be [N, {(n_q + 2 * n_kv) * head_dim}], got {tuple(qkv.shape)}")
    if k_pages.dtype != qkv.dtype or v_pages.dtype != qkv.dtype:
        raise ValueError(f"qkv is {qkv.dtype} but the pages are {k_pages.dtype} / {v_pages.dtype}")
    check_page_size(k_pages.shape[2])
    q, k, v = _append_ref(qkv, n_q, n_kv, head_dim, q_scale, k_scale, cos, sin, positions, slots, k_pages, v_pages, eps)
    return (q, k, v) if return_kv else q


def _attention_ref(q, k_pages, v_pages, block_tables, positions, rows, window_left, alibi_slopes, scale):  # noqa: ANN001, ANN202
    n, hq, d = q.shape
    n_pages, hkv, page_size = k_pages.shape[:3]
    rows = torch.arange(n, device=q.device) if rows is None else rows.long()
    pos = torch.where((rows >= 0) & (rows < block_tables.shape[0]), positions.long(), -1)
    out = torch.zeros_like(q)
    for i in range(n):  # one query at a time: memory stays at one request's keys
        last = int(pos[i])
        if last < 0:
            continue
        if last >= block_tables.shape[1] * page_size:
            raise ValueError(f"paged_attention: position {last} is beyond block_tables ({block_tables.shape[1]} pages)")
        first = max(0, last - window_left) if window_left >= 0 else 0
        j = torch.arange(first, last + 1, device=q.device)
        page = block_tables[rows[i], j // page_size].long()
        if bool((page < 0).any()) or bool((page >= n_pages).any()):
            raise ValueError("paged_attention: page beyond the pool")
        k = k_pages[page, :, j % page_size].float()
        v = v_pages[page, :, j % page_size].float()
        s = torch.einsum("hgd,khd->hgk", q[i].float().view(hkv, hq // hkv, d), k) * scale
        if alibi_slopes is not None:
            s = s - alibi_slopes.float().view(hkv, hq // hkv, 1) * (last - j).float()
        out[i] = torch.einsum("hgk,khd->hgd", torch.softmax(s, dim=-1), v).reshape(hq, d).to(q.dtype)
    return out


def paged_attention(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_tables: torch.Tensor,
    positions: torch.Tensor,
    rows: torch.Tensor | None = None,
    *,
    window_left: int = -1,
    alibi_slopes: torch.Tensor | None = None,
    scale: float | None = None,
) -> torch.Tensor:
    """Attention of ``q`` [N, Hq, D] over the paged cache; returns [N, Hq, D].

    Query ``i`` belongs to request ``rows[i]`` (default: ``i``) at ``positions[i]`` and sees that
    request's keys ``j <= positions[i]`` with ``positions[i] - j <= window_left`` (when
    ``window_left >= 0``); each KV head serves ``Hq / Hkv`` query heads. ``alibi_slopes`` (fp32 [Hq])
    adds ``slope * (j - position)`` to the scores. Queries with position -1 (or a row out of range)
    return zeros. Whatever the pages hold outside the keys seen is ignored, NaN included. Several
    queries of one request may be passed: each is computed on its own.

    A position beyond the table, or a page beyond the pool among the keys seen, raises ValueError for CPU
    tensors; on CUDA it is "bad kernel argument" in the device status word, and that output means nothing."""
    scale = scale if scale is not None else 1.0 / math.sqrt(q.shape[-1])
    if _ext.use_cuda_kernels(q):
        if q.dtype in _KERNEL_DTYPES and q.shape[-1] in _HEAD_DIMS:
            return _ext.require().paged_attention(q.contiguous(), k_pages, v_pages, block_tables, positions, rows,
                                                  window_left, alibi_slopes, scale)
        _ext.fallback("paged_attention", "dtype / head_dim without a kernel")
    _inference_only("paged_attention", q, k_pages, v_pages, alibi_slopes)
    if q.dim() != 3 or k_pages.dim() != 4 or q.shape[1] % k_pages.shape[1] or q.shape[2] != k_pages.shape[3]:
        raise ValueError(f"paged_attention: q {tuple(q.shape)} does not fit k_pages {tuple(k_pages.shape)}")
    if k_pages.dtype != q.dtype or v_pages.dtype != q.dtype:
        raise ValueError(f"q is {q.dtype} but the pages are {k_pages.dtype} / {v_pages.dtype}")
    if rows is None and block_tables.shape[0] != q.shape[0]:
        raise ValueError("paged_attention: without rows, block_tables has one row per query")
    check_page_size(k_pages.shape[2])
    return _attention_ref(q, k_pages, v_pages, block_tables, positions, rows, window_left, alibi_slopes, scale)
