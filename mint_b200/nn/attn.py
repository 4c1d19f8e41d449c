"""Grouped-query / multi-head attention (mint/nn/attn.py:10-141).

Bias-free q/k/v/o projections, per-head QK-RMSNorm, positional encoding, causal attention
with an optional left window. The q/k/v projections run as one GEMM over ``[Wq; Wk; Wv]``
and QK-norm + RoPE run as one fused kernel. Under tensor parallelism the module holds
``n_heads / tp`` query heads and ``n_kv_heads / tp`` KV heads (column-parallel q/k/v,
row-parallel o).
"""

from __future__ import annotations

import torch
from torch import nn

from mint_b200.kvcache.base import KVCache
from mint_b200.kvcache.paged import PagedLayer
from mint_b200.nn.base import compute_dtype
from mint_b200.nn.flashattn import FlashAttention
from mint_b200.nn.norm import RMSNorm
from mint_b200.nn.pos import ALiBiPositionalBias, NoPE, PosEmbeddings, RoPE
from mint_b200.ops.attention import has_kernel
from mint_b200.ops.linear import linear
from mint_b200.ops.paged import has_kernels, paged_attention, qk_norm_rope_paged
from mint_b200.ops.rope import qk_norm_rope
from mint_b200.parallel import fused as fused_tp
from mint_b200.parallel import tp as tpc


class GroupedQueryAttention(nn.Module):
    def __init__(
        self,
        n_heads: int,
        n_kv_heads: int,
        head_dim: int,
        embed_dim: int,
        pos_embeddings: PosEmbeddings,
        dtype: torch.dtype,
        window_size: int = -1,
    ) -> None:
        super().__init__()
        self.n_heads = n_heads
        self.n_kv_heads = n_kv_heads
        self.head_dim = head_dim
        self.window_size = window_size
        self.pos_embeddings = pos_embeddings
        self.attention = FlashAttention(use_custom_fa=True)
        self.wq = nn.Linear(embed_dim, n_heads * head_dim, bias=False, dtype=dtype)
        self.wk = nn.Linear(embed_dim, n_kv_heads * head_dim, bias=False, dtype=dtype)
        self.wv = nn.Linear(embed_dim, n_kv_heads * head_dim, bias=False, dtype=dtype)
        self.wo = nn.Linear(n_heads * head_dim, embed_dim, bias=False, dtype=dtype)
        self.q_norm = RMSNorm(head_dim)
        self.k_norm = RMSNorm(head_dim)
        self.tp: tpc.TPInfo | None = None

    def _fusable(self) -> bool:
        return all(type(m) is nn.Linear for m in (self.wq, self.wk, self.wv)) and (
            self.pos_embeddings.fused_kind in ("rope", "none")
        )

    def _norm_rope(self, qkv: torch.Tensor, start_pos: int):  # noqa: ANN202
        """QK-RMSNorm + RoPE on the fused projection ``[B, T, (hq + 2 hkv) * hd]`` -> q, k, v."""
        pe = self.pos_embeddings
        cos, sin = pe.tables() if isinstance(pe, RoPE) else (None, None)
        q, k, v = qk_norm_rope(
            qkv, self.n_heads, self.n_kv_heads, self.head_dim, self.q_norm.scale, self.k_norm.scale, cos, sin,
            start_pos=start_pos, eps=self.q_norm.eps,
        )
        return q, k, v, None

    def _project(self, x: torch.Tensor, dt: torch.dtype, start_pos: int):  # noqa: ANN202
        bsz, seqlen = x.shape[0], x.shape[1]
        hq, hkv, hd = self.n_heads, self.n_kv_heads, self.head_dim
        if self._fusable():
            qkv = linear(x, self.wq.weight, self.wk.weight, self.wv.weight, compute_dtype=dt)
            pe = self.pos_embeddings
            if isinstance(pe, RoPE):
                cos, sin = pe.tables()
            else:
                cos = sin = None
            return self._norm_rope(qkv, start_pos)
        q = self.wq(x).view(bsz, seqlen, hq, hd)
        k = self.wk(x).view(bsz, seqlen, hkv, hd)
        v = self.wv(x).view(bsz, seqlen, hkv, hd)
        q = self.q_norm(q)
        k = self.k_norm(k)
        q, k, bias = self.pos_embeddings(q, k, start_pos=start_pos)
        return q, k, v, bias

    def _forward_paged(self, x: torch.Tensor, layer: PagedLayer) -> torch.Tensor:
        """One step over a paged cache: ``x`` [1, N, E] holds the packed tokens of ``layer.step``.

        When every request of the step is new, its prompts need not read the pages: they are the documents of one
        packed row where the FlashAttention kernel takes them. Heads and types that only the paged kernel takes,
        ALiBi models, and steps with older requests attend over the pages. What neither kernel takes (and CPU
        tensors) attends prompt by prompt, so that no mask spans prompts that do not see each other."""
        if x.shape[0] != 1:
            raise ValueError(f"paged steps pack all tokens into one row, got a batch of {x.shape[0]}")
        if tpc.active(self.tp):
            raise ValueError("paged caches are not supported under tensor parallelism")
        dt = compute_dtype(x)
        step, n = layer.step, x.shape[1]
        pe = self.pos_embeddings
        cos = sin = slopes = None
        if isinstance(pe, RoPE):
            cos, sin = pe.tables()
        elif isinstance(pe, ALiBiPositionalBias):
            slopes = pe.slopes.reshape(-1).float()
        elif not isinstance(pe, NoPE):
            raise ValueError(f"paged caches take rope, linear_rope, alibi or nope positions, not {type(pe).__name__}")
        if all(type(m) is nn.Linear for m in (self.wq, self.wk, self.wv)):
            qkv = linear(x, self.wq.weight, self.wk.weight, self.wv.weight, compute_dtype=dt)
        else:
            qkv = torch.cat([self.wq(x), self.wk(x), self.wv(x)], dim=-1)
        dense = x.is_cuda and has_kernel(qkv.dtype, self.head_dim)
        prompts = step.fresh and max(step.new_lens, default=0) > 1 and slopes is None
        if prompts and not dense and x.is_cuda:
            prompts = not has_kernels(qkv.dtype, self.head_dim)
        out = qk_norm_rope_paged(
            qkv.view(n, -1), self.n_heads, self.n_kv_heads, self.head_dim, self.q_norm.scale, self.k_norm.scale, cos, sin,
            step.plan.positions, step.plan.slots, layer.k_pages, layer.v_pages, eps=self.q_norm.eps, return_kv=prompts,
        )
        window = self.window_size if self.window_size > 0 else -1
        if prompts:
            q, k, v = (t.unsqueeze(0) for t in out)
            if dense:
                out = self.attention(q, k, v, causal=True, window_size=(window, -1), doc_ids=step.doc_ids)
            else:
                out, end = torch.zeros_like(q), 0
                for length in step.new_lens:
                    at, end = slice(end, end + length), end + length
                    if length:
                        out[:, at] = self.attention(q[:, at], k[:, at], v[:, at], causal=True, window_size=(window, -1))
        else:
            out = paged_attention(out, layer.k_pages, layer.v_pages, step.block_tables, step.plan.positions,
                                  step.plan.rows, window_left=window, alibi_slopes=slopes)
        out = out.reshape(1, n, -1)
        return linear(out, self.wo.weight, compute_dtype=dt) if type(self.wo) is nn.Linear else self.wo(out)

    def forward(
        self,
        x: torch.Tensor,
        kv_cache: KVCache | PagedLayer | None = None,
        start_pos: int = 0,
        base_attn_mask: torch.Tensor | None = None,
        doc_ids: torch.Tensor | None = None,
    ) -> torch.Tensor:
        if isinstance(kv_cache, PagedLayer):
            if start_pos != 0 or base_attn_mask is not None or doc_ids is not None:
                raise ValueError("a paged step has its own positions and requests: no start_pos, attention mask or doc_ids")
            return self._forward_paged(x, kv_cache)
        dt = compute_dtype(x)
        # TP on CUDA: QKV GEMM with its all-gather (SP) or backward all-reduce (no SP), wo GEMM with its
        # reduce-scatter (SP) or all-reduce (no SP), each as fused kernels
        fuse = (kv_cache is None and self._fusable() and type(self.wo) is nn.Linear and dt == torch.bfloat16
                and fused_tp.enabled(self.tp, x))
        if fuse:
            bsz, seqlen = x.shape[0], x.shape[1] * (self.tp.size if self.tp.sp else 1)
            qkv = fused_tp.column_parallel_linear(x, (self.wq.weight, self.wk.weight, self.wv.weight), self.tp)
            q, k, v, bias = self._norm_rope(qkv, start_pos)
        else:
            x = tpc.enter_column_parallel(x, self.tp)
            bsz, seqlen = x.shape[0], x.shape[1]
            q, k, v, bias = self._project(x, dt, start_pos)
        if bias is not None and bias.shape[1] != q.shape[2] and self.tp is not None and self.tp.size > 1:
            per = q.shape[2]
            bias = bias[:, self.tp.rank * per : (self.tp.rank + 1) * per]
        window = (self.window_size, -1) if self.window_size > 0 else (-1, -1)
        out = self.attention(
            q, k, v, causal=True, window_size=window, kv_cache=kv_cache,
            base_attn_mask=base_attn_mask, doc_ids=doc_ids, bias=bias, start_pos=start_pos,
        )
        out = out.reshape(bsz, seqlen, -1)
        if fuse:
            return fused_tp.row_parallel_linear(out, self.wo.weight, self.tp)
        if type(self.wo) is nn.Linear:
            y = linear(out, self.wo.weight, compute_dtype=dt)
        else:
            y = self.wo(out)
        return tpc.exit_row_parallel(y, self.tp)


class MultiHeadAttention(GroupedQueryAttention):
    """MHA: every query head has its own KV head (``n_kv_heads == n_heads``)."""

    def __init__(
        self,
        n_heads: int,
        head_dim: int,
        embed_dim: int,
        pos_embeddings: PosEmbeddings,
        dtype: torch.dtype,
        window_size: int = -1,
    ) -> None:
        super().__init__(n_heads, n_heads, head_dim, embed_dim, pos_embeddings, dtype, window_size)


class MultiQueryAttention(GroupedQueryAttention):
    """MQA: a single shared KV head (``n_kv_heads == 1``)."""

    def __init__(
        self,
        n_heads: int,
        head_dim: int,
        embed_dim: int,
        pos_embeddings: PosEmbeddings,
        dtype: torch.dtype,
        window_size: int = -1,
    ) -> None:
        super().__init__(n_heads, 1, head_dim, embed_dim, pos_embeddings, dtype, window_size)
