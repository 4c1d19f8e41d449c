"""Paged KV cache for ragged batches of requests.

One pool of pages per layer and operand, ``[n_pages, n_kv_heads, page_size, head_dim]``, shared by up to
``max_batch`` requests of different lengths: memory follows the tokens that exist, not
``max_batch * max_seq_len`` as in the dense :class:`~mint_b200.kvcache.base.KVCache`
(mint/kvcache/base.py:4-65), and the pages of a finished request serve the next one.

The block tables, lengths and free list live on the device and are advanced by one kernel per step
(:func:`mint_b200.ops.paged_plan`); the host keeps a mirror of the lengths to know what fits. A step is::

    step = cache.plan([5, 0, 1, ...])      # new tokens per request; packed tokens in request order
    logits = model(tokens[None], kv_caches=step.layers)

and ``cache.release([row, ...])`` returns the pages of finished requests.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from mint_b200.ops.paged import PagedPlan, check_page_size, paged_plan


class PagedKVCache:
    def __init__(
        self,
        n_layers: int,
        n_pages: int,
        page_size: int = 16,
        n_kv_heads: int = 4,
        head_dim: int = 128,
        max_batch: int = 32,
        max_seq_len: int = 2048,
        dtype: torch.dtype = torch.float32,
        device: str | torch.device = "cpu",
    ) -> None:
        check_page_size(page_size)
        if min(n_layers, n_pages, n_kv_heads, head_dim, max_batch, max_seq_len) < 1:
            raise ValueError("PagedKVCache sizes must be positive")
        self.n_layers, self.n_pages, self.page_size = n_layers, n_pages, page_size
        self.max_batch, self.max_seq_len = max_batch, max_seq_len
        self.dtype = dtype
        self.device = torch.device(device)
        shape = (n_layers, n_pages, n_kv_heads, page_size, head_dim)
        self.k_pages = torch.zeros(shape, dtype=dtype, device=device)
        self.v_pages = torch.zeros(shape, dtype=dtype, device=device)
        i32 = {"dtype": torch.int32, "device": device}
        self.block_tables = torch.zeros(max_batch, (max_seq_len + page_size - 1) // page_size, **i32)
        self.seq_lens = torch.zeros(max_batch, **i32)
        self.free_pages = torch.arange(n_pages, **i32)  # entries from free_head on are free
        self.free_head = torch.zeros(1, **i32)
        self.lens = [0] * max_batch  # host mirror of seq_lens
        self._free = n_pages  # host mirror: pages left

    def pages_for(self, tokens: int) -> int:
        return (tokens + self.page_size - 1) // self.page_size

    @property
    def n_free_pages(self) -> int:
        return self._free

    def plan(self, new_lens: list[int], n_tokens: int | None = None) -> PagedStep:
        """Make room for ``new_lens[b]`` more tokens of every request and return the step's layout.

        ``n_tokens`` is the packed length (default: their sum); a larger one pads. Raises ValueError, with
        nothing changed, when the pages or a request's ``max_seq_len`` do not suffice."""
        new_lens = list(new_lens) + [0] * (self.max_batch - len(new_lens))
        if len(new_lens) > self.max_batch or min(new_lens) < 0:
            raise ValueError(f"one non-negative count for each of at most {self.max_batch} requests")
        total = sum(new_lens)
        n_tokens = total if n_tokens is None else n_tokens
        if n_tokens < total:
            raise ValueError(f"{total} new tokens do not fit n_tokens={n_tokens}")
        after = [a + n for a, n in zip(self.lens, new_lens)]
        if max(after) > self.max_seq_len:
            raise ValueError(f"KV cache overflow: {max(after)} > max_seq_len={self.max_seq_len}")
        need = sum(self.pages_for(a) - self.pages_for(b) for a, b in zip(after, self.lens))
        if need > self._free:
            raise ValueError(f"KV cache overflow: {need} pages needed, {self._free} of {self.n_pages} free")
        fresh = all(b == 0 for b, n in zip(self.lens, new_lens) if n > 0)
        step = self.plan_on_device(torch.tensor(new_lens, dtype=torch.int32).to(self.device, non_blocking=True), n_tokens)
        step.fresh, step.new_lens = fresh, new_lens
        self.lens, self._free = after, self._free - need
        return step

    def plan_on_device(self, new_lens: torch.Tensor, n_tokens: int) -> PagedStep:
        """:meth:`plan` for an int32 ``[max_batch]`` tensor of counts, without the host's checks and mirror
        (no host synchronization: it can be captured in a CUDA graph)."""
        p = paged_plan(self.seq_lens, new_lens, self.block_tables, self.free_pages, self.free_head,
                       page_size=self.page_size, n_tokens=n_tokens)
        self.seq_lens.copy_(p.seq_lens)
        self.free_head.copy_(p.free_head)
        return PagedStep(self, p)

    def advance(self, new_lens: list[int]) -> None:
        """Bring the host mirror up to date with a replayed :meth:`plan_on_device`."""
        after = [a + n for a, n in zip(self.lens, new_lens)]
        self._free -= sum(self.pages_for(a) - self.pages_for(b) for a, b in zip(after, self.lens))
        self.lens = after

    def release(self, rows: list[int]) -> None:
        """Forget the requests in ``rows``; their pages are free again."""
        for row in rows:
            n = self.pages_for(self.lens[row])
            head = self.n_pages - self._free
            if n:
                self.free_pages[head - n : head] = self.block_tables[row, :n]
            self._free += n
            self.lens[row] = 0
            self.seq_lens[row] = 0
        self.free_head.fill_(self.n_pages - self._free)

    def reset(self) -> None:
        self.free_pages.copy_(torch.arange(self.n_pages, dtype=torch.int32))
        self.free_head.zero_()
        self.seq_lens.zero_()
        self.lens = [0] * self.max_batch
        self._free = self.n_pages


@dataclass
class PagedLayer:
    """One layer's pools within one step: what the attention modules take as ``kv_cache``."""

    k_pages: torch.Tensor
    v_pages: torch.Tensor
    step: PagedStep


class PagedStep:
    """The packed tokens of one step and every layer's view of the cache (``layers``)."""

    def __init__(self, cache: PagedKVCache, plan: PagedPlan) -> None:
        self.plan = plan
        self.doc_ids = plan.rows.unsqueeze(0)  # the requests as documents of the packed row
        self.block_tables = cache.block_tables
        self.fresh = False  # every request with new tokens had none before
        self.new_lens: list[int] = []  # new tokens of every request, if the host knows them
        self.layers = [PagedLayer(cache.k_pages[i], cache.v_pages[i], self) for i in range(cache.n_layers)]
