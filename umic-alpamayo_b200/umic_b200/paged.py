"""Paged KV cache: one pool of pages for requests of different lengths.

Beside InplaceKVCache (one dense slab whose rows share a length), for serving: requests
come, grow by a token a step and end on their own, and the cache hands out pages as they
do. Every layer's K and V pages are views of one slab [layers, 2, num_pages, kv_heads,
page_size, head_dim] (bf16, or float8_e4m3fn with a scale per layer and KV head); the
block table, the lengths and the ring of free pages live on the device and are advanced
there, so a step needs no length on the host and one captured CUDA graph serves every
step of the same batch:

    step = cache.step(new_tokens, capacity)      # once a step: table, slots, positions
    for layer ...:
        q = cache.write(layer, q, k, v, step, positions, inv_freq, sections, ...)
        out = cache.attend(layer, q, scale)      # one new token per request

A step's q, k and v have `capacity` rows: the requests' new tokens one request behind the
other, and rows of any content behind the last. `attend` takes one query row per request,
over all that is cached. So prompts are attended by the model's own attention, on the dense
k and v of the step; a prompt that continues a cached request has no attention over the
pages other than one token a step.
"""

from __future__ import annotations

import torch

from .kernels.paged import (E4M3, PagedPlan, paged_attention, paged_kv_append, paged_plan,
                            qk_norm_mrope_kv)


class PagedKVCache:
    """A pool of pages and the requests on it.

    slab: the pages of every layer; block_table int32 [max_requests, max_pages]; kv_lens
    int32 [max_requests], the cached lengths; free_ring / free_span: the ring of free pages
    and its ends; k_scale / v_scale fp32 [layers, kv_heads] for e4m3 pages, else None.
    Calls on one cache must be ordered on one stream.
    """

    def __init__(self, slab: torch.Tensor, max_requests: int, max_pages: int) -> None:
        if slab.dim() != 6 or slab.shape[1] != 2:
            raise ValueError("PagedKVCache: the slab must be [layers, 2, num_pages, kv_heads, "
                             f"page_size, head_dim], got {tuple(slab.shape)}")
        layers, _, pages, heads, self.page_size, _ = slab.shape
        dev = slab.device
        self.slab = slab
        self.block_table = torch.full((max_requests, max_pages), -1, dtype=torch.int32,
                                      device=dev)
        self.kv_lens = torch.zeros(max_requests, dtype=torch.int32, device=dev)
        self.free_ring = torch.arange(pages, dtype=torch.int32, device=dev)
        self.free_span = torch.tensor([0, pages], dtype=torch.int64, device=dev)
        self.k_scale = self.v_scale = None
        if slab.dtype == E4M3:
            self.k_scale = torch.ones(layers, heads, dtype=torch.float32, device=dev)
            self.v_scale = torch.ones(layers, heads, dtype=torch.float32, device=dev)

    @classmethod
    def allocate(cls, num_layers: int, num_pages: int, heads: int, head_dim: int,
                 page_size: int, max_requests: int, max_pages: int, device,
                 dtype=torch.bfloat16) -> "PagedKVCache":
        """An empty cache: `num_pages` pages of `page_size` tokens per layer, shared by up to
        `max_requests` requests of up to `max_pages` pages each."""
        slab = torch.empty(num_layers, 2, num_pages, heads, page_size, head_dim, device=device,
                           dtype=dtype)
        return cls(slab, max_requests, max_pages)

    # ---------------------------------------------------------------- step

    def step(self, new_tokens: torch.Tensor, capacity: int) -> PagedPlan:
        """Advances the requests: new_tokens int32 [max_requests] on the device says how many
        tokens each appends (0: none; negative: drops that many, -kv_lens ends it).
        `capacity` bounds the step's tokens, which are numbered request by request, and is
        the number of the plan's slots and of the rows that `write` and `append` take. Requests
        that find no page, row or capacity keep their length and their tokens' slots are -1
        (umic_b200.device_errors() then holds DEVERR_PAGES). Returns the plan; its kv_lens
        is this cache's."""
        return paged_plan(self.kv_lens, new_tokens, self.block_table, self.free_ring,
                          self.free_span, self.page_size, capacity, out_lens=self.kv_lens,
                          out_span=self.free_span)

    def free_pages(self) -> int:
        """Pages on the ring (reads the device: synchronises)."""
        head, tail = self.free_span.tolist()
        return tail - head

    # -------------------------------------------------------------- layers

    def pages(self, layer: int) -> tuple[torch.Tensor, torch.Tensor]:
        return self.slab[layer, 0], self.slab[layer, 1]

    def scales(self, layer: int) -> dict:
        if self.k_scale is None:
            return {}
        return {"k_scale": self.k_scale[layer], "v_scale": self.v_scale[layer]}

    def write(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
              plan: PagedPlan, positions: torch.Tensor, inv_freq: torch.Tensor, sections,
              **kwargs) -> torch.Tensor:
        """Norms and rotates q and k [capacity, heads, head_dim] and writes k and v at the
        plan's slots (rows whose slot is -1 are not written); returns the rotated q
        (qk_norm_mrope_kv's arguments; positions [axes, capacity])."""
        k_pages, v_pages = self.pages(layer)
        return qk_norm_mrope_kv(q, k, v, positions, inv_freq, sections, k_pages=k_pages,
                                v_pages=v_pages, slots=plan.slots, **self.scales(layer),
                                **kwargs)[0]

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, plan: PagedPlan) -> None:
        """Writes finished keys and values [capacity, kv_heads, head_dim] at the plan's
        slots, e.g. those of a dense prefill."""
        paged_kv_append(*self.pages(layer), k, v, plan.slots, **self.scales(layer))

    def attend(self, layer: int, q: torch.Tensor, scale: float, *,
               return_lse: bool = False):
        """Attention of one new token per request, q [max_requests, heads, head_dim], over
        everything cached; rows of requests without tokens come out as zeros."""
        return paged_attention(q, *self.pages(layer), self.block_table, self.kv_lens, scale,
                               return_lse=return_lse, **self.scales(layer))
