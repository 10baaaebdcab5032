"""Serving over a paged KV cache (C ABI: umic_paged_plan, umic_qk_norm_mrope_kv,
umic_paged_attention).

A pool of pages [num_pages, kv_heads, page_size, head_dim] (bf16, or float8_e4m3fn with
one fp32 scale per KV head) holds the keys and values of requests of different lengths;
a request's row of the block table lists its pages. One serving step is
  paged_plan         grows the rows and says where each new token goes, on the device
  qk_norm_mrope_kv   norms and rotates q and k and writes k and v at those slots
                     (paged_kv_append: the write alone)
  paged_attention    attends one new token per request over its pages
and nothing of it needs a length on the host, so one captured CUDA graph serves every
step. `PagedKVCache` (umic_b200.paged) keeps the pool and runs them together.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib
from ._common import require_bf16, require_cuda, stats
from .rmsnorm import _w_dtype

E4M3 = torch.float8_e4m3fn


class PagedPlan(NamedTuple):
    """A step's plan: kv_lens [R] and free_span [2] after it, cu_tokens [R + 1], and the
    slot and position of each of the step's tokens (-1: none)."""

    kv_lens: torch.Tensor
    free_span: torch.Tensor
    cu_tokens: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor


def _require(name: str, what: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple) -> None:
    if t.dtype != dtype:
        raise TypeError(f"{name}: {what} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name}: {what} {tuple(t.shape)}, expected {shape}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: {what} must be contiguous")


def paged_plan(kv_lens: torch.Tensor, new_tokens: torch.Tensor, block_table: torch.Tensor,
               free_ring: torch.Tensor, free_span: torch.Tensor, page_size: int, capacity: int,
               *, out_lens: torch.Tensor | None = None,
               out_span: torch.Tensor | None = None) -> PagedPlan:
    """Block table, slots and free pages of one step, from request lengths on the device.

    kv_lens / new_tokens int32 [R]: cached lengths, and what each request appends (n > 0)
    or drops from its end (n < 0). block_table int32 [R, max_pages] (rows may be strided)
    and free_ring int32 [num_pages] change in place; free_span int64 [2] holds the ring
    positions of the first free page and behind the last. Requests are served in order
    while free pages, table width and `capacity` (tokens of the step) last; one that is
    not keeps what it had, gets slots of -1 and sets DEVERR_PAGES (umic_b200.device_errors).
    out_lens may be kv_lens and out_span may be free_span (then they advance in place).
    """
    dev = require_cuda("paged_plan", kv_lens, new_tokens, block_table, free_ring, free_span,
                       out_lens, out_span)
    n = kv_lens.shape[0] if kv_lens.dim() == 1 else -1
    _require("paged_plan", "kv_lens", kv_lens, torch.int32, (n,))
    _require("paged_plan", "new_tokens", new_tokens, torch.int32, (n,))
    _require("paged_plan", "free_span", free_span, torch.int64, (2,))
    pages = free_ring.numel()
    _require("paged_plan", "free_ring", free_ring, torch.int32, (pages,))
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != n \
            or (block_table.stride(1) != 1 and block_table.shape[1] > 1):
        raise ValueError(f"paged_plan: block_table must be int32 [{n}, max_pages] with its rows "
                         f"contiguous, got {block_table.dtype} {tuple(block_table.shape)}")
    capacity = int(capacity)
    if capacity < 0:
        raise ValueError(f"paged_plan: capacity {capacity}")
    # one allocation: span (2 x int64), token offsets, lengths, slots, positions
    buf = torch.empty(5 + 2 * n + 2 * capacity, dtype=torch.int32, device=dev)
    span, cu, lens, slots, positions = buf.split((4, n + 1, n, capacity, capacity))
    if out_lens is None:
        out_lens = lens
    else:
        _require("paged_plan", "out_lens", out_lens, torch.int32, (n,))
    if out_span is None:
        out_span = span.view(torch.int64)
    else:
        _require("paged_plan", "out_span", out_span, torch.int64, (2,))
    _lib.call("umic_paged_plan", dev, kv_lens.data_ptr(), new_tokens.data_ptr(), n,
              block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
              free_ring.data_ptr(), pages, free_span.data_ptr(), int(page_size),
              out_lens.data_ptr(), out_span.data_ptr(), cu.data_ptr(), slots.data_ptr(),
              positions.data_ptr(), capacity)
    stats["umic_paged_plan"] += 1
    return PagedPlan(out_lens, out_span, cu, slots, positions)


def _check_pages(name: str, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 k_scale: torch.Tensor | None, v_scale: torch.Tensor | None) -> int:
    """Checks a pool and its scales; returns its dtype code."""
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or \
            k_pages.stride() != v_pages.stride() or k_pages.dtype != v_pages.dtype:
        raise ValueError(f"{name}: k_pages and v_pages must be [num_pages, kv_heads, page_size, "
                         "head_dim] of one shape, strides and dtype")
    if k_pages.stride(3) != 1:
        raise ValueError(f"{name}: head_dim must be contiguous in the pages")
    if k_pages.dtype == torch.bfloat16:
        if k_scale is not None or v_scale is not None:
            raise ValueError(f"{name}: scales belong to {E4M3} pages")
        return _lib.DTYPE_BF16
    if k_pages.dtype != E4M3:
        raise TypeError(f"{name}: pages must be bfloat16 or {E4M3}, got {k_pages.dtype}")
    for what, s in (("k_scale", k_scale), ("v_scale", v_scale)):
        if s is not None:
            _require(name, what, s, torch.float32, (k_pages.shape[1],))
    return _lib.DTYPE_E4M3


def _input(name, q, k, v, positions, inv_freq, sections, interleaved, scaling, q_weight,
           k_weight, q_eps, k_eps, k_pages, v_pages, slots, k_scale, v_scale, q_out, k_out):
    dev = require_cuda(name, q, k, v, positions, inv_freq, q_weight, k_weight, k_pages, v_pages,
                       slots, k_scale, v_scale, q_out, k_out)
    require_bf16(name, q, k, v, q_out, k_out)
    if k.dim() != 3:
        raise ValueError(f"{name}: k must be [tokens, heads, head_dim], got {tuple(k.shape)}")
    t, hk, d = k.shape
    for what, x in (("q", q), ("k", k), ("v", v), ("q_out", q_out), ("k_out", k_out)):
        if x is None:
            continue
        if x.dim() != 3 or x.shape[0] != t or x.shape[2] != d or x.stride(2) != 1 or \
                (what not in ("q", "q_out") and x.shape[1] != hk):
            raise ValueError(f"{name}: {what} {tuple(x.shape)} / strides {x.stride()} does not "
                             f"match k {tuple(k.shape)} (head_dim contiguous)")
    if q_out is not None and q_out.shape != q.shape:
        raise ValueError(f"{name}: q_out {tuple(q_out.shape)} for q {tuple(q.shape)}")
    if k_pages is None:
        if v_pages is not None or slots is not None or k_scale is not None or \
                v_scale is not None:
            raise ValueError(f"{name}: v_pages, slots and scales go with k_pages")
        pool, dt, slots_ptr = (0, 0, 0, 0, 0), _lib.DTYPE_BF16, None
    else:
        if v is None or v_pages is None or slots is None:
            raise ValueError(f"{name}: a cache write needs v, v_pages and slots")
        dt = _check_pages(name, k_pages, v_pages, k_scale, v_scale)
        if k_pages.shape[1] != hk or k_pages.shape[3] != d:
            raise ValueError(f"{name}: pages {tuple(k_pages.shape)} do not match k "
                             f"{tuple(k.shape)}")
        _require(name, "slots", slots, torch.int32, (t,))
        pool = (*k_pages.stride()[:3], k_pages.shape[0], k_pages.shape[2])
        slots_ptr = slots.data_ptr()
    w = q_weight if q_weight is not None else k_weight
    if w is not None:
        for what, x in (("q_weight", q_weight), ("k_weight", k_weight)):
            if x is not None:
                _require(name, what, x, w.dtype, (d,))
    if positions is None:
        rot = (None, 4, 0, 0, None, 0, 1, 0, 0, 0, 0)
    else:
        if positions.dim() == 1:
            positions = positions[None]
        axes = positions.shape[0]
        if positions.dtype not in (torch.int32, torch.int64) or positions.dim() != 2 or \
                positions.shape[1] != t or not 1 <= axes <= 3 or len(sections) != axes:
            raise ValueError(f"{name}: positions must be int32 or int64 [axes, {t}] with one of "
                             f"{len(sections)} sections per axis (1 to 3), got "
                             f"{positions.dtype} {tuple(positions.shape)}")
        half = inv_freq.numel()
        _require(name, "inv_freq", inv_freq, torch.float32, (half,))
        sec = (*map(int, sections), 0, 0)
        rot = (positions.data_ptr(), positions.element_size(),
               positions.stride(0), positions.stride(1), inv_freq.data_ptr(),
               2 * half, axes, sec[0], sec[1], sec[2], int(interleaved))
    if q is None:
        qa, qo = (None, 0, 0, 0), (None, 0, 0)
    else:
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        qa = (q.data_ptr(), q.stride(0), q.stride(1), q.shape[1])
        qo = (q_out.data_ptr(), q_out.stride(0), q_out.stride(1))
    if k_pages is None:
        if k_out is None:
            k_out = torch.empty(k.shape, dtype=k.dtype, device=dev)
        ko = (k_out.data_ptr(), k_out.stride(0), k_out.stride(1))
    else:
        k_out, ko = None, (None, 0, 0)
    va = (v.data_ptr(), v.stride(0), v.stride(1)) if v is not None else (None, 0, 0)
    _lib.call("umic_qk_norm_mrope_kv", dev, *qa, k.data_ptr(), k.stride(0), k.stride(1), *va, hk,
              *qo, *ko, _lib.ptr(q_weight), _lib.ptr(k_weight),
              _w_dtype(w) if w is not None else _lib.DTYPE_BF16, q_eps, k_eps, *rot, scaling,
              _lib.ptr(k_pages), _lib.ptr(v_pages), *pool, dt, _lib.ptr(k_scale),
              _lib.ptr(v_scale), slots_ptr, t, d)
    return q_out, k_out


def qk_norm_mrope_kv(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor | None,
                     positions: torch.Tensor, inv_freq: torch.Tensor, sections, *,
                     interleaved: bool = False, scaling: float = 1.0,
                     q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                     q_eps: float = 1e-6, k_eps: float = 1e-6,
                     k_pages: torch.Tensor | None = None, v_pages: torch.Tensor | None = None,
                     slots: torch.Tensor | None = None, k_scale: torch.Tensor | None = None,
                     v_scale: torch.Tensor | None = None, q_out: torch.Tensor | None = None,
                     k_out: torch.Tensor | None = None):
    """Per-head RMSNorm, rotary positions with several axes, and the paged K/V write.

    q [T, Hq, D], k / v [T, Hk, D] bf16 (any token and head strides, D contiguous).
    positions [axes, T] (or [T]) int32 / int64 holds one coordinate per axis -- (time,
    height, width) of an image patch, three equal ones for text -- and inv_freq [r / 2]
    fp32 the frequencies of the r rotated elements; `sections` says how many frequencies
    each axis turns, in runs (t..t h..h w..w) or, with interleaved, as t h w t h w ... t t.
    cos and sin are multiplied by `scaling`. Norms run where a weight [D] is given.

    With k_pages / v_pages [P, Hk, page, D], k and v are written at slots [T] int32 (-1
    skips a token; two tokens must not share a slot) and (q_out, None) is returned;
    without, (q_out, k_out), and v is not touched. q_out may be q and k_out k.
    """
    if positions is None or inv_freq is None:
        raise ValueError("qk_norm_mrope_kv: positions and inv_freq are needed")
    out = _input("qk_norm_mrope_kv", q, k, v, positions, inv_freq, sections, interleaved,
                 scaling, q_weight, k_weight, q_eps, k_eps, k_pages, v_pages, slots, k_scale,
                 v_scale, q_out, k_out)
    stats["umic_qk_norm_mrope_kv"] += 1
    return out


def paged_kv_append(k_pages: torch.Tensor, v_pages: torch.Tensor, k_new: torch.Tensor,
                    v_new: torch.Tensor, slots: torch.Tensor, *,
                    k_scale: torch.Tensor | None = None,
                    v_scale: torch.Tensor | None = None) -> None:
    """Writes finished keys and values [T, Hk, D] at slots [T] of the pages, e.g. to move a
    dense prefix (InplaceKVCache) into them; the same write as qk_norm_mrope_kv's."""
    _input("paged_kv_append", None, k_new, v_new, None, None, (), False, 1.0, None, None, 0.0,
           0.0, k_pages, v_pages, slots, k_scale, v_scale, None, None)
    stats["umic_paged_kv_append"] += 1


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    block_table: torch.Tensor, kv_lens: torch.Tensor, scale: float, *,
                    k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                    return_lse: bool = False, out: torch.Tensor | None = None):
    """softmax(scale * q k^T) v of one new token per request over its pages.

    q [B, Hq, D] bf16 (D contiguous), pages [P, Hk, page, D], block_table int32
    [B, max_pages], kv_lens int32 [B] (read on the device). Returns out [B, Hq, D], with
    return_lse also the log of each row's sum of exponentials, fp32 [B, Hq]. Requests
    without tokens come out as zeros (lse -inf). D 64, 80, 96, 128 or 256; page a multiple
    of 16; any number of query heads per KV head.
    """
    dev = require_cuda("paged_attention", q, k_pages, v_pages, block_table, kv_lens, k_scale,
                       v_scale, out)
    require_bf16("paged_attention", q, out)
    dt = _check_pages("paged_attention", k_pages, v_pages, k_scale, v_scale)
    if q.dim() != 3 or q.stride(2) != 1 or q.shape[2] != k_pages.shape[3]:
        raise ValueError(f"paged_attention: q {tuple(q.shape)} (head_dim contiguous) for pages "
                         f"{tuple(k_pages.shape)}")
    b, hq, d = q.shape
    p, hk, page, _ = k_pages.shape
    _require("paged_attention", "kv_lens", kv_lens, torch.int32, (b,))
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != b \
            or (block_table.stride(1) != 1 and block_table.shape[1] > 1):
        raise ValueError(f"paged_attention: block_table must be int32 [{b}, max_pages] with its "
                         f"rows contiguous, got {block_table.dtype} "
                         f"{tuple(block_table.shape)}")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.stride(2) != 1:
        raise ValueError(f"paged_attention: out {tuple(out.shape)} for q {tuple(q.shape)}")
    lse = torch.empty((b, hq), dtype=torch.float32, device=dev) if return_lse else None
    # its own workspace for every call: calls on several streams, and graphs captured
    # apart, never share one
    _lib._ensure_device(dev)
    need = _lib.lib().umic_paged_attention_workspace_bytes(
        b, hq, hk, d, block_table.shape[1], page, dt)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _lib.call("umic_paged_attention", dev, q.data_ptr(), q.stride(0), q.stride(1),
              k_pages.data_ptr(), v_pages.data_ptr(), *k_pages.stride()[:3], p, page, dt,
              _lib.ptr(k_scale), _lib.ptr(v_scale), block_table.data_ptr(),
              block_table.stride(0), block_table.shape[1], kv_lens.data_ptr(), out.data_ptr(),
              out.stride(0), out.stride(1), _lib.ptr(lse), b, hq, hk, d, scale, ws.data_ptr(),
              need)
    stats["umic_paged_attention"] += 1
    return (out, lse) if return_lse else out
