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

import functools
import struct
from typing import NamedTuple

import torch

from .. import _lib
from ._common import require_cuda, stats
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


# The checks below are most of what a small call costs on the host: each reads a tensor's
# shape, strides, dtype and device once.

def _one_device(name: str, first: torch.Tensor, *rest: torch.Tensor | None) -> torch.device:
    dev = first.device
    for t in rest:
        if t is not None and t.device != dev:
            require_cuda(name, first, *rest)
    if not first.is_cuda:
        require_cuda(name, first)
    return dev


def _require(name: str, what: str, t: torch.Tensor, dtype: torch.dtype, *shape: int) -> None:
    if t.dtype is not dtype:
        raise TypeError(f"{name}: {what} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name}: {what} {tuple(t.shape)}, expected {shape}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: {what} must be contiguous")


def _table(name: str, table: torch.Tensor, n: int) -> tuple[int, int]:
    """Row stride and width of a block table of n rows."""
    if table.dtype is torch.int32 and table.ndim == 2:
        rows, width = table.shape
        stride, unit = table.stride()
        if rows == n and (unit == 1 or width <= 1):
            return stride, width
    raise ValueError(f"{name}: block_table must be int32 [{n}, max_pages] with its rows "
                     f"contiguous, got {table.dtype} {tuple(table.shape)}")


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
    dev = _one_device("paged_plan", kv_lens, new_tokens, block_table, free_ring, free_span,
                      out_lens, out_span)
    n, pages = kv_lens.numel(), free_ring.numel()
    _require("paged_plan", "kv_lens", kv_lens, torch.int32, n)
    _require("paged_plan", "new_tokens", new_tokens, torch.int32, n)
    _require("paged_plan", "free_span", free_span, torch.int64, 2)
    _require("paged_plan", "free_ring", free_ring, torch.int32, pages)
    stride, width = _table("paged_plan", block_table, n)
    capacity = int(capacity)
    if capacity < 0:
        raise ValueError(f"paged_plan: capacity {capacity}")
    if out_lens is None:
        out_lens = torch.empty_like(kv_lens)
    else:
        _require("paged_plan", "out_lens", out_lens, torch.int32, n)
    if out_span is None:
        out_span = torch.empty_like(free_span)
    else:
        _require("paged_plan", "out_span", out_span, torch.int64, 2)
    cu, slots = kv_lens.new_empty(n + 1), kv_lens.new_empty(capacity)
    positions = kv_lens.new_empty(capacity)
    _lib.call("umic_paged_plan", dev, kv_lens.data_ptr(), new_tokens.data_ptr(), n,
              block_table.data_ptr(), stride, width, free_ring.data_ptr(), pages,
              free_span.data_ptr(), page_size, out_lens.data_ptr(), out_span.data_ptr(),
              cu.data_ptr(), slots.data_ptr(), positions.data_ptr(), capacity)
    stats["umic_paged_plan"] += 1
    return PagedPlan(out_lens, out_span, cu, slots, positions)


def _check_pages(name: str, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 k_scale: torch.Tensor | None, v_scale: torch.Tensor | None) -> tuple:
    """Checks a pool and its scales; returns its dtype code, shape and strides."""
    shape, strides, dtype = k_pages.shape, k_pages.stride(), k_pages.dtype
    if len(shape) != 4 or shape != v_pages.shape or strides != v_pages.stride() or \
            dtype is not v_pages.dtype:
        raise ValueError(f"{name}: k_pages and v_pages must be [num_pages, kv_heads, page_size, "
                         "head_dim] of one shape, strides and dtype")
    if strides[3] != 1:
        raise ValueError(f"{name}: head_dim must be contiguous in the pages")
    if dtype is torch.bfloat16:
        if k_scale is not None or v_scale is not None:
            raise ValueError(f"{name}: scales belong to {E4M3} pages")
        return _lib.DTYPE_BF16, shape, strides
    if dtype is not E4M3:
        raise TypeError(f"{name}: pages must be bfloat16 or {E4M3}, got {dtype}")
    if k_scale is not None:
        _require(name, "k_scale", k_scale, torch.float32, shape[1])
    if v_scale is not None:
        _require(name, "v_scale", v_scale, torch.float32, shape[1])
    return _lib.DTYPE_E4M3, shape, strides


def _rows(name: str, what: str, x: torch.Tensor, t: int, heads: int | None, d: int) -> tuple:
    """(pointer, token stride, head stride, heads) of [t, heads, d] bf16 rows."""
    if x.dtype is not torch.bfloat16:
        raise TypeError(f"{name}: {what} must be bfloat16, got {x.dtype}")
    shape, strides = x.shape, x.stride()
    if len(shape) != 3 or shape[0] != t or shape[2] != d or strides[2] != 1 or \
            (heads is not None and shape[1] != heads):
        raise ValueError(f"{name}: {what} {tuple(shape)} / strides {strides}, expected "
                         f"[{t}, {'heads' if heads is None else heads}, {d}] with head_dim "
                         "contiguous")
    return x.data_ptr(), strides[0], strides[1], shape[1]


def _input(name, q, k, v, positions, inv_freq, sections, interleaved, scaling, q_weight,
           k_weight, q_eps, k_eps, k_pages, v_pages, slots, k_scale, v_scale, q_out, k_out):
    dev = _one_device(name, k, q, v, positions, inv_freq, q_weight, k_weight, k_pages, v_pages,
                      slots, k_scale, v_scale, q_out, k_out)
    shape, strides = k.shape, k.stride()
    if len(shape) != 3:
        raise ValueError(f"{name}: k must be [tokens, heads, head_dim], got {tuple(shape)}")
    t, hk, d = shape
    if k.dtype is not torch.bfloat16 or strides[2] != 1:
        _rows(name, "k", k, t, hk, d)
    k_st, k_sh, _ = strides
    if v is None:
        v_ptr = v_st = v_sh = 0
    else:
        v_ptr, v_st, v_sh, _ = _rows(name, "v", v, t, hk, d)
    kp = vp = pg_sp = pg_sh = pg_ss = num_pages = page = ks = vs = slots_ptr = 0
    ko = ko_st = ko_sh = 0
    dt = _lib.DTYPE_BF16
    if k_pages is None:
        if v_pages is not None or slots is not None or k_scale is not None or \
                v_scale is not None:
            raise ValueError(f"{name}: v_pages, slots and scales go with k_pages")
        if k_out is None:
            k_out = k.new_empty(shape)
        ko, ko_st, ko_sh, _ = _rows(name, "k_out", k_out, t, hk, d)
    else:
        if v is None or v_pages is None or slots is None:
            raise ValueError(f"{name}: a cache write needs v, v_pages and slots")
        if k_out is not None:
            raise ValueError(f"{name}: k_out goes without k_pages")
        dt, (num_pages, heads, page, dim), (pg_sp, pg_sh, pg_ss, _) = _check_pages(
            name, k_pages, v_pages, k_scale, v_scale)
        if heads != hk or dim != d:
            raise ValueError(f"{name}: pages {tuple(k_pages.shape)} do not match k "
                             f"{tuple(shape)}")
        _require(name, "slots", slots, torch.int32, t)
        kp, vp, slots_ptr = k_pages.data_ptr(), v_pages.data_ptr(), slots.data_ptr()
        if k_scale is not None:
            ks = k_scale.data_ptr()
        if v_scale is not None:
            vs = v_scale.data_ptr()
    if q is None:
        q_ptr = q_st = q_sh = hq = qo = qo_st = qo_sh = 0
    else:
        q_ptr, q_st, q_sh, hq = _rows(name, "q", q, t, None, d)
        if q_out is None:
            q_out = q.new_empty((t, hq, d))
            qo, qo_st, qo_sh = q_out.data_ptr(), hq * d, d
        else:
            qo, qo_st, qo_sh, _ = _rows(name, "q_out", q_out, t, hq, d)
    qw = kw = wdt = 0
    if q_weight is not None:
        wdt = _w_dtype(q_weight)
        _require(name, "q_weight", q_weight, q_weight.dtype, d)
        qw = q_weight.data_ptr()
    if k_weight is not None:
        wdt = _w_dtype(k_weight)
        _require(name, "k_weight", k_weight, k_weight.dtype if qw == 0 else q_weight.dtype, d)
        kw = k_weight.data_ptr()
    pos = inv = p_sa = p_st = s0 = s1 = s2 = half = 0
    pos_bytes = axes = 1
    if positions is not None:
        p_shape, dtype, n = positions.shape, positions.dtype, len(sections)
        pos_bytes = 8 if dtype is torch.int64 else 4
        if p_shape == (n, t):
            axes, (p_sa, p_st) = n, positions.stride()
        elif n == 1 and p_shape == (t,):
            p_st, = positions.stride()
        else:
            axes = 0
        if not 1 <= axes <= 3 or (dtype is not torch.int64 and dtype is not torch.int32):
            raise ValueError(f"{name}: positions must be int32 or int64 [axes, {t}] with one of "
                             f"{n} sections per axis (1 to 3), got {dtype} {tuple(p_shape)}")
        half = inv_freq.numel()
        _require(name, "inv_freq", inv_freq, torch.float32, half)
        s0, s1, s2 = (*sections, 0, 0)[:3]
        pos, inv = positions.data_ptr(), inv_freq.data_ptr()
    try:
        args = _lib.pack_mrope_args(
            q_ptr, k.data_ptr(), v_ptr, qo, ko, qw, kw, pos, inv, kp, vp, ks, vs, slots_ptr,
            q_st, q_sh, k_st, k_sh, v_st, v_sh, qo_st, qo_sh, ko_st, ko_sh, p_sa, p_st, pg_sp,
            pg_sh, pg_ss, num_pages, page, t, hq, hk, d, wdt, pos_bytes, 2 * half, axes, s0, s1,
            s2, 1 if interleaved else 0, dt, q_eps, k_eps, scaling)
    except struct.error as e:
        raise ValueError(f"{name}: {e}") from None
    _lib.call("umic_qk_norm_mrope_kv", dev, args)
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

    q [T, Hq, D], k / v [T, Hk, D] bf16 (D contiguous, token and head strides multiples of 8
    elements, 16-byte aligned; so are outputs and pages, whose rows must lie apart).
    positions [axes, T] (or [T]) int32 / int64 holds one coordinate per axis -- (time,
    height, width) of an image patch, three equal ones for text -- and inv_freq [r / 2]
    fp32 the frequencies of the r rotated elements. `sections`, one per axis, sum to r / 2:
    the axes turn that many frequencies each, in runs (t..t h..h w..w); with interleaved,
    frequency i is turned by axis i % axes while i < axes * section of that axis, else by the
    first (t h w t h w ... t t), so (24, 20, 20) turns as many of each but (10, 27, 27) turns
    22, 21 and 21, as transformers does. cos and sin are multiplied by `scaling`. Norms run
    where a weight [D] is given.

    With k_pages / v_pages [P, Hk, page, D], k and v are written at slots [T] int32 (one per
    row; -1 skips a token; two tokens must not share a slot) and (q_out, None) is returned;
    without, (q_out, k_out), and v is not touched. q_out may be q and k_out k. e4m3 pages
    hold the fp32 value divided by its head's scale, rounded once, saturated at +-448.
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


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(dev: torch.device, *sizes: int) -> int:
    _lib._ensure_device(dev)
    return _lib.lib().umic_paged_attention_workspace_bytes(*sizes)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    block_table: torch.Tensor, kv_lens: torch.Tensor, scale: float, *,
                    k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                    return_lse: bool = False, out: torch.Tensor | None = None):
    """softmax(scale * q k^T) v of one new token per request over its pages.

    q [B, Hq, D] bf16 (D contiguous), pages [P, Hk, page, D], block_table int32
    [B, max_pages], kv_lens int32 [B] (read on the device). Returns out [B, Hq, D] (a given
    `out` may be q), with
    return_lse also the log of each row's sum of exponentials, fp32 [B, Hq]. Requests
    without tokens come out as zeros (lse -inf). D 64, 80, 96, 128 or 256; page a multiple
    of 16; any number of query heads per KV head; strides multiples of 16 bytes. Sums are
    fp32; weights are held to 2^-17 of themselves over bf16 pages, to 2^-11 over e4m3 ones.

    There is one query row per request: a prompt that continues a cached request can be
    planned and written, but its tokens cannot be attended here except one step each.
    """
    dev = _one_device("paged_attention", q, k_pages, v_pages, block_table, kv_lens, k_scale,
                      v_scale, out)
    dt, (p, hk, page, dp), (sp, sh, ss, _) = _check_pages("paged_attention", k_pages, v_pages,
                                                          k_scale, v_scale)
    if q.ndim != 3 or q.shape[2] != dp:
        raise ValueError(f"paged_attention: q {tuple(q.shape)} for pages {tuple(k_pages.shape)}")
    b, hq, d = q.shape
    qa = _rows("paged_attention", "q", q, b, hq, d)
    _require("paged_attention", "kv_lens", kv_lens, torch.int32, b)
    stride, width = _table("paged_attention", block_table, b)
    if out is None:
        out = q.new_empty((b, hq, d))
        oa = (out.data_ptr(), hq * d, d)
    else:
        oa = _rows("paged_attention", "out", out, b, hq, d)
    lse = torch.empty((b, hq), dtype=torch.float32, device=dev) if return_lse else None
    # its own workspace for every call: calls on several streams, and graphs captured
    # apart, never share one
    need = _workspace_bytes(dev, b, hq, hk, d, width, page, dt)
    ws = q.new_empty((need + 1) // 2)
    try:
        args = _lib.pack_paged_attention_args(
            qa[0], k_pages.data_ptr(), v_pages.data_ptr(),
            0 if k_scale is None else k_scale.data_ptr(),
            0 if v_scale is None else v_scale.data_ptr(), block_table.data_ptr(),
            kv_lens.data_ptr(), oa[0], 0 if lse is None else lse.data_ptr(), ws.data_ptr(),
            qa[1], qa[2], sp, sh, ss, p, page, stride, width, oa[1], oa[2], b, need, hq, hk, d,
            dt, scale)
    except struct.error as e:
        raise ValueError(f"paged_attention: {e}") from None
    _lib.call("umic_paged_attention", dev, args)
    stats["umic_paged_attention"] += 1
    return (out, lse) if return_lse else out
