"""The paged-cache serving operators restated on the CPU in 64 bits (test infrastructure).

No reference counterpart: the reference keeps one dense buffer per layer whose rows share
a length (src/umic/cache.py:25-160). The rotary formula is checked against transformers'
own three-axis rotary module in tests/test_paged_cpu.py.
"""

from __future__ import annotations

import torch


def paged_plan(kv_lens, new_tokens, table, ring, span, page, capacity):
    """The step plan, request by request. Lists and CPU tensors in, dict of CPU tensors out
    (table and ring are copied)."""
    lens, new = [int(x) for x in kv_lens], [int(x) for x in new_tokens]
    table, ring = table.clone().cpu(), ring.clone().cpu()
    head, tail = int(span[0]), int(span[1])
    size, width = ring.numel(), table.shape[1]
    free = min(max(tail - head, 0), size)
    source = ring.clone()
    pages = lambda x: -(-x // page)  # noqa: E731
    slots = torch.full((capacity,), -1, dtype=torch.int32)
    positions = slots.clone()
    out_lens, cu = [], [0]
    need = count = taken = given = 0
    unserved = False
    for r, (old, d) in enumerate(zip(lens, new)):
        ok = old >= 0 and old + d >= 0 and pages(old) <= width and pages(old + d) <= width
        d = d if ok else 0
        before, after = (pages(old), pages(old + d)) if ok else (0, 0)
        first = need
        need += max(after - before, 0)
        start = count
        count += max(d, 0)
        cu.append(min(count, 2 ** 31 - 1))
        ok = ok and (after <= before or need <= free) and (d <= 0 or count <= capacity)
        if not ok:
            unserved = True
            out_lens.append(old)
            continue
        out_lens.append(old + d)
        for j in range(before, after):
            table[r, j] = source[(head + first + j - before) % size]
            taken = max(taken, first + j - before + 1)
        for j in range(after, before):
            ring[(tail + given) % size] = table[r, j]
            given += 1
        for i in range(max(d, 0)):
            pos = old + i
            slots[start + i] = int(table[r, pos // page]) * page + pos % page
            positions[start + i] = pos
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return {"kv_lens": i32(out_lens), "free_span": torch.tensor([head + taken, tail + given]),
            "cu_tokens": i32(cu), "slots": slots, "positions": positions, "table": table,
            "ring": ring, "unserved": unserved}


def mrope_axes(sections, interleaved: bool) -> list[int]:
    """The axis that turns each frequency."""
    half = sum(sections)
    if interleaved:
        n = len(sections)
        return [i % n if i < n * sections[i % n] else 0 for i in range(half)]
    return [a for a, s in enumerate(sections) for _ in range(s)]


def norm_mrope(x, weight, eps, positions, inv_freq, sections, interleaved, scaling=1.0):
    """(y, magnitude) in fp64 of x [T, H, D]: the normalised, rotated rows and, for error
    bounds, |a| + |b| of the pair that each output is made of."""
    x = x.detach().cpu().double()
    if weight is not None:
        x = x * (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt() * weight.detach().cpu().double()
    if positions is None:
        return x, x.abs()
    axes = mrope_axes(sections, interleaved)
    pos = positions.detach().cpu().double()
    angle = pos[axes].t() * inv_freq.detach().cpu().double()  # [T, half]
    cos, sin = (angle.cos() * scaling)[:, None], (angle.sin() * scaling)[:, None]
    half = len(axes)
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    y = torch.cat((a * cos - b * sin, b * cos + a * sin, rest), -1)
    mag = (a.abs() + b.abs()) * abs(scaling)
    return y, torch.cat((mag, mag, rest.abs()), -1)


def paged_attention(q, k_pages, v_pages, table, lens, scale, k_scale=None, v_scale=None,
                    device="cpu"):
    """(out, lse, spread, reach) in fp64 CPU tensors, computed on `device`; a row's tokens on
    pages outside the pool are left out. For error bounds: spread = sum_j p_j |v_j|, and
    reach = max_j scale * sum |q| |k_j|."""
    q = q.detach().to(device).double()
    b, hq, d = q.shape
    num, hk, page, _ = k_pages.shape

    def values(pages, s, ids, at):
        x = pages.detach().to(device)
        x = x.view(torch.uint8)[ids, :, at].view(x.dtype) if x.element_size() == 1 else x[ids, :, at]
        x = (x.float() if x.element_size() == 1 else x).double().transpose(0, 1)
        return x if s is None else x * s.detach().to(device).double().view(-1, 1, 1)

    out, spread = torch.zeros(b, hq, d).double(), torch.zeros(b, hq, d).double()
    lse, reach = torch.full((b, hq), float("-inf")).double(), torch.zeros(b, hq).double()
    for r in range(b):
        n = min(max(int(lens[r]), 0), table.shape[1] * page)
        j = torch.arange(n)
        ids, at = table[r].cpu().long()[j // page], j % page
        there = (ids >= 0) & (ids < num)
        if not bool(there.any()):
            continue
        ids, at = ids[there].to(device), at[there].to(device)
        k, v = values(k_pages, k_scale, ids, at), values(v_pages, v_scale, ids, at)
        qr = q[r].view(hk, hq // hk, d)
        s = qr @ k.transpose(1, 2) * scale
        lse[r] = torch.logsumexp(s, -1).reshape(hq)
        w = torch.softmax(s, -1)
        out[r] = (w @ v).reshape(hq, d)
        spread[r] = (w @ v.abs()).reshape(hq, d)
        reach[r] = (qr.abs() @ k.abs().transpose(1, 2) * abs(scale)).amax(-1).reshape(hq)
    return out, lse, spread, reach
