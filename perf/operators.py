"""The paged-cache serving operators, as cases that can be timed and compared.

Three operators, called as a serving step calls them:
  plan    block tables, slot map and free pages of a step, from request lengths
  input   attention input of ragged tokens: per-head RMSNorm, rotary positions with
          several axes, and the write of K and V into the pages by slot
  attend  attention of one new token per request over its pages

`own = False` computes them in plain torch (32 bits, angles in 64), `own = True` calls
umic_b200. Tensors: q / k / v [tokens, heads, head_dim] bf16, pages
[num_pages, kv_heads, page_size, head_dim] bf16 or float8_e4m3fn with one fp32 scale per
KV head, lengths and tables int32.
"""

import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "umic-alpamayo_b200")


def _umic():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import umic_b200.kernels as kernels

    return kernels


# ------------------------------------------------------------------------ cases

def listed():
    lm = {"hq": 32, "hk": 8, "d": 128}
    expert = {"hq": 16, "hk": 8, "d": 128}
    return [
        # one decode step of a car's few episodes: latency is all that counts
        {"name": "plan_decode_8", "op": "plan", "requests": 8, "page": 16, "longest": 3264,
         "new": 1, "ends": 0.0, "short": False},
        # one decode step of a loaded server; a part of the requests end and give pages back
        {"name": "plan_decode_1024", "op": "plan", "requests": 1024, "page": 32,
         "longest": 4100, "new": 1, "ends": 0.1, "short": False},
        # the prompts of 32 episodes admitted at once
        {"name": "plan_prefill_32", "op": "plan", "requests": 32, "page": 64, "longest": 3300,
         "new": 3100, "ends": 0.0, "short": False},
        # attention input of one layer in a decode step of 8 episodes
        {"name": "input_decode_8", "op": "input", "tokens": 8, "page": 16, "norm": True,
         "axes": 3, "interleaved": True, "rotary": 128, "paged": True, "e4m3": False, **lm},
        # the same layer in the prefill of one episode: text and camera frames
        {"name": "input_prefill_3100", "op": "input", "tokens": 3100, "page": 32, "norm": True,
         "axes": 3, "interleaved": True, "rotary": 128, "paged": True, "e4m3": False, **lm},
        # the prefill of 8 episodes into an 8-bit cache
        {"name": "input_prefill_24800_e4m3", "op": "input", "tokens": 24800, "page": 64,
         "norm": True, "axes": 3, "interleaved": True, "rotary": 128, "paged": True,
         "e4m3": True, **lm},
        # vision tower: height and width positions of 16 images' patches, no norm, no cache
        {"name": "input_vision_16384", "op": "input", "tokens": 16384, "page": 16,
         "norm": False, "axes": 2, "interleaved": False, "rotary": 80, "paged": False,
         "e4m3": False, "hq": 16, "hk": 16, "d": 80},
        # a dense prefix of two episodes moved into pages: no norm, no rotation
        {"name": "append_6200", "op": "append", "tokens": 6200, "page": 16, "e4m3": False,
         "hk": 8, "d": 128},
        # one layer's decode attention: a single episode after its prompt
        {"name": "attend_1x3164", "op": "attend", "requests": 1, "longest": 3164,
         "ragged": False, "page": 16, "e4m3": False, **lm},
        # 8 episodes
        {"name": "attend_8x3164", "op": "attend", "requests": 8, "longest": 3164,
         "ragged": False, "page": 32, "e4m3": False, **lm},
        # a loaded server over an 8-bit cache, lengths from one token up, some slots empty
        {"name": "attend_256_e4m3", "op": "attend", "requests": 256, "longest": 4096,
         "ragged": True, "page": 64, "e4m3": True, **expert},
        # long contexts up to the model's position limit
        {"name": "attend_32x32768", "op": "attend", "requests": 32, "longest": 32768,
         "ragged": True, "page": 64, "e4m3": False, **lm},
    ]


# (query heads, kv heads, head dim, rotary dim of the text form)
_HEADS = [(32, 8, 128, 128), (16, 8, 128, 128), (8, 4, 128, 128), (28, 4, 128, 128),
          (16, 16, 80, 80), (12, 12, 64, 64), (16, 2, 64, 32), (20, 4, 96, 96),
          (16, 1, 128, 64), (8, 2, 256, 64)]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["plan", "input", "input", "append", "attend", "attend", "attend"])
    page = rng.choice([16, 32, 48, 64, 128])
    if op == "plan":
        requests = _spread(rng, 1, 1024)
        new = 1 if rng.random() < 0.5 else _spread(rng, 2, max(2, min(3100, 99200 // requests)))
        return {"op": "plan", "requests": requests, "page": page,
                "longest": new + _spread(rng, 1, 4100), "new": new,
                "ends": rng.choice([0.0, 0.1, 0.3]), "short": rng.random() < 0.3}
    hq, hk, d, rotary = rng.choice(_HEADS)
    e4m3 = rng.random() < 0.4
    if op == "append":
        return {"op": "append", "tokens": _spread(rng, 1, 24800), "page": page, "e4m3": e4m3,
                "hk": hk, "d": d}
    if op == "input":
        axes = rng.choice([1, 2, 3, 3])
        paged = rng.random() < 0.7
        return {"op": "input", "tokens": _spread(rng, 1, 24800 * 5120 // max(5120, hq * d)),
                "page": page, "norm": rng.random() < 0.7, "axes": axes,
                "interleaved": axes == 3 and rng.random() < 0.7, "rotary": rotary,
                "paged": paged, "e4m3": paged and e4m3, "hq": hq, "hk": hk, "d": d}
    requests = _spread(rng, 1, 256)
    most = min(32768, 32 * 32768 * 1024 // (requests * max(1024, hk * d)))
    return {"op": "attend", "requests": requests, "longest": _spread(rng, 1, most),
            "ragged": rng.random() < 0.7, "page": page, "e4m3": e4m3, "hq": hq, "hk": hk,
            "d": d}


# ----------------------------------------------------------------------- inputs

def _lengths(case, gen, dev):
    """Request lengths: all about the longest, or ragged from one token up with some empty."""
    n, longest = case["requests"], case["longest"]
    u = torch.rand(n, generator=gen, device=dev)
    if not case["ragged"]:
        low = max(1, longest - 64)
        lens = (low + u * (longest - low + 1)).long().clamp(max=longest)
    else:
        lens = (1 + u * longest).long().clamp(max=longest)
        empty = torch.rand(n, generator=gen, device=dev) < 0.03
        lens = torch.where(empty, torch.zeros_like(lens), lens)
    lens[0] = longest
    return lens.to(torch.int32)


def _pool(case, pages, gen, dev):
    """K and V pages and, for 8-bit ones, the scales of their KV heads."""
    shape = (2, pages, case["hk"], case["page"], case["d"])
    if not case["e4m3"]:
        pool = torch.randn(shape, generator=gen, device=dev, dtype=torch.bfloat16)
        return pool[0], pool[1], None, None
    pool = torch.randn(shape, generator=gen, device=dev, dtype=torch.float16).mul_(48.0)
    pool = pool.clamp_(-448, 448).to(torch.float8_e4m3fn)
    scales = (0.8 + 0.4 * torch.rand(2, case["hk"], generator=gen, device=dev)) / 48.0
    return pool[0], pool[1], scales[0].contiguous(), scales[1].contiguous()


def _slots(tokens, page, pages, gen, dev):
    """The slots of `tokens` tokens that fill shuffled pages from the front."""
    order = torch.randperm(pages, generator=gen, device=dev)
    t = torch.arange(tokens, device=dev)
    return (order[t // page] * page + t % page).to(torch.int32)


def _positions(case, gen, dev):
    """Positions [axes, tokens] of text runs of 28 tokens and frames of 16 x 16 patches (or,
    with two axes, of 32 x 32 patches per image), episodes of 3100 tokens far into a drive."""
    t = torch.arange(case["tokens"], device=dev)
    if case["axes"] == 2:
        inside = t % 1024
        return torch.stack((inside // 32, inside % 32))
    episode, j = t // 3100, t % 3100
    start = torch.randint(0, 29000, (int(case["tokens"] // 3100) + 1,), generator=gen,
                          device=dev)[episode]
    block, r = j // 284, j % 284
    base = start + block * 44
    if case["axes"] == 1:
        return (start + j)[None].contiguous()
    text = r < 28
    patch = (r - 28).clamp(min=0)
    return torch.stack((torch.where(text, base + r, base + 28),
                        torch.where(text, base + r, base + 28 + patch // 16),
                        torch.where(text, base + r, base + 28 + patch % 16)))


def _sections(case):
    half = case["rotary"] // 2
    if case["axes"] == 1:
        return (half,)
    if case["axes"] == 2:
        return (half // 2, half - half // 2)
    side = (half * 5) // 16  # 24 + 20 + 20 of 64
    return (half - 2 * side, side, side)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    page = case["page"]
    state = {"case": case, "page": page}
    if case["op"] == "plan":
        n = case["requests"]
        width = -(-case["longest"] // page)
        room = case["longest"] - case["new"]
        u = torch.rand(n, generator=gen, device=dev)
        lens = (u * (room + 1)).long().clamp(max=room)
        if case["new"] > 1:  # prompts: most requests are new, some continue
            lens = torch.where(torch.rand(n, generator=gen, device=dev) < 0.8,
                               torch.zeros_like(lens), lens)
        low = case["new"] if case["new"] == 1 else max(1, case["new"] // 2)
        new = torch.randint(low, case["new"] + 1, (n,), generator=gen, device=dev)
        ends = torch.rand(n, generator=gen, device=dev) < case["ends"]
        new = torch.where(ends, -lens, new)
        used = (lens + page - 1) // page
        asked = ((lens + new + page - 1) // page - used).clamp(min=0)
        free = int(asked.sum())
        spare = 16 + n // 4
        pages = n * width + spare  # a pool that could hold them all at their longest
        order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
        j = torch.arange(width, device=dev)[None]
        at = (used.cumsum(0) - used)[:, None] + j
        mine = j < used[:, None]
        table = torch.where(mine, order[at.clamp(max=pages - 1)], -1).to(torch.int32)
        in_use = int(used.sum())
        head = int(torch.randint(0, pages, (1,), generator=gen, device=dev))
        ring = torch.full((pages,), -1, dtype=torch.int32, device=dev)
        ring[(head + torch.arange(pages - in_use, device=dev)) % pages] = order[in_use:]
        count = (free * 3) // 4 if case["short"] else free + spare
        state.update(lens=lens.to(torch.int32), new=new.to(torch.int32), table=table, ring=ring,
                     span=torch.tensor([head, head + count], dtype=torch.int64, device=dev),
                     capacity=n * case["new"])
        return state
    if case["op"] == "attend":
        lens = _lengths(case, gen, dev)
        used = (lens.long() + page - 1) // page
        total = int(used.sum())
        width = -(-case["longest"] // page)
        k, v, ks, vs = _pool(case, total + 3, gen, dev)
        order = torch.randperm(total + 3, generator=gen, device=dev)
        j = torch.arange(width, device=dev)[None]
        at = (used.cumsum(0) - used)[:, None] + j
        table = torch.where(j < used[:, None], order[at.clamp(max=total + 2)], -1)
        q = torch.randn(case["requests"], case["hq"], case["d"], generator=gen, device=dev)
        state.update(q=(1.5 * q).to(torch.bfloat16), k_pages=k, v_pages=v, k_scale=ks,
                     v_scale=vs, table=table.to(torch.int32), lens=lens,
                     scale=case["d"] ** -0.5)
        return state
    tokens, hk, d = case["tokens"], case["hk"], case["d"]
    hq = case.get("hq", 0)
    qkv = torch.randn(tokens, hq + 2 * hk, d, generator=gen, device=dev).to(torch.bfloat16)
    state.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hk], v=qkv[:, hq + hk:])
    if case["op"] == "append" or case["paged"]:
        pages = -(-tokens // page) + 3
        kp, vp, ks, vs = _pool(case, pages, gen, dev)
        state.update(k_pages=kp, v_pages=vp, k_scale=ks, v_scale=vs,
                     slots=_slots(tokens, page, pages, gen, dev))
    if case["op"] == "input":
        half = case["rotary"] // 2
        i = torch.arange(half, device=dev, dtype=torch.float64)
        if case["axes"] == 2:  # each axis has its own run of frequencies
            i, n, theta = i % (half // 2), half // 2, 1e4
        else:
            n, theta = half, 1e6
        state.update(positions=_positions(case, gen, dev),
                     inv_freq=(theta ** (-i / n)).float(), sections=_sections(case),
                     interleaved=case["interleaved"], qw=None, kw=None)
        if case["norm"]:
            w = 1 + 0.1 * torch.randn(2, d, generator=gen, device=dev)
            w = w.to(torch.bfloat16)
            state.update(qw=w[0].contiguous(), kw=w[1].contiguous())
    return state


# ------------------------------------------------------------------ plain forms

def _plan(s):
    page, table, ring = s["page"], s["table"], s["ring"]
    old, new = s["lens"].long(), s["new"].long()
    head, tail = s["span"][0], s["span"][1]
    size, width = ring.numel(), table.shape[1]

    def pages(x):
        return (x + page - 1) // page

    valid = ((old >= 0) & (pages(old) <= width)
             & (old + new >= 0) & (pages(old + new) <= width))
    new = torch.where(valid, new, 0)
    before, after = pages(old), pages(old + new)
    need, give = (after - before).clamp(min=0), (before - after).clamp(min=0)
    count = new.clamp(min=0)
    need_end, give_end, count_end = need.cumsum(0), give.cumsum(0), count.cumsum(0)
    served = (valid & ((need == 0) | (need_end <= tail - head))
              & ((count == 0) | (count_end <= s["capacity"])))
    take = head + need_end - need

    start = count_end - count
    t = torch.arange(s["capacity"], device=old.device)
    r = torch.searchsorted(count_end, t, right=True).clamp(max=old.numel() - 1)
    pos = old[r] + t - start[r]
    at = pos // page
    fresh = ring[(take[r] + at - before[r]) % size]
    kept = table[r, at.clamp(0, width - 1)]
    slot = torch.where(at >= before[r], fresh, kept).long() * page + pos % page
    fine = served[r] & (t < count_end[-1])
    slots = torch.where(fine, slot, -1).to(torch.int32)
    positions = torch.where(fine, pos, -1).to(torch.int32)

    j = torch.arange(width, device=old.device)[None]
    came = served[:, None] & (j >= before[:, None]) & (j < after[:, None])
    left = served[:, None] & (j >= after[:, None]) & (j < before[:, None])
    taken = ring[(take[:, None] + j - before[:, None]) % size]
    place = (tail + (give_end - give)[:, None] + j - after[:, None]) % size
    longer = torch.cat((ring, ring[:1]))  # one more place, for what is not given back
    longer[torch.where(left, place, size)] = table
    ring.copy_(longer[:-1])
    table.copy_(torch.where(came, taken, table))
    lens = torch.where(served, old + new, old).to(torch.int32)
    cu = torch.cat((count_end[:1] * 0, count_end)).to(torch.int32)
    span = torch.stack((head + torch.where(served, need, 0).sum(),
                        tail + torch.where(served, give, 0).sum()))
    return {"kv_lens": lens, "slots": slots, "positions": positions, "cu_tokens": cu,
            "free_span": span, "block_table": table, "free_ring": ring}


def _to_pages(pages, slots, page, x, scale):
    """Writes x [tokens, heads, dim] (32 bits) at its slots, rounded to the pages' type."""
    at = slots.long()
    if scale is not None:
        x = (x / scale[:, None]).clamp(-448, 448)
    x = x.to(pages.dtype)
    if scale is not None:  # index writes go by bytes
        pages, x = pages.view(torch.uint8), x.view(torch.uint8)
    pages[at // page, :, at % page] = x


def _axis_of(s, half, dev):
    i = torch.arange(half, device=dev)
    sec = s["sections"]
    if s["interleaved"]:
        n = len(sec)
        per = torch.tensor(sec, device=dev)[i % n]
        return torch.where(i < n * per, i % n, 0)
    edges = torch.tensor(sec, device=dev).cumsum(0)
    return torch.searchsorted(edges, i, right=True)


def _rotated(x, weight, cos, sin, eps):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.float()
    half = cos.shape[-1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, rest), -1)


def _input(s):
    dev = s["k"].device
    half = s["inv_freq"].numel()
    pos = s["positions"][_axis_of(s, half, dev)].t().double()  # [tokens, half]
    angle = pos * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q = _rotated(s["q"], s["qw"], cos, sin, 1e-6).to(torch.bfloat16)
    k = _rotated(s["k"], s["kw"], cos, sin, 1e-6)
    if "slots" not in s:
        return {"q": q, "k": k.to(torch.bfloat16)}
    _to_pages(s["k_pages"], s["slots"], s["page"], k, s["k_scale"])
    _to_pages(s["v_pages"], s["slots"], s["page"], s["v"].float(), s["v_scale"])
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _append(s):
    _to_pages(s["k_pages"], s["slots"], s["page"], s["k"].float(), s["k_scale"])
    _to_pages(s["v_pages"], s["slots"], s["page"], s["v"].float(), s["v_scale"])
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _gathered(pages, table, scale):
    """[requests, heads, tokens, dim] in 32 bits."""
    x = pages.view(torch.uint8) if scale is not None else pages
    x = x[table.long().clamp(min=0)]  # [requests, width, heads, page, dim]
    x = x.view(pages.dtype).float() if scale is not None else x.float()
    x = x.transpose(1, 2).flatten(2, 3)
    return x if scale is None else x * scale[None, :, None, None]


def _attend(s):
    b, hq, d = s["q"].shape
    hk = s["k_pages"].shape[1]
    q = s["q"].float().view(b, hk, hq // hk, d)
    k = _gathered(s["k_pages"], s["table"], s["k_scale"])
    score = (q @ k.transpose(-1, -2)) * s["scale"]
    del k
    j = torch.arange(score.shape[-1], device=q.device)
    away = j >= s["lens"].long()[:, None, None, None]
    score = score.masked_fill(away, float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = (score - top).exp()
    total = p.sum(-1, keepdim=True)
    v = _gathered(s["v_pages"], s["table"], s["v_scale"])
    v = v.masked_fill(away[:, :, 0, :, None], 0.0)
    out = (p @ v) / total.clamp(min=torch.finfo(torch.float32).tiny)
    lse = torch.where(total > 0, top + total.log(), float("-inf"))
    return {"out": out.reshape(b, hq, d).to(torch.bfloat16), "lse": lse.reshape(b, hq)}


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"plan": _plan, "input": _input, "append": _append, "attend": _attend}[op](state)
    kernels = _umic()
    s = state
    if op == "plan":
        p = kernels.paged_plan(s["lens"], s["new"], s["table"], s["ring"], s["span"],
                               s["page"], s["capacity"])
        return {"kv_lens": p.kv_lens, "slots": p.slots, "positions": p.positions,
                "cu_tokens": p.cu_tokens, "free_span": p.free_span, "block_table": s["table"],
                "free_ring": s["ring"]}
    if op == "attend":
        out, lse = kernels.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"],
                                           s["lens"], s["scale"], k_scale=s["k_scale"],
                                           v_scale=s["v_scale"], return_lse=True)
        return {"out": out, "lse": lse}
    if op == "append":
        kernels.paged_kv_append(s["k_pages"], s["v_pages"], s["k"], s["v"], s["slots"],
                                k_scale=s["k_scale"], v_scale=s["v_scale"])
        return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if "slots" not in s:
        q, k = kernels.qk_norm_mrope_kv(s["q"], s["k"], None, s["positions"], s["inv_freq"],
                                        s["sections"], interleaved=s["interleaved"],
                                        q_weight=s["qw"], k_weight=s["kw"])
        return {"q": q, "k": k}
    q, _ = kernels.qk_norm_mrope_kv(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"],
                                    s["sections"], interleaved=s["interleaved"],
                                    q_weight=s["qw"], k_weight=s["kw"], k_pages=s["k_pages"],
                                    v_pages=s["v_pages"], slots=s["slots"],
                                    k_scale=s["k_scale"], v_scale=s["v_scale"])
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


# ------------------------------------------------------------------------- work

def work(case):
    if case["op"] == "plan":
        n, cap = case["requests"], case["requests"] * case["new"]
        # lengths and asks in, lengths and offsets out; slot and position of each token;
        # an entry of the table and of the ring for each page that changes hands
        return {"bytes": 16 * n + 8 * cap + 8 * (cap // case["page"] + 1) + 32, "flops": 0}
    hk, d, e = case["hk"], case["d"], 1 if case["e4m3"] else 2
    if case["op"] == "attend":
        b, longest = case["requests"], case["longest"]
        tokens = b * longest
        if case["ragged"]:
            tokens = longest + int((b - 1) * 0.97 * (longest + 1) / 2)
        return {"bytes": 2 * tokens * hk * d * e + b * case["hq"] * (4 * d + 4),
                "flops": 4 * tokens * case["hq"] * d}
    t = case["tokens"]
    if case["op"] == "append":
        return {"bytes": t * (2 * hk * d * (2 + e) + 4), "flops": 0}
    paged = case["paged"]
    rows = case["hq"] * 4 + hk * ((2 + e) * 2 if paged else 4)
    return {"bytes": t * (rows * d + 8 * case["axes"] + (4 if paged else 0)),
            "flops": t * (case["hq"] + hk) * d * (7 if case["norm"] else 3)}


# ------------------------------------------------------------------------ exact

def exact(case, seed):
    """The operators from their definitions in 64 bits."""
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    page = case["page"]
    if case["op"] == "attend":
        b, hq, d = s["q"].shape
        hk = case["hk"]
        out = torch.zeros(b, hq, d, dtype=torch.float64, device="cuda")
        lse = torch.full((b, hq), float("-inf"), dtype=torch.float64, device="cuda")
        for r, n in enumerate(s["lens"].tolist()):
            if n == 0:
                continue
            ids = s["table"][r, :-(-n // page)].long()
            kv = []
            for pages, scale in ((s["k_pages"], s["k_scale"]), (s["v_pages"], s["v_scale"])):
                if scale is None:
                    x = pages[ids].double()
                else:
                    x = pages.view(torch.uint8)[ids].view(pages.dtype).double()
                    x = x * scale.double().view(1, hk, 1, 1)
                kv.append(x.permute(1, 0, 2, 3).reshape(hk, -1, d)[:, :n])
            q = s["q"][r].double().view(hk, hq // hk, d)
            logit = torch.einsum("hgd,htd->hgt", q, kv[0]) * s["scale"]
            lse[r] = torch.logsumexp(logit, -1).reshape(hq)
            out[r] = torch.einsum("hgt,htd->hgd", torch.softmax(logit, -1), kv[1]).reshape(hq, d)
        return {"out": out, "lse": lse}

    def stored(pages, scale, x):
        flat = pages.double().permute(0, 2, 1, 3).reshape(-1, case["hk"], case["d"]).clone()
        if scale is not None:
            x = torch.clamp(x / scale.double().view(1, -1, 1), -448.0, 448.0)
        flat[s["slots"].long()] = x
        return flat.view(-1, page, case["hk"], case["d"]).permute(0, 2, 1, 3)

    if case["op"] == "append":
        return {"k_pages": stored(s["k_pages"], s["k_scale"], s["k"].double()),
                "v_pages": stored(s["v_pages"], s["v_scale"], s["v"].double())}
    half = case["rotary"] // 2
    axis = []
    for i in range(half):
        if case["interleaved"]:
            a = i % 3
            axis.append(a if a and i < 3 * s["sections"][a] else 0)
        else:
            a, edge = 0, s["sections"][0]
            while i >= edge:
                a += 1
                edge += s["sections"][a]
            axis.append(a)
    theta = torch.stack([s["positions"][a].double() * s["inv_freq"][i].double()
                         for i, a in enumerate(axis)], -1)
    turn = torch.polar(torch.ones_like(theta), theta)[:, None]

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6) * w.double()
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
        return torch.cat((z.real, z.imag, x[..., 2 * half:]), -1)

    q, k = turned(s["q"], s["qw"]), turned(s["k"], s["kw"])
    if not case["paged"]:
        return {"q": q, "k": k}
    return {"q": q, "k_pages": stored(s["k_pages"], s["k_scale"], k),
            "v_pages": stored(s["v_pages"], s["v_scale"], s["v"].double())}
