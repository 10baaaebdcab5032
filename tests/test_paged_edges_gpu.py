"""GPU tests of the paged-cache serving operators at the edges of what their documentation
allows: layouts, the largest tables, borders of the cache's type, requests that a long walk
of one warp covers."""

import itertools

import pytest
import torch

from oracle import paged as oracle
from umic_b200 import _lib
from umic_b200.kernels import paged_attention, paged_kv_append, qk_norm_mrope_kv

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _ordered(shape, order, dev, pad=0):
    """Zeros of `shape` [..., D] whose leading axes lie in memory in `order`; the innermost
    of them with `pad` unused elements behind each row."""
    dims = [shape[a] for a in order]
    wide = torch.zeros(*dims, shape[-1] + pad, dtype=torch.bfloat16, device=dev)[..., :shape[-1]]
    back = [order.index(a) for a in range(len(order))]
    return wide.permute(*back, len(order))


# ----------------------------------------------------------------- layouts

@pytest.mark.parametrize("pad", [0, 8])
def test_input_writes_rows_in_any_order_of_axes(cuda, pad):
    """Rotated q and k, and pages, in every order of their axes, tight or with room between
    the rows: the bits of the plain layout."""
    g = _gen(41)
    t, hq, hk, d, page = 37, 6, 3, 64, 16
    q, k, v = (torch.randn(t, h, d, generator=g).to(torch.bfloat16).to(cuda)
               for h in (hq, hk, hk))
    pos = torch.randint(0, 5000, (3, t), generator=g).to(cuda)
    inv = (1e6 ** (-torch.arange(32) / 32)).to(cuda)
    slots = torch.randperm(5 * page, generator=g)[:t].int().to(cuda)
    args = (q, k, v, pos, inv, (12, 10, 10))
    want_q, want_k = qk_norm_mrope_kv(q, k, None, *args[3:])
    kp = torch.zeros(5, hk, page, d, dtype=torch.bfloat16, device=cuda)
    vp = torch.zeros_like(kp)
    qk_norm_mrope_kv(*args, k_pages=kp, v_pages=vp, slots=slots)
    for order in itertools.permutations(range(2)):
        q_out = _ordered((t, hq, d), order, cuda, pad=pad)
        k_out = _ordered((t, hk, d), order, cuda, pad=pad)
        qk_norm_mrope_kv(q, k, None, *args[3:], q_out=q_out, k_out=k_out)
        assert torch.equal(q_out, want_q) and torch.equal(k_out, want_k)
    for order in itertools.permutations(range(3)):
        kx, vx = (_ordered(kp.shape, order, cuda, pad=pad) for _ in range(2))
        q_out, _ = qk_norm_mrope_kv(*args, k_pages=kx, v_pages=vx, slots=slots)
        assert torch.equal(q_out, want_q)
        assert torch.equal(kx, kp) and torch.equal(vx, vp)


def test_single_entries_need_no_stride(cuda):
    """The stride of an axis of one entry is never used: one token, one head, one page."""
    d = 64
    g = _gen(42)
    k = torch.randn(1, 2, d, generator=g).to(torch.bfloat16).to(cuda)
    pages = torch.zeros(2 * 16 * d, dtype=torch.bfloat16, device=cuda)
    kp = pages.as_strided((1, 2, 16, d), (0, 16 * d, d, 1))
    vp = torch.zeros_like(pages).as_strided((1, 2, 16, d), (0, 16 * d, d, 1))
    slots = torch.tensor([7], dtype=torch.int32, device=cuda)
    paged_kv_append(kp, vp, k, -k, slots)
    assert torch.equal(kp[0, :, 7], k[0]) and torch.equal(vp[0, :, 7], -k[0])
    assert int((pages != 0).sum()) <= 2 * d


def test_attention_writes_rows_in_any_order_of_axes(cuda):
    g = _gen(43)
    kp, vp = torch.randn(2, 6, 2, 16, 64, generator=g).to(torch.bfloat16).to(cuda)
    q = torch.randn(3, 8, 64, generator=g).to(torch.bfloat16).to(cuda)
    table = torch.randperm(6, generator=g).int().view(3, 2).to(cuda)
    lens = torch.tensor([32, 0, 19], dtype=torch.int32, device=cuda)
    want = paged_attention(q, kp, vp, table, lens, 0.2)
    for order, pad in itertools.product(itertools.permutations(range(2)), (0, 8)):
        out = _ordered((3, 8, 64), order, cuda, pad=pad)
        out.fill_(9.0)
        paged_attention(q, kp, vp, table, lens, 0.2, out=out)
        assert torch.equal(out, want)


# ------------------------------------------------------------ longest rows

@pytest.mark.parametrize("e4m3", [False, True])
def test_attention_over_the_longest_row(cuda, e4m3):
    """A row of 2^31 - 16 tokens (262657 entries that name one page of 8176), beside a short
    one. All scores are 0 and V of a dim is the same in every token, so the output is that
    value and the lse the length's logarithm.

    Bounds: a warp sums its share of the line, one product of 16 tokens after the other, each
    off by at most a step of the running sum (2^-23), and the output is rounded once (2^-8).
    The weights are 1 and their sums whole numbers, exact in a lane; about 200 partial sums
    are joined (2^-24 of the sum each), and the logarithm, 22 at most, is good to four half
    steps.
    """
    page, width, d = 8176, 262657, 64
    n = page * width
    assert n == 2 ** 31 - 16
    dt = torch.float8_e4m3fn if e4m3 else torch.bfloat16
    dims = (torch.arange(d) % 3).float()
    kp = torch.ones(1, 1, page, d).to(dt).to(cuda)
    vp = dims.expand(1, 1, page, d).contiguous().to(dt).to(cuda)
    table = torch.zeros(2, width, dtype=torch.int32, device=cuda)
    lens = torch.tensor([n, 40], dtype=torch.int32, device=cuda)
    q = torch.zeros(2, 3, d, dtype=torch.bfloat16, device=cuda)
    out, lse = paged_attention(q, kp, vp, table, lens, 0.3, return_lse=True)
    warps = torch.cuda.get_device_properties(cuda).multi_processor_count * 8
    rel = 2.0 ** -8 + (n / 16 / warps + 200) * 2.0 ** -23
    assert bool(((out.cpu().float() - dims).abs() <= dims * rel).all())
    want = lens.cpu().double().log()[:, None].expand(2, 3)
    assert bool(((lse.cpu().double() - want).abs() <= (200 + 4 * 22) * 2.0 ** -24).all())


# ------------------------------------------------------- borders of e4m3

def _border_scales():
    """(scales, values) fp32 of quotients value / scale that lie on or next to the middle of
    two e4m3 values: value 128 .. 255 over 17, 19 .. 31, and the neighbours of that scale."""
    x = torch.arange(128, 256).float().repeat_interleave(8)
    s = x / torch.arange(17, 33, 2).float().repeat(128)
    up, down = (torch.nextafter(s, s + d) for d in (1.0, -1.0))
    return torch.cat((down, s, up)), x.repeat(3)


def _stored(x, s):
    """The page's bytes for x over s: the quotient in fp32, saturated, rounded to e4m3."""
    return (x / s).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


@pytest.mark.parametrize("form", ["append", "rotated", "normed"])
def test_e4m3_pages_hold_the_rounded_quotient(cuda, form):
    """K and V in e4m3 pages are the value divided by its head's scale, not multiplied by the
    scale's rounded inverse, bit for bit: as they are, rotated by position 0, and (V) beside a
    normed K. A product with the inverse stores the neighbour of some of these quotients."""
    scale, x = _border_scales()
    assert bool((_stored(x, scale) != _stored(x * (1 / scale), torch.ones_like(x))).any())
    hk, d = len(x), 16
    rows = x[:, None] * 2.0 ** -torch.arange(d).float()  # the border at every exponent, then
    rows[:, 1::2] *= -1                                  # smaller values, subnormal at last
    k = rows.to(torch.bfloat16)[None].repeat(3, 1, 1)
    k[1] *= 8  # up to 248 and, over the border of the type, saturated
    k[2] *= 32
    pages = torch.zeros(2, 1, hk, 16, d, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)
    slots = torch.tensor([3, 0, 9], dtype=torch.int32, device=cuda)
    kd, s = k.to(cuda), scale.to(cuda)
    if form == "append":
        paged_kv_append(pages[0], pages[1], kd, -kd, slots, k_scale=s, v_scale=s)
    else:
        w = torch.ones(d, dtype=torch.bfloat16, device=cuda) if form == "normed" else None
        qk_norm_mrope_kv(None, kd, -kd, torch.zeros(1, 3, dtype=torch.int32, device=cuda),
                         torch.ones(8, device=cuda), (8,), k_weight=w, k_pages=pages[0],
                         v_pages=pages[1], slots=slots, k_scale=s, v_scale=s)
    want = _stored(k.float(), scale[:, None])
    got = pages.view(torch.uint8)[:, 0][:, :, [3, 0, 9]].transpose(1, 2).cpu()
    assert torch.equal(got[1], want ^ 0x80)
    if form != "normed":
        assert torch.equal(got[0], want)


@pytest.mark.parametrize("rotated", [False, True])
def test_e4m3_pages_keep_special_values(cuda, rotated):
    """Zeros of both signs, infinities (saturated), NaN and the smallest and largest bf16
    values, over scales from 2^-100 to 2^100 and 1e-30."""
    big, small = torch.finfo(torch.bfloat16).max, torch.finfo(torch.bfloat16).tiny
    x = torch.tensor([0.0, -0.0, float("inf"), -float("inf"), float("nan"), big, -big, small,
                      -small, 448.0, -449.0, 464.0, 465.0, 1.0, -(2.0 ** -9), 2.0 ** -10])
    scale = torch.tensor([2.0 ** -100, 1e-30, 2.0 ** -10, 1.0, 0.3, 7.0, 2.0 ** 100])
    k = x.to(torch.bfloat16).expand(1, len(scale), 16).contiguous().to(cuda)
    pages = torch.zeros(2, 1, len(scale), 16, 16, dtype=torch.uint8, device=cuda)
    pool, s = pages.view(torch.float8_e4m3fn), scale.to(cuda)
    slots = torch.tensor([2], dtype=torch.int32, device=cuda)
    if rotated:  # pairs of a finite element and one that is not are NaN: no rotation of pairs
        k = torch.where(k.isfinite(), k, 1.0)
        qk_norm_mrope_kv(None, k, k, torch.zeros(1, 1, dtype=torch.int32, device=cuda),
                         torch.ones(8, device=cuda), (8,), k_pages=pool[0], v_pages=pool[1],
                         slots=slots, k_scale=s, v_scale=s)
    else:
        paged_kv_append(pool[0], pool[1], k, k, slots, k_scale=s, v_scale=s)
    want = _stored(k[0].float().cpu(), scale[:, None])
    got = pages[:, 0, :, 2].cpu()
    nan = (want & 0x7f) == 0x7f
    assert bool(((got & 0x7f)[:, nan] == 0x7f).all())
    same = got == want
    if rotated:  # x - y * 0 of K may lose the sign of a zero
        same[0] |= ((got[0] | want) & 0x7f) == 0
    assert bool((same | nan).all())


# ------------------------------------------------------------- long walks

WALKS = [
    # hq, hk, d, rotary sections, interleaved
    (32, 8, 128, (24, 20, 20), True),
    (16, 16, 80, (20, 20), False),
    (12, 3, 96, (8, 4, 4), True),
    (6, 2, 256, (128,), False),
]


@pytest.mark.parametrize("walk", WALKS, ids=lambda w: "x".join(map(str, w[:3])))
@pytest.mark.parametrize("tokens", [9001, 24800])
@pytest.mark.parametrize("form", ["bf16", "e4m3", "plain", "append", "append_e4m3"])
def test_input_of_many_tokens_a_warp(cuda, walk, tokens, form):
    """So many tokens that a warp walks over several (10 and more of 24800): every row and
    every slot has the bits of calls on 400 tokens, of which a warp sees no more than two, and
    tokens picked at random agree with the 64-bit oracle. Values differ by token, head, dim and
    kind of row; slots are shuffled, some tokens have none, and other slots keep what they held.
    """
    hq, hk, d, sections, inter = walk
    e4m3, append = "e4m3" in form, "append" in form
    g = torch.Generator(device=cuda).manual_seed(tokens + d)
    qkv = torch.randn(tokens, hq + 2 * hk, d, generator=g, device=cuda).to(torch.bfloat16)
    q, k, v = qkv.split((hq, hk, hk), 1)
    half = sum(sections)
    inv = (1e6 ** (-torch.arange(half, device=cuda) / half)).float()
    pos = torch.randint(0, 32768, (len(sections), tokens), generator=g, device=cuda)
    weights = (1 + 0.2 * torch.randn(2, d, generator=g, device=cuda)).to(torch.bfloat16)
    norm = dict(q_weight=weights[0], k_weight=weights[1]) if form != "plain" else {}
    page = 16
    pages = tokens // page + 3
    slots = torch.randperm(pages * page, generator=g, device=cuda)[:tokens].int()
    slots[3::11] = -1
    scales = (0.5 + torch.rand(2, hk, generator=g, device=cuda)) / 40

    def filled():
        x = torch.full((2, pages, hk, page, d), 0x3c, dtype=torch.uint8, device=cuda)
        return x.view(torch.float8_e4m3fn) if e4m3 else x.to(torch.bfloat16)

    def call(pool, a, b):
        kwargs = {}
        if e4m3:
            kwargs = dict(k_scale=scales[0], v_scale=scales[1])
        if append:
            return paged_kv_append(pool[0], pool[1], k[a:b], v[a:b], slots[a:b], **kwargs)
        if form != "plain":
            kwargs.update(k_pages=pool[0], v_pages=pool[1], slots=slots[a:b])
        return qk_norm_mrope_kv(q[a:b], k[a:b], v[a:b], pos[:, a:b], inv, sections,
                                interleaved=inter, **norm, **kwargs)

    pool, parts = filled(), filled()
    whole = call(pool, 0, tokens)
    pieces = [call(parts, a, min(a + 400, tokens)) for a in range(0, tokens, 400)]
    as_bytes = lambda x: x.view(torch.uint8) if e4m3 else x  # noqa: E731
    assert torch.equal(as_bytes(pool), as_bytes(parts))
    free = torch.ones(pages * page, dtype=torch.bool, device=cuda)
    free[slots[slots >= 0].long()] = False
    untouched = as_bytes(pool).transpose(2, 3).flatten(1, 2)[:, free]
    assert bool((untouched == 0x3c).all())
    on = torch.nonzero(slots >= 0)[:, 0]
    at = slots[on].long()
    if not e4m3:
        stored = pool[1].transpose(1, 2).flatten(0, 1)
        if form != "plain":
            assert torch.equal(stored[at], v[on])
        if append:
            assert torch.equal(pool[0].transpose(1, 2).flatten(0, 1)[at], k[on])
    elif append:
        for kind, x in enumerate((k, v)):
            want = (x[on].float() / scales[kind][:, None]).clamp(-448, 448)
            got = as_bytes(pool)[kind].transpose(1, 2).flatten(0, 1)[at]
            assert torch.equal(got, want.to(torch.float8_e4m3fn).view(torch.uint8))
    if append:
        return
    assert torch.equal(whole[0], torch.cat([x[0] for x in pieces]))
    pick = torch.randperm(tokens, generator=_gen(d))[:300].to(cuda)
    args = (pos[:, pick], inv, sections, inter)
    u = 2.0 ** -24  # 40 roundings in fp32 of |a| + |b|, then half a step of the output's type
    y, mag = oracle.norm_mrope(q[pick], norm.get("q_weight"), 1e-6, *args)
    bound = mag * 40 * u
    bound = bound + (y.abs() + bound) * 2.0 ** -8
    assert bool(((whole[0][pick].cpu().double() - y).abs() <= bound).all())
    y, mag = oracle.norm_mrope(k[pick], norm.get("k_weight"), 1e-6, *args)
    if form == "plain":
        assert torch.equal(whole[1], torch.cat([x[1] for x in pieces]))
        got, scale = whole[1][pick].cpu().double(), 1.0
    else:
        there = (slots[pick] >= 0).cpu()
        y, mag = y[there], mag[there]
        got = as_bytes(pool)[0].transpose(1, 2).flatten(0, 1)[slots[pick].long()[there.to(cuda)]]
        got = (got.view(torch.float8_e4m3fn).float() if e4m3 else got).cpu().double()
        scale = scales[0].cpu().double()[:, None] if e4m3 else 1.0
    bound = mag * 40 * u / scale
    y = (y / scale).clamp(-448, 448) if e4m3 else y
    half_step = torch.clamp((y.abs() + bound) * 2.0 ** -4, min=2.0 ** -10) if e4m3 else \
        (y.abs() + bound) * 2.0 ** -8
    assert bool(((got - y).abs() <= bound + half_step).all())


# ----------------------------------------------------------------- streams

@pytest.mark.parametrize("raw", [True, False])
def test_calls_go_to_the_current_stream(cuda, raw, monkeypatch):
    """The handle passed to the library is torch's current stream: the default one, a side
    stream, the one that a graph is captured on; with and without torch's short cut to it."""
    if not raw:
        monkeypatch.setattr(_lib, "_raw_stream", None)
    anywhere = torch.device("cuda")
    side = torch.cuda.Stream()
    for dev in (cuda, anywhere):
        assert _lib.stream_ptr(dev) == torch.cuda.current_stream(cuda).cuda_stream
        with torch.cuda.stream(side):
            assert _lib.stream_ptr(dev) == side.cuda_stream
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        assert _lib.stream_ptr(cuda) == torch.cuda.current_stream(cuda).cuda_stream != 0
        torch.zeros(1, device=cuda)


# ---------------------------------------------------------------- sections

@pytest.mark.parametrize("sections", [(24, 20, 20), (10, 27, 27), (0, 32, 32), (64, 0, 0)])
def test_interleaved_sections_past_the_frequencies(cuda, sections):
    """Interleaved sections of every reach turn what the documented rule says."""
    g = _gen(51)
    x = torch.randn(64, 3, 128, generator=g).to(torch.bfloat16)
    pos = torch.randint(0, 32768, (3, 64), generator=g)
    inv = 1e6 ** (-torch.arange(64) / 64)
    got, _ = qk_norm_mrope_kv(x.to(cuda), x[:, :1].to(cuda), None, pos.to(cuda), inv.to(cuda),
                              sections, interleaved=True)
    y, mag = oracle.norm_mrope(x, None, 0.0, pos, inv, sections, True)
    bound = mag * 40 * 2.0 ** -24  # roundings in fp32, then half a step of bf16
    bound = bound + (y.abs() + bound) * 2.0 ** -8
    assert bool(((got.cpu().double() - y).abs() <= bound).all())


# --------------------------------------------------------------- infinity

@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_infinite_values_reach_their_rows(cuda, sign):
    """An infinity in V of a token in use comes out as an infinity or NaN in its dim of the
    heads of its KV head, and nowhere else."""
    g = _gen(53)
    kp, vp = torch.randn(2, 4, 2, 16, 64, generator=g).to(torch.bfloat16).to(cuda)
    q = torch.randn(2, 6, 64, generator=g).to(torch.bfloat16).to(cuda)
    table = torch.arange(4, dtype=torch.int32, device=cuda).view(2, 2)
    lens = torch.tensor([32, 20], dtype=torch.int32, device=cuda)
    clean = paged_attention(q, kp, vp, table, lens, 0.1)
    vp[1, 1, 3, 17] = sign * float("inf")
    out = paged_attention(q, kp, vp, table, lens, 0.1)
    assert not bool(out[0, 3:, 17].isfinite().any())
    out[0, 3:, 17] = clean[0, 3:, 17]
    assert torch.equal(out, clean)


# ------------------------------------------------- optional and shared arguments

def _e4m3_pool(g, pages, heads, page, d, dev):
    x = (torch.randn(2, pages, heads, page, d, generator=g) * 3).clamp(-448, 448)
    return x.to(torch.float8_e4m3fn).to(dev)


@pytest.mark.parametrize("given", ["none", "k", "v"])
def test_e4m3_pages_without_scales(cuda, given):
    """A scale that is not given is 1, for K and V each, in the write and in the attention."""
    g = _gen(57)
    pool = _e4m3_pool(g, 5, 2, 16, 64, cuda)
    other = pool.view(torch.uint8).clone().view(pool.dtype)
    s = (0.5 + torch.rand(2, generator=g)).to(cuda)
    one = torch.ones(2, device=cuda)
    some = {} if given == "none" else {f"{given}_scale": s}
    full = {"k_scale": one, "v_scale": one, **some}
    k, v = torch.randn(2, 9, 2, 64, generator=g).to(torch.bfloat16).to(cuda)
    slots = torch.randperm(80, generator=g)[:9].int().to(cuda)
    paged_kv_append(pool[0], pool[1], k, v, slots, **some)
    paged_kv_append(other[0], other[1], k, v, slots, **full)
    assert torch.equal(pool.view(torch.uint8), other.view(torch.uint8))
    q = torch.randn(2, 8, 64, generator=g).to(torch.bfloat16).to(cuda)
    table = torch.tensor([[4, 1, 0], [2, 3, 0]], dtype=torch.int32, device=cuda)
    lens = torch.tensor([40, 17], dtype=torch.int32, device=cuda)
    a = paged_attention(q, pool[0], pool[1], table, lens, 0.1, return_lse=True, **some)
    b = paged_attention(q, pool[0], pool[1], table, lens, 0.1, return_lse=True, **full)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_attention_tables_of_every_kind(cuda):
    """A table of no columns, one row for all requests, rows far apart; no requests at all."""
    g = _gen(59)
    kp, vp = torch.randn(2, 6, 2, 16, 64, generator=g).to(torch.bfloat16).to(cuda)
    q = torch.randn(3, 4, 64, generator=g).to(torch.bfloat16).to(cuda)
    lens = torch.tensor([33, 48, 5], dtype=torch.int32, device=cuda)
    row = torch.tensor([[3, 0, 5]], dtype=torch.int32, device=cuda)
    want, lse = paged_attention(q, kp, vp, row.repeat(3, 1), lens, 0.2, return_lse=True)
    assert torch.equal(paged_attention(q, kp, vp, row.expand(3, 3), lens, 0.2), want)
    wide = torch.full((3, 11), -1, dtype=torch.int32, device=cuda)
    wide[:, 4:7] = row
    assert torch.equal(paged_attention(q, kp, vp, wide[:, 4:7], lens, 0.2), want)
    none = torch.zeros(3, 0, dtype=torch.int32, device=cuda)
    out, lse = paged_attention(q, kp, vp, none, torch.zeros_like(lens), 0.2, return_lse=True)
    assert bool((out == 0).all()) and bool((lse == float("-inf")).all())
    out, lse = paged_attention(q[:0], kp, vp, row[:0], lens[:0], 0.2, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


def test_attention_over_its_own_queries(cuda):
    """out may be q: whole, split and empty requests, the bits of a separate output."""
    g = _gen(61)
    for d, lens in ((64, [500, 0, 3, 16]), (80, [37, 1200, 1, 20]), (128, [90] * 40)):
        lens = torch.tensor(lens, dtype=torch.int32)
        b, width = len(lens), -(-int(lens.max()) // 16)
        kp, vp = torch.randn(2, b * width, 2, 16, d, generator=g).to(torch.bfloat16).to(cuda)
        table = torch.randperm(b * width, generator=g).int().view(b, width).to(cuda)
        q = torch.randn(b, 8, d, generator=g).to(torch.bfloat16).to(cuda)
        want = paged_attention(q, kp, vp, table, lens.to(cuda), 0.1)
        got = paged_attention(q, kp, vp, table, lens.to(cuda), 0.1, out=q)
        assert got is q and torch.equal(got, want)


def test_first_calls_of_no_tokens(cuda):
    """Steps and writes of no tokens leave everything as it is."""
    from umic_b200.paged import PagedKVCache

    cache = PagedKVCache.allocate(1, 4, 2, 64, 16, 3, 2, cuda)
    cache.slab.zero_()
    plan = cache.step(torch.zeros(3, dtype=torch.int32, device=cuda), 0)
    x = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=cuda)
    assert plan.slots.numel() == 0 and plan.cu_tokens.tolist() == [0] * 4
    q = cache.write(0, x, x, x, plan, plan.positions.expand(3, -1), torch.ones(32, device=cuda),
                    (12, 10, 10))
    cache.append(0, x, x, plan)
    assert q.shape == (0, 2, 64) and cache.kv_lens.tolist() == [0] * 3
    assert cache.free_pages() == 4 and not bool(cache.slab.any())
    assert _lib.device_errors(cuda) == 0
