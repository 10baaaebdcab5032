"""GPU parity of the paged-cache serving operators against the 64-bit oracle.

Whole numbers (the plan) must be equal. Floating outputs are held to one rounding of the
output's type -- half a step: 2^-8 of the value for bf16, 2^-4 (and 2^-10 below the
smallest normal) for e4m3 -- plus a bound on the fp32 arithmetic before it, derived at
each use from the number of roundings it makes.
"""

import pytest
import torch

from oracle import paged as oracle
from umic_b200 import _lib
from umic_b200.kernels import (paged_attention, paged_kv_append, paged_plan, qk_norm_mrope_kv,
                               stats)

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
U = 2.0 ** -24  # half a step of fp32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# --------------------------------------------------------------------- plan

def _plan_case(seed, requests, page, width, new_max, ends, free_share, spare=5, head=None):
    """A consistent pool: every page is in one row or in the ring. Returns CPU tensors."""
    g = _gen(seed)
    room = width * page
    lens = torch.randint(0, room + 1, (requests,), generator=g)
    lens[torch.rand(requests, generator=g) < 0.3] = 0
    new = torch.minimum(torch.randint(0, new_max + 1, (requests,), generator=g), room - lens)
    cut = torch.rand(requests, generator=g) < ends
    drop = (torch.rand(requests, generator=g) * (lens + 1)).long().clamp(max=lens)
    drop = torch.where(torch.rand(requests, generator=g) < 0.5, lens, drop)
    new = torch.where(cut, -drop, new)
    used = -(-lens // page)
    asked = int((-(-(lens + new) // page) - used).clamp(min=0).sum())
    pages = int(used.sum()) + asked + spare
    order = torch.randperm(pages, generator=g).int()
    table = torch.full((requests, width), -7, dtype=torch.int32)
    at = 0
    for r in range(requests):
        n = int(used[r])
        table[r, :n] = order[at:at + n]
        at += n
    free = min(int(asked * free_share) + (spare if free_share >= 1 else 0), pages - at)
    ring = torch.full((pages,), -1, dtype=torch.int32)
    head = int(torch.randint(0, 3 * pages, (1,), generator=g)) if head is None else head
    for i in range(free):
        ring[(head + i) % pages] = order[at + i]
    return lens.int(), new.int(), table, ring, torch.tensor([head, head + free])


def _check_plan(cuda, lens, new, table, ring, span, page, capacity, strided=False,
                in_place=False, err=None):
    want = oracle.paged_plan(lens, new, table, ring, span, page, capacity)
    _lib.device_errors(cuda)
    t = table.to(cuda)
    if strided:
        wide = torch.full((table.shape[0], table.shape[1] + 3), -9, dtype=torch.int32,
                          device=cuda)
        wide[:, :-3] = t
        t = wide[:, :-3]
    rg, sp, ln = ring.to(cuda), span.to(cuda), lens.to(cuda)
    kw = {"out_lens": ln, "out_span": sp} if in_place else {}
    p = paged_plan(ln, new.to(cuda), t, rg, sp, page, capacity, **kw)
    got = {**p._asdict(), "table": t, "ring": rg}
    for k, v in want.items():
        if k != "unserved":
            assert torch.equal(got[k].cpu().long(), v.long()), k
    if strided:
        assert bool((wide[:, -3:] == -9).all())
    if in_place:
        assert p.kv_lens is ln and p.free_span is sp
    expected = (_lib.DEVERR_PAGES if want["unserved"] else 0) if err is None else err
    assert _lib.device_errors(cuda) == expected


@pytest.mark.parametrize("requests,page,width,new_max", [
    (1, 16, 1, 16), (1, 1, 7, 3), (7, 16, 5, 1), (33, 48, 9, 100), (256, 16, 21, 1),
    (1000, 32, 6, 5), (1025, 7, 4, 3), (3, 64, 300, 9000), (8192, 16, 2, 2)])
@pytest.mark.parametrize("ends,free_share", [(0.0, 1.0), (0.3, 1.0), (0.2, 0.5), (0.0, 0.0)])
def test_plan_matches_oracle(cuda, requests, page, width, new_max, ends, free_share):
    c = _plan_case(requests + page, requests, page, width, new_max, ends, free_share)
    asked = int(c[1].clamp(min=0).sum())
    _check_plan(cuda, *c, page, asked + 13, strided=ends > 0, in_place=free_share == 0.5)


@pytest.mark.parametrize("room", [0, 1, 40, 41])
def test_plan_capacity_ends_the_step(cuda, room):
    """Requests whose tokens no longer fit the slots are not served; the slots of a request
    that is cut in the middle are all -1."""
    c = _plan_case(5, 12, 16, 8, 20, 0.0, 1.0)
    _check_plan(cuda, *c, 16, room)


def test_plan_refuses_single_requests_by_value(cuda):
    """Negative lengths, crops below zero, rows too narrow and lengths past the row: those
    requests keep what they had, the others are served."""
    lens = torch.tensor([5, -1, 16, 3, 40, 64, 2], dtype=torch.int32)
    new = torch.tensor([1, 1, -17, 62, -8, 0, 2 ** 31 - 1], dtype=torch.int32)
    table = torch.arange(28, dtype=torch.int32).view(7, 4)
    ring = torch.full((40,), -1, dtype=torch.int32)
    ring[:12] = torch.arange(28, 40)
    _check_plan(cuda, lens, new, table, ring, torch.tensor([0, 12]), 16, 64)
    lens[3] = 100  # behind the row's four pages
    new[3] = -99
    _check_plan(cuda, lens, new, table, ring, torch.tensor([0, 12]), 16, 64)


def test_plan_bad_pages_get_no_slot(cuda):
    """A ring entry outside the pool is not turned into a slot."""
    lens, new = torch.zeros(2).int(), torch.tensor([16, 16]).int()
    table = torch.full((2, 1), -1, dtype=torch.int32)
    ring = torch.tensor([1, 77, 0], dtype=torch.int32)
    _lib.device_errors(cuda)
    p = paged_plan(lens.to(cuda), new.to(cuda), table.to(cuda), ring.to(cuda),
                   torch.tensor([0, 3], device=cuda), 16, 32)
    assert p.slots.tolist() == list(range(16, 32)) + [-1] * 16
    assert _lib.device_errors(cuda) == _lib.DEVERR_BAD_PAGE


# -------------------------------------------------------------------- input

def _pool(seed, pages, hk, page, d, e4m3, dev, order="phsd"):
    """(k_pages, v_pages, k_scale, v_scale); `order` is the memory order of the axes."""
    g = _gen(seed)
    x = torch.randn(2, pages, hk, page, d, generator=g)
    x = (x * 40).clamp(-448, 448).to(E4M3) if e4m3 else x.to(torch.bfloat16)
    x = x.view(torch.uint8) if e4m3 else x
    if order == "pshd":
        x = x.transpose(2, 3).contiguous().to(dev).transpose(2, 3)
    else:
        x = x.to(dev)
    x = x.view(E4M3) if e4m3 else x
    s = ((0.5 + torch.rand(2, hk, generator=g)) / 40).to(dev) if e4m3 else (None, None)
    return x[0], x[1], s[0], s[1]


def _bound(y, mag, roundings, e4m3, scale=1.0):
    """Half a step of the type around y, after an fp32 error of `roundings` half steps of
    mag; y and mag in the stored units (divided by scale)."""
    err = mag * roundings * U / scale
    y = y.abs() / scale + err
    return err + (torch.clamp(y * 2.0 ** -4, min=2.0 ** -10) if e4m3 else y * 2.0 ** -8)


# fp32 roundings on the way to an output of |a| + |b|: the sum of D squares (16 in a lane
# and 4 shuffles at most, or D / 32 and 5: under 24) halved by the root, rsqrt 2, eps and
# mean 2, two products 2; angle to 32 bits (2^-25 turns = 2 pi 2^-25 rad: under 7 half
# steps), sincospi 2, scaling 1, rotation 3, division by the scale 1: under 36 in all.
ROUNDINGS = 40


def _mrope_positions(g, axes, tokens):
    pos = torch.randint(0, 32768, (axes, tokens), generator=g)
    pos[:, ::5] = pos[:1, ::5]
    return pos


MROPE = [
    # hq, hk, d, rotary, sections, interleaved
    (32, 8, 128, 128, (24, 20, 20), True),
    (16, 8, 128, 128, (24, 20, 20), False),
    (16, 16, 80, 80, (20, 20), False),
    (4, 2, 16, 16, (2, 3, 3), True),
    (3, 1, 48, 32, (16,), False),
    (28, 4, 96, 64, (8, 0, 24), False),
    (2, 2, 256, 256, (44, 42, 42), True),
    (5, 5, 64, 0, (), False),
]


@pytest.mark.parametrize("shape", MROPE, ids=lambda s: f"{s[0]}x{s[1]}x{s[2]}r{s[3]}")
@pytest.mark.parametrize("tokens", [1, 3, 77, 1031])
@pytest.mark.parametrize("form", ["bf16", "e4m3", "plain"])
def test_input_matches_oracle(cuda, shape, tokens, form):
    hq, hk, d, rotary, sections, inter = shape
    g = _gen(tokens + d)
    dev = cuda
    norm = tokens != 3
    qkv = torch.randn(tokens, hq + 2 * hk, d, generator=g).to(torch.bfloat16).to(dev)
    q, k, v = qkv.split((hq, hk, hk), 1)
    before = qkv.clone()
    wdt = torch.float32 if hk % 2 else torch.bfloat16
    qw, kw = ((1 + 0.2 * torch.randn(2, d, generator=g)).to(wdt).to(dev) if norm
              else (None, None))
    half = rotary // 2
    inv = (1e6 ** (-torch.arange(half) / max(half, 1))).to(dev)
    pos = _mrope_positions(g, len(sections) or 1, tokens).to(dev)
    if tokens % 2:
        pos = pos.int()
    scaling = 1.25 if form == "plain" else 1.0
    page, e4m3 = 16, form == "e4m3"
    if form == "plain":
        if not rotary:
            pytest.skip("neither rotation nor cache")
        q2, k2 = qk_norm_mrope_kv(q, k, None, pos, inv, sections, interleaved=inter,
                                  scaling=scaling, q_weight=qw, k_weight=kw, q_eps=1e-5,
                                  k_eps=1e-3)
    else:
        pages = tokens // page + 4
        kp, vp, ks, vs = _pool(tokens, pages, hk, page, d, e4m3, dev,
                               "pshd" if tokens == 77 else "phsd")
        slots = torch.randperm(pages * page, generator=g)[:tokens].int()
        slots[1::7] = -1
        kp0, vp0 = kp.float().cpu(), vp.float().cpu()
        kwargs = dict(k_scale=ks, v_scale=vs)
        if rotary:
            q2, none = qk_norm_mrope_kv(q, k, v, pos, inv, sections, interleaved=inter,
                                        q_weight=qw, k_weight=kw, q_eps=1e-5, k_eps=1e-3,
                                        k_pages=kp, v_pages=vp, slots=slots.to(dev), **kwargs)
            assert none is None
        else:
            kw = None
            paged_kv_append(kp, vp, k, v, slots.to(dev), **kwargs)
    assert torch.equal(qkv, before)  # the inputs are left as they were
    args = (pos if rotary else None, inv, sections, inter, scaling)
    if rotary:
        y, mag = oracle.norm_mrope(q, qw, 1e-5, *args)
        assert bool(((q2.cpu().double() - y).abs() <= _bound(y, mag, ROUNDINGS, False)).all())
    y, mag = oracle.norm_mrope(k, kw, 1e-3, *args)
    if form == "plain":
        assert bool(((k2.cpu().double() - y).abs() <= _bound(y, mag, ROUNDINGS, False)).all())
        return
    for pages_now, pages_then, val, size, scale in (
            (kp, kp0, y, mag, ks), (vp, vp0, v.cpu().double(), v.cpu().double().abs(), vs)):
        now = pages_now.float().cpu().double()
        expect = pages_then.double().clone()
        bound = torch.zeros_like(expect)
        sc = scale.cpu().double()[:, None] if scale is not None else 1.0
        on = slots >= 0
        at, off = slots[on].long() // page, slots[on].long() % page
        stored = val[on] / sc
        expect[at, :, off] = stored.clamp(-448, 448) if e4m3 else stored
        bound[at, :, off] = _bound(val[on], size[on], ROUNDINGS, e4m3, sc)
        assert bool(((now - expect).abs() <= bound).all())


def test_input_in_place_and_expanded_positions(cuda):
    """q and k rotated over themselves, one position row shared by the three axes, equal
    the copies' results bit for bit."""
    g = _gen(3)
    q = torch.randn(50, 8, 128, generator=g).to(torch.bfloat16).to(cuda)
    k = torch.randn(50, 2, 128, generator=g).to(torch.bfloat16).to(cuda)
    pos = torch.randint(0, 9999, (1, 50), generator=g).to(cuda)
    inv = (1e6 ** (-torch.arange(64) / 64)).to(cuda)
    a = qk_norm_mrope_kv(q, k, None, pos.expand(3, 50), inv, (24, 20, 20), interleaved=True)
    b = qk_norm_mrope_kv(q, k, None, pos[0], inv, (64,))
    c = qk_norm_mrope_kv(q, k, None, pos.expand(3, 50), inv, (24, 20, 20), interleaved=True,
                         q_out=q, k_out=k)
    assert c[0] is q and c[1] is k
    for x, y, z in zip(a, b, c):
        assert torch.equal(x, y) and torch.equal(x, z)


def test_input_far_positions(cuda):
    """Positions up to 2^31: the angle keeps 64 bits' accuracy (2^-52 of itself, half a step
    each for the product here and in the oracle, and one for the constant)."""
    g = _gen(31)
    x = torch.randn(64, 4, 128, generator=g).to(torch.bfloat16).to(cuda)
    pos = torch.randint(1 << 30, (1 << 31) - 1, (2, 64), generator=g)
    inv = (1e4 ** (-torch.arange(64) / 64)).to(cuda)
    for p in (pos.to(cuda), pos.int().to(cuda)):
        got, _ = qk_norm_mrope_kv(x, x[:, :1], None, p, inv, (20, 44), q_weight=None)
        y, mag = oracle.norm_mrope(x, None, 0.0, pos, inv, (20, 44), False)
        bound = _bound(y, mag, ROUNDINGS, False) + mag * 2.0 ** 31 * 2.0 ** -51
        assert bool(((got.cpu().double() - y).abs() <= bound).all())


@pytest.mark.parametrize("tokens", [2367, 2368, 2369, 9000])
def test_input_every_token_once(cuda, tokens):
    """More and fewer tokens than resident warps, with one head and with many: every row is
    written, and only rows that a slot names."""
    for hk, d in ((1, 32), (9, 80)):
        k = torch.full((tokens, hk, d), 2.0, dtype=torch.bfloat16, device=cuda)
        pages = tokens // 16 + 2
        kp = torch.zeros(pages, hk, 16, d, dtype=torch.bfloat16, device=cuda)
        vp = torch.zeros_like(kp)
        slots = torch.arange(tokens, dtype=torch.int32, device=cuda) + 5
        paged_kv_append(kp, vp, k, -k, slots)
        flat = kp.transpose(1, 2).reshape(-1, hk, d)
        assert bool((flat[5:5 + tokens] == 2).all())
        assert bool((flat[:5] == 0).all()) and bool((flat[5 + tokens:] == 0).all())
        assert torch.equal(vp, -kp)


def test_input_special_values(cuda):
    """e4m3 saturates at 448 and keeps NaN; -1 and bad slots write nothing."""
    kp, vp, ks, vs = _pool(1, 3, 1, 16, 16, True, cuda)
    k0 = kp.float().clone()
    k = torch.zeros(6, 1, 16, dtype=torch.bfloat16, device=cuda)
    k[0, 0, :4] = torch.tensor([1e6, -1e6, float("inf"), float("nan")])
    k[2:] = 7.0
    slots = torch.tensor([5, 6, -1, 48, -2, 1 << 30], dtype=torch.int32, device=cuda)
    _lib.device_errors(cuda)
    paged_kv_append(kp, vp, k, k, slots, k_scale=ks, v_scale=vs)
    assert _lib.device_errors(cuda) == _lib.DEVERR_BAD_PAGE
    got = kp.float()
    row = got[0, 0, 5]
    assert row[:3].tolist() == [448.0, -448.0, 448.0] and bool(row[3].isnan())
    assert bool((row[4:] == 0).all()) and bool((got[0, 0, 6] == 0).all())
    got[0, 0, 5:7] = k0[0, 0, 5:7]
    assert torch.equal(got, k0)


# ---------------------------------------------------------------- attention

def _attend_case(seed, lens, hq, hk, d, page, e4m3, dev, order="phsd", spare=2, width=None):
    g = _gen(seed)
    lens = torch.tensor(lens, dtype=torch.int32)
    used = -(-lens // page)
    need = int(used.sum())
    kp, vp, ks, vs = _pool(seed, need + spare, hk, page, d, e4m3, dev, order)
    perm = torch.randperm(need + spare, generator=g)
    width = max(1, int(used.max())) if width is None else width
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(used.tolist()):
        table[r, :n] = perm[at:at + n]
        at += n
    q = (1.5 * torch.randn(len(lens), hq, d, generator=g)).to(torch.bfloat16).to(dev)
    return q, kp, vp, table, lens, d ** -0.5, ks, vs


def _check_attend(cuda, q, kp, vp, table, lens, scale, ks, vs, device="cpu", **kw):
    want, lse, spread, reach = oracle.paged_attention(q, kp, vp, table, lens, scale, ks, vs,
                                                      device)
    out, got_lse = paged_attention(q, kp, vp, table.to(cuda), lens.to(cuda), scale, k_scale=ks,
                                   v_scale=vs, return_lse=True, **kw)
    d, longest = q.shape[2], int(lens.max())
    # a score: D products summed in fp32 (truncating sums: a whole step each), scaled
    # (2 roundings) and taken to base 2; exp2 2 steps. A weight moves by that much, and the
    # sums of weights and of weighted values by a step per tile joined (len / 16, and under
    # 200 partial results). Weights are held to 2^-17 for bf16 pages and to 2^-11 (half a
    # step of fp16) for e4m3 ones.
    score = reach * (d + 6) * 2 * U
    sums = (longest / 16 + 200 + 16) * 2 * U
    held = 2.0 ** -11 if ks is not None else 2.0 ** -17
    rel = 2 * score + sums + held + 8 * U
    bound = spread * rel[..., None]
    bound = bound + (want.abs() + bound) * 2.0 ** -8
    off = (out.cpu().double() - want).abs()
    assert bool((off <= bound).all()), float((off - bound).max())
    there = torch.isfinite(lse)
    assert torch.equal(got_lse.cpu().isfinite(), there)
    off = (got_lse.cpu().double() - lse).abs()[there]
    assert bool((off <= (score + sums + 8 * U + lse.abs() * 4 * U)[there]).all())
    assert bool((out.cpu()[~there] == 0).all()) and bool((got_lse.cpu()[~there] < 0).all())
    return out, got_lse


HEADS = [(32, 8, 128), (16, 16, 80), (8, 1, 64), (28, 4, 96), (16, 1, 128), (6, 3, 256),
         (40, 1, 64), (17, 1, 256)]


@pytest.mark.parametrize("heads", HEADS, ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens,page", [
    ([1], 16), ([0, 15, 16, 17, 0, 33], 16), ([129, 1, 64, 63, 65], 64), ([700], 48),
    ([5, 0, 900, 31], 128)])
def test_attend_matches_oracle(cuda, heads, e4m3, lens, page):
    c = _attend_case(len(lens) + page, lens, *heads, page, e4m3, cuda,
                     "pshd" if page == 48 else "phsd")
    _check_attend(cuda, *c)


@pytest.mark.parametrize("batch,longest,e4m3", [(1, 5000, False), (3, 4097, True),
                                                (64, 300, False), (300, 40, True)])
def test_attend_long_and_many(cuda, batch, longest, e4m3):
    """Requests long enough to be split over every SM, and more requests than workers."""
    g = _gen(batch)
    lens = torch.randint(0, longest + 1, (batch,), generator=g).tolist()
    lens[batch // 2] = longest
    c = _attend_case(batch, lens, 8, 2, 128, 16, e4m3, cuda)
    _check_attend(cuda, *c)


@pytest.mark.parametrize("heads", HEADS[:7], ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens", [[0, 0, 0], [1, 0, 0], [40, 700, 0], [2000, 3, 1100]])
def test_attend_wide_table(cuda, heads, e4m3, lens):
    """A table whose rows could hold far more than the requests do."""
    c = _attend_case(7, lens, *heads, 64, e4m3, cuda, width=40000)
    _check_attend(cuda, *c)


@pytest.mark.parametrize("heads,e4m3,batch,longest", [
    ((32, 8, 128), False, 40, 4500), ((16, 8, 128), True, 300, 2000), ((16, 1, 64), False, 3, 900000),
    ((24, 3, 256), True, 5, 52000), ((16, 16, 80), False, 1, 90000)])
def test_attend_large(cuda, heads, e4m3, batch, longest):
    """Enough tiles that the warps claim their work; the same bits every time."""
    g = _gen(batch)
    lens = (torch.rand(batch, generator=g) * longest).long()
    lens[batch // 2], lens[-1] = longest, longest - 5
    lens[3::17] = 0
    c = _attend_case(batch, lens.tolist(), *heads, 64, e4m3, cuda)
    out, lse = _check_attend(cuda, *c, device=cuda)
    q, kp, vp, table, lens, scale, ks, vs = c
    for _ in range(3):
        again = paged_attention(q, kp, vp, table.to(cuda), lens.to(cuda), scale, k_scale=ks,
                                v_scale=vs, return_lse=True)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)


def test_attend_every_length_of_a_tile(cuda):
    c = _attend_case(9, list(range(0, 70)), 8, 4, 64, 32, False, cuda)
    _check_attend(cuda, *c)


@pytest.mark.parametrize("e4m3", [False, True])
def test_attend_ignores_what_lies_behind(cuda, e4m3):
    """NaN and infinity behind a request's length, on pages of nobody and in table entries
    behind its pages change nothing."""
    q, kp, vp, table, lens, scale, ks, vs = _attend_case(4, [37, 0, 1, 16], 8, 2, 128, 16, e4m3,
                                                         cuda, width=6)
    clean = paged_attention(q, kp, vp, table.to(cuda), lens.to(cuda), scale, k_scale=ks,
                            v_scale=vs)
    keep = torch.zeros(kp.shape[0], 16, dtype=torch.bool)
    for r, n in enumerate(lens.tolist()):
        for j in range(n):
            keep[table[r, j // 16], j % 16] = True
    gone = (~keep).to(cuda)[:, None, :, None].expand(kp.shape)
    if e4m3:
        kp.view(torch.uint8)[gone] = 0x7f
        vp.view(torch.uint8)[gone] = 0xff
    else:
        kp[gone] = float("nan")
        vp[gone] = float("inf")
    table[:, 3:] = torch.tensor([1 << 30, -5, 0])
    _lib.device_errors(cuda)
    again = paged_attention(q, kp, vp, table.to(cuda), lens.to(cuda), scale, k_scale=ks,
                            v_scale=vs)
    assert torch.equal(clean, again)
    assert _lib.device_errors(cuda) == 0


def test_attend_bad_pages_are_left_out(cuda):
    q, kp, vp, table, lens, scale, ks, vs = _attend_case(6, [100, 40, 16], 8, 2, 128, 16, False,
                                                         cuda)
    table[0, 2], table[0, 6], table[2, 0] = -1, 1 << 30, kp.shape[0]
    lens[1] = 4000  # past its row: cut there
    table[1, 3:] = table[1, 0]
    _lib.device_errors(cuda)
    out, lse = _check_attend(cuda, q, kp, vp, table, lens, scale, ks, vs)
    assert _lib.device_errors(cuda) == _lib.DEVERR_BAD_PAGE
    assert bool((out[2] == 0).all()) and bool((lse[2] == float("-inf")).all())


def test_attend_extreme_scores(cuda):
    """Scores of +-1000 leave one token with all the weight; a page shared by two requests
    serves both; NaN in a valid token reaches its own head only."""
    q, kp, vp, table, lens, scale, ks, vs = _attend_case(8, [50, 20], 4, 2, 64, 16, False, cuda)
    q[0] = 0
    q[0, :, 0] = 100.0
    kp[..., 0] = -80.0
    kp[table[0, 1], :, 3, 0] = 80.0
    table[1, :2] = table[0, :2]
    out, lse = _check_attend(cuda, q, kp, vp, table, lens, scale, ks, vs)
    for h in range(4):
        assert torch.equal(out[0, h], vp[table[0, 1], h // 2, 3])
    vp[table[0, 0], 1, 2, 5] = float("nan")
    out2 = paged_attention(q, kp, vp, table.to(cuda), lens.to(cuda), scale)
    assert torch.equal(out2[:, :2], out[:, :2])
    assert bool(out2[1, 2:, 5].isnan().all())
    assert bool(out2[1, 2:, :5].isfinite().all())


@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("code", [0x7f, 0xff])
def test_attend_e4m3_nan_and_largest(cuda, d, code):
    """NaN of either sign in a valid token: in V it makes its dim NaN for the heads of its
    KV head, in K their whole rows, whatever the sign of q; +-448 are values like others."""
    c = _attend_case(13, [50, 20, 700], 8, 2, d, 16, True, cuda)
    q, kp, vp, table, lens, scale, ks, vs = c
    kp.view(torch.uint8)[table[0, 0], :, 3, ::7] = 0x7e
    vp.view(torch.uint8)[table[0, 1], :, 2, ::5] = 0xfe
    _check_attend(cuda, *c)
    args = (table.to(cuda), lens.to(cuda), scale)
    clean = paged_attention(q, kp, vp, *args, k_scale=ks, v_scale=vs)
    vp.view(torch.uint8)[table[0, 2], 1, 1, 9] = code
    kp.view(torch.uint8)[table[2, 30], 0, 5, 11] = code
    out, lse = paged_attention(q, kp, vp, *args, k_scale=ks, v_scale=vs, return_lse=True)
    assert bool(out[0, 4:, 9].isnan().all()) and bool(out[2, :4].isnan().all())
    assert bool(lse[2, :4].isnan().all()) and bool(lse[0].isfinite().all())
    out[0, 4:, 9], out[2, :4] = clean[0, 4:, 9], clean[2, :4]
    assert torch.equal(out, clean)


def test_attend_strided_q_and_out(cuda):
    """q as a slice of a packed projection, out into a wider buffer left alone around it."""
    c = _attend_case(12, [33, 80], 8, 2, 128, 16, False, cuda)
    q, rest = c[0], c[1:]
    packed = torch.zeros(2, 12, 128, dtype=torch.bfloat16, device=cuda)
    packed[:, :8] = q
    wide = torch.full((2, 10, 128), 3.0, dtype=torch.bfloat16, device=cuda)
    a, _ = _check_attend(cuda, q, *rest)
    b, _ = _check_attend(cuda, packed[:, :8], *rest, out=wide[:, 1:9])
    assert torch.equal(a, b) and bool((wide[:, 0] == 3).all() and (wide[:, 9] == 3).all())


def test_attend_is_deterministic(cuda):
    c = _attend_case(21, [3000, 5, 800, 0, 77], 32, 8, 128, 16, False, cuda)
    q, kp, vp, table, lens, scale, _, _ = c
    runs = [paged_attention(q, kp, vp, table.to(cuda), lens.to(cuda), scale) for _ in range(5)]
    assert all(torch.equal(runs[0], r) for r in runs[1:])


def test_attend_offsets_past_32_bits(cuda):
    """A pool of more than 2^32 elements, its last pages in use."""
    hk, page, d = 8, 64, 128
    pages = (1 << 32) // (hk * page * d) + 8
    pool = torch.zeros(2, pages, hk, page, d, dtype=torch.bfloat16, device=cuda)
    g = _gen(2)
    small = torch.randn(2, 6, hk, page, d, generator=g).to(torch.bfloat16)
    at = torch.tensor([pages - 1, 0, pages - 3, 5, pages - 2, 1])
    pool[:, at.to(cuda)] = small.to(cuda)
    q = torch.randn(2, 16, d, generator=g).to(torch.bfloat16).to(cuda)
    lens = torch.tensor([190, 150], dtype=torch.int32)
    big = at.int().view(2, 3)
    tiny = torch.arange(6).int().view(2, 3)
    a = paged_attention(q, pool[0], pool[1], big.to(cuda), lens.to(cuda), 0.1)
    b = paged_attention(q, *small.to(cuda), tiny.to(cuda), lens.to(cuda), 0.1)
    assert torch.equal(a, b)
    k = torch.randn(5, hk, d, generator=g).to(torch.bfloat16).to(cuda)
    slots = (pages - 2) * page + torch.arange(5)
    paged_kv_append(pool[0], pool[1], k, -k, slots.int().to(cuda))
    assert torch.equal(pool[0, pages - 2, :, :5].transpose(0, 1), k)
    assert torch.equal(pool[1, pages - 2, :, :5].transpose(0, 1), -k)


def test_calls_are_counted_natively(cuda):
    before = stats["umic_paged_attention"]
    c = _attend_case(1, [3], 8, 2, 64, 16, False, cuda)
    paged_attention(*c[:3], c[3].to(cuda), c[4].to(cuda), c[5])
    assert stats["umic_paged_attention"] == before + 1


# ----------------------------------------------------------------- refusals

def _z(dev, *shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype, device=dev)


def test_plan_wrapper_refusals(cuda):
    i = lambda *s, dtype=torch.int32: _z(cuda, *s, dtype=dtype)  # noqa: E731
    good = dict(kv_lens=i(2), new_tokens=i(2), block_table=i(2, 3), free_ring=i(9),
                free_span=i(2, dtype=torch.int64), page_size=16, capacity=4)
    paged_plan(**good)
    for error, change in [
            (TypeError, dict(kv_lens=i(2, dtype=torch.int64))),
            (TypeError, dict(free_span=i(2))), (ValueError, dict(new_tokens=i(3))),
            (ValueError, dict(block_table=i(3, 3))), (ValueError, dict(kv_lens=i(2, 1))),
            (ValueError, dict(block_table=i(3, 2).t())), (ValueError, dict(capacity=-1)),
            (ValueError, dict(new_tokens=i(4)[::2])), (ValueError, dict(out_lens=i(3))),
            (TypeError, dict(out_span=i(2))), (RuntimeError, dict(page_size=0)),
            (RuntimeError, dict(free_ring=torch.zeros(9, dtype=torch.int32)))]:
        with pytest.raises(error):
            paged_plan(**{**good, **change})


def test_input_wrapper_refusals(cuda):
    z = lambda *s, dtype=torch.bfloat16: _z(cuda, *s, dtype=dtype)  # noqa: E731
    i32 = torch.int32
    good = dict(q=z(3, 4, 64), k=z(3, 2, 64), v=z(3, 2, 64), positions=z(3, 3, dtype=i32),
                inv_freq=z(32, dtype=torch.float32), sections=(12, 10, 10),
                k_pages=z(4, 2, 16, 64), v_pages=z(4, 2, 16, 64), slots=z(3, dtype=i32) - 1)
    qk_norm_mrope_kv(**good)
    e = z(4, 2, 16, 64, dtype=torch.uint8).view(E4M3)
    for error, change in [
            (TypeError, dict(q=z(3, 4, 64).half())), (ValueError, dict(q=z(4, 4, 64))),
            (ValueError, dict(k=z(3, 2, 128)[..., ::2])), (ValueError, dict(v=z(3, 1, 64))),
            (ValueError, dict(v=None)), (ValueError, dict(slots=None)),
            (TypeError, dict(slots=z(3, dtype=torch.int64))),
            (ValueError, dict(sections=(16, 16))), (RuntimeError, dict(sections=(16, 16, 1))),
            (ValueError, dict(positions=z(3, 4, dtype=i32))),
            (ValueError, dict(positions=z(3, 3, dtype=torch.float32))),
            (ValueError, dict(positions=None)), (TypeError, dict(inv_freq=z(32))),
            (ValueError, dict(k_pages=None)), (ValueError, dict(v_pages=z(5, 2, 16, 64))),
            (ValueError, dict(k_pages=z(4, 3, 16, 64), v_pages=z(4, 3, 16, 64))),
            (ValueError, dict(k_scale=z(2, dtype=torch.float32))),
            (ValueError, dict(k_pages=e, v_pages=e, k_scale=z(3, dtype=torch.float32))),
            (TypeError, dict(k_pages=e, v_pages=e, k_scale=z(2))),
            (TypeError, dict(k_pages=e.view(torch.float8_e5m2), v_pages=e.view(torch.float8_e5m2))),
            (ValueError, dict(q_weight=z(65))), (ValueError, dict(q_out=z(3, 5, 64))),
            (RuntimeError, dict(q_out=z(3, 1, 64).expand(3, 4, 64))),
            (ValueError, dict(sections=(1 << 40, 10, 10))), (ValueError, dict(k_out=z(3, 2, 64))),
            (TypeError, dict(q_weight=z(64), k_weight=z(64, dtype=torch.float32)))]:
        with pytest.raises(error):
            qk_norm_mrope_kv(**{**good, **change})


def test_attend_wrapper_refusals(cuda):
    z = lambda *s, dtype=torch.bfloat16: _z(cuda, *s, dtype=dtype)  # noqa: E731
    i32 = torch.int32
    good = dict(q=z(2, 4, 64), k_pages=z(4, 2, 16, 64), v_pages=z(4, 2, 16, 64),
                block_table=z(2, 2, dtype=i32), kv_lens=z(2, dtype=i32), scale=0.1)
    paged_attention(**good)
    pages = z(4, 2, 24, 64)
    for error, change in [
            (TypeError, dict(q=z(2, 4, 64).half())), (ValueError, dict(q=z(2, 4, 128))),
            (ValueError, dict(q=z(2, 64))), (RuntimeError, dict(q=z(2, 5, 64))),
            (ValueError, dict(block_table=z(3, 2, dtype=i32))),
            (ValueError, dict(block_table=z(2, 2, dtype=torch.int64))),
            (TypeError, dict(kv_lens=z(2, dtype=torch.int64))),
            (ValueError, dict(kv_lens=z(3, dtype=i32))), (ValueError, dict(out=z(2, 5, 64))),
            (RuntimeError, dict(out=z(2, 1, 64).expand(2, 4, 64))),
            (ValueError, dict(scale="0.1")),
            (RuntimeError, dict(k_pages=pages, v_pages=pages)),
            (ValueError, dict(v_pages=z(4, 2, 16, 64).transpose(1, 2)))]:
        with pytest.raises(error):
            paged_attention(**{**good, **change})


def test_attend_many_requests(cuda):
    """More requests than threads of a CTA: each equals the same request in a small batch."""
    g = _gen(77)
    lens = torch.randint(0, 17, (20000,), generator=g)
    kp, vp, _, _ = _pool(3, 300, 2, 16, 64, False, cuda)
    table = torch.randint(0, 300, (20000, 1), generator=g).int().to(cuda)
    q = torch.randn(20000, 4, 64, generator=g).to(torch.bfloat16).to(cuda)
    lens = lens.int().to(cuda)
    out = paged_attention(q, kp, vp, table, lens, 0.125)
    for a in range(0, 20000, 4000):
        s = slice(a, a + 100)
        assert torch.equal(out[s], paged_attention(q[s], kp, vp, table[s], lens[s], 0.125))
    assert bool((out[lens == 0] == 0).all())
