"""CPU checks of the paged-cache serving operators: the oracle against independent forms
(transformers' three-axis rotary module, a dense softmax, a pool that is walked step by
step) and every refusal that the host decides before a launch."""

import ctypes

import pytest
import torch

from oracle import paged as oracle
from umic_b200 import _lib
from umic_b200.kernels import (paged_attention, paged_kv_append, paged_plan, qk_norm_mrope_kv)

F = ctypes.c_void_p(4096)  # never dereferenced: the check under test fails first


# ------------------------------------------------------------------- oracle

def test_rotary_oracle_is_transformers_three_axis_rotary():
    import transformers.models.qwen3_vl.modeling_qwen3_vl as hf

    from umic_b200.workloads import text_config

    rot = hf.Qwen3VLTextRotaryEmbedding(text_config())
    g = torch.Generator().manual_seed(0)
    pos = torch.randint(0, 500, (3, 1, 40), generator=g)
    x = torch.randn(1, 5, 40, 128, generator=g)
    cos, sin = rot(x, pos)
    want = (x * cos[:, None]
            + torch.cat((-x[..., 64:], x[..., :64]), -1) * sin[:, None])[0].transpose(0, 1)
    got, _ = oracle.norm_mrope(x[0].transpose(0, 1), None, 0.0, pos[:, 0], rot.inv_freq,
                               (24, 20, 20), True)
    # fp32 angles up to 500 rad: 2^-24 of them, times |a| + |b| < 10
    assert float((got - want.double()).abs().max()) < 500 * 2.0 ** -23 * 10


def test_rotary_oracle_is_transformers_vision_rotary():
    import transformers.models.qwen3_vl.modeling_qwen3_vl as hf

    dim = 40
    freqs = hf.Qwen3VLVisionRotaryEmbedding(dim)
    hw = torch.stack((torch.arange(30) // 6, torch.arange(30) % 6))
    table = freqs(32)
    emb = torch.cat((table[hw[0]], table[hw[1]]), -1)
    emb = torch.cat((emb, emb), -1)
    x = torch.randn(30, 2, 80, generator=torch.Generator().manual_seed(1))
    want = hf.apply_rotary_pos_emb_vision(x, x, emb.cos(), emb.sin())[0]
    inv = torch.cat((freqs.inv_freq, freqs.inv_freq))
    got, _ = oracle.norm_mrope(x, None, 0.0, hw, inv, (20, 20), False)
    assert float((got - want.double()).abs().max()) < 1e-4


def test_attention_oracle_is_a_dense_softmax():
    g = torch.Generator().manual_seed(2)
    kp, vp = torch.randn(2, 4, 2, 16, 8, generator=g).double()
    q = torch.randn(1, 4, 8, generator=g).double()
    table = torch.tensor([[2, 0, 3]])
    out, lse, _, _ = oracle.paged_attention(q, kp, vp, table, torch.tensor([37]), 0.3)
    k = torch.cat([kp[i] for i in (2, 0, 3)], 1)[:, :37].repeat_interleave(2, 0)
    v = torch.cat([vp[i] for i in (2, 0, 3)], 1)[:, :37].repeat_interleave(2, 0)
    s = (q[0][:, None] * k).sum(-1) * 0.3
    assert torch.allclose(out[0], torch.softmax(s, -1)[:, None].matmul(v)[:, 0])
    assert torch.allclose(lse[0], torch.logsumexp(s, -1))


def test_plan_oracle_keeps_every_page_in_one_place():
    """Random steps of appends, crops and ends: each page of the pool stays in exactly one
    row or in the ring, and a token's slot never changes while it is cached."""
    g = torch.Generator().manual_seed(3)
    r, width, page, pages = 5, 4, 3, 11
    lens = torch.zeros(r, dtype=torch.int32)
    table = torch.full((r, width), -1, dtype=torch.int32)
    ring, span = torch.arange(pages).int(), torch.tensor([0, pages])
    held = [[] for _ in range(r)]
    for _ in range(200):
        d = torch.randint(-6, 6, (r,), generator=g)
        got = oracle.paged_plan(lens, d, table, ring, span, page, 14)
        lens, table, ring, span = (got[k] for k in ("kv_lens", "table", "ring", "free_span"))
        cu = got["cu_tokens"].tolist()
        for i in range(r):
            n = int(lens[i])
            held[i] = held[i][:n]
            held[i] += [s for s in got["slots"][cu[i]:cu[i + 1]].tolist() if s >= 0]
            assert len(held[i]) == n
            assert held[i] == [int(table[i, j // page]) * page + j % page for j in range(n)]
        rows = [int(table[i, j]) for i in range(r) for j in range(-(-int(lens[i]) // page))]
        free = [int(ring[i % pages]) for i in range(int(span[0]), int(span[1]))]
        assert sorted(rows + free) == list(range(pages))


# -------------------------------------------------------------- C refusals

def _plan(requests=2, stride=4, max_pages=4, num_pages=8, page=16, cap=8, lens=F, span=F,
          slots=F):
    return _lib.lib().umic_paged_plan(lens, F, requests, F, stride, max_pages, F, num_pages,
                                      span, page, F, F, F, slots, F, cap, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(requests=0), 1, "requests=0"), (dict(page=0), 1, "page_size=0"),
    (dict(max_pages=0), 1, "max_pages=0"), (dict(num_pages=-1), 1, "num_pages=-1"),
    (dict(cap=-1), 1, "capacity=-1"), (dict(lens=None), 1, "null"), (dict(slots=None), 1, "null"),
    (dict(stride=3), 1, "overlap"), (dict(requests=8193), 2, "8192"),
    (dict(num_pages=1 << 27), 2, "2^31"), (dict(max_pages=1 << 28, stride=1 << 28), 2, "2^31"),
    (dict(cap=1 << 31), 2, "2^31"), (dict(span=ctypes.c_void_p(4100)), 3, "8-byte")])
def test_plan_refusals(kw, code, text):
    assert _plan(**kw) == code
    assert text in _lib.last_message()


def _at(p):
    return 0 if p is None else p.value


def _mrope(q=F, q_st=512, hq=4, k=F, k_st=256, v=F, hk=2, k_out=None, w=0, positions=F, pos=8,
           rot=128, axes=3, sec=(24, 20, 20), kp=F, pg=(8192, 2048, 128), num=8, page=16, dt=0,
           slots=F, tokens=4, d=128):
    args = _lib.pack_mrope_args(
        _at(q), _at(k), _at(v), _at(F), _at(k_out), 0, 0, _at(positions), _at(F), _at(kp),
        _at(kp), 0, 0, _at(slots), q_st, d, k_st, d, k_st, d, 512, d, 256, d, 4, 1, *pg, num,
        page, tokens, hq, hk, d, w, pos, rot, axes, *sec, 1, dt, 1e-6, 1e-6, 1.0)
    return _lib.lib().umic_qk_norm_mrope_kv(args, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(hk=0), 1, "hk=0"), (dict(hq=-1), 1, "hq=-1"), (dict(tokens=-1), 1, "tokens=-1"),
    (dict(d=120), 2, "head_dim 120"), (dict(d=272), 2, "head_dim 272"),
    (dict(rot=136), 2, "rotary_dim 136"), (dict(rot=24), 2, "rotary_dim 24"),
    (dict(rot=-16), 2, "rotary_dim -16"), (dict(axes=4), 2, "4 position axes"),
    (dict(axes=0), 2, "0 position axes"), (dict(sec=(24, 20, 19)), 1, "sum to 64"),
    (dict(axes=2), 1, "sections"), (dict(sec=(-1, 45, 20)), 1, "sections"),
    (dict(pos=2), 1, "2 bytes"), (dict(w=2), 1, "w_dtype"), (dict(dt=1), 1, "cache_dtype"),
    (dict(num=0), 2, "num_pages 0"), (dict(num=1 << 28), 2, "2^31"),
    (dict(tokens=1 << 31), 2, "too many"), (dict(q=None), 1, "null"), (dict(k=None), 1, "null"),
    (dict(positions=None), 1, "null"), (dict(v=None), 1, "null"), (dict(slots=None), 1, "null"),
    (dict(kp=None), 1, "null"), (dict(q_st=516), 3, "alignment"),
    (dict(pg=(8192, 64, 128)), 1, "overlap"),
    (dict(pg=(8192, 2048, 0)), 1, "overlap"), (dict(pg=(0, 2048, 128)), 1, "overlap"),
    (dict(k=ctypes.c_void_p(4104)), 3, "alignment"), (dict(pg=(8192, 2048, 132)), 3, "alignment"),
    (dict(dt=2, pg=(8192, 2048, 136)), 3, "alignment")])
def test_input_refusals(kw, code, text):
    assert _mrope(**kw) == code
    assert text in _lib.last_message()


def test_input_of_no_tokens_is_a_noop():
    assert _mrope(tokens=0, q=None, k=None) == 0
    assert _lib.lib().umic_qk_norm_mrope_kv(None, None) == 1


def _attend(q=F, q_sb=512, kp=F, pg=(8192, 2048, 128), num=8, page=16, dt=0, table=F, width=4,
            lens=F, out=F, batch=2, hq=4, hk=2, d=128, ws=F, ws_bytes=1 << 30):
    args = _lib.pack_paged_attention_args(
        _at(q), _at(kp), _at(kp), 0, 0, _at(table), _at(lens), _at(out), 0, _at(ws), q_sb, 128,
        *pg, num, page, width, width, 512, 128, batch, ws_bytes, hq, hk, d, dt, 0.1)
    return _lib.lib().umic_paged_attention(args, None)


def test_structs_match_the_header():
    """The packed formats against the header's fields, in order and by type."""
    import re
    from pathlib import Path

    header = (Path(__file__).resolve().parent.parent / "include" / "umic_b200.h").read_text()
    for name, fmt in (("umic_mrope_args", "14Q18q12i3f"), ("umic_paged_attention_args",
                                                          "10Q13q4if")):
        body = re.search(r"typedef struct " + name + r" \{(.*?)\} " + name + ";", header,
                         re.S).group(1)
        kinds = ""
        for line in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
            n = len(line.split(",")) if line.strip() else 0
            kind = "Q" if "*" in line else "q" if "int64_t" in line else \
                "i" if "int32_t" in line else "f"
            kinds += kind * n
        assert kinds == "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([Qqif])", fmt))


@pytest.mark.parametrize("kw,code,text", [
    (dict(batch=-1), 1, "batch=-1"), (dict(hk=0), 1, "hkv=0"), (dict(num=0), 1, "num_pages=0"),
    (dict(width=-1), 1, "max_pages=-1"), (dict(dt=1), 1, "cache_dtype"),
    (dict(hq=5), 2, "5 query heads"), (dict(d=112), 2, "head_dim 112"),
    (dict(page=24), 2, "page_size 24"), (dict(num=1 << 27), 2, "2^31"),
    (dict(width=1 << 27), 2, "2^31"), (dict(batch=1 << 30), 2, "2^31"), (dict(q=None), 1, "null"),
    (dict(lens=None), 1, "null"), (dict(table=None), 1, "null"), (dict(out=None), 1, "null"),
    (dict(q_sb=516), 3, "alignment"), (dict(d=256), 1, "overlap"),
    (dict(batch=1 << 14, num=1 << 20, width=1 << 16), 2, "2^30"), (dict(pg=(8192, 2052, 128)), 3, "alignment"),
    (dict(dt=2, pg=(8192, 2056, 128)), 3, "alignment"),
    (dict(out=ctypes.c_void_p(4098)), 3, "alignment"), (dict(ws=None), 1, "workspace"),
    (dict(ws_bytes=4), 1, "workspace"), (dict(ws=ctypes.c_void_p(4100)), 1, "workspace")])
def test_attend_refusals(kw, code, text):
    assert _attend(**kw) == code
    assert text in _lib.last_message()


def test_attend_of_no_requests_is_a_noop():
    assert _attend(batch=0, q=None) == 0
    assert _lib.lib().umic_paged_attention(None, None) == 1


# -------------------------------------------------------- wrapper refusals

def _z(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def test_wrappers_refuse_cpu_tensors():
    i = _z(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        paged_plan(i, i, _z(2, 3, dtype=torch.int32), i, _z(2, dtype=torch.int64), 16, 4)
    x, pages = _z(3, 2, 64), _z(4, 2, 16, 64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        qk_norm_mrope_kv(x, x, None, _z(3, dtype=torch.int64), torch.ones(32), (32,))
    with pytest.raises(RuntimeError, match="no CPU path"):
        paged_kv_append(pages, pages, x, x, _z(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        paged_attention(x, pages, pages, _z(3, 2, dtype=torch.int32), _z(3, dtype=torch.int32),
                        0.1)


def test_paged_cache_refuses_other_slabs():
    from umic_b200.paged import PagedKVCache

    with pytest.raises(ValueError, match="slab"):
        PagedKVCache(_z(2, 3, 4, 2, 16, 64), 2, 3)
    with pytest.raises(ValueError, match="slab"):
        PagedKVCache(_z(2, 4, 2, 16, 64), 2, 3)
