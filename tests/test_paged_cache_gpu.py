"""PagedKVCache on the GPU: the operators run together over serving steps, eager, captured
and on other streams, against a dense cache kept on the side in 64 bits."""

import pytest
import torch

from oracle import paged as oracle
from umic_b200 import _lib
from umic_b200.paged import PagedKVCache

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
HQ, HK, D, LAYERS, PAGE, R, WIDTH = 8, 2, 64, 2, 16, 6, 5
SECTIONS = (12, 10, 10)


def _inv(dev):
    return (1e6 ** (-torch.arange(32) / 32)).to(dev)


def _cache(dev, dtype=torch.bfloat16, pages=20):
    c = PagedKVCache.allocate(LAYERS, pages, HK, D, PAGE, R, WIDTH, dev, dtype)
    c.slab.view(torch.uint8).fill_(0x7f)  # NaN wherever nothing was written
    if c.k_scale is not None:
        c.k_scale.uniform_(0.01, 0.03)
        c.v_scale.uniform_(0.01, 0.03)
    return c


def _inputs(g, tokens, dev):
    return [torch.randn(tokens, h, D, generator=g).to(torch.bfloat16).to(dev)
            for h in (HQ, HK, HK)]


class Dense:
    """Each request's rotated keys and its values, per layer, as the pages hold them."""

    def __init__(self, cache):
        self.c = cache
        self.k = [[torch.zeros(0, HK, D).double() for _ in range(R)] for _ in range(LAYERS)]
        self.v = [[torch.zeros(0, HK, D).double() for _ in range(R)] for _ in range(LAYERS)]

    def held(self, x, layer, scale):
        """bf16 or e4m3 rounding of 64-bit values."""
        if scale is None:
            return x.to(torch.bfloat16).double()
        s = scale[layer].cpu().double()[:, None]
        return (x / s).float().clamp(-448, 448).to(E4M3).float().double() * s

    def crop(self, r, n):
        for layer in range(LAYERS):
            self.k[layer][r], self.v[layer][r] = self.k[layer][r][:n], self.v[layer][r][:n]

    def add(self, layer, r, k, v):
        self.k[layer][r] = torch.cat((self.k[layer][r], self.held(k, layer, self.c.k_scale)))
        self.v[layer][r] = torch.cat((self.v[layer][r], self.held(v, layer, self.c.v_scale)))

    def attend(self, layer, q, scale):
        out = torch.zeros(R, HQ, D).double()
        for r in range(R):
            k = self.k[layer][r].repeat_interleave(HQ // HK, 1)
            v = self.v[layer][r].repeat_interleave(HQ // HK, 1)
            if len(k):
                w = torch.softmax(torch.einsum("hd,thd->ht", q[r], k) * scale, -1)
                out[r] = torch.einsum("ht,thd->hd", w, v)
        return out


def _run_step(cache, dense, g, asks, capacity, dev, scale=0.125):
    """One step of every layer; returns the worst error of the attention rows."""
    old = cache.kv_lens.tolist()
    want = oracle.paged_plan(old, asks, cache.block_table.cpu(), cache.free_ring.cpu(),
                             cache.free_span.cpu(), PAGE, capacity)
    plan = cache.step(torch.tensor(asks, dtype=torch.int32, device=dev), capacity)
    assert torch.equal(plan.slots.cpu(), want["slots"])
    new = cache.kv_lens.tolist()
    assert new == want["kv_lens"].tolist()
    for r in range(R):
        if new[r] < old[r]:
            dense.crop(r, new[r])
    inv = _inv(dev)
    pos = plan.positions.expand(3, -1)
    cu, slots = plan.cu_tokens.tolist(), plan.slots.tolist()
    worst = 0.0
    for layer in range(LAYERS):
        q, k, v = _inputs(g, capacity, dev)
        w = (1 + 0.1 * torch.randn(2, D, generator=g)).to(torch.bfloat16).to(dev)
        rotated = cache.write(layer, q, k, v, plan, pos, inv, SECTIONS, interleaved=True,
                              q_weight=w[0], k_weight=w[1])
        kr, _ = oracle.norm_mrope(k, w[1], 1e-6, pos, inv, SECTIONS, True)
        for r in range(R):
            on = [t for t in range(cu[r], min(cu[r + 1], capacity)) if slots[t] >= 0]
            if on:
                dense.add(layer, r, kr[on], v.cpu().double()[on])
        last = torch.tensor([max(min(cu[r + 1], capacity) - 1, 0) for r in range(R)])
        qs = rotated[last.to(dev)]
        out = cache.attend(layer, qs, scale)
        ref = dense.attend(layer, qs.cpu().double(), scale)
        worst = max(worst, float((out.cpu().double() - ref).abs().max()))
        empty = torch.tensor([n == 0 for n in new])
        assert bool((out.cpu()[empty] == 0).all())
    return worst


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_serving_steps(cuda, dtype):
    """Prompts, single tokens, crops, ends, new requests, an exhausted pool."""
    cache = _cache(cuda, dtype)
    dense = Dense(cache)
    g = torch.Generator().manual_seed(5)
    _lib.device_errors(cuda)
    steps = [([40, 0, 17, 1, 0, 0], 64), ([1, 1, 1, 1, 0, 0], 6), ([-9, 30, 1, -2, 16, 0], 50),
             ([1] * 6, 6), ([-32, -1, 1, 1, 1, 1], 6), ([70, 1, 1, 0, 1, 1], 80),
             ([0, 60, 60, 60, 60, 60], 300), ([1, 1, 1, 1, 1, 1], 6)]
    # Values of at most about 4, weights summing to 1: half a step of bf16 at 4 is 2^-7 for
    # the output; the pages hold the rounded keys and values that the dense side holds, up
    # to a rounding border (a whole step of one key element, bf16 2^-7 or e4m3 2^-3 of it,
    # moves a score by at most 2^-3 * 4 * 4 / 8 and one weight by that much).
    bound = 2.0 ** -6 if dtype == torch.bfloat16 else 2.0 ** -5
    for asks, capacity in steps:
        assert _run_step(cache, dense, g, asks, capacity, cuda) <= bound
    assert _lib.device_errors(cuda) == _lib.DEVERR_PAGES  # the step of 60s did not all fit
    ends = [-n for n in cache.kv_lens.tolist()]
    cache.step(torch.tensor(ends, dtype=torch.int32, device=cuda), 1)
    assert cache.free_pages() == 20 and cache.kv_lens.tolist() == [0] * R
    at, end = cache.free_span.tolist()
    assert sorted(cache.free_ring[i % 20].item() for i in range(at, end)) == list(range(20))


def _decode(cache, one, q, k, v, scale=0.125):
    """A decode step as it is captured: every length is read on the device."""
    plan = cache.step(one, R)
    pos = plan.positions.expand(3, -1)
    outs = []
    for layer in range(LAYERS):
        rq = cache.write(layer, q, k, v, plan, pos, _decode.inv, SECTIONS, interleaved=True)
        outs.append(cache.attend(layer, rq, scale))
    return outs


def _clone(cache, dev):
    other = _cache(dev, cache.slab.dtype, cache.slab.shape[2])
    for name in ("slab", "block_table", "kv_lens", "free_ring", "free_span"):
        a, b = getattr(other, name), getattr(cache, name)
        a.view(torch.uint8).copy_(b.view(torch.uint8))
    if cache.k_scale is not None:
        other.k_scale.copy_(cache.k_scale)
        other.v_scale.copy_(cache.v_scale)
    return other


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_one_graph_serves_every_step(cuda, dtype):
    """A captured step, replayed while lengths grow over page borders, equals eager steps
    bit for bit; two graphs of two caches replay on two streams at once."""
    _decode.inv = _inv(cuda)
    g = torch.Generator().manual_seed(6)
    start = _cache(cuda, dtype)
    asks = torch.tensor([15, 0, 31, 1, 40, 7], dtype=torch.int32, device=cuda)
    plan = start.step(asks, 96)
    q, k, v = _inputs(g, 96, cuda)
    for layer in range(LAYERS):
        start.write(layer, q, k, v, plan, plan.positions.expand(3, -1), _decode.inv, SECTIONS)
    one = torch.tensor([1, 0, 1, 1, 1, 1], dtype=torch.int32, device=cuda)
    static = _inputs(g, R, cuda)
    data = [_inputs(g, R, cuda) for _ in range(20)]

    eager = _clone(start, cuda)
    want = []
    for x in data:
        want.append([o.clone() for o in _decode(eager, one, *x)])

    caches = [_clone(start, cuda) for _ in range(2)]
    ins = [[t.clone() for t in static] for _ in range(2)]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _decode(_clone(start, cuda), one, *static)  # warm-up
    torch.cuda.current_stream().wait_stream(side)
    for c, x in zip(caches, ins):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_decode(c, one, *x))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i, x in enumerate(data):
        for graph, dst, s in zip(graphs, ins, streams):
            with torch.cuda.stream(s):
                for a, b in zip(dst, x):
                    a.copy_(b)
                graph.replay()
        torch.cuda.synchronize()
        for got in outs:
            assert all(torch.equal(a, b) for a, b in zip(got, want[i])), i
    for c in caches:
        assert torch.equal(c.kv_lens, eager.kv_lens)
        assert torch.equal(c.block_table, eager.block_table)
        assert torch.equal(c.slab.view(torch.uint8), eager.slab.view(torch.uint8))


def test_calls_on_several_streams_at_once(cuda):
    """Attention of two requests sets on two streams, interleaved, each with its own
    workspace."""
    _decode.inv = _inv(cuda)
    g = torch.Generator().manual_seed(8)
    c = _cache(cuda)
    plan = c.step(torch.tensor([60, 33, 2, 47, 0, 64], dtype=torch.int32, device=cuda), 206)
    q, k, v = _inputs(g, 206, cuda)
    c.append(0, k, v, plan)
    qs = [torch.randn(R, HQ, D, generator=g).to(torch.bfloat16).to(cuda) for _ in range(8)]
    want = [c.attend(0, x, 0.2) for x in qs]
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for i, x in enumerate(qs):
            with torch.cuda.stream(streams[i % 4]):
                got.append((i, c.attend(0, x, 0.2)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i, o in got)


def test_dense_prefix_moves_into_pages(cuda):
    """An InplaceKVCache prefix appended to pages is attended like the dense one."""
    from umic_b200.cache import InplaceKVCache

    g = torch.Generator().manual_seed(9)
    dense = InplaceKVCache.allocate(1, 2, HK, D, 64, cuda)
    kd, vd = (torch.randn(2, HK, 50, D, generator=g).to(torch.bfloat16).to(cuda)
              for _ in range(2))
    dense.layers[0].update(kd, vd)
    c = _cache(cuda)
    plan = c.step(torch.tensor([50, 50, 0, 0, 0, 0], dtype=torch.int32, device=cuda), 100)
    keys, values = dense.layers[0].keys, dense.layers[0].values
    c.append(0, keys.transpose(1, 2).reshape(100, HK, D), values.transpose(1, 2).reshape(
        100, HK, D), plan)
    q = torch.randn(R, HQ, D, generator=g).to(torch.bfloat16).to(cuda)
    out = c.attend(0, q, 0.125)
    ref = torch.nn.functional.scaled_dot_product_attention(
        q[:2, :, None].double(), keys.double().repeat_interleave(4, 1),
        values.double().repeat_interleave(4, 1), scale=0.125)[:, :, 0]
    # outputs of at most about 2: half a step of bf16 there, and as much again for the
    # weights' and sums' fp32 (2^-17 of the values)
    assert float((out[:2].double() - ref).abs().max()) < 2.0 ** -7
    assert bool((out[2:] == 0).all())
