"""CPU check of interleaved sections that reach past the frequencies: which axis turns what,
in the oracle that the kernels are held to, is what transformers' rotary module does."""

import pytest
import torch

from oracle import paged as oracle


@pytest.mark.parametrize("sections,turned", [
    ((24, 20, 20), (24, 20, 20)), ((10, 27, 27), (22, 21, 21)), ((0, 32, 32), (22, 21, 21)),
    ((64, 0, 0), (64, 0, 0)), ((44, 0, 20), (44, 0, 20))])
def test_interleaved_sections_are_transformers(sections, turned):
    import transformers.models.qwen3_vl.modeling_qwen3_vl as hf

    from umic_b200.workloads import text_config

    axes = oracle.mrope_axes(sections, True)
    assert tuple(axes.count(a) for a in range(3)) == turned
    rot = hf.Qwen3VLTextRotaryEmbedding(text_config())
    rot.mrope_section = list(sections)
    g = torch.Generator().manual_seed(0)
    pos = torch.randint(0, 500, (3, 1, 40), generator=g)
    x = torch.randn(40, 2, 128, generator=g)
    cos, sin = (t[0, :, None] for t in rot(x, pos))
    want = x * cos + torch.cat((-x[..., 64:], x[..., :64]), -1) * sin
    got, _ = oracle.norm_mrope(x, None, 0.0, pos[:, 0], rot.inv_freq, sections, True)
    # fp32 angles up to 500 rad: 2^-24 of them, times |a| + |b| < 10
    assert float((got - want.double()).abs().max()) < 500 * 2.0 ** -23 * 10
