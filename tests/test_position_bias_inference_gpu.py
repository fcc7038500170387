"""``maisi.spatial_attention`` with a learned position bias: the block that inference runs, against the one that learned it."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grid", [(8, 8, 4), (3, 7, 5)], ids=str)
def test_the_learned_bias_is_applied(ctmr, dev, grid):
    c, heads, m, f = 64, 2, ctmr.maisi, ctmr.differentiable
    g = torch.Generator(device=dev).manual_seed(1)
    r = lambda *s: torch.randn(*s, device=dev, generator=g)
    w = {"norm.weight": 1 + 0.1 * r(c), "norm.bias": 0.1 * r(c), "attn.position_bias": r(3, 8, heads).requires_grad_()}
    for n in ("to_q", "to_k", "to_v", "out_proj"):
        w[f"attn.{n}.weight"], w[f"attn.{n}.bias"] = r(c, c) / math.sqrt(c), 0.1 * r(c)
    x = r(2, *grid, c)
    args = dict(num_groups=16, eps=1e-6, num_head_channels=c // heads, include_fc=True)
    buckets = f.PackedVolumes([grid], dev).buckets(num_buckets=8, max_distance=6)
    got = m.spatial_attention(x, w, buckets=buckets, **args)
    want = torch.stack([m.spatial_attention_volumes([item], w, buckets=buckets, **args)[0].detach() for item in x])
    # the same fp32 operators but for the group norm's, whose values agree to some half steps; through the scores (of some
    # ten units), the products and sums over c channels a few tens of half steps of the largest values
    bound = 64 * 2.0 ** -24 * float(want.abs().max())
    assert not got.requires_grad and float((got - want).abs().max()) <= bound
    plain = m.spatial_attention(x, {n: t for n, t in w.items() if n != "attn.position_bias"}, **args)
    assert float((got - plain).abs().max()) > 1e3 * bound
