"""CPU tests: a learned position bias is never left out silently."""

from __future__ import annotations

import pytest
import torch


def _weights(c=64, heads=2):
    w = {f"attn.{n}.{part}": torch.zeros(*shape) for n in ("to_q", "to_k", "to_v", "out_proj")
         for part, shape in (("weight", (c, c)), ("bias", (c,)))}
    return w | {"norm.weight": torch.ones(c), "norm.bias": torch.zeros(c), "attn.position_bias": torch.zeros(3, 8, heads)}


def test_attention_without_buckets_refuses_a_table(ctmr, monkeypatch):
    tokens, w = torch.zeros(1, 60, 64), _weights()
    for module in (ctmr.fast_fp32, ctmr.differentiable):
        with pytest.raises(ValueError, match="attn.position_bias needs buckets"):
            module.self_attention_tokens(tokens, w, heads=2, scale=0.2, include_fc=True)
    monkeypatch.setattr(ctmr.fast_fp32, "group_norm", lambda x, *a, **kw: x)
    with pytest.raises(ValueError, match="attn.position_bias needs buckets"):
        ctmr.maisi.spatial_attention(torch.zeros(1, 3, 4, 5, 64), w, num_groups=16, eps=1e-6, num_head_channels=32,
                                     include_fc=True)


def test_the_networks_refuse_a_table(ctmr, monkeypatch):
    m = ctmr.maisi
    monkeypatch.setattr(ctmr.fast_fp32, "group_norm", lambda x, *a, **kw: x)
    monkeypatch.setattr(m, "_time_projections", lambda w: (torch.zeros(0, 4), torch.zeros(0), {}))
    monkeypatch.setattr(m, "_block_major_index", lambda *a: (torch.zeros(0, dtype=torch.int64), {}))
    prefixed = {f"mid.{k}": v for k, v in _weights().items()}
    _, attention = m._blocks(prefixed, torch.zeros(1, 4), 16, 1e-6, True)
    with pytest.raises(ValueError, match="attn.position_bias needs buckets"):
        attention(torch.zeros(1, 3, 4, 5, 64), "mid", 32)
