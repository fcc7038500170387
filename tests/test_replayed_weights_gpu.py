"""The networks' inference between replays of a captured ``AdamW`` step of the same weights."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _weights(dev, c, seed=3):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=dev, generator=g)
    w = {"norm.weight": 1 + 0.1 * r(c), "norm.bias": 0.1 * r(c)}
    for n in ("to_q", "to_k", "to_v", "out_proj"):
        w[f"attn.{n}.weight"], w[f"attn.{n}.bias"] = r(c, c) / math.sqrt(c), 0.1 * r(c)
    return w | {"conv.weight": r(c, c, 3, 3, 3) / math.sqrt(27 * c), "conv.bias": 0.1 * r(c)}


def _infer(ctmr, x, w):
    y = ctmr.maisi.spatial_attention(x, w, num_groups=16, eps=1e-6, num_head_channels=32, include_fc=True)
    return ctmr.fast_fp32.conv3d(y, w["conv.weight"], w["conv.bias"], padding=1)


@pytest.mark.parametrize("precision", ["fp32", "bf16"])
def test_inference_follows_captured_steps(ctmr, dev, precision):
    """Eager and recorded inference on weights that replays change equal inference on copies, which nothing is kept of."""
    ff, c = ctmr.fast_fp32, 64
    x, w = torch.randn(1, 6, 7, 8, c, device=dev), _weights(dev, c)
    copies = lambda: {n: t.clone() for n, t in w.items()}
    optimizer = ctmr.differentiable.AdamW(list(w.values()), lr=1e-2)
    grads = [torch.randn_like(t) for t in w.values()]
    with ff.precision(precision):
        before = _infer(ctmr, x, w)  # packs and fuses the weights
        assert torch.equal(_infer(ctmr, x, w), before)
        optimizer.step(grads)
        assert torch.equal(_infer(ctmr, x, w), _infer(ctmr, x, copies()))
        step, pass_ = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(step):
            optimizer.step(grads)
        with torch.cuda.graph(pass_):
            recorded = _infer(ctmr, x, w)
        last = _infer(ctmr, x, w)
        for _ in range(3):
            step.replay()
            got = _infer(ctmr, x, w)
            pass_.replay()
            want = _infer(ctmr, x, copies())
            assert not torch.equal(want, last)
            assert torch.equal(got, want) and torch.equal(recorded, want)
            last = want
        ff.settle_weights(w.values())
        assert torch.equal(_infer(ctmr, x, w), last)
        kept = ff.cache_size()
        assert torch.equal(_infer(ctmr, x, w), last) and ff.cache_size() == kept
        ff.drop_packed_weights(w.values())
