"""``differentiable.attention`` under caps far above the scores: the capped score keeps its bits whatever the cap, and
approaches the score itself."""

from __future__ import annotations

import attention_oracle as oracle
import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs(dev, n, hq, hk, lq, lk, d, dtype, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    make = lambda l, h: torch.randn(n, l, h, d, device=dev, generator=g).to(dtype).transpose(1, 2)
    return make(lq, hq), make(lk, hk), make(lk, hk), make(lq, hq)


def _want(q, k, v, dout, **kw):
    """``[(value, bound)]``: fp32's bound, whose capped scores are off by a share of themselves, and the 16-bit roundings
    as they are without a cap (which moves the weights, scores of up to s, by 2 s^3 / (3 cap^2) of themselves at most:
    below 1 % for s = 10 and a cap of 300)."""
    cap = kw.pop("softcap")
    exact = oracle.attention(*(t.float() for t in (q, k, v)), dout=dout.float(), softcap=cap, **kw)
    if q.dtype == torch.float32:
        return exact
    rounded = oracle.attention(q, k, v, dout=dout, **kw)
    return [(value, 1.02 * (bound + more)) for (value, bound), (_, more) in zip(exact, rounded)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("softcap", [300.0, 1e4, 1e6, 1e9, 1e25])
@pytest.mark.parametrize("shape", [(1, 4, 2, 150, 190, 64), (1, 2, 2, 140, 300, 128), (2, 4, 1, 70, 130, 24), (1, 8, 2, 2, 700, 64)],
                         ids=str)
def test_scores_keep_their_bits(ctmr, dev, shape, softcap, dtype):
    q, k, v, dout = _inputs(dev, *shape, dtype)
    d, lq, lk = shape[-1], shape[3], shape[4]
    slopes = torch.linspace(0.0, 0.05, shape[1], device=dev)
    for kw in ({}, {"slopes": slopes, "prefix": 40}):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = ctmr.differentiable.attention(*leaves, scale=d ** -0.5, softcap=softcap, **kw)
        got = [out.detach(), *torch.autograd.grad(out, leaves, dout)]
        mask = oracle.visible(shape[0], lq, lk, dev, prefix=kw.pop("prefix", None))
        for g, w, name in zip(got, _want(q, k, v, dout, scale=d ** -0.5, softcap=softcap, mask=mask, **kw),
                              ("out", "dq", "dk", "dv")):
            oracle.check(g, w, name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_scores_of_the_cap_s_own_size(ctmr, dev, dtype):
    """Scores of some thousands under a cap of a thousand, on both bends of the tangent and between."""
    q, k, v, dout = _inputs(dev, 1, 2, 2, 100, 200, 64, dtype, seed=1)
    kw = dict(scale=100.0, softcap=1000.0)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ctmr.differentiable.attention(*leaves, **kw)
    got = [out.detach(), *torch.autograd.grad(out, leaves, dout)]
    for g, w in zip(got, oracle.attention(q, k, v, dout=dout, **kw)):
        oracle.check(g, w)
