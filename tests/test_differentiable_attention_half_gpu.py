"""Gradients of ``differentiable.attention`` in fp16, whose range ds would leave, and of ragged rows whose distance bias
grows, against 64 bits (``attention_oracle``)."""

from __future__ import annotations

import math

import attention_oracle as oracle
import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs(dev, n, hq, hk, lq, lk, d, dtype, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    make = lambda l, h: torch.randn(n, l, h, d, device=dev, generator=g).to(dtype).transpose(1, 2)
    return make(lq, hq), make(lk, hk), make(lk, hk), make(lq, hq)


def _compare(ctmr, q, k, v, dout, *, ids=None, prefix=None, **kw):
    f = ctmr.differentiable
    kw = {"scale": q.shape[-1] ** -0.5} | kw
    mask = oracle.visible(q.shape[0], q.shape[2], k.shape[2], q.device, ids, ids, prefix)
    want = oracle.attention(q, k, v, mask=mask, dout=dout, **kw)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = f.attention(*leaves, prefix=prefix, documents=None if ids is None else f.Documents(ids), **kw)
    got = [out.detach(), *torch.autograd.grad(out, leaves, dout)]
    for t, w, name in zip(got, want, ("out", "dq", "dk", "dv")):
        assert t.dtype == q.dtype
        oracle.check(t, w, name)
    return got


@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1, 8), (2, 4, 2, 130, 130, 64), (1, 8, 8, 129, 257, 32), (1, 6, 2, 200, 77, 128),
                                   (2, 2, 1, 300, 300, 96), (1, 16, 4, 2, 900, 128), (1, 4, 1, 2100, 2100, 24)], ids=str)
@pytest.mark.parametrize("size", [1.0, 2.0 ** -18, 2.0 ** 12])
def test_gradients_of_every_size(ctmr, dev, shape, size):
    """Output gradients of 4e-6 and of 4000 times the ordinary: ds is kept in range by what they and v are."""
    q, k, v, dout = _inputs(dev, *shape, torch.float16)
    _compare(ctmr, q, k, v, (dout.float() * size).half())


@pytest.mark.parametrize("kw", [{"softcap": 3.0}, {"slopes": True}, {"prefix": 40}, {"ids": True},
                                {"softcap": 3.0, "slopes": True, "prefix": 40, "ids": True}], ids=str)
def test_masks_and_biases(ctmr, dev, kw):
    q, k, v, dout = _inputs(dev, 2, 4, 2, 210, 210, 64, torch.float16, seed=1)
    kw = dict(kw)
    if kw.get("slopes"):
        kw["slopes"] = torch.linspace(0.01, 0.3, 4, device=dev)
    if kw.get("ids"):
        ids = torch.full((2, 210), -1, dtype=torch.int32)
        ids[:, :70], ids[:, 70:190] = 0, 1
        kw["ids"] = ids.to(dev)
    _compare(ctmr, q, k, v, dout, **kw)


def test_padding_does_not_lower_the_gradients(ctmr, dev):
    """Padding of the type's largest values would take ds of ordinary rows below the type's least."""
    q, k, v, dout = (t.contiguous() for t in _inputs(dev, 1, 2, 2, 200, 200, 64, torch.float16, seed=2))
    dout = (dout.float() * 2.0 ** -10).half()
    ids = torch.zeros(1, 200, dtype=torch.int32, device=dev)
    ids[:, 150:] = -1
    clean = _compare(ctmr, q, k, v, dout, ids=ids)
    for value in (65504.0, -65504.0, math.inf, math.nan):
        for t in (q, k, v, dout):
            t[:, :, 150:] = value
        again = _compare(ctmr, q, k, v, dout, ids=ids)
        assert all(torch.equal(a, b) for a, b in zip(clean, again))


def test_rows_that_see_nothing_do_not_lower_the_gradients(ctmr, dev):
    q, k, v, dout = (t.contiguous() for t in _inputs(dev, 1, 2, 1, 150, 100, 32, torch.float16, seed=3))
    dout = (dout.float() * 2.0 ** -10).half()
    clean = _compare(ctmr, q, k, v, dout, prefix=0)  # the first 50 rows see no key
    dout[:, :, :50] = 65504.0
    again = _compare(ctmr, q, k, v, dout, prefix=0)
    assert all(torch.equal(a, b) for a, b in zip(clean, again))


def test_documents_without_keys_do_not_lower_the_gradients(ctmr, dev):
    f = ctmr.differentiable
    q, k, v, dout = (t.contiguous() for t in _inputs(dev, 2, 2, 1, 70, 900, 32, torch.float16, seed=6))
    dout = (dout.float() * 2.0 ** -10).half()
    ids, key_ids = (torch.zeros(2, l, dtype=torch.int32, device=dev) for l in (70, 900))
    ids[:, 40:] = 7  # no key is of it
    documents, mask = f.Documents(ids, key_ids), oracle.visible(2, 70, 900, dev, ids, key_ids)
    results = []
    for value in (None, 65504.0):
        if value is not None:
            dout[:, :, 40:] = value
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = f.attention(*leaves, scale=0.2, documents=documents)
        results.append([out.detach(), *torch.autograd.grad(out, leaves, dout)])
        for t, w in zip(results[-1], oracle.attention(q, k, v, scale=0.2, mask=mask, dout=dout)):
            oracle.check(t, w)
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_visible_infinity_and_nan_show(ctmr, dev):
    for value in (math.inf, math.nan):
        q, k, v, dout = (t.contiguous() for t in _inputs(dev, 1, 1, 1, 70, 70, 32, torch.float16, seed=4))
        dout[0, 0, 3, 5] = value
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = ctmr.differentiable.attention(*leaves, scale=0.2)
        dq, dk, dv = torch.autograd.grad(out, leaves, dout)
        assert not bool(dv[0, 0, :, 5].isfinite().any()) and bool(dv[0, 0, :, 6].isfinite().all())
        assert not bool(dq[0, 0, 3].isfinite().all()) and bool(dq[0, 0, 4].isfinite().all())


def test_captured_and_replayed(ctmr, dev):
    make = lambda seed: [t.clone() for t in _inputs(dev, 2, 4, 2, 260, 700, 64, torch.float16, seed)]
    documents = ctmr.differentiable.Documents(torch.zeros(2, 260, dtype=torch.int32, device=dev),
                                              torch.zeros(2, 700, dtype=torch.int32, device=dev))

    def step(q, k, v, dout):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = ctmr.differentiable.attention(*leaves, scale=0.125, documents=documents)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    static = make(0)
    step(*static)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*static)
    for seed in range(1, 5):
        fresh = make(seed)
        fresh[3] *= 2.0 ** (4 - 5 * seed)  # another power of two each time
        for s, t in zip(static, fresh):
            s.copy_(t)
        graph.replay()
        eager = step(*fresh)
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("documents", [False, True])
def test_a_bias_that_grows_with_the_distance(ctmr, dev, dtype, documents):
    """Slopes below zero: rows past the end of a ragged tile have weights past every range, and add nothing."""
    q, k, v, dout = _inputs(dev, 1, 2, 2, 200, 200, 32, dtype, seed=5)
    slopes = torch.tensor([-1.0, 0.5], device=dev)
    ids = torch.zeros(1, 200, dtype=torch.int32, device=dev) if documents else None
    _compare(ctmr, q, k, v, dout, slopes=slopes, ids=ids)
