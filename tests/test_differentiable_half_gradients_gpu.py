"""fp16 gradients of ``differentiable.attention`` whose rows differ far in size: what one document, head or row has in its
output gradient or values does not decide how many bits another keeps.  And the shapes, masks and strides of the other
types' gradients, in fp16."""

from __future__ import annotations

import math

import attention_oracle as oracle
import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs(dev, n, hq, hk, lq, lk, d, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    make = lambda l, h: torch.randn(n, l, h, d, device=dev, generator=g).half().transpose(1, 2)
    return make(lq, hq), make(lk, hk), make(lk, hk), make(lq, hq)


def _run(ctmr, q, k, v, dout, **kw):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ctmr.differentiable.attention(*leaves, **kw)
    return [out.detach(), *torch.autograd.grad(out, leaves, dout)]


def _compare(ctmr, q, k, v, dout, *, ids=None, key_ids=None, prefix=None, scale=None, **kw):
    f = ctmr.differentiable
    kw["scale"] = q.shape[-1] ** -0.5 if scale is None else scale
    mask = oracle.visible(q.shape[0], q.shape[2], k.shape[2], q.device, ids, key_ids, prefix)
    want = oracle.attention(q, k, v, mask=mask, dout=dout, **kw)
    got = _run(ctmr, q, k, v, dout, prefix=prefix, documents=None if ids is None else f.Documents(ids, key_ids), **kw)
    for t, w, name in zip(got, want, ("out", "dq", "dk", "dv")):
        oracle.check(t, w, name)
    return got


def _two(dev, first, total):
    ids = torch.zeros(1, total, dtype=torch.int32, device=dev)
    ids[:, first:] = 1
    return ids


@pytest.mark.parametrize("first", [150, 1024, 64])
@pytest.mark.parametrize(("d", "softcap"), [(64, 0.0), (32, 0.0), (128, 3.0), (128, 0.0)])
def test_documents_keep_their_own_bits(ctmr, dev, first, d, softcap):
    """A document beside one whose output gradient is 2^20 times its own: as exact as alone, and the same bits as beside
    one of its own size."""
    total = 2 * first
    q, k, v, dout = (t.contiguous() for t in _inputs(dev, 1, 2, 1, total, total, d, seed=first))
    dout *= 2.0 ** -10
    ids = _two(dev, first, total)
    f, kw = ctmr.differentiable, dict(scale=d ** -0.5, softcap=softcap)
    beside = _run(ctmr, q, k, v, dout, documents=f.Documents(ids), **kw)
    dout[:, :, first:] *= 2.0 ** 20
    got = _run(ctmr, q, k, v, dout, documents=f.Documents(ids), **kw)
    for half in (slice(0, first), slice(first, total)):
        want = oracle.attention(*(t[:, :, half] for t in (q, k, v)), dout=dout[:, :, half], **kw)
        for t, w, name in zip(got, want, ("out", "dq", "dk", "dv")):
            oracle.check(t[:, :, half], w, (name, half))
    assert all(torch.equal(a[:, :, :first], b[:, :, :first]) for a, b in zip(got, beside))


def test_values_that_no_row_sees(ctmr, dev):
    """The type's largest values under an id that no query row has."""
    q, k, v, dout = (t.contiguous() for t in _inputs(dev, 1, 2, 2, 200, 400, 64, seed=1))
    dout *= 2.0 ** -12
    ids = torch.zeros(1, 200, dtype=torch.int32, device=dev)
    key_ids = torch.zeros(1, 400, dtype=torch.int32, device=dev)
    key_ids[:, 300:] = 5
    clean = _compare(ctmr, q, k, v, dout, ids=ids, key_ids=key_ids)
    v[:, :, 300:] = 65504.0
    k[:, :, 300:] = 65504.0
    assert all(torch.equal(a, b) for a, b in zip(clean, _compare(ctmr, q, k, v, dout, ids=ids, key_ids=key_ids)))


@pytest.mark.parametrize("d", [32, 64, 128])
def test_rows_and_heads_keep_their_own_bits(ctmr, dev, d):
    """dq of a row does not depend on other rows and heads, dk and dv of a key that only small rows see neither."""
    q, k, v, dout = (t.contiguous() for t in _inputs(dev, 2, 4, 2, 300, 300, d, seed=2))
    dout *= 2.0 ** -10
    small = _compare(ctmr, q, k, v, dout, prefix=0)
    dout[:, 1] *= 2.0 ** 20  # the other query head of key head 0
    dout[1] *= 2.0 ** 3
    dout[:, 2:, :200] *= 2.0 ** 20  # rows before the last keys
    got = _compare(ctmr, q, k, v, dout, prefix=0)
    assert torch.equal(got[1][0, 0], small[1][0, 0])
    assert torch.equal(got[1][0, 2:, 200:], small[1][0, 2:, 200:])
    assert all(torch.equal(a[0, 1, 200:], b[0, 1, 200:]) for a, b in zip(got[2:], small[2:]))


@pytest.mark.parametrize("order", ["rising", "falling", "one"])
def test_output_gradients_over_the_whole_range(ctmr, dev, order):
    """Rows from 2^-14 to 2^13 in one call: the keys' sums are moved to another power of two on the way, or never."""
    q, k, v, dout = (t.contiguous() for t in _inputs(dev, 1, 4, 2, 520, 520, 64, seed=3))
    power = torch.linspace(-14, 13, 520, device=dev).round()
    power = {"rising": power, "falling": power.flip(0), "one": torch.where(torch.arange(520, device=dev) == 300, 13.0, -14.0)}[order]
    dout = (dout.float() * torch.exp2(power)[:, None]).half()
    _compare(ctmr, q, k, v, dout)
    _compare(ctmr, q, k, v, dout, prefix=17, softcap=5.0, slopes=torch.rand(4, device=dev))


def test_zero_output_gradients(ctmr, dev):
    q, k, v, dout = _inputs(dev, 1, 2, 1, 140, 140, 32)
    assert all(bool((t == 0).all()) for t in _run(ctmr, q, k, v, torch.zeros_like(dout), scale=0.2)[1:])


SHAPES = [(1, 2, 1, 63, 65, 32), (1, 8, 8, 129, 257, 32), (1, 4, 1, 200, 130, 96), (1, 2, 2, 300, 300, 128),
          (2, 8, 2, 77, 513, 40), (1, 3, 3, 191, 64, 72), (1, 16, 4, 260, 260, 128), (1, 6, 2, 33, 1000, 64),
          (1, 1, 1, 1, 5, 32), (2, 8, 2, 1, 700, 64), (1, 4, 4, 3, 4001, 128), (1, 8, 1, 4, 130, 48)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("softcap", [0.0, 2.0])
def test_shapes(ctmr, dev, shape, softcap):
    q, k, v, dout = _inputs(dev, *shape, seed=4)
    _compare(ctmr, q, k, v, dout, softcap=softcap)
    _compare(ctmr, q, k, v, dout, softcap=softcap, prefix=shape[4] // 3, slopes=torch.rand(shape[1], device=dev))


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("lengths", [[64, 64, 64], [1, 62, 130, 2], [5]], ids=str)
def test_documents(ctmr, dev, lengths, d):
    q, k, v, dout = _inputs(dev, 2, 4, 2, 300, 300, d, seed=5)
    ids = torch.full((2, 300), -1, dtype=torch.int32)
    at = 0
    for i, length in enumerate(lengths):
        ids[:, at:at + length] = i
        at += length
    ids[1] = ids[1].flip(0)
    _compare(ctmr, q, k, v, dout, ids=ids.to(dev))
    _compare(ctmr, q, k, v, dout, ids=ids.to(dev), prefix=70, softcap=3.0, slopes=torch.rand(4, device=dev))


def test_strides(ctmr, dev):
    n, l, h, d = 2, 140, 2, 32
    g = torch.Generator(device=dev).manual_seed(6)
    fused = torch.randn(n, l, 3 * h * d, device=dev, generator=g).half()
    q, k, v = (fused[..., i * h * d:(i + 1) * h * d].unflatten(-1, (h, d)).transpose(1, 2) for i in range(3))
    dout = _inputs(dev, n, h, h, l, l, d, seed=7)[3]
    _compare(ctmr, q, k, v, dout)
    _compare(ctmr, q, k[:1].expand(n, h, l, d), k[:, :, :1].expand(n, h, l, d), dout[:, :, 5:6].expand(n, h, l, d))
    _compare(ctmr, q, k, v, torch.ones((), device=dev, dtype=torch.float16).expand(n, h, l, d))


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_masked_places_hold_has_no_effect(ctmr, dev, value):
    f = ctmr.differentiable
    q, k, v, dout = (t.contiguous() for t in _inputs(dev, 2, 4, 2, 300, 300, 64, seed=8))
    ids = torch.full((2, 300), -1, dtype=torch.int32, device=dev)
    ids[:, :100], ids[:, 100:190], ids[:, 190:250] = 0, 1, 2
    kw = dict(scale=0.125, documents=f.Documents(ids))
    clean = _run(ctmr, q, k, v, dout, **kw)
    for t in (q, k, v, dout):
        t.transpose(1, 2)[(ids == 1) | (ids < 0)] = value
    keep = (ids != 1)[:, None, :, None]
    for got, want in zip(_run(ctmr, q, k, v, dout, **kw), clean):
        assert torch.equal(got[keep.expand_as(got)], want[keep.expand_as(got)])
