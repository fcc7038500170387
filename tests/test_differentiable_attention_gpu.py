"""``differentiable.attention`` and its gradients against 64 bits (``attention_oracle``): types, grouped heads, odd
lengths, every mask, both forward forms, strides, what masked places hold, graphs and streams."""

from __future__ import annotations

import math

import attention_oracle as oracle
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _heads(dev, n, l, h, d, dtype, seed, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (scale * torch.randn(n, l, h, d, device=dev, generator=g)).to(dtype).transpose(1, 2)


def _inputs(dev, n, hq, hk, lq, lk, d, dtype, seed=0):
    return (_heads(dev, n, lq, hq, d, dtype, 4 * seed), _heads(dev, n, lk, hk, d, dtype, 4 * seed + 1),
            _heads(dev, n, lk, hk, d, dtype, 4 * seed + 2), _heads(dev, n, lq, hq, d, dtype, 4 * seed + 3))


def _rows(dev, n, lengths, total, start=0):
    """(n, total) ids of documents side by side, the rest padding; each item's ids turned by one document."""
    out = torch.full((n, total), -1, dtype=torch.int32)
    for b in range(n):
        at = 0
        for i, length in enumerate(lengths[b % len(lengths):] + lengths[:b % len(lengths)]):
            out[b, at:at + length] = start + i
            at += length
    return out.to(dev)


def _run(f, q, k, v, dout, **kw):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = f.attention(*leaves, **kw)
    return [out.detach(), *torch.autograd.grad(out, leaves, dout)]


def _compare(ctmr, q, k, v, dout, *, scale=None, softcap=0.0, slopes=None, prefix=None, ids=None, key_ids=None):
    f = ctmr.differentiable
    b, _, lq, d = q.shape
    lk = k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    documents = None if ids is None else f.Documents(ids, key_ids)
    kw = dict(scale=scale, softcap=softcap, slopes=slopes, prefix=prefix, documents=documents)
    mask = oracle.visible(b, lq, lk, q.device, ids, key_ids, prefix)
    train = q.dtype != torch.float16
    want = oracle.attention(q, k, v, scale=scale, softcap=softcap, slopes=slopes, mask=mask, dout=dout if train else None)
    with torch.no_grad():
        out = f.attention(q, k, v, **kw)
    assert out.dtype == q.dtype and out.transpose(1, 2).is_contiguous()
    oracle.check(out, want[0], "out")
    empty = ~mask.any(-1)
    assert bool((out.transpose(1, 2)[empty] == 0).all())
    if not train:
        return
    got = _run(f, q, k, v, dout, **kw)
    assert torch.equal(got[0], out)
    for g, w, name in zip(got, want, ("out", "dq", "dk", "dv")):
        oracle.check(g, w, name)
    assert bool((got[1].transpose(1, 2)[empty] == 0).all())
    unseen = ~mask.any(-2)
    assert bool((got[2].transpose(1, 2)[unseen] == 0).all()) and bool((got[3].transpose(1, 2)[unseen] == 0).all())


# (n, hq, hk, lq, lk, d): one row and key; tile edges and off by one; head widths between the kernels'; grouped
# heads; other lengths of rows and keys; eight and more items (the XCD order)
SHAPES = [(1, 1, 1, 1, 1, 8), (1, 2, 1, 63, 65, 32), (2, 4, 2, 128, 128, 64), (1, 8, 8, 129, 257, 32),
          (1, 4, 1, 200, 130, 96), (1, 2, 2, 300, 300, 128), (2, 8, 2, 77, 513, 40), (1, 3, 3, 191, 64, 72),
          (1, 16, 4, 260, 260, 128), (1, 6, 2, 33, 1000, 64)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_every_key(ctmr, dev, shape, dtype):
    _compare(ctmr, *_inputs(dev, *shape, dtype))


# few rows (their own kernel): one token, a group of tokens, keys split over workgroups and not
FEW = [(1, 1, 1, 1, 5, 32), (2, 8, 2, 1, 700, 64), (1, 4, 4, 3, 4001, 128), (4, 32, 8, 1, 2500, 128),
       (1, 8, 1, 4, 130, 48), (3, 2, 2, 31, 333, 32), (1, 32, 1, 1, 64, 32)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", FEW, ids=str)
def test_few_rows(ctmr, dev, shape, dtype):
    q, k, v, dout = _inputs(dev, *shape, dtype)
    _compare(ctmr, q, k, v, dout)
    n, hq, _, lq, lk, _ = shape
    lengths = torch.randint(0, lk + 1, (n,), generator=torch.Generator().manual_seed(5))
    key_ids = torch.where(torch.arange(lk) < lengths[:, None], 0, -1).int().to(dev)
    ids = torch.zeros(n, lq, dtype=torch.int32, device=dev)
    slopes = torch.rand(hq, device=dev)
    _compare(ctmr, q, k, v, dout, ids=ids, key_ids=key_ids, softcap=5.0)
    _compare(ctmr, q, k, v, dout, prefix=lk // 2, slopes=slopes, ids=ids, key_ids=key_ids)


def test_long_keys_split_over_workgroups(ctmr, dev):
    for shape in ((1, 4, 2, 150, 9000, 64), (1, 1, 1, 40, 20000, 32)):
        for dtype in (torch.bfloat16, torch.float32):
            q, k, v, dout = _inputs(dev, *shape, dtype)
            _compare(ctmr, q, k, v, dout)
            _compare(ctmr, q, k, v, dout, prefix=100, ids=_rows(dev, 1, [30, 60], shape[3]),
                     key_ids=_rows(dev, 1, [shape[4] - 700, 600], shape[4]))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("lengths", [[64, 64, 64], [1, 62, 130, 2], [5], [200, 3, 90]], ids=str)
def test_documents(ctmr, dev, lengths, d, dtype):
    l = 300
    q, k, v, dout = _inputs(dev, 2, 4, 2, l, l, d, dtype)
    ids = _rows(dev, 2, lengths, l, start=3)
    _compare(ctmr, q, k, v, dout, ids=ids)
    _compare(ctmr, q, k, v, dout, ids=ids, prefix=70, softcap=3.0, slopes=torch.rand(4, device=dev))


def test_documents_in_any_order(ctmr, dev):
    l = 350
    q, k, v, dout = _inputs(dev, 2, 2, 2, l, l, 64, torch.bfloat16)
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(-1, 4, (2, l), generator=g).int().to(dev)
    _compare(ctmr, q, k, v, dout, ids=ids)
    _compare(ctmr, q[:, :, :100], k, v, dout[:, :, :100], ids=ids[:, :100].contiguous(), key_ids=ids.flip(1))
    large = torch.tensor([2 ** 31 - 1, 0, 7], dtype=torch.int32)[torch.randint(0, 3, (2, l), generator=g)].to(dev)
    large[large == 7] = -(2 ** 31)
    _compare(ctmr, q, k, v, dout, ids=large)


def test_every_row_padding(ctmr, dev):
    q, k, v, dout = _inputs(dev, 2, 2, 1, 70, 70, 32, torch.bfloat16)
    ids = torch.full((2, 70), -1, dtype=torch.int32, device=dev)
    ids[1] = 0
    _compare(ctmr, q, k, v, dout, ids=ids)
    _compare(ctmr, q[:, :, :4], k, v, dout[:, :, :4], ids=ids[:, :4].contiguous(), key_ids=ids)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(2, 4, 2, 200, 200, 64), (2, 2, 2, 130, 300, 32), (2, 4, 1, 300, 131, 128)], ids=str)
def test_prefix(ctmr, dev, shape, dtype):
    """None, causal, inside a tile, everything, one for each item; more rows than keys leave the first rows empty."""
    q, k, v, dout = _inputs(dev, *shape, dtype)
    for prefix in (0, 1, 77, 10 ** 6, torch.tensor([150, -3], dtype=torch.int32, device=dev)):
        if isinstance(prefix, int):
            _compare(ctmr, q, k, v, dout, prefix=prefix)
        else:
            _compare(ctmr, q, k, v, dout, prefix=prefix, softcap=2.0)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_cap_and_distance(ctmr, dev, dtype):
    q, k, v, dout = _inputs(dev, 1, 4, 2, 150, 190, 64, dtype)
    slopes = torch.tensor([0.0, 0.01, 0.5, 4.0], device=dev)
    _compare(ctmr, q, k, v, dout, softcap=1.5)
    _compare(ctmr, q, k, v, dout, slopes=slopes)
    _compare(ctmr, q, k, v, dout, softcap=30.0, slopes=slopes, scale=2.0)


def test_large_scores(ctmr, dev):
    """Scores of some hundreds: one key takes nearly all of a row, and the reference maximum moves often."""
    for dtype in TYPES:
        q, k, v, dout = _inputs(dev, 1, 2, 2, 100, 400, 64, dtype)
        _compare(ctmr, (4 * q.float()).to(dtype), (4 * k.float()).to(dtype), v, dout, scale=0.5)
        ramp = k * torch.linspace(0.1, 3, 400, device=dev).to(dtype)[:, None]  # later keys score higher
        _compare(ctmr, q, ramp.to(dtype), v, dout, scale=1.0)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_strides(ctmr, dev, dtype):
    """Columns of a fused projection, keys shared over the batch, an odd address, a transposed head, one-row views."""
    n, l, h, d = 2, 140, 2, 32
    g = torch.Generator(device=dev).manual_seed(1)
    fused = torch.randn(n, l, 3 * h * d, device=dev, generator=g).to(dtype)
    q, k, v = (fused[..., i * h * d:(i + 1) * h * d].unflatten(-1, (h, d)).transpose(1, 2) for i in range(3))
    dout = _heads(dev, n, l, h, d, dtype, 9)
    _compare(ctmr, q, k, v, dout)
    wide = k[:1].expand(n, h, l, d)
    _compare(ctmr, q, wide, wide, dout)
    same = k[:, :, :1].expand(n, h, l, d)  # one row for every key
    _compare(ctmr, q, same, v, dout[:, :, 5:6].expand(n, h, l, d))
    flat = torch.zeros(q.numel() + 1, device=dev, dtype=dtype)
    odd = flat[1:].view(n, h, l, d)
    odd.copy_(q)
    _compare(ctmr, odd, odd, v, dout)
    turned = torch.randn(n, h, d, l, device=dev, generator=g).to(dtype).transpose(2, 3)
    _compare(ctmr, turned, k, turned, torch.ones((), device=dev, dtype=dtype).expand(n, h, l, d))
    _compare(ctmr, q[:, :, 7:8], k[:, :, 3:], v[:, :, 3:], dout[:, :, 7:8])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("lq", [300, 2])
def test_what_masked_places_hold_has_no_effect(ctmr, dev, value, dtype, lq):
    """Padding and another document's tokens hold NaN or infinities, inside the same tiles."""
    f = ctmr.differentiable
    n, hq, hk, lk, d = 2, 4, 2, 300, 64
    q, k, v, dout = (t.clone() for t in _inputs(dev, n, hq, hk, lq, lk, d, dtype))
    key_ids = _rows(dev, n, [100, 90, 60], lk)
    ids = key_ids[:, :lq].contiguous() if lq == lk else torch.zeros(n, lq, dtype=torch.int32, device=dev)
    documents = f.Documents(ids, key_ids)
    kw = dict(scale=d ** -0.5, documents=documents)
    clean = f.attention(q, k, v, **kw)
    grads = _run(f, q, k, v, dout, **kw) if dtype != torch.float16 else None
    for t, t_ids in ((q, ids), (k, key_ids), (v, key_ids), (dout, ids)):
        t.transpose(1, 2)[(t_ids == 1) | (t_ids < 0)] = value
    out = f.attention(q, k, v, **kw)
    keep = (ids != 1)[:, None, :, None].expand_as(out)
    assert torch.equal(out[keep], clean[keep])
    if grads is None:
        return
    for got, want, t_ids in zip(_run(f, q, k, v, dout, **kw), grads, (ids, ids, key_ids, key_ids)):
        keep = (t_ids != 1)[:, None, :, None].expand_as(got)
        assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("lq", [200, 1])
def test_visible_nan_and_infinity_show(ctmr, dev, dtype, lq):
    f = ctmr.differentiable
    q, k, v, dout = (t.clone() for t in _inputs(dev, 1, 2, 2, lq, 200, 32, dtype))
    key_ids = _rows(dev, 1, [90, 70], 200)
    ids = key_ids if lq == 200 else torch.zeros(1, 1, dtype=torch.int32, device=dev)
    kw = dict(scale=32 ** -0.5, documents=f.Documents(ids, key_ids))
    clean = f.attention(q, k, v, **kw)
    v[0, 0, 5, 3], v[0, 0, 6, 4], v[0, 1, 7, 9] = math.inf, math.nan, -math.inf
    out = f.attention(q, k, v, **kw)
    seen = (ids[0] == 0)
    want = clean.clone()
    want[0, 0, seen, 3], want[0, 0, seen, 4], want[0, 1, seen, 9] = math.inf, math.nan, -math.inf
    assert torch.equal(out.nan_to_num(7e3, 8e3, 9e3), want.nan_to_num(7e3, 8e3, 9e3))
    if dtype != torch.float16:
        dout[0, 0, 0, 2] = math.inf
        dv = _run(f, q, k, clean.new_zeros(v.shape), dout, **kw)[3]
        col = dv[0, 0, :, 2]
        assert bool((col[key_ids[0] == 0] == math.inf).all()) and bool(col[key_ids[0] != 0].isfinite().all())


def test_infinity_in_a_single_row(ctmr, dev):
    """What a tile holds past its only row is nothing, not the row again."""
    f = ctmr.differentiable
    for dtype in TYPES:
        q, k, v, dout = (t.clone() for t in _inputs(dev, 1, 1, 1, 1, 1, 32, dtype))
        v[..., 3] = math.inf
        out = f.attention(q, k, v, scale=0.1)
        assert torch.equal(out, v)
        if dtype != torch.float16:
            v.zero_()
            dout[..., 4] = -math.inf
            assert torch.equal(_run(f, q, k, v, dout, scale=0.1)[3], dout)


@pytest.mark.parametrize("kw", [{}, {"softcap": 2.0}, {"prefix": 20}, {"slopes": True}, {"ids": True}], ids=str)
def test_differences(ctmr, dev, kw):
    f = ctmr.differentiable
    q, k, v, dout = _inputs(dev, 1, 4, 2, 80, 80, 32, torch.float32)
    kw = dict(kw)
    if kw.pop("ids", None):
        kw["documents"] = f.Documents(_rows(dev, 1, [30, 41], 80))
    if kw.get("slopes"):
        kw["slopes"] = torch.rand(4, device=dev)
    grads = _run(f, q, k, v, dout, scale=0.3, **kw)[1:]
    h = 1e-2
    for i, g in enumerate(grads):
        u = torch.randn(g.shape, device=dev, generator=torch.Generator(device=dev).manual_seed(40 + i))
        at = lambda s: float((f.attention(*[t + s * h * u if j == i else t for j, t in enumerate((q, k, v))], scale=0.3,
                                          **kw).double() * dout.double()).sum())
        slope = (at(1.0) - at(-1.0)) / (2 * h)
        # cut-off h^2 / 6 of a third derivative of the scores' scale cubed, below 10 times the slope's size; noise
        # 10240^(1/2) 2^-22 / h
        assert abs(slope - float((g.double() * u.double()).sum())) <= 2e-3 * float(g.norm() * u.norm())


def test_only_the_wanted_gradients(ctmr, dev):
    f = ctmr.differentiable
    q, k, v, dout = _inputs(dev, 1, 4, 2, 100, 120, 64, torch.bfloat16)
    every = _run(f, q, k, v, dout, scale=0.1)
    for i in range(3):
        leaves = [t.detach().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        out = f.attention(*leaves, scale=0.1)
        assert torch.equal(torch.autograd.grad(out, leaves[i], dout)[0], every[1 + i])


def test_the_same_tensor_three_times(ctmr, dev):
    f = ctmr.differentiable
    x, _, _, dout = _inputs(dev, 1, 2, 2, 90, 90, 32, torch.float32)
    leaf = x.detach().requires_grad_()
    got, = torch.autograd.grad(f.attention(leaf, leaf, leaf, scale=0.2), leaf, dout)
    parts = oracle.attention(x, x, x, scale=0.2, dout=dout)[1:]
    value, bound = (sum(p[i] for p in parts) for i in range(2))
    oracle.check(got, (value, bound + 4 * oracle.U * value.abs()))


@pytest.mark.parametrize("lq", [260, 1])
def test_repeats_streams_and_graph(ctmr, dev, lq):
    f = ctmr.differentiable
    make = lambda seed: [t.clone() for t in _inputs(dev, 2, 4, 2, lq, 1100, 64, torch.bfloat16, seed)]
    key_ids = _rows(dev, 2, [500, 400], 1100)
    ids = key_ids[:, :lq].contiguous()
    documents = f.Documents(ids, key_ids)
    prefix = torch.tensor([10, 300], dtype=torch.int32, device=dev)
    step = lambda q, k, v, dout: _run(f, q, k, v, dout, scale=0.125, documents=documents, prefix=prefix)
    static = make(0)
    want = step(*static)
    assert all(torch.equal(a, b) for a, b in zip(want, step(*static)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step(*static)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    graphs, outs = [], []
    for _ in range(2):  # two captures: each has workspaces of its own
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(*static))
    for seed in range(1, 4):
        fresh = make(seed)
        for s, t in zip(static, fresh):
            s.copy_(t)
        for graph in graphs:
            graph.replay()
        eager = step(*fresh)
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_documents_keep_their_own_copy(ctmr, dev):
    f = ctmr.differentiable
    q, k, v, dout = _inputs(dev, 1, 2, 2, 100, 100, 32, torch.bfloat16)
    ids = _rows(dev, 1, [40, 50], 100)
    documents = f.Documents(ids)
    want = f.attention(q, k, v, scale=0.2, documents=documents)
    ids.zero_()
    assert torch.equal(f.attention(q, k, v, scale=0.2, documents=documents), want)


def test_empty(ctmr, dev):
    f = ctmr.differentiable
    for n, h, lq, lk in ((0, 2, 5, 5), (1, 2, 0, 5), (1, 2, 5, 0)):
        q, k, v = (torch.ones(n, h, l, 16, device=dev, requires_grad=True) for l in (lq, lk, lk))
        out = f.attention(q, k, v, scale=1.0)
        assert out.shape == q.shape and bool((out == 0).all())
        for g, t in zip(torch.autograd.grad(out, (q, k, v), torch.ones_like(out)), (q, k, v)):
            assert g.shape == t.shape and bool((g == 0).all())


def test_refuses_foreign_documents(ctmr, dev):
    f = ctmr.differentiable
    q, k, v, _ = _inputs(dev, 1, 2, 2, 8, 8, 16, torch.float16)
    with pytest.raises(ValueError, match="documents are for"):
        f.attention(q, k, v, scale=1.0, documents=f.Documents(torch.zeros(1, 9, dtype=torch.int32, device=dev)))
