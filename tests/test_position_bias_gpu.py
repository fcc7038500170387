"""``attention`` with a position bias, and its gradients, against 64 bits (``position_bias_oracle``): types, grouped heads,
extents, every mask, both forward forms, places of their own, what is not finite, graphs and streams."""

from __future__ import annotations

import math

import attention_oracle
import position_bias_oracle as oracle
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _heads(dev, n, l, h, d, dtype, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn(n, l, h, d, device=dev, generator=g).to(dtype).transpose(1, 2)


def _inputs(dev, n, hq, hk, lq, lk, d, dtype, seed=0):
    return [_heads(dev, n, l, h, d, dtype, 4 * seed + i) for i, (l, h) in enumerate(((lq, hq), (lk, hk), (lk, hk), (lq, hq)))]


def _table(dev, extents, buckets, hq, dtype, seed=9, scale=0.7):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (scale * torch.randn(len(extents), buckets, hq, device=dev, generator=g)).to(dtype)


def _places(dev, items, l, extents, seed=3, beyond=0):
    """Places drawn from the extents; ``beyond``: as many more on both sides."""
    g = torch.Generator().manual_seed(seed)
    t = torch.stack([torch.randint(-beyond, e + beyond, (items or 1, l), generator=g) for e in extents], -1).int().to(dev)
    return t if items else t[0]


def _grid(dev, shape):
    return torch.stack(torch.meshgrid(*(torch.arange(s) for s in shape), indexing="ij"), -1).reshape(-1, len(shape)).int().to(dev)


def dtype_bits(t):
    return 8 * t.element_size()


def _run(f, q, k, v, table, dout, **kw):
    leaves = [t.detach().requires_grad_() for t in (q, k, v, table)]
    out = f.attention(*leaves[:3], position_bias=leaves[3], **kw)
    return [out.detach(), *torch.autograd.grad(out, leaves, dout)]


def _compare(ctmr, q, k, v, dout, table, places, key_places=None, *, extents, num_buckets=None, max_distance=10, softcap=0.0,
             slopes=None, prefix=None, ids=None, key_ids=None):
    f = ctmr.differentiable
    b, _, lq, d = q.shape
    lk, num_buckets = k.shape[2], table.shape[1]
    plan = f.PositionBuckets(places, key_places, extents=extents, num_buckets=num_buckets, max_distance=max_distance)
    kw = dict(scale=d ** -0.5, softcap=softcap, slopes=slopes, prefix=prefix, buckets=plan,
              documents=None if ids is None else f.Documents(ids, key_ids))
    which = oracle.numbers(places, places if key_places is None else key_places, extents, num_buckets, max_distance)
    mask = attention_oracle.visible(b, lq, lk, q.device, ids, key_ids, prefix)
    want = oracle.attention(q, k, v, table, which, scale=kw["scale"], softcap=softcap, slopes=slopes, mask=mask, dout=dout)
    with torch.no_grad():
        out = f.attention(q, k, v, position_bias=table, **kw)
    assert out.dtype == q.dtype and out.transpose(1, 2).is_contiguous()
    attention_oracle.check(out, want[0], "out")
    empty = ~mask.any(-1)
    assert bool((out.transpose(1, 2)[empty] == 0).all())
    got = _run(f, q, k, v, table, dout, **kw)
    if dtype_bits(q) == 32:
        assert torch.equal(got[0], out)
    else:  # weights of twice the bits where the table's gradient is wanted; without it the bits are the same
        leaf = q.detach().requires_grad_()
        assert torch.equal(f.attention(leaf, k, v, position_bias=table, **kw), out)
    assert got[4].dtype == table.dtype and got[4].shape == table.shape
    for g, w, name in zip(got, want, ("out", "dq", "dk", "dv", "dtable")):
        attention_oracle.check(g, w, name)
    assert bool((got[1].transpose(1, 2)[empty] == 0).all())
    return got


# (n, hq, hk, lq, lk, d), extents, buckets, items of places: one row and key; tile edges and off by one; one to four axes,
# both widths of the columns; places of each item and shared
SHAPES = [((1, 1, 1, 1, 1, 8), (1,), 4, 0), ((1, 2, 1, 63, 65, 32), (9, 7), 8, 0), ((2, 4, 2, 128, 128, 64), (16, 16, 8), 32, 0),
          ((1, 8, 8, 129, 257, 32), (20, 21, 23), 16, 0), ((2, 4, 1, 200, 130, 96), (40, 40, 48), 32, 2),
          ((1, 2, 2, 300, 300, 128), (24, 24, 16), 32, 0), ((2, 8, 2, 77, 513, 40), (5, 6, 7, 8), 6, 2),
          ((1, 3, 3, 191, 64, 72), (128,), 64, 0), ((1, 8, 4, 260, 260, 128), (32, 33, 1, 62), 10, 1),
          ((1, 6, 2, 33, 1000, 64), (10, 10, 10), 32, 0), ((3, 2, 2, 150, 150, 24), (6, 5, 5), 4, 3)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize(("shape", "extents", "buckets", "items"), SHAPES, ids=str)
def test_every_key(ctmr, dev, shape, extents, buckets, items, dtype):
    n, hq, hk, lq, lk, d = shape
    table = _table(dev, extents, buckets, hq, dtype if lq % 2 else torch.float32)
    _compare(ctmr, *_inputs(dev, *shape, dtype), table, _places(dev, items, lq, extents, beyond=2),
             _places(dev, items, lk, extents, seed=4), extents=extents, max_distance=buckets)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize(("grid", "d"), [((8, 8, 4), 32), ((6, 7, 9), 64), ((5, 40, 3), 128), ((12, 25), 16)], ids=str)
def test_voxels_of_a_grid(ctmr, dev, grid, d, dtype):
    l = math.prod(grid)
    table = _table(dev, grid, 16, 4, dtype)
    _compare(ctmr, *_inputs(dev, 2, 4, 2, l, l, d, dtype), table, _grid(dev, grid), extents=grid, max_distance=9)


# few rows (their own kernel): one token, a group of tokens, keys split over workgroups and not
FEW = [((1, 1, 1, 1, 5, 32), (5,)), ((2, 8, 2, 1, 700, 64), (10, 10, 7)), ((1, 4, 4, 3, 4001, 128), (30, 30, 30)),
       ((4, 32, 8, 1, 2500, 128), (16, 16, 10)), ((1, 8, 1, 4, 130, 48), (70, 50)), ((3, 2, 2, 31, 333, 32), (7, 7, 7))]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize(("shape", "extents"), FEW, ids=str)
def test_few_rows(ctmr, dev, shape, extents, dtype):
    n, hq, _, lq, lk, _ = shape
    args = (*_inputs(dev, *shape, dtype), _table(dev, extents, 32, hq, torch.float32), _places(dev, n, lq, extents),
            _places(dev, 0, lk, extents, seed=4))
    _compare(ctmr, *args, extents=extents)
    lengths = torch.randint(0, lk + 1, (n,), generator=torch.Generator().manual_seed(5))
    key_ids = torch.where(torch.arange(lk) < lengths[:, None], 0, -1).int().to(dev)
    ids = torch.zeros(n, lq, dtype=torch.int32, device=dev)
    _compare(ctmr, *args, extents=extents, ids=ids, key_ids=key_ids, softcap=5.0)
    _compare(ctmr, *args, extents=extents, prefix=lk // 2, slopes=torch.rand(hq, device=dev), ids=ids, key_ids=key_ids)


def _rows(dev, n, lengths, total):
    """(n, total) ids of documents side by side, the rest padding; each item's ids turned by one document."""
    out = torch.full((n, total), -1, dtype=torch.int32)
    for b in range(n):
        at = 0
        for i, length in enumerate(lengths[b % len(lengths):] + lengths[:b % len(lengths)]):
            out[b, at:at + length] = i
            at += length
    return out.to(dev)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize(("softcap", "prefix", "slopes", "lengths"),
                         [(0.0, None, False, [100, 3, 190]), (7.0, None, False, None), (400.0, None, False, [320]),
                          (0.0, 0, False, None), (5.0, 70, True, [64, 128, 1]), (0.0, None, True, [1, 1, 1])], ids=str)
@pytest.mark.parametrize("extents", [(9, 8, 7), (50, 40, 30)], ids=str)
def test_masks_caps_and_slopes(ctmr, dev, dtype, softcap, prefix, slopes, lengths, extents):
    n, hq, l = 2, 4, 321
    ids = None if lengths is None else _rows(dev, n, lengths, l)
    _compare(ctmr, *_inputs(dev, n, hq, 2, l, l, 64, dtype), _table(dev, extents, 16, hq, torch.float32),
             _places(dev, 0, l, extents), extents=extents, softcap=softcap, prefix=prefix, ids=ids,
             slopes=0.1 * torch.rand(hq, device=dev) if slopes else None)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d", [32, 120, 128])
@pytest.mark.parametrize(("softcap", "prefix", "lengths"), [(7.0, 40, [100, 29, 64]), (400.0, 0, [130, 71]), (0.0, 150, [90, 110])],
                         ids=str)
def test_masks_and_caps_of_narrow_and_wide_heads(ctmr, dev, dtype, d, softcap, prefix, lengths):
    n, hq, l, extents = 2, 4, 205, (43, 43, 41)
    prefix = torch.tensor([prefix, 3], dtype=torch.int32, device=dev)
    _compare(ctmr, *_inputs(dev, n, hq, 2, l, l, d, dtype), _table(dev, extents, 32, hq, dtype), _places(dev, n, l, extents),
             extents=extents, max_distance=40, softcap=softcap, prefix=prefix, ids=_rows(dev, n, lengths, l))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_long_rows_split_over_workgroups(ctmr, dev, dtype):
    for shape, extents in (((1, 4, 2, 150, 5000, 64), (30, 20, 20)), ((1, 2, 1, 2500, 40, 32), (60, 60))):
        _compare(ctmr, *_inputs(dev, *shape, dtype), _table(dev, extents, 32, shape[1], torch.float32),
                 _places(dev, 0, shape[3], extents), _places(dev, 0, shape[4], extents, seed=4), extents=extents)


@pytest.mark.parametrize("kw", [{}, {"softcap": 2.0}, {"prefix": 20}, {"ids": True}], ids=str)
def test_differences(ctmr, dev, kw):
    f, extents, kw = ctmr.differentiable, (8, 10), dict(kw)
    q, k, v, dout = _inputs(dev, 1, 4, 2, 80, 80, 32, torch.float32)
    table = _table(dev, extents, 8, 4, torch.float32)
    if kw.pop("ids", None):
        kw["documents"] = f.Documents(_rows(dev, 1, [30, 41], 80))
    kw |= {"buckets": f.PositionBuckets(_grid(dev, extents), extents=extents, num_buckets=8, max_distance=7), "scale": 0.3}
    grads = _run(f, q, k, v, table, dout, **kw)[1:]
    h = 1e-2
    for i, g in enumerate(grads):
        u = torch.randn(g.shape, device=dev, generator=torch.Generator(device=dev).manual_seed(40 + i))

        def at(by):
            x = [t + by * h * u if j == i else t for j, t in enumerate((q, k, v, table))]
            return float((f.attention(*x[:3], position_bias=x[3], **kw).double() * dout.double()).sum())

        # cut-off: h^2 / 6 = 1.7e-5 of a third derivative, that of scores that move by 2 or 3 at most below 100 slopes'
        # sizes; noise 10240^(1/2) 2^-24 / h = 6e-4
        slope = (at(1.0) - at(-1.0)) / (2 * h)
        assert abs(slope - float((g.double() * u.double()).sum())) <= 2e-3 * float(g.norm() * u.norm())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_zeros_change_nothing_but_rounding_and_the_bias_moves_weights(ctmr, dev, dtype):
    """A table of one large value gives all weight to the keys of its bucket."""
    f, extents = ctmr.differentiable, (9, 9)
    q, k, v, _ = _inputs(dev, 1, 2, 2, 81, 81, 32, dtype)
    plan = f.PositionBuckets(_grid(dev, extents), extents=extents, num_buckets=16, max_distance=8)
    table = torch.zeros(2, 16, 2, device=dev)
    assert torch.equal(f.attention(q, k, v, scale=0.2, position_bias=table, buckets=plan), f.attention(q, k, v, scale=0.2))
    table[:, 0] = 1000.0  # both distances zero: the voxel itself
    got = f.attention(q, k, v, scale=0.2, position_bias=table, buckets=plan).double()
    # all other weights are below e^-900.  The voxel's own is 2^(s - m) of a score of 2000 log2(e) = 2885 and its maximum m,
    # both rounded to half a step at most: 2 2885 2^-24 ln 2 off one.  fp32 heads divide the same weight out again (a product,
    # a reciprocal and a product of half a step each); 16 bits round it to one first, and the output to their type.
    u, step = 2.0 ** -24, torch.finfo(dtype).eps / 2
    bound = 3 * u + (2 * 2885 * u * math.log(2) + step + 2.0 ** -25 / v.abs().double() if dtype != torch.float32 else 0.0)
    assert bool(((got - v.double()).abs() <= v.double().abs() * bound).all())


@pytest.mark.parametrize("want", [(True, False, False, False), (False, True, False, False), (False, False, False, True),
                                  (True, False, True, True)], ids=str)
def test_gradients_of_some(ctmr, dev, want):
    f, extents = ctmr.differentiable, (10, 12)
    tensors = [*_inputs(dev, 2, 4, 2, 333, 333, 64, torch.bfloat16)]
    dout = tensors.pop()
    tensors.append(_table(dev, extents, 8, 4, torch.bfloat16))
    plan = f.PositionBuckets(_places(dev, 0, 333, extents), extents=extents, num_buckets=8, max_distance=9)
    docs = f.Documents(_rows(dev, 2, [200, 100], 333))
    every = _run(f, *tensors, dout, scale=0.2, buckets=plan, documents=docs)[1:]
    if not want[3]:  # the forward call's weights are rounded once then, and so is delta
        leaves = [t.detach().requires_grad_() for t in tensors[:3]]
        out = f.attention(*leaves, position_bias=tensors[3], scale=0.2, buckets=plan, documents=docs)
        every = (*torch.autograd.grad(out, leaves, dout), None)
    leaves = [t.detach().requires_grad_(w) for t, w in zip(tensors, want)]
    out = f.attention(*leaves[:3], position_bias=leaves[3], scale=0.2, buckets=plan, documents=docs)
    got = torch.autograd.grad(out, [t for t in leaves if t.requires_grad], dout)
    for g, e in zip(got, [e for e, w in zip(every, want) if w]):
        assert torch.equal(g, e)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_a_bias_of_minus_infinity_hides(ctmr, dev, dtype):
    """As a mask would: whole rows among them, in the weights and in the gradients."""
    f, extents = ctmr.differentiable, (11, 13)
    q, k, v, dout = _inputs(dev, 1, 2, 2, 143, 143, 32, dtype)
    places = _grid(dev, extents)
    plan = f.PositionBuckets(places, extents=extents, num_buckets=8, max_distance=6)
    which = oracle.numbers(places, places, extents, 8, 6)
    for least in (-math.inf, torch.finfo(dtype).min if dtype != torch.float16 else -math.inf):
        table = _table(dev, extents, 8, 2, dtype)
        table[1, [0, 4, 5, 6, 7]] = least  # the same column and those to one side: the last column's rows see nothing
        table[1, 1:4] = 0.25
        mask = (which[..., 1] >= 1) & (which[..., 1] < 4)
        finite = torch.where(table > -1e30, table, 0.0)
        want = oracle.attention(q, k, v, finite, which, scale=0.2, mask=mask, dout=dout)
        got = _run(f, q, k, v, table, dout, scale=0.2, buckets=plan)
        empty = ~mask.any(-1)
        assert bool(empty.any()) and bool((got[0].transpose(1, 2)[empty] == 0).all())
        assert bool((got[1].transpose(1, 2)[empty] == 0).all())
        for g, w, name in zip(got, want, ("out", "dq", "dk", "dv", "dtable")):
            attention_oracle.check(g, w, name)


def test_a_bias_that_is_no_number_stays_in_its_reach(ctmr, dev):
    f, extents = ctmr.differentiable, (8, 16)
    q, k, v, dout = _inputs(dev, 1, 2, 2, 128, 128, 32, torch.bfloat16)
    plan = f.PositionBuckets(_grid(dev, extents), extents=extents, num_buckets=32, max_distance=16)
    table = _table(dev, extents, 32, 2, torch.float32)
    clean = f.attention(q, k, v, scale=0.2, position_bias=table, buckets=plan)
    table[1, 16 + 7, 1] = math.nan  # seven to the right, of the second head: rows of the columns up to the ninth
    got = f.attention(q, k, v, scale=0.2, position_bias=table, buckets=plan)
    reach = torch.arange(128, device=dev) % 16 <= 8
    assert torch.equal(got[:, 0], clean[:, 0]) and torch.equal(got[:, 1, ~reach], clean[:, 1, ~reach])
    assert bool(got[:, 1, reach].isnan().all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_what_masked_places_hold_has_no_effect(ctmr, dev, dtype):
    f, extents, l = ctmr.differentiable, (9, 9, 3), 243
    ids = _rows(dev, 1, [100, 60], l)
    plan = f.PositionBuckets(_grid(dev, extents), extents=extents, num_buckets=8, max_distance=7)
    table, results = _table(dev, extents, 8, 4, torch.float32), []
    for fill in (None, math.nan, math.inf, -math.inf):
        q, k, v, dout = _inputs(dev, 1, 4, 2, l, l, 64, dtype)
        if fill is not None:
            for t in (q, k, v, dout):
                t[:, :, 160:] = fill
        results.append(_run(f, q, k, v, table, dout, scale=0.2, buckets=plan, documents=f.Documents(ids)))
    for other in results[1:]:
        assert all(torch.equal(a[:, :, :160], b[:, :, :160]) for a, b in zip(results[0][:4], other[:4]))
        assert torch.equal(results[0][4], other[4])


def test_strided_heads_and_tables(ctmr, dev):
    f, extents, l = ctmr.differentiable, (10, 10), 100
    x = torch.randn(2, l, 3, 4, 32, device=dev, dtype=torch.bfloat16)
    q, k, v = x.permute(2, 0, 3, 1, 4).unbind(0)
    wide = _table(dev, extents, 32, 8, torch.float32)
    table = wide[:, ::2, ::2]
    plan = f.PositionBuckets(_grid(dev, extents), extents=extents, num_buckets=16, max_distance=9)
    args = dict(scale=0.3, buckets=plan)
    got = f.attention(q, k, v, position_bias=table, **args)
    assert torch.equal(got, f.attention(q.contiguous(), k.contiguous(), v.contiguous(), position_bias=table.contiguous(), **args))
    leaf = wide.requires_grad_()
    grad, = torch.autograd.grad(f.attention(q, k, v, position_bias=leaf[:, ::2, ::2], **args).sum(), leaf)
    assert grad.shape == wide.shape and not bool(grad[:, 1::2].any())


def test_same_bits_again_and_copied_places(ctmr, dev):
    f, extents, l = ctmr.differentiable, (16, 16, 8), 2048
    q, k, v, dout = _inputs(dev, 1, 4, 4, l, l, 32, torch.bfloat16)
    places = _grid(dev, extents)
    plan = f.PositionBuckets(places, extents=extents)
    places.fill_(0)
    table = _table(dev, extents, 32, 4, torch.float32)
    first = _run(f, q, k, v, table, dout, scale=0.2, buckets=plan)
    again = f.PositionBuckets(_grid(dev, extents), extents=extents)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, _run(f, q, k, v, table, dout, scale=0.2, buckets=again)))


def test_captured_step_and_another_stream(ctmr, dev):
    f, extents, l = ctmr.differentiable, (12, 11, 5), 660
    q, k, v, dout = _inputs(dev, 1, 4, 4, l, l, 64, torch.bfloat16)
    table = _table(dev, extents, 16, 4, torch.float32)
    places = _grid(dev, extents)

    def step():
        plan = f.PositionBuckets(places, extents=extents, num_buckets=16)
        return _run(f, q, k, v, table, dout, scale=0.125, buckets=plan)

    want = step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = step()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        for t in got:
            t.zero_()
        table.mul_(1.0 + 0.1 * i)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step(), got)), i


def test_a_plan_outlives_its_owner_on_another_stream(ctmr, dev):
    f, extents, l = ctmr.differentiable, (16, 16, 8), 2048
    q, k, v, _ = _inputs(dev, 2, 8, 8, l, l, 64, torch.bfloat16)
    table = _table(dev, extents, 32, 8, torch.float32)
    places = _grid(dev, extents)
    want = f.attention(q, k, v, scale=0.2, position_bias=table, buckets=f.PositionBuckets(places, extents=extents))
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    plan = f.PositionBuckets(places, extents=extents)
    size = plan.plan.numel()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(20):
            got = f.attention(q, k, v, scale=0.2, position_bias=table, buckets=plan)
    del plan
    torch.full((size,), 255, dtype=torch.uint8, device=dev)  # would lie where the plan was
    torch.cuda.synchronize()
    assert torch.equal(got, want)
