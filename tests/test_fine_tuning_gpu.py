"""The operators of a fine-tuning step run together: ``maisi.spatial_attention_volumes`` with a learned position bias, its
gradients, their clipping and ``AdamW``, eager and captured, against the same step in 64 bits."""

from __future__ import annotations

import math

import position_bias_oracle as oracle
import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPES = [(6, 5, 4), (3, 8, 5), (1, 1, 7), (9, 4, 6)]
BUCKETS = dict(num_buckets=8, max_distance=6)


def _weights(dev, c, heads, dtype, seed=3):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=dev, generator=g)
    w = {}
    for n in ("to_q", "to_k", "to_v", "out_proj"):
        w[f"attn.{n}.weight"], w[f"attn.{n}.bias"] = (r(c, c) / math.sqrt(c)).to(dtype), (0.1 * r(c)).to(dtype)
    return w | {"norm.weight": 1 + 0.1 * r(c), "norm.bias": 0.1 * r(c), "attn.position_bias": 0.5 * r(3, 8, heads)}


def _volumes(dev, c, dtype, seed=5):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [torch.randn(*s, c, device=dev, generator=g).to(dtype) for s in SHAPES]


def _block(volumes, w, heads, noise):
    """The block in 64 bits; ``noise`` stands in for the rounding of each intermediate."""
    out = []
    for x in volumes:
        c = x.shape[-1]
        g = x.reshape(-1, 16, c // 16)
        var, mean = torch.var_mean(g, dim=(0, 2), keepdim=True, correction=0)
        t = noise(((g - mean) / torch.sqrt(var + 1e-6)).reshape(-1, c) * w["norm.weight"] + w["norm.bias"])
        lin = lambda t, n: noise(t @ w[f"attn.{n}.weight"].T + w[f"attn.{n}.bias"])
        q, k, v = (lin(t, n).reshape(-1, heads, c // heads).transpose(0, 1) for n in ("to_q", "to_k", "to_v"))
        at = torch.stack(torch.meshgrid(*(torch.arange(s) for s in x.shape[:3]), indexing="ij"), -1).reshape(-1, 3).to(x.device)
        extents = [max(axis) for axis in zip(*SHAPES)]
        which = oracle.numbers(at, at, extents, BUCKETS["num_buckets"], BUCKETS["max_distance"])[0]
        s = q @ k.transpose(1, 2) * (c // heads) ** -0.5
        for a in range(3):
            s = s + w["attn.position_bias"][a][which[..., a]].permute(2, 0, 1)
        merged = noise(noise(torch.softmax(s, -1)) @ v).transpose(0, 1).reshape(-1, c)
        out.append(noise(x + lin(merged, "out_proj").reshape(x.shape)))
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize(("c", "heads"), [(64, 2), (128, 2)])
def test_block_and_its_gradients(ctmr, dev, dtype, c, heads):
    leaves = lambda ts, ws: ([t.detach().clone().requires_grad_() for t in ts],
                             {n: t.detach().clone().requires_grad_() for n, t in ws.items()})
    volumes, w = leaves(_volumes(dev, c, dtype), _weights(dev, c, heads, dtype))
    douts = _volumes(dev, c, dtype, seed=7)
    packed = ctmr.differentiable.PackedVolumes(SHAPES, dev)
    got = ctmr.maisi.spatial_attention_volumes(volumes, w, num_groups=16, eps=1e-6, num_head_channels=c // heads,
                                               include_fc=True, packed=packed, buckets=packed.buckets(**BUCKETS))
    got = [t.detach() for t in got] + list(torch.autograd.grad(got, [*volumes, *w.values()], douts))
    u = torch.finfo(dtype).eps / 2

    def run(noise):
        v, m = leaves([t.double() for t in volumes], {n: t.double() for n, t in w.items()})
        out = _block(v, m, heads, noise)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, [*v, *m.values()], [d.double() for d in douts]))

    torch.manual_seed(0)
    want, off = run(lambda t: t), run(lambda t: t * (1 + u * (2 * torch.rand_like(t) - 1)))
    names = [*(f"out{i}" for i in range(len(SHAPES))), *(f"d{i}" for i in range(len(SHAPES))), *w]
    rows = sum(math.prod(s) for s in SHAPES)
    # The products are summed in fp32, which 16-bit roundings hide: a sum of k terms rounds k - 1 partial sums by half a step
    # each, of either sign, sqrt(k) half steps of the sum's size; the longest sums are over all rows.
    sums = math.sqrt(rows) if dtype == torch.float32 else 1.0
    for name, g, e, o in zip(names, got, want, off):
        # as many independent errors of half a step give the same size; the backward products round as many values again.  Four
        # times it, over a whole tensor, is far outside.  The bias of to_k moves every score of a row alike: its gradient is
        # nothing but the errors, of a size that to_q's bias gradient has, relative to that.
        size = sums * max(float((o - e).norm()), u * float(e.norm()))
        if name == "attn.to_k.bias":
            size = u * math.sqrt(rows) * float(want[names.index("attn.to_q.bias")].norm())
        assert float((g.double() - e).norm()) <= 4 * size + 1e-12, (name, float((g.double() - e).norm()), 4 * size)


def _step(f, maisi, volumes, target, packed, buckets, w, optimizer):
    leaves = {n: t.detach().requires_grad_() for n, t in w.items()}
    out = maisi.spatial_attention_volumes(volumes, leaves, num_groups=16, eps=1e-6, num_head_channels=32, include_fc=True,
                                          packed=packed, buckets=buckets)
    grads = torch.autograd.grad(out, list(leaves.values()), [o.detach() - t for o, t in zip(out, target)])
    return optimizer.step(grads), [o.detach() for o in out]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_captured_steps_are_the_eager_ones(ctmr, dev, dtype):
    """Forward, backward, clipping and update in one graph, replayed with eager work between."""
    f, maisi = ctmr.differentiable, ctmr.maisi
    volumes, target = _volumes(dev, 64, dtype), _volumes(dev, 64, dtype, seed=7)
    packed = f.PackedVolumes(SHAPES, dev)
    buckets = packed.buckets(**BUCKETS)

    def make():
        w = _weights(dev, 64, 2, dtype)
        return w, f.AdamW(list(w.values()), lr=1e-2, max_norm=1.0)

    eager, optimizer = make()
    want = []
    for _ in range(5):
        norm, outs = _step(f, maisi, volumes, target, packed, buckets, eager, optimizer)
        want.append([t.clone() for t in (norm, *outs, *eager.values(), *optimizer.state_dict().values())])
    assert not torch.equal(want[0][0], want[1][0]) and int(optimizer.steps) == 5
    w, optimizer = make()
    first = {n: t.clone() for n, t in w.items()}
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):  # loads every kernel before the capture, on weights of its own
        _step(f, maisi, volumes, target, packed, buckets, *make())
    torch.cuda.current_stream().wait_stream(stream)
    with torch.cuda.graph(graph):
        norm, outs = _step(f, maisi, volumes, target, packed, buckets, w, optimizer)
    for i, expected in enumerate(want):
        graph.replay()
        torch.cuda.synchronize()
        _step(f, maisi, volumes, target, packed, buckets, *make())
        f.clip_gradients([t.clone() for t in volumes], 1.0)
        for a, b in zip((norm, *outs, *w.values(), *optimizer.state_dict().values()), expected):
            assert torch.equal(a, b), i
    assert all(not torch.equal(w[n], t) for n, t in first.items())


def test_two_captured_steps_have_workspaces_of_their_own(ctmr, dev):
    """Two graphs of the same block on other weights, replayed in turn and on streams of their own at once."""
    f, maisi, dtype = ctmr.differentiable, ctmr.maisi, torch.bfloat16
    volumes, target = _volumes(dev, 64, dtype), _volumes(dev, 64, dtype, seed=7)
    packed = f.PackedVolumes(SHAPES, dev)
    buckets = packed.buckets(**BUCKETS)
    make = lambda seed: (w := _weights(dev, 64, 2, dtype, seed=seed), f.AdamW(list(w.values()), lr=1e-2, max_norm=1.0))
    want = []
    for seed in (1, 2):
        w, o = make(seed)
        for _ in range(4):
            _step(f, maisi, volumes, target, packed, buckets, w, o)
        want.append([t.clone() for t in w.values()])
    sides = []
    for seed in (1, 2):
        w, o = make(seed)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _step(f, maisi, volumes, target, packed, buckets, w, o)
        sides.append((graph, w, torch.cuda.Stream()))
    for graph, _, _ in sides * 2:
        graph.replay()
    torch.cuda.synchronize()
    for graph, _, stream in sides * 2:
        with torch.cuda.stream(stream):
            graph.replay()
    torch.cuda.synchronize()
    for (_, w, _), expected in zip(sides, want):
        assert all(torch.equal(a, b) for a, b in zip(w.values(), expected))


def test_a_capture_refuses_a_table_that_an_eager_graph_holds(ctmr, dev):
    f = ctmr.differentiable
    q = torch.randn(1, 2, 60, 32, device=dev)
    plan = f.PositionBuckets(f.PackedVolumes([(3, 4, 5)], dev).positions, extents=(3, 4, 5))
    table = torch.zeros(3, 32, 2, device=dev, requires_grad=True)
    held = f.attention(q, q, q, scale=0.2, position_bias=table, buckets=plan)
    with pytest.raises(RuntimeError, match="outside this capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            f.attention(q, q, q, scale=0.2, position_bias=table, buckets=plan)
    torch.cuda.synchronize()
    assert held.grad_fn is not None
    assert torch.isfinite(f.attention(q, q, q, scale=0.2, position_bias=table, buckets=plan)).all()
