"""Group norm, rotary positions and masked attention run together as ``maisi.spatial_attention_volumes``: values and
gradients against the same block in 64 bits, volumes that do not touch each other, a captured training step."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPES = [(6, 5, 7), (1, 1, 1), (3, 4, 4), (2, 9, 11)]


class _Noise(torch.autograd.Function):
    """The value, and its gradient on the way back, off by up to ``u`` of themselves."""

    @staticmethod
    def forward(ctx, t, u):
        ctx.u = u
        return t + u * t * (2 * torch.rand_like(t) - 1)

    @staticmethod
    def backward(ctx, g):
        return g + ctx.u * g * (2 * torch.rand_like(g) - 1), None


def _block(volumes, w, heads, groups, sections, dtype=None):
    """The block in 64 bits, volume by volume from the formulas.  With ``dtype`` every value that a run in this type
    stores, and every gradient of one, is off by up to half a step; fp32 takes the square root of the terms of a sum
    (the channels) as its steps, since its sums round as often."""
    c = volumes[0].shape[-1]
    if dtype is None:
        noise = lambda t: t
    else:
        u = 2.0 ** -24 * math.sqrt(c) if dtype == torch.float32 else torch.finfo(dtype).eps / 2
        noise = lambda t: _Noise.apply(t, u)
    lin = lambda t, name: noise(t @ noise(w[f"attn.{name}.weight"]).T + noise(w[f"attn.{name}.bias"]))
    out = []
    for x in volumes:
        x = noise(x)
        g = x.reshape(-1, groups, c // groups)
        var, mean = torch.var_mean(g, dim=(0, 2), keepdim=True, correction=0)
        h = noise(((g - mean) / torch.sqrt(var + 1e-6)).reshape(-1, c) * noise(w["norm.weight"]) + noise(w["norm.bias"]))
        q, k, v = (lin(h, n).reshape(-1, heads, c // heads).transpose(0, 1) for n in ("to_q", "to_k", "to_v"))
        if sections is not None:
            at = torch.cartesian_prod(*(torch.arange(s, device=x.device) for s in x.shape[:3])).double()
            turned = []
            for t in (q, k):
                parts, start = [], 0
                for axis, width in enumerate(sections):
                    angle = at[:, axis, None] * 1e4 ** (torch.arange(0, width, 2, device=x.device).double() / -width)
                    a, b = t[..., start:start + width].chunk(2, -1)
                    parts += [a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()]
                    start += width
                turned.append(noise(torch.cat([*parts, t[..., start:]], -1)))
            q, k = turned
        s = noise(q @ k.transpose(1, 2)) * (c // heads) ** -0.5
        merged = noise(noise(torch.softmax(s, -1)) @ v).transpose(0, 1).reshape(-1, c)
        out.append(noise(x + lin(merged, "out_proj").reshape(x.shape)))
    return out


def _weights(dev, c, dtype, seed=3):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=dev, generator=g)
    w = {}
    for n in ("to_q", "to_k", "to_v", "out_proj"):
        w[f"attn.{n}.weight"], w[f"attn.{n}.bias"] = (r(c, c) / math.sqrt(c)).to(dtype), (0.1 * r(c)).to(dtype)
    return w | {"norm.weight": 1 + 0.1 * r(c), "norm.bias": 0.1 * r(c)}


def _volumes(dev, shapes, c, dtype, seed=5):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [torch.randn(*s, c, device=dev, generator=g).to(dtype) for s in shapes]


def _leaves(volumes, w):
    return [t.detach().clone().requires_grad_() for t in volumes], {n: t.detach().clone().requires_grad_() for n, t in w.items()}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize(("c", "width", "sections"), [(64, 32, (8, 12, 12)), (128, 64, (20, 20, 20)), (96, 24, None)])
def test_block_and_its_gradients(ctmr, dev, dtype, c, width, sections):
    volumes, w = _leaves(_volumes(dev, SHAPES, c, dtype), _weights(dev, c, dtype))
    douts = _volumes(dev, SHAPES, c, dtype, seed=7)
    packed = ctmr.differentiable.PackedVolumes(SHAPES, dev)
    got = ctmr.maisi.spatial_attention_volumes(volumes, w, num_groups=16, eps=1e-6, num_head_channels=width, include_fc=True,
                                               packed=packed, sections=sections)
    got = [t.detach() for t in got] + list(torch.autograd.grad(got, [*volumes, *w.values()], douts))

    def run(kind):
        v, m = _leaves([t.double() for t in volumes], {n: t.double() for n, t in w.items()})
        out = _block(v, m, c // width, 16, sections, kind)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, [*v, *m.values()], [d.double() for d in douts]))

    torch.manual_seed(0)
    want, off = run(None), run(dtype)
    names = [*(f"out{i}" for i in range(len(SHAPES))), *(f"d{i}" for i in range(len(SHAPES))), *w]
    for name, g, e, o in zip(names, got, want, off):
        # the same count of independent errors gives the same size; four times it, over a whole tensor, is far outside.
        # The bias of to_k moves every score of a row alike, so its gradient is nothing but the errors.
        bound = 4 * float((o - e).norm()) + 1e-12
        assert float((g.double() - e).norm()) <= bound, (name, float((g.double() - e).norm()), bound)


def test_fp16_without_gradients_and_one_volume(ctmr, dev):
    args = dict(num_groups=16, eps=1e-6, num_head_channels=32, include_fc=True, sections=(8, 12, 12))
    w = _weights(dev, 64, torch.float16)
    volumes = _volumes(dev, SHAPES, 64, torch.float16)
    with torch.no_grad():
        got = ctmr.maisi.spatial_attention_volumes(volumes, w, **args)
        alone = [ctmr.maisi.spatial_attention_volumes([v], w, **args)[0] for v in volumes]
    torch.manual_seed(0)
    exact = [t.double() for t in volumes], {n: t.double() for n, t in w.items()}
    want, off = _block(*exact, 2, 16, (8, 12, 12)), _block(*exact, 2, 16, (8, 12, 12), torch.float16)
    for g, a, e, o in zip(got, alone, want, off):
        assert g.dtype == torch.float16
        assert float((g.double() - e).norm()) <= 4 * float((o - e).norm())
        assert float((a.double() - e).norm()) <= 4 * float((o - e).norm())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_volumes_do_not_touch_each_other(ctmr, dev, dtype):
    w, douts = _weights(dev, 64, dtype), _volumes(dev, SHAPES, 64, dtype, seed=7)
    results = []
    for fill in (None, math.nan):
        volumes, m = _leaves(_volumes(dev, SHAPES, 64, dtype), w)
        if fill is not None:
            with torch.no_grad():
                volumes[2].fill_(fill)
        out = ctmr.maisi.spatial_attention_volumes(volumes, m, num_groups=16, eps=1e-6, num_head_channels=32,
                                                   include_fc=True, sections=(8, 12, 12))
        results.append(([t.detach() for t in out], torch.autograd.grad(out, volumes, douts)))
    for clean, other in zip(*results):
        for i in (0, 1, 3):
            assert torch.equal(clean[i], other[i]), i
    assert bool(results[1][0][2].isnan().all())


def test_captured_training_step(ctmr, dev):
    """Forward, backward and an update in one graph, replayed with eager work between, against the eager steps."""
    dtype = torch.bfloat16
    first, x = _weights(dev, 64, dtype), _volumes(dev, SHAPES, 64, dtype)
    target = _volumes(dev, SHAPES, 64, dtype, seed=7)
    packed = ctmr.differentiable.PackedVolumes(SHAPES, dev)

    def step(w):
        leaves = {n: t.detach().requires_grad_() for n, t in w.items()}
        out = ctmr.maisi.spatial_attention_volumes(x, leaves, num_groups=16, eps=1e-6, num_head_channels=32, include_fc=True,
                                                   packed=packed, sections=(8, 12, 12))
        grads = torch.autograd.grad(out, list(leaves.values()), [o.detach() - t for o, t in zip(out, target)])
        for t, g in zip(w.values(), grads):
            t.sub_(g, alpha=1e-4)

    eager = {n: t.clone() for n, t in first.items()}
    steps = []
    for _ in range(4):
        step(eager)
        steps.append({n: t.clone() for n, t in eager.items()})
    w = {n: t.clone() for n, t in first.items()}
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(w)  # loads every kernel before the capture
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(w)
    for want in steps[1:]:
        graph.replay()
        torch.cuda.synchronize()
        ctmr.maisi.spatial_attention_volumes(x, first, num_groups=16, eps=1e-6, num_head_channels=32, include_fc=True)
        for n in w:
            assert torch.equal(w[n], want[n]), n
