"""``gradient_norm``, ``clip_gradients`` and ``AdamW`` against 64 bits: types, odd sizes and addresses, more tensors than a
launch takes, ends of the range, what is not finite, skipped steps, graphs and streams."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24  # half a step of fp32
SIZES = [(1,), (3,), (4097,), (64, 65), (0,), (255,), (4096,), (7, 11, 13), (1 << 14,), (12289,)]


def _list(dev, sizes, dtype, seed=0, scale=1.0, offset=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    out = []
    for s in sizes:
        n = math.prod(s)
        row = (scale * torch.randn(n + offset, device=dev, generator=g)).to(dtype)
        out.append(row[offset:].view(s))
    return out


def _norm(tensors, scale=1.0):
    return math.sqrt(sum(float((scale * t.double()).square().sum()) for t in tensors))


def _least(dtype):
    """Half of the least step that a type's values have."""
    return {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}[dtype]


def _check_norm(got, want):
    # fp64 sums of up to 2^20 terms (2^-53 each, of either sign) and one rounding to fp32
    assert abs(float(got) - want) <= (U + 2.0 ** -40) * want, (float(got), want)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_norm_and_clipping(ctmr, dev, dtype, offset):
    f = ctmr.differentiable
    grads = _list(dev, SIZES, dtype, offset=offset)
    want = _norm(grads)
    norm = f.gradient_norm([None, *grads])
    assert norm.shape == () and norm.dtype == torch.float32
    _check_norm(norm, want)
    before = [t.double() for t in grads]
    got = f.clip_gradients(grads, 2.0)
    assert torch.equal(got, norm)
    factor = 2.0 / (want + 1e-6)
    u = torch.finfo(dtype).eps / 2
    for b, t in zip(before, grads):
        # the norm, its sum with 1e-6 and the quotient, half a step each; the product, of fp32, and its rounding
        bound = (b * factor).abs() * (4 * U + u * (dtype != torch.float32) + U) + _least(dtype)
        assert bool(((t.double() - b * factor).abs() <= bound).all())


def test_neighbours_of_views_are_left_alone(ctmr, dev):
    flat = torch.ones(1000, device=dev, dtype=torch.bfloat16)
    ctmr.differentiable.clip_gradients([flat[5:98], flat[99:700]], 1e-3)
    kept = torch.cat([flat[:5], flat[98:99], flat[700:]])
    assert bool((kept == 1).all()) and float(flat[5:98].max()) < 1e-3 and float(flat[99:700].max()) < 1e-3


def test_small_norms_are_left_as_they_are(ctmr, dev):
    grads = _list(dev, SIZES, torch.float16, scale=1e-4)
    before = [t.clone() for t in grads]
    ctmr.differentiable.clip_gradients(grads, 1.0)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    ctmr.differentiable.clip_gradients(grads, math.inf)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))


@pytest.mark.parametrize("count", [1, 159, 160, 161, 500])
def test_more_tensors_than_a_launch_takes(ctmr, dev, count):
    g = torch.Generator().manual_seed(count)
    sizes = [(int(torch.randint(0, 300, (), generator=g)),) for _ in range(count - 1)] + [(9000,)]
    kinds = [TYPES[i % 3] for i in range(count)]
    grads = [_list(dev, [s], k, seed=i)[0] for i, (s, k) in enumerate(zip(sizes, kinds))]
    want, before = _norm(grads), [t.double() for t in grads]
    _check_norm(ctmr.differentiable.clip_gradients(grads, 1.0), want)
    for b, t in zip(before, grads):
        assert bool(((t.double() - b / want).abs() <= (b / want).abs() * (1e-5 + torch.finfo(t.dtype).eps / 2)
                     + _least(t.dtype)).all())


def test_many_values(ctmr, dev):
    grads = _list(dev, [(5000, 7001), (1 << 22,), (3,)], torch.bfloat16)
    _check_norm(ctmr.differentiable.gradient_norm(grads), _norm(grads))


@pytest.mark.parametrize(("dtype", "scale"), [(torch.float32, 1e30), (torch.float32, 1e-30), (torch.bfloat16, 1e30),
                                              (torch.bfloat16, 1e-30), (torch.float16, 1e-6)], ids=str)
def test_squares_past_the_range_of_fp32(ctmr, dev, dtype, scale):
    grads = _list(dev, [(1000,), (33,)], dtype, scale=scale)
    _check_norm(ctmr.differentiable.gradient_norm(grads), _norm(grads))


def test_other_layouts(ctmr, dev):
    f = ctmr.differentiable
    base = torch.randn(6, 10, device=dev)
    grads = [base.t(), torch.randn(4, 3, 2, device=dev).permute(2, 0, 1), torch.randn(3, device=dev).expand(5, 3),
             torch.randn(8, 8, device=dev)[:, ::2], torch.randn((), device=dev)]
    _check_norm(f.gradient_norm(grads), _norm(grads))
    want = _norm(grads[:2])
    before = [t.clone() for t in grads[:2]]
    _check_norm(f.clip_gradients(grads[:2], 0.5), want)
    assert all(torch.allclose(t, b * (0.5 / want), rtol=1e-6, atol=0) for t, b in zip(grads, before))


def test_what_is_not_finite(ctmr, dev):
    f = ctmr.differentiable
    t = torch.ones(3000, device=dev)
    t[7] = math.inf
    assert f.clip_gradients([t], 1.0) == math.inf
    assert bool(t[7].isnan()) and bool((t[:7] == 0).all()) and bool((t[8:] == 0).all())
    t = torch.ones(3000, device=dev, dtype=torch.float16)
    t[2999] = math.nan
    assert bool(f.clip_gradients([t, torch.ones(5, device=dev)], 1.0).isnan()) and bool(t.isnan().all())


def test_without_a_limit_what_is_not_finite_stays_where_it_is(ctmr, dev):
    f = ctmr.differentiable
    t = torch.ones(3000, device=dev)
    t[7], t[8] = math.inf, math.nan
    kept = t.clone()
    assert bool(f.clip_gradients([t], math.inf).isnan()) and torch.equal(t.nan_to_num(9.0), kept.nan_to_num(9.0))
    p = torch.zeros(3000, device=dev)
    o = f.AdamW([p], lr=0.5, weight_decay=0.0)
    o.step([t], gradient_scale=2.0)
    # every finite gradient moves its value by the rate, to the roundings of a step and eps 1e-8
    assert bool(((p[9:] + 0.5).abs() < 1e-6).all()) and bool(((p[:7] + 0.5).abs() < 1e-6).all())
    assert bool(p[7:9].isnan().all())


def test_same_bits_again(ctmr, dev):
    grads = _list(dev, [(300001,), (777,)], torch.float32)
    first = ctmr.differentiable.gradient_norm(grads)
    assert all(torch.equal(first, ctmr.differentiable.gradient_norm(grads)) for _ in range(5))


# ---------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------
def _step(p, g, m, v, w, t, factor, lr, betas, eps, decay):
    """One step in 64 bits: (value, bound) of the moments, the copy and the parameter."""
    b1, b2 = betas
    g = g.double() * factor
    m0, v0 = b1 * m.double(), b2 * v.double()
    m1, v1 = m0 + (1 - b1) * g, v0 + (1 - b2) * g * g
    # in half steps: the factor 4 and its product 1; a beta and its product 2 (1 - beta as well); the sum 1
    em = U * (2 * m0.abs() + 7 * ((1 - b1) * g).abs() + m1.abs()) + 2.0 ** -149
    ev = U * (2 * v0 + 13 * (1 - b2) * g * g + v1) + 2.0 ** -149
    by = (v1 / (1 - b2 ** t)).sqrt() + eps
    # sqrt: half of v's error and its own step, the correction 1, the sum with eps 2
    eby = (ev / (1 - b2 ** t)).sqrt().clamp(max=1e300).minimum(0.5 * ev / v1.clamp(min=1e-300) * by) + 5 * U * by
    rate = lr / (1 - b1 ** t)
    move = rate * m1 / by
    emove = rate * em / by + move.abs() * (eby / by + 4 * U)
    w1 = w.double() - (lr * decay * w.double() + move)
    ew = emove + 3 * U * (lr * decay * w.double()).abs() + U * (lr * decay * w.double() + move).abs() + U * w1.abs() + 2.0 ** -149
    u = torch.finfo(p.dtype).eps / 2
    ep = ew + (u * w1.abs() + _least(p.dtype) if p.dtype != torch.float32 else 0.0)
    return (m1, em), (v1, ev), (w1, ew), (w1, ep)


def _inside(got, want, name):
    value, bound = want
    err = (got.double().reshape(-1) - value.reshape(-1)).abs()
    assert bool((err <= 1.01 * bound.reshape(-1)).all()), (name, float((err / bound.reshape(-1)).max()))


def _state(o, i):
    p = o.parameters[i]
    n, at, m = p.numel(), o._starts[i], o._master_starts[i]
    w = p.flatten() if p.dtype == torch.float32 else o.master[m:m + n]
    return o.exp_avg[at:at + n].clone(), o.exp_avg_sq[at:at + n].clone(), w.clone()


@pytest.mark.parametrize("kinds", [[torch.float32], [torch.bfloat16], [torch.float16], TYPES], ids=str)
@pytest.mark.parametrize(("max_norm", "offset"), [(None, 0), (0.7, 1)])
def test_steps(ctmr, dev, kinds, max_norm, offset):
    f = ctmr.differentiable
    params = [_list(dev, [s], kinds[i % len(kinds)], seed=i, scale=0.1, offset=offset)[0] for i, s in enumerate(SIZES)]
    args = dict(lr=3e-3, betas=(0.8, 0.95), eps=1e-7, weight_decay=0.1)
    o = f.AdamW(params, max_norm=max_norm, **args)
    for t in range(1, 4):
        grads = [_list(dev, [p.shape], p.dtype, seed=100 * t + i, scale=0.02, offset=(t + i) % 3)[0]
                 for i, p in enumerate(params)]
        scale = 0.5 if t == 2 else 1.0
        want = _norm(grads, scale)
        factor = scale * (1.0 if max_norm is None else min(1.0, max_norm / (want + 1e-6)))
        assert max_norm is None or want > max_norm
        before = [(*_state(o, i), p.clone()) for i, p in enumerate(params)]
        _check_norm(o.step(grads, gradient_scale=scale), want)
        assert int(o.steps) == t
        for i, (p, g, (m, v, w, _)) in enumerate(zip(params, grads, before)):
            bounds = _step(p, g.flatten(), m, v, w, t, factor, args["lr"], args["betas"], args["eps"], args["weight_decay"])
            for name, got, b in zip(("m", "v", "w", "p"), (*_state(o, i), p), bounds):
                _inside(got, b, (i, name, t))


def test_the_library_optimizer_agrees(ctmr, dev):
    """Steps with clipping against torch's own, in fp32 and over more parameters than a launch takes."""
    sizes = [((i * 37) % 90 + 1, (i * 11) % 30 + 1) for i in range(170)]
    ours = [torch.nn.Parameter(t) for t in _list(dev, sizes, torch.float32, scale=0.1)]
    theirs = [torch.nn.Parameter(t.detach().double()) for t in ours]
    o = ctmr.differentiable.AdamW(ours, lr=1e-2, weight_decay=0.05, max_norm=1.0)
    r = torch.optim.AdamW(theirs, lr=1e-2, weight_decay=0.05)
    for t in range(5):
        grads = _list(dev, sizes, torch.float32, seed=t + 1)
        o.step(grads)
        for p, g in zip(theirs, grads):
            p.grad = g.double()
        torch.nn.utils.clip_grad_norm_(theirs, 1.0)
        r.step()
    for a, b in zip(ours, theirs):
        # five steps, each with the roundings counted in _step: at most some ten half steps of what a step moves (about
        # the rate each) and one of the value
        assert bool(((a.double() - b).abs() <= 5 * (12 * U * 5e-2 + U * (b.abs() + 0.1))).all())


def test_small_steps_of_16_bits_are_not_lost(ctmr, dev):
    p = torch.ones(100, device=dev, dtype=torch.bfloat16)
    o = ctmr.differentiable.AdamW([p], lr=1e-4, weight_decay=0.0)
    for _ in range(100):
        o.step([torch.ones_like(p)])
    assert bool((p == torch.tensor(0.99, dtype=torch.bfloat16)).all())


def test_none_keeps_a_parameter_and_its_moments(ctmr, dev):
    params = _list(dev, [(100,), (50,), (70,)], torch.bfloat16)
    o = ctmr.differentiable.AdamW(params)
    kept = params[1].clone()
    o.step([torch.ones_like(params[0]), None, torch.ones_like(params[2])])
    assert torch.equal(params[1], kept) and not bool(o.exp_avg[128:192].any()) and bool(o.exp_avg[192:262].all())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_steps_that_are_skipped(ctmr, dev, bad):
    params = _list(dev, [(5000,), (50,)], torch.float16)
    grads = _list(dev, [(5000,), (50,)], torch.float16, seed=1)
    o = ctmr.differentiable.AdamW(params, max_norm=1.0, skip_non_finite=True)
    o.step(grads)
    before = [t.clone() for t in (*params, *o.state_dict().values())]
    grads[1][3] = bad
    norm = o.step(grads)
    assert not math.isfinite(float(norm))
    assert all(torch.equal(a, b) for a, b in zip(before, (*params, *o.state_dict().values())))
    grads[1][3] = 0
    o.step(grads)
    assert int(o.steps) == 2 and not torch.equal(params[0], before[0])


def test_changes_are_seen_by_autograd(ctmr, dev):
    p = torch.nn.Parameter(torch.ones(4, device=dev))
    y = (p * p).sum()
    ctmr.differentiable.AdamW([p]).step([torch.ones_like(p)])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    g = torch.ones(4, device=dev)
    z = (torch.ones(4, device=dev, requires_grad=True) * g).sum()
    ctmr.differentiable.clip_gradients([g], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_captured_steps(ctmr, dev):
    """A step with a rate on the device and its clipping in one graph, replayed with eager work between."""
    f = ctmr.differentiable

    def make():
        params = _list(dev, [(3001,), (64, 64)], torch.bfloat16)
        lr = torch.tensor(1e-3, device=dev)
        return params, lr, f.AdamW(params, lr=lr, max_norm=0.5)

    batches = [_list(dev, [(3001,), (64, 64)], torch.bfloat16, seed=s) for s in range(1, 6)]
    params, lr, o = make()
    want = []
    for i, grads in enumerate(batches):
        lr.fill_(1e-3 / (i + 1))
        norm = o.step(grads)
        clipped = [t.clone() for t in grads]
        f.clip_gradients(clipped, 0.25)
        want.append([t.clone() for t in (norm, *params, *o.state_dict().values(), *clipped)])
    params, lr, o = make()
    grads = [t.clone() for t in batches[0]]
    clipped = [t.clone() for t in grads]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = o.step(grads)
        f.clip_gradients(clipped, 0.25)
    for i, batch in enumerate(batches):
        for t, c, b in zip(grads, clipped, batch):
            t.copy_(b)
            c.copy_(b)
        lr.fill_(1e-3 / (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        f.gradient_norm(batch)
        for a, b in zip((norm, *params, *o.state_dict().values(), *clipped), want[i]):
            assert torch.equal(a, b), i


def test_on_another_stream(ctmr, dev):
    f = ctmr.differentiable
    grads = _list(dev, [(200001,)], torch.float32)
    want = [f.gradient_norm(grads)]
    clipped = [t.clone() for t in grads]
    f.clip_gradients(clipped, 1.0)
    other = [t.clone() for t in grads]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = f.clip_gradients(other, 1.0)
        o = f.AdamW([other[0].clone()])
        o.step(clipped)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want[0]) and torch.equal(other[0], clipped[0]) and int(o.steps) == 1
