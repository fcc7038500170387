"""``differentiable.group_norm`` and its gradients against 64 bits: types, ragged shapes, channel counts that
no vector divides, both forms of the kernels, strides, graphs and streams."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24  # half a step of fp32


def _inputs(dev, shape, groups, dtype, ptype, seed=0, mean=0.3):
    g = torch.Generator(device=dev).manual_seed(seed)
    c = shape[-1]
    r = lambda *s: torch.randn(*s, device=dev, generator=g)
    x = (r(*shape) * torch.exp(0.4 * r(c)) + mean * r(c)).to(dtype)
    return x, (1 + 0.2 * r(c)).to(ptype), (0.2 * r(c)).to(ptype), r(*shape).to(dtype)


def _exact(x, w, b, dy, groups, eps, silu):
    """(y, dx, dw, db) in 64 bits by autograd, and the quantities that the tolerances count."""
    leaves = [t.detach().double().requires_grad_() for t in (x, w, b)]
    xd, wd, bd = leaves
    n, c = x.shape[0], x.shape[-1]
    g = xd.reshape(n, -1, groups, c // groups)
    var, mean = torch.var_mean(g, dim=(1, 3), keepdim=True, correction=0)
    rstd = 1 / torch.sqrt(var + eps)
    xhat = ((g - mean) * rstd).reshape(x.shape)
    z = xhat * wd + bd
    y = z * torch.sigmoid(z) if silu else z
    grads = torch.autograd.grad(y, leaves, dy.double())
    full = rstd.expand_as(g).reshape(x.shape)
    return y.detach(), grads, xhat.detach(), z.detach(), full.detach()


def _check(y, grads, x, w, b, dy, groups, eps, silu):
    ref, (rx, rw, rb), xhat, z, rstd = _exact(x, w, b, dy, groups, eps, silu)
    half = torch.finfo(x.dtype).eps / 2
    wd = w.double()
    # z: four fp32 roundings of gamma xhat (difference, low mean, rstd, product) and one of the sum; SiLU
    # has a slope below 1.1 and the hardware's exponential and reciprocal are within 1e-6
    ez = 5 * U * (wd * xhat).abs() + 2 * U * z.abs() + U
    tol = half * ref.abs() + 1.1 * ez + 1e-6 * ref.abs()
    if x.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half a step below the normal range
    assert bool(((y.double() - ref).abs() <= tol).all())
    if grads is None:
        return
    # dz = dy silu'(z): sigmoid to 1e-6 (1 + |z|) relative, and silu'' below 0.5 of an error in z
    edz = dy.double().abs() * ((1e-6 * (1 + z.abs()) + 0.5 * ez) if silu else U)
    dz_abs = dy.double().abs() * 1.1
    n, c = x.shape[0], x.shape[-1]
    over = tuple(range(x.dim() - 1))
    group_mean = lambda t: t.reshape(n, -1, groups, c // groups).mean((1, 3), keepdim=True).expand(
        n, t.numel() // n // c, groups, c // groups).reshape(x.shape)
    exh = 4 * U * xhat.abs()
    # sums over voxels: up to 32 terms are added in fp32 before they join an fp64 sum, at most 31 roundings of partial
    # sums that the terms' sizes bound, and one of each product
    batch = 32 * U
    ea = group_mean(wd.abs() * (edz + batch * dz_abs))
    eb = group_mean(wd.abs() * (edz * xhat.abs() + dz_abs * exh + batch * dz_abs * xhat.abs()))
    a, bb = group_mean((wd.abs() * dz_abs)), group_mean(wd.abs() * dz_abs * xhat.abs())
    tol = half * rx.abs() + rstd * (wd.abs() * edz + ea + eb * xhat.abs() + bb * exh
                                    + 6 * U * (wd.abs() * dz_abs + a + bb * xhat.abs()))
    if x.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    assert bool(((grads[0].double() - rx).abs() <= tol).all())
    half = torch.finfo(w.dtype).eps / 2
    assert bool(((grads[2].double() - rb).abs() <= (edz + batch * dz_abs).sum(over) + half * rb.abs() + U).all())
    assert bool(((grads[1].double() - rw).abs() <= (edz * xhat.abs() + dz_abs * exh + batch * dz_abs * xhat.abs()).sum(over) + half * rw.abs() + U).all())


# (shape, groups): one voxel; ragged; channel counts that 8, 4 and 2 do not divide; one channel a group; one group;
# more channel vectors than threads; the chunked form with ragged chunks; many items
SHAPES = [((1, 1, 32), 4), ((2, 3, 5, 7, 64), 32), ((1, 11, 13, 9, 36), 6), ((2, 17, 35), 5), ((3, 6, 10), 2),
          ((1, 300, 24), 24), ((2, 50, 40), 1), ((1, 9, 2600), 8), ((1, 45, 31, 29, 128), 32), ((2, 20011, 96), 32),
          ((1, 30001, 35), 7), ((70, 4, 64), 16), ((2, 16, 16, 8, 512), 32), ((1, 40000, 6), 3)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape,groups", SHAPES, ids=str)
@pytest.mark.parametrize("silu", [True, False])
def test_values_and_gradients(ctmr, dev, shape, groups, dtype, silu):
    f = ctmr.differentiable
    ptype = dtype if groups % 2 else torch.float32
    x, w, b, dy = _inputs(dev, shape, groups, dtype, ptype)
    for t in (x, w, b):
        t.requires_grad_()
    y = f.group_norm(x, w, b, num_groups=groups, eps=1e-6, apply_silu=silu)
    assert y.dtype == dtype and y.shape == x.shape
    grads = torch.autograd.grad(y, (x, w, b), dy)
    assert [g.dtype for g in grads] == [dtype, ptype, ptype]
    _check(y.detach(), grads, x, w, b, dy, groups, 1e-6, silu)
    with torch.no_grad():
        assert torch.equal(f.group_norm(x, w, b, num_groups=groups, eps=1e-6, apply_silu=silu), y)


@pytest.mark.parametrize("rows", [200, 30000])
def test_mean_far_above_the_spread(ctmr, dev, rows):
    """A mean of 1000 spreads: fp32 sums of squares would keep one digit of the variance."""
    f = ctmr.differentiable
    x, w, b, dy = _inputs(dev, (1, rows, 32), 4, torch.float32, torch.float32, mean=0.0)
    x = (x + 1000.0).requires_grad_()
    y = f.group_norm(x, w, b, num_groups=4, eps=1e-6, apply_silu=True)
    _check(y.detach(), None, x, w, b, dy, 4, 1e-6, True)


def test_constant_group_has_no_nan(ctmr, dev):
    x = torch.full((1, 64, 8), 3.0, device=dev, requires_grad=True)
    w, b = torch.ones(8, device=dev), torch.zeros(8, device=dev)
    y = ctmr.differentiable.group_norm(x, w, b, num_groups=2, eps=1e-6)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert bool((y == 0).all()) and bool((dx == 0).all())


@pytest.mark.parametrize("rows", [256, 40000])
def test_nan_stays_in_its_group(ctmr, dev, rows):
    f = ctmr.differentiable
    x, w, b, _ = _inputs(dev, (2, rows, 64), 8, torch.bfloat16, torch.float32)
    clean = f.group_norm(x, w, b, num_groups=8, eps=1e-6, apply_silu=True)
    x[1, rows // 2, 17] = math.nan
    y = f.group_norm(x, w, b, num_groups=8, eps=1e-6, apply_silu=True)
    assert bool(y[1, :, 16:24].isnan().all())
    y[1, :, 16:24] = clean[1, :, 16:24]
    assert torch.equal(y, clean)


def test_strides_offsets_and_odd_addresses(ctmr, dev):
    f = ctmr.differentiable
    for dtype in TYPES:
        x, w, b, dy = _inputs(dev, (2, 33, 64), 8, dtype, torch.float32)
        flat = torch.zeros(x.numel() + 1, device=dev, dtype=dtype)
        odd = flat[1:].view(x.shape)  # an address that no vector divides
        odd.copy_(x)
        spread = torch.zeros(2, 64, 33, device=dev, dtype=dtype).transpose(1, 2)
        spread.copy_(x)
        want = None
        for t in (x, odd, spread):
            t = t.detach().requires_grad_()
            y = f.group_norm(t, w, b, num_groups=8, eps=1e-6, apply_silu=True)
            grad, = torch.autograd.grad(y, t, dy.transpose(1, 2).contiguous().transpose(1, 2))
            _check(y.detach(), None, x, w, b, dy, 8, 1e-6, True)
            if want is not None:
                # the vector width moves the sums' order by an fp64 rounding only
                assert bool(((grad.double() - want.double()).abs() <= torch.finfo(dtype).eps * want.double().abs()
                             + 1e-6).all())
            want = grad


def test_only_the_wanted_gradients(ctmr, dev):
    f = ctmr.differentiable
    for rows in (64, 40000):
        x, w, b, dy = _inputs(dev, (2, rows, 64), 8, torch.bfloat16, torch.float32)
        run = lambda *leaves: torch.autograd.grad(
            f.group_norm(x, w, b, num_groups=8, eps=1e-6, apply_silu=True), leaves, dy)
        for t in (x, w, b):
            t.requires_grad_()
        every = run(x, w, b)
        for i, t in enumerate((x, w, b)):
            for o in (x, w, b):
                o.requires_grad_(o is t)
            assert torch.equal(run(t)[0], every[i])


def test_broadcast_input_and_shared_weight(ctmr, dev):
    """Gradients of an expanded input and of a weight used twice add up as autograd's do."""
    f = ctmr.differentiable
    x, w, b, _ = _inputs(dev, (1, 40, 32), 4, torch.float32, torch.float32)
    x, w = x.requires_grad_(), w.requires_grad_()
    wide = x.expand(3, 40, 32)
    y = f.group_norm(wide, w, b, num_groups=4, eps=1e-6, apply_silu=True)
    y = f.group_norm(y, w, b, num_groups=4, eps=1e-6)
    dy = torch.randn(y.shape, device=dev, generator=torch.Generator(device=dev).manual_seed(3))
    got = torch.autograd.grad(y, (x, w), dy)
    xd, wd = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()

    def norm(t, silu):
        g = t.reshape(3, 40, 4, 8)
        var, mean = torch.var_mean(g, dim=(1, 3), keepdim=True, correction=0)
        z = ((g - mean) / torch.sqrt(var + 1e-6)).reshape(t.shape) * wd + b.double()
        return z * torch.sigmoid(z) if silu else z

    want = torch.autograd.grad(norm(norm(xd.expand(3, 40, 32), True), False), (xd, wd), dy.double())
    # two norms in fp32: their errors of some 1e-6 relative to the gradients' scale, 3 x 40 terms a weight
    for g, r in zip(got, want):
        assert float((g.double() - r).abs().max()) <= 2e-5 * float(r.abs().max())


def test_differences(ctmr, dev):
    f = ctmr.differentiable
    x, w, b, dy = _inputs(dev, (2, 65, 48), 6, torch.float32, torch.float32)
    run = lambda *t: f.group_norm(*t, num_groups=6, eps=1e-6, apply_silu=True)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(run(*leaves), leaves, dy)
    h = 1e-2
    for i, g in enumerate(grads):
        u = torch.randn(g.shape, device=dev, generator=torch.Generator(device=dev).manual_seed(7 + i))
        at = lambda s: float((run(*[t + s * h * u if j == i else t for j, t in enumerate((x, w, b))]).double()
                              * dy.double()).sum())
        slope = (at(1.0) - at(-1.0)) / (2 * h)
        # cut-off h^2 / 6 of a third derivative that is a few times the values' scale; noise 6240^(1/2) U / h
        assert abs(slope - float((g.double() * u.double()).sum())) <= 1e-3 * float(g.norm() * u.norm())


@pytest.mark.parametrize("rows", [128, 40000])
def test_repeats_streams_and_graph(ctmr, dev, rows):
    f = ctmr.differentiable
    x, w, b, dy = _inputs(dev, (2, rows, 64), 8, torch.bfloat16, torch.float32)

    def step(x, w, b, dy):
        x, w, b = (t.detach().requires_grad_() for t in (x, w, b))
        y = f.group_norm(x, w, b, num_groups=8, eps=1e-6, apply_silu=True)
        return [t.detach() for t in (y, *torch.autograd.grad(y, (x, w, b), dy))]

    want = step(x, w, b, dy)
    assert all(torch.equal(a, c) for a, c in zip(want, step(x, w, b, dy)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step(x, w, b, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(want, again))
    static = [t.clone() for t in (x, w, b, dy)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for seed in range(3):
        fresh = _inputs(dev, (2, rows, 64), 8, torch.bfloat16, torch.float32, seed=10 + seed)
        for s, t in zip(static, fresh):
            s.copy_(t)
        graph.replay()
        assert all(torch.equal(a, c) for a, c in zip(out, step(*fresh)))


def test_empty(ctmr, dev):
    f = ctmr.differentiable
    w, b = torch.ones(8, device=dev, requires_grad=True), torch.zeros(8, device=dev)
    for shape in ((0, 5, 8), (2, 0, 8)):
        x = torch.empty(shape, device=dev, requires_grad=True)
        y = f.group_norm(x, w, b, num_groups=2, eps=1e-6, apply_silu=True)
        dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
        assert y.shape == dx.shape == shape and bool((dw == 0).all())
