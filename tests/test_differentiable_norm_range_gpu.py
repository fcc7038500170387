"""``differentiable.group_norm`` of values whose squares leave fp32's range, in both forms of the kernels."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of fp32


def _exact(x, w, b, dy, groups, eps):
    leaves = [t.detach().double().requires_grad_() for t in (x, w, b)]
    n, c = x.shape[0], x.shape[-1]
    g = leaves[0].reshape(n, -1, groups, c // groups)
    var, mean = torch.var_mean(g, dim=(1, 3), keepdim=True, correction=0)
    xhat = ((g - mean) / torch.sqrt(var + eps)).reshape(x.shape)
    y = xhat * leaves[1] + leaves[2]
    return y.detach(), torch.autograd.grad(y, leaves, dy.double()), xhat.detach()


def _inputs(dev, rows, dtype, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=dev, generator=g)
    return r(1, rows, 32), 1 + 0.2 * r(32), 0.2 * r(32), r(1, rows, 32).to(dtype)


def _compare(ctmr, x, w, b, dy, eps):
    x, w, b = (t.detach().requires_grad_() for t in (x, w, b))
    y = ctmr.differentiable.group_norm(x, w, b, num_groups=4, eps=eps)
    grads = torch.autograd.grad(y, (x, w, b), dy)
    ref, want, xhat = _exact(x, w, b, dy, 4, eps)
    half = torch.finfo(x.dtype).eps / 2
    xw = (xhat * w.double()).abs()
    # x less the mean, its low part, times rstd (rounded itself) and gamma, plus beta: five roundings of the product and
    # one of the sum; then the type's
    assert bool(((y.detach().double() - ref).abs() <= half * ref.abs() + 6 * U * xw + 2 * U * ref.abs() + U).all())
    # sums over the voxels of dy and dy xhat: 32 terms in fp32 (31 roundings) and xhat's four
    n = dy.double().abs()
    over = (0, 1)
    assert bool(((grads[2].double() - want[2]).abs() <= 33 * U * n.sum(over) + U).all())
    assert bool(((grads[1].double() - want[1]).abs() <= 38 * U * (n * xhat.abs()).sum(over) + U).all())
    mean = lambda t: t.reshape(1, -1, 4, 8).mean((1, 3), keepdim=True).expand(1, x.shape[1], 4, 8).reshape(x.shape)
    wn = w.double().abs() * n
    size = wn + mean(wn) + xhat.abs() * mean(wn * xhat.abs())
    scale = 1 / torch.sqrt(torch.var(x.detach().double().reshape(1, -1, 4, 8), dim=(1, 3), correction=0, keepdim=True) + eps)
    scale = scale.expand(1, x.shape[1], 4, 8).reshape(x.shape)
    least = torch.finfo(x.dtype).smallest_normal * half  # half a step below the normal numbers
    assert bool(((grads[0].double() - want[0]).abs() <= half * want[0].abs() + 45 * U * scale * size + least).all())


@pytest.mark.parametrize("rows", [200, 30000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("size", [1e17, 1e20, 1e30, 3e37])
def test_spreads_whose_squares_overflow(ctmr, dev, rows, dtype, size):
    x, w, b, dy = _inputs(dev, rows, dtype)
    x = (x * size).to(dtype)
    # the output gradient as large: dx is of its size over the spread's, which fp32 holds as normal numbers
    _compare(ctmr, x, w, b, (dy.float() * min(size, 1e10)).to(dtype), 1e-6)


@pytest.mark.parametrize("rows", [200, 30000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("size", [1e-15, 1e-20, 1e-25, 1e-30])
def test_spreads_whose_squares_underflow(ctmr, dev, rows, dtype, size):
    """Without eps the statistics are those of the values however small."""
    x, w, b, dy = _inputs(dev, rows, dtype, seed=1)
    _compare(ctmr, (x * size).to(dtype), w, b, dy, 0.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_a_few_large_values_and_channels(ctmr, dev, dtype):
    """Some rows of one channel, and one whole channel, leave the range; the others of their groups do not."""
    x, w, b, dy = _inputs(dev, 20001, dtype, seed=2)
    x[:, 300:310, 3] *= 1e22
    x[:, :, 9] *= 1e25
    x[:, 0, 17] = 3e38  # the value that the others are taken less of
    x[:, 1, 17] = -3e38
    _compare(ctmr, x.to(dtype), w, b, dy, 1e-6)


@pytest.mark.parametrize("rows", [200, 30000])
def test_a_constant_channel_without_eps(ctmr, dev, rows):
    """Zero variance and zero eps: not finite, in that group alone."""
    x, w, b, _ = _inputs(dev, rows, torch.float32, seed=3)
    f = ctmr.differentiable
    clean = f.group_norm(x, w, b, num_groups=4, eps=0.0)
    x[..., 8:16] = 2.0
    y = f.group_norm(x, w, b, num_groups=4, eps=0.0)
    assert bool(y[..., 8:16].isnan().all())
    assert torch.equal(y[..., :8], clean[..., :8]) and torch.equal(y[..., 16:], clean[..., 16:])
    assert math.isfinite(float(clean.abs().max()))
