"""The position bias table's gradient over long rows, where errors that sums do not average out show: rows of both signs,
weights and scores' gradients in parts, values of the bias in fp32."""

from __future__ import annotations

import math

import position_bias_oracle as oracle
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24  # half a step of fp32
BUCKETS = dict(num_buckets=32, max_distance=16)


def _grid(dev, shape):
    return torch.stack(torch.meshgrid(*(torch.arange(s) for s in shape), indexing="ij"), -1).reshape(-1, len(shape)).int().to(dev)


def _heads(dev, l, h, d, dtype, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn(1, l, h, d, device=dev, generator=g).to(dtype).transpose(1, 2)


def _table_gradient(f, q, k, v, table, dout, plan, softcap=0.0):
    leaf = table.detach().requires_grad_()
    out = f.attention(q, k, v, scale=q.shape[-1] ** -0.5, softcap=softcap, position_bias=leaf, buckets=plan)
    return torch.autograd.grad(out, leaf, dout)[0]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize(("d", "grid", "softcap"), [(32, (16, 16, 8), 0.0), (64, (40, 30), 0.0), (128, (9, 16, 16), 0.0),
                                                    (64, (16, 16, 8), 20.0), (32, (20, 20, 7), 400.0)], ids=str)
def test_neighbours_of_other_sign_cancel(ctmr, dev, dtype, d, grid, softcap):
    """Rows 2 i and 2 i + 1 with the same q and place and opposite gradients: whatever the sums round, and to which side, the
    table's gradient is zero to the last bit."""
    f, places = ctmr.differentiable, _grid(dev, grid)
    l = places.shape[0]
    even = torch.arange(l, device=dev) // 2 * 2
    q, dout = _heads(dev, l, 2, d, dtype, 1)[:, :, even], _heads(dev, l, 2, d, dtype, 4)[:, :, even].clone()
    dout[:, :, 1::2] *= -1
    k, v = (_heads(dev, l, 2, d, dtype, seed) for seed in (2, 3))
    table = torch.randn(len(grid), 32, 2, device=dev)
    plan = f.PositionBuckets(places[even].contiguous(), places, extents=grid, **BUCKETS)
    assert not bool(_table_gradient(f, q, k, v, table, dout, plan, softcap).any())
    assert bool(_table_gradient(f, q, k, v, table, dout.abs(), plan, softcap).any())


def _exact(q, k, v, table, dout, places, grid):
    """The table's gradient in 64 bits, a head at a time, and the largest score."""
    which, axes = oracle.numbers(places, places, grid, *BUCKETS.values())[0], range(len(grid))
    total, top = torch.zeros(table.shape, dtype=torch.float64, device=q.device), 0.0
    for h in range(q.shape[1]):
        a, b, c, g, t = (x.detach().double() for x in (q[0, h], k[0, h], v[0, h], dout[0, h], table[:, :, h]))
        s = a @ b.T / math.sqrt(a.shape[-1])
        for axis in axes:
            s += t[axis][which[..., axis]]
        top = max(top, float(s.abs().max()))
        p = torch.softmax(s, -1)
        ds = p * (g @ c.T - (g * (p @ c)).sum(-1, keepdim=True))
        for axis in axes:
            for n in range(table.shape[1]):
                total[axis, n, h] = torch.where(which[..., axis] == n, ds, 0.0).sum()
    return total, top


def _long(ctmr, dev, dtype, table_type, d, grid, scale=0.5):
    f, places = ctmr.differentiable, _grid(dev, grid)
    q, k, v, dout = (_heads(dev, places.shape[0], 4, d, dtype, seed) for seed in range(4))
    g = torch.Generator(device=dev).manual_seed(9)
    table = (scale * torch.randn(len(grid), 32, 4, device=dev, generator=g)).to(table_type)
    got = _table_gradient(f, q, k, v, table, dout, f.PositionBuckets(places, extents=grid, **BUCKETS))
    return (got, *_exact(q, k, v, table, dout, places, grid))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize(("d", "grid"), [(32, (16, 16, 8)), (64, (16, 16, 16)), (128, (16, 16, 16))], ids=str)
def test_tables_of_fp32_get_all_of_its_bits(ctmr, dev, dtype, d, grid):
    """Over the whole gradient, in half steps U of fp32, each the mean of many independent roundings (3^-1/2 of the largest):

    * a product of d terms rounds its running sum, which grows like a random walk (2^-1/2 of the last size in the mean), once
      for each matrix step: (steps / 6)^1/2, steps of 16 terms, of 2 with fp32 heads.  g . v has that relative to its size;
      a score s, to whose error its weight's relative one is equal, |s| times it, and where the weights' squares e^2s are, s
      of a normal distribution is 2 +- 1: 5^1/2 times it;
    * the exponent's argument (1.6), the exponential and the difference g . v - delta (one each): 2.2 together;
    * a column of a row is added to by 768 one-hot products at most (256 keys of a place in three parts): (768 / 6)^1/2.

    A third more is left.  That is 0.9e-6 with 16-bit heads; two parts of a bf16 weight are 1.2e-6 off, of a score's gradient
    2.3e-6, rows of one sign 2.5e-6 (at 4096 rows of 64)."""
    got, want, _ = _long(ctmr, dev, dtype, torch.float32, d, grid)
    steps = d / (2 if dtype == torch.float32 else 16)
    bound = 4 / 3 * math.sqrt((5 + 1) * steps / 6 + 2.2 ** 2 + 768 / 6) * U
    assert float((got.double() - want).norm()) <= bound * float(want.norm())


@pytest.mark.parametrize(("dtype", "share"), [(torch.bfloat16, 0.01), (torch.float16, 0.05)], ids=str)
def test_tables_of_16_bits_get_rounded_gradients(ctmr, dev, dtype, share):
    """An error of 2.5e-6 (two parts) takes a value over the border between two of its type's where it lies as near, 2.5e-6 of
    steps of 2^-8 (bf16) or 2^-11 (fp16) relative at least: 0.06 % and 0.5 % of values of the mean size, for values of a
    tenth of it ten times as many.  One part (4.6e-4, 5.8e-5) would move 12 % of either and more."""
    got, want, _ = _long(ctmr, dev, dtype, dtype, 64, (16, 16, 16))
    assert float((got != want.to(dtype)).double().mean()) <= share


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_large_biases_keep_their_bits(ctmr, dev, dtype):
    """A weight's relative error is its score's: the value in the scores' units, the sum of a pair, that of both pairs and of the
    product, and the exponent's argument are rounded to half a step of the score's size at most, 5^1/2 3^-1/2 of it in the mean.
    Four half steps of the largest score are far above; two bf16 parts of the bias, 2^-18 of it, are 64 of them."""
    got, want, top = _long(ctmr, dev, dtype, torch.float32, 64, (16, 16, 8), scale=6.0)
    assert top > 20 and float((got.double() - want).norm()) <= 4 * U * top * float(want.norm())
