"""The position bias table's gradient over long rows, where errors that sums do not average out show."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
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
