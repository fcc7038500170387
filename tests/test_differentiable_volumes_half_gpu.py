"""``maisi.spatial_attention_volumes`` and its gradients in fp16, against the same block in 64 bits, also where the volumes'
output gradients differ far in size."""

from __future__ import annotations

import pytest
import torch
from test_differentiable_volumes_gpu import SHAPES, _block, _leaves, _volumes, _weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sizes", [(1.0, 1.0, 1.0, 1.0), (2.0 ** -6, 2.0 ** 9, 1.0, 2.0 ** 3)], ids=["alike", "apart"])
@pytest.mark.parametrize(("c", "width", "sections"), [(64, 32, (8, 12, 12)), (128, 64, (20, 20, 20)), (96, 24, None)])
def test_block_and_its_gradients(ctmr, dev, c, width, sections, sizes):
    dtype = torch.float16
    volumes, w = _leaves(_volumes(dev, SHAPES, c, dtype), _weights(dev, c, dtype))
    douts = [(d.float() * s).half() for d, s in zip(_volumes(dev, SHAPES, c, dtype, seed=7), sizes)]
    got = ctmr.maisi.spatial_attention_volumes(volumes, w, num_groups=16, eps=1e-6, num_head_channels=width, include_fc=True,
                                               sections=sections)
    got = [t.detach() for t in got] + list(torch.autograd.grad(got, [*volumes, *w.values()], douts))

    def run(kind):
        v, m = _leaves([t.double() for t in volumes], {n: t.double() for n, t in w.items()})
        out = _block(v, m, c // width, 16, sections, kind)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, [*v, *m.values()], [d.double() for d in douts]))

    torch.manual_seed(0)
    want, off = run(None), run(dtype)
    names = [*(f"out{i}" for i in range(len(SHAPES))), *(f"d{i}" for i in range(len(SHAPES))), *w]
    for name, g, e, o in zip(names, got, want, off):
        # as many independent errors of the same size, four times over, and half a step of the least fp16 numbers for
        # each value of the tensor and of the two that its gradient went through
        bound = 4 * float((o - e).norm()) + 3 * 2.0 ** -25 * g.numel() ** 0.5
        assert g.dtype == w.get(name, volumes[0]).dtype
        assert float((g.double() - e).norm()) <= bound, (name, float((g.double() - e).norm()), bound)
