"""Padding rows and keys of ``differentiable.attention`` that share their 32 rows with two documents, in layouts where the
other side holds whole tiles of one of them: padding sees and is seen by nothing, whatever it holds."""

from __future__ import annotations

import math

import attention_oracle as oracle
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
P = -1

# (query runs, key runs or None for the same) of (id, rows)
LAYOUTS = {
    "keys of long documents": ([(0, 70), (1, 10), (P, 48)], [(0, 64), (1, 320), (P, 16)]),
    "rows of long documents": ([(0, 64), (1, 320), (P, 16)], [(0, 70), (1, 10), (P, 48)]),
    "padding between": ([(0, 70), (1, 10), (P, 16), (1, 200)], None),
    "a block that starts with padding": ([(P, 40), (0, 30), (1, 10), (P, 16), (1, 200), (0, 128)], None),
    "padding first in its rows": ([(0, 64), (P, 3), (0, 20), (1, 9), (1, 256), (0, 64)], None),
    "three documents": ([(2, 64), (0, 10), (1, 10), (P, 3), (2, 9), (1, 192), (0, 192)], None),
}


def _ids(dev, runs):
    return torch.cat([torch.full((rows,), i, dtype=torch.int32) for i, rows in runs])[None].to(dev)


def _inputs(dev, lq, lk, d, dtype, hq=2, hk=1):
    g = torch.Generator(device=dev).manual_seed(lq + lk + d)
    make = lambda l, h: torch.randn(1, l, h, d, device=dev, generator=g).to(dtype).transpose(1, 2)
    return make(lq, hq), make(lk, hk), make(lk, hk), make(lq, hq)


def _compare(ctmr, dev, ids, key_ids, d, dtype, value=0.0, **kw):
    """Values and gradients with ``value`` in every place of the padding, against 64 bits."""
    f = ctmr.differentiable
    q, k, v, dout = _inputs(dev, ids.shape[1], key_ids.shape[1], d, dtype)
    for t, i in ((q, ids), (k, key_ids), (v, key_ids), (dout, ids)):
        t.transpose(1, 2)[i < 0] = value
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = f.attention(*leaves, scale=d ** -0.5, documents=f.Documents(ids, key_ids), **kw)
    got = [out.detach(), *torch.autograd.grad(out, leaves, dout)]
    mask = oracle.visible(1, ids.shape[1], key_ids.shape[1], dev, ids, key_ids, kw.get("prefix"))
    want = oracle.attention(q, k, v, scale=d ** -0.5, mask=mask, dout=dout, **{n: t for n, t in kw.items() if n != "prefix"})
    for g, w, i, name in zip(got, want, (ids, ids, key_ids, key_ids), ("out", "dq", "dk", "dv")):
        assert bool((g.transpose(1, 2)[i < 0] == 0).all()), (name, "of padding")
        oracle.check(g, w, name)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
@pytest.mark.parametrize("d", [32, 128])
def test_padding_sees_nothing(ctmr, dev, layout, d, dtype):
    rows, keys = (None if r is None else _ids(dev, r) for r in LAYOUTS[layout])
    keys = rows if keys is None else keys
    for value in (1.0, math.nan):
        _compare(ctmr, dev, rows, keys, d, dtype, value)
    _compare(ctmr, dev, rows, keys, d, dtype, math.inf, prefix=100, softcap=4.0)


@pytest.mark.parametrize("seed", range(12))
def test_random_layouts(ctmr, dev, seed):
    """Runs of three documents and padding of any length, the lengths drawn over their logarithm."""
    g = torch.Generator().manual_seed(seed)
    draw = lambda n: int(torch.randint(0, n, (1,), generator=g))

    def layout(total):
        runs, left = [], total
        while left > 0:
            rows = min(left, int(2 ** (8 * float(torch.rand(1, generator=g)))))
            runs.append((draw(4) - 1, rows))
            left -= rows
        return _ids(dev, runs)

    rows = layout(200 + draw(300))
    _compare(ctmr, dev, rows, rows if seed % 2 else layout(200 + draw(300)), 32, TYPES[seed % 3], math.nan)
