"""Few rows with a position bias whose values, a head of a group behind the other, take most of LDS, or more than it has."""

from __future__ import annotations

import pytest
import test_position_bias_gpu as base
import torch

pytestmark = pytest.mark.gpu


# (n, hq, hk, lq, lk, d): 127, 63 and 32 KB of values (the few-row form), 254 KB and, in fp32, heads of 128 (the tiled form)
@pytest.mark.parametrize("dtype", base.TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 8, 2, 1, 900, 32), (2, 4, 2, 5, 300, 64), (1, 3, 3, 2, 2000, 128), (1, 16, 2, 1, 700, 32),
                                   (1, 8, 1, 2, 500, 128)], ids=str)
def test_values_that_fill_lds(ctmr, dev, shape, dtype):
    n, hq, _, lq, lk, _ = shape
    extents = (32, 32, 32, 32)
    base._compare(ctmr, *base._inputs(dev, *shape, dtype), base._table(dev, extents, 32, hq, torch.float32),
                  base._places(dev, n, lq, extents), base._places(dev, 0, lk, extents, seed=4), extents=extents)
