"""CPU tests of the differentiable operators' guards: caps, forward-mode tangents, leaves in captures, threads, tracing."""

from __future__ import annotations

import ctypes

import pytest
import torch


@pytest.mark.parametrize(("softcap", "scale", "good"), [(1e29, 1.0, True), (2e30, 1.0, False), (3e38, 1.0, False),
                                                        (1e20, 1e-9, True), (1e20, 1e-11, False), (257.0, 0.1, True)])
def test_caps_at_the_end_of_the_range(ctmr, native_loaded, softcap, scale, good):
    L, t = ctmr._lib, torch.zeros(1, 1, 4, 16)
    with pytest.raises(ValueError, match="on the GPU" if good else "too large"):
        ctmr.differentiable.attention(t, t, t, scale=scale, softcap=softcap)
    d = L.MaskedAttentionDesc(1, 4, 4, 1, 1, 16, 0, 0, 0, scale, softcap, 0, *([(64, 64, 16)] * 4))
    code = native_loaded.ctmr_masked_attention_workspace_bytes(ctypes.byref(d))
    assert code == 0 if good else code == L.E_INVALID
