"""CPU tests of ``AdamW``'s public settings and state, changed between steps: what the kernels would read is checked."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch


@pytest.fixture
def launched(ctmr, monkeypatch):
    """The arguments of each launch; nothing is launched."""
    f, calls = ctmr.differentiable, []
    monkeypatch.setattr(f, "_on_gpu", lambda t, name: None)
    monkeypatch.setattr(f, "_stream_of", lambda t: None)
    monkeypatch.setattr(f.ops, "adamw", lambda *a: calls.append(a) or torch.zeros(()))
    return calls


def _optimizer(ctmr, **kw):
    params = [torch.zeros(4, 6), torch.zeros(70, dtype=torch.bfloat16)]
    return ctmr.differentiable.AdamW(params, **kw), [torch.zeros_like(p) for p in params]


@pytest.mark.parametrize(
    ("name", "value", "message"),
    [("lr", lambda t: torch.tensor(1e-4, dtype=torch.float64), "lr"), ("lr", lambda t: torch.tensor([1e-4]), "lr"),
     ("lr", lambda t: torch.empty((), device="meta"), "lr"), ("lr", lambda t: math.nan, "lr"), ("lr", lambda t: -1.0, "lr"),
     ("betas", lambda t: (0.9, 1.0), "betas"), ("betas", lambda t: (math.nan, 0.9), "betas"), ("eps", lambda t: math.inf, "eps"),
     ("weight_decay", lambda t: -0.1, "weight_decay"), ("max_norm", lambda t: 0.0, "max_norm"),
     *((n, change, "keep their shapes") for n in ("exp_avg", "exp_avg_sq", "master", "steps", "missed") for change in (
         lambda t: t.double() if t.dim() else t.int(), lambda t: torch.zeros(3, dtype=t.dtype),
         lambda t: torch.stack([t, t], -1)[..., 0] if t.dim() else t[None], lambda t: t.tolist(),
         lambda t: t.to_sparse() if t.dim() else None))])
def test_what_is_bound_anew_is_checked(ctmr, launched, name, value, message):
    o, grads = _optimizer(ctmr)
    before = getattr(o, name)
    setattr(o, name, value(before))
    for _ in range(2):
        with pytest.raises(ValueError, match=message):
            o.step(grads)
    assert not launched
    setattr(o, name, before)
    o.step(grads)
    assert len(launched) == 1


@pytest.mark.parametrize("name", ["lr", "exp_avg", "exp_avg_sq", "master", "steps", "missed"])
def test_host_tensors_are_refused(ctmr, monkeypatch, name):
    from torch._subclasses.fake_tensor import FakeTensorMode

    monkeypatch.setattr(ctmr.differentiable.ops, "adamw", None)
    with FakeTensorMode():
        params = [torch.empty(4, 6, device="cuda"), torch.empty(70, dtype=torch.bfloat16, device="cuda")]
        o = ctmr.differentiable.AdamW(params, lr=torch.empty((), device="cuda"))
        value = getattr(o, name)
        setattr(o, name, torch.empty(value.shape, dtype=value.dtype))
        with pytest.raises(ValueError, match="device"):
            o.step([torch.empty_like(p) for p in params])


def test_parameters_of_another_count(ctmr, launched):
    o, grads = _optimizer(ctmr)
    o.parameters.append(torch.zeros(3))
    with pytest.raises(ValueError, match="3 parameters where there were 2"):
        o.step([*grads, torch.zeros(3)])
    assert not launched


def test_good_changes_are_taken(ctmr, launched):
    o, grads = _optimizer(ctmr)
    o.lr, o.betas, o.eps, o.weight_decay, o.max_norm, o.skip_non_finite = torch.tensor(0.25), [0.5, 0.25], 1, 0, None, 1
    o.exp_avg, o.steps = torch.ones_like(o.exp_avg), torch.tensor(7)
    o.step(grads)
    call, = launched
    assert call[2] is o.exp_avg and call[5] is o.steps and call[6] is o.lr
    assert call[11:19] == (0.0, 0.5, 0.25, 1.0, 0.0, 1.0, math.inf, True)


def test_numbers_of_the_parameters_with_gradients(ctmr, launched):
    o, grads = _optimizer(ctmr)
    o.step(grads)
    o.step([None, grads[1]])
    assert [list(call[20]) for call in launched] == [[], [1]] and all(call[19] is o.missed for call in launched)


def test_a_state_without_missed_steps(ctmr, launched):
    o, _ = _optimizer(ctmr)
    o.missed += 3
    old = {n: t + 1 for n, t in o.state_dict().items() if n != "missed"}
    o.load_state_dict(old)
    assert o.missed.tolist() == [0, 0] and int(o.steps) == 1


def test_host_checks_of_counted_steps(ctmr, native_loaded):
    L, lib, p = ctmr._lib, native_loaded, 4096
    space = lambda sizes, parameters: lib.ctmr_adamw_workspace_bytes(len(sizes), (ctypes.c_int64 * len(sizes))(*sizes), parameters)
    assert space([4096, 1], 2) == 64 + 16 + 16 and space([4096], 3) == 64 + 16 + 32 and space([], 0) == 64
    assert space([4096, 1], 1) == space([-1], 1) == L.E_INVALID and space([1], (1 << 24) + 1) == L.E_UNSUPPORTED

    def step(numbers=(0, 2), parameters=3, missed=p, ws=p, nbytes=1 << 20, desc=True):
        d = L.AdamwDesc(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, scale=1.0, most=1.0)
        two = lambda kind, v: (kind * 2)(v, v)
        given = None if numbers is None else (ctypes.c_int32 * 2)(*numbers)
        return lib.ctmr_adamw_counted(ctypes.byref(d) if desc else None, 2, two(ctypes.c_void_p, p), two(ctypes.c_void_p, p),
                                      two(ctypes.c_int64, 9), two(ctypes.c_int32, 0), two(ctypes.c_int64, 0), None, p, p, None, p,
                                      parameters, given, missed, None, None, ws, nbytes, None)

    for kw in ({"numbers": (0, 3)}, {"numbers": (1, 1)}, {"numbers": (2, 1)}, {"numbers": (-1, 1)}, {"parameters": 1},
               {"parameters": -1}, {"missed": None}, {"desc": False}):
        assert step(**kw) == L.E_INVALID, kw
    assert step(parameters=1 << 25) == L.E_UNSUPPORTED
    assert step(nbytes=64 + 16 + 16) == step(ws=None) == step(ws=p + 8) == L.E_WORKSPACE
