"""CPU tests of the operators on lists of tensors: what they refuse, the library's host checks, tracing."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch


def _calls(f):
    return {"norm": f.gradient_norm, "clip": lambda t: f.clip_gradients(t, 1.0), "adamw": f.AdamW}


@pytest.mark.parametrize("name", ["norm", "clip", "adamw"])
@pytest.mark.parametrize(
    ("tensors", "message"),
    [([], "no tensor"), ([None], "no tensor|dense"), (torch.zeros(3), "list of tensors"), ([1.0], "dense"),
     ([torch.zeros(3, dtype=torch.float64)], "float32, bfloat16"), ([torch.zeros(3, dtype=torch.int32)], "float32"),
     ([torch.zeros(3).to_sparse()], "dense"),
 ([torch.zeros(3)], "on the GPU"),
     ([torch.zeros(3), torch.zeros(3, device="meta")], "cpu and meta")])
def test_lists_are_refused(ctmr, name, tensors, message):
    with pytest.raises(ValueError, match=message):
        _calls(ctmr.differentiable)[name](tensors)


@pytest.mark.parametrize("name", ["norm", "clip", "adamw"])
def test_forward_mode_is_refused(ctmr, name):
    t = torch.zeros(4)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        _calls(ctmr.differentiable)[name]([t, torch.autograd.forward_ad.make_dual(t, t)])


@pytest.fixture
def on_cpu(ctmr, monkeypatch):
    """The checks behind the one that asks for the GPU; nothing is launched."""
    f = ctmr.differentiable
    monkeypatch.setattr(f, "_on_gpu", lambda t, name: None)
    monkeypatch.setattr(f, "_stream_of", lambda t: None)
    launched = []
    monkeypatch.setattr(f.ops, "adamw", lambda *a: launched.append(a) or torch.zeros(()))
    f.launched = launched
    yield f
    del f.launched


def test_shared_memory_and_gaps_are_refused(on_cpu):
    flat = torch.zeros(64)
    for tensors in ([flat[:32], flat[31:]], [flat, flat], [flat[:8].expand(4, 8)], [flat.view(8, 8)[:, :4]],
                    [flat.view(8, 8)[::2]]):
        for call in (lambda t: on_cpu.clip_gradients(t, 1.0), on_cpu.AdamW):
            with pytest.raises(ValueError, match="share memory|without gaps"):
                call(tensors)
    on_cpu._apart([flat[:32], flat[32:], torch.zeros(4, 3, 2).permute(2, 0, 1), torch.zeros(0), flat[5:5]], "gradients",
                  False)


@pytest.mark.parametrize("value", [0.0, -1.0, math.nan])
def test_limits_are_refused(on_cpu, value):
    with pytest.raises(ValueError, match="max_norm"):
        on_cpu.clip_gradients([torch.zeros(3)], value)
    with pytest.raises(ValueError, match="max_norm"):
        on_cpu.AdamW([torch.zeros(3)], max_norm=value)


@pytest.mark.parametrize(
    ("kw", "message"),
    [({"betas": (1.0, 0.9)}, "betas"), ({"betas": (0.9, -0.1)}, "betas"), ({"betas": (0.9, math.nan)}, "betas"),
     ({"eps": -1.0}, "eps"), ({"eps": math.inf}, "eps"), ({"weight_decay": -0.1}, "weight_decay"), ({"lr": -1.0}, "lr"),
     ({"lr": math.nan}, "lr"), ({"lr": torch.zeros(1)}, "lr"), ({"lr": torch.zeros((), dtype=torch.float64)}, "lr")])
def test_settings_are_refused(on_cpu, kw, message):
    with pytest.raises(ValueError, match=message):
        on_cpu.AdamW([torch.zeros(3)], **kw)


def test_steps_are_refused(on_cpu):
    p, h = torch.zeros(4, 6), torch.zeros(5, dtype=torch.bfloat16)
    o = on_cpu.AdamW([p, h])
    good = [torch.zeros(4, 6), torch.zeros(5, dtype=torch.bfloat16)]
    for grads, kw, message in (([good[0]], {}, "1 gradients for 2"), ([torch.zeros(6, 4), good[1]], {}, "gradient 0"),
                               ([good[0], torch.zeros(5)], {}, "gradient 1"), ([None, None], {}, "no tensor"),
                               ([good[0], torch.zeros(5, dtype=torch.float64)], {}, "float32, bfloat16"),
                               (good, {"lr": -1.0}, "lr"), (good, {"gradient_scale": math.inf}, "gradient_scale")):
        with pytest.raises(ValueError, match=message):
            o.step(grads, **kw)
    assert not on_cpu.launched
    o.step(good)
    o.step([None, good[1]])
    assert [len(a[0]) for a in on_cpu.launched] == [2, 1] and on_cpu.launched[1][9] == [64]
    p.data = torch.zeros(6, 4).t()
    with pytest.raises(ValueError, match="parameter 0 has become"):
        o.step(good)


def test_gradients_in_another_order_of_axes_are_brought_into_the_parameters(on_cpu):
    p = torch.zeros(6, 4).t()
    g = torch.arange(24.0).view(4, 6)
    on_cpu.AdamW([p]).step([g])
    taken, = on_cpu.launched[0][1]
    assert taken.stride() == p.stride() and torch.equal(taken, g)


def test_state_is_loaded_and_laid_out(on_cpu):
    params = [torch.full((3,), 1.5, dtype=torch.bfloat16), torch.zeros(70), torch.full((2, 2), 2.0, dtype=torch.float16).t()]
    o = on_cpu.AdamW(params)
    assert o._starts == [0, 64, 192] and o._master_starts == [0, 0, 64]
    assert o.exp_avg.shape == o.exp_avg_sq.shape == (256,) and o.master.shape == (128,)
    assert o.master[:3].tolist() == [1.5] * 3 and o.master[64:68].tolist() == [2.0] * 4
    state = {n: t + 1 for n, t in o.state_dict().items()}
    o.load_state_dict(state)
    assert all(torch.equal(t, state[n]) for n, t in o.state_dict().items())
    assert params[0].tolist() == [2.5] * 3 and params[2].flatten().tolist() == [3.0] * 4 and not params[1].any()
    for bad in ({}, state | {"more": state["steps"]}, state | {"master": torch.zeros(4)}, state | {"steps": torch.zeros(())}):
        with pytest.raises(ValueError, match="other parameters"):
            o.load_state_dict(bad)


def test_host_checks(ctmr, native_loaded):
    L, lib, p = ctmr._lib, native_loaded, 4096
    inf = math.inf

    def norm(count=2, ptrs=(p, 0), sizes=(10, 0), elems=(1, 0), most=inf, scale=1.0, out=p, ws=p, nbytes=1 << 20):
        n = max(count, 0)
        return lib.ctmr_gradient_norm(count, (ctypes.c_void_p * n)(*ptrs[:n]), (ctypes.c_int64 * n)(*sizes[:n]),
                                      (ctypes.c_int32 * n)(*elems[:n]), scale, most, out, ws, nbytes, None)

    for kw in ({"count": -1}, {"sizes": (10, -1)}, {"elems": (1, 3)}, {"ptrs": (p, 0), "sizes": (10, 1)}, {"ptrs": (p + 1, 0)},
               {"ptrs": (p, p + 2)}, {"most": 0.0}, {"most": math.nan}, {"scale": math.nan}, {"out": None}):
        assert norm(**kw) == L.E_INVALID, kw
    assert norm(sizes=(1 << 41, 0)) == L.E_UNSUPPORTED and norm(sizes=(1 << 36, 0)) == L.E_UNSUPPORTED
    for kw in ({"ws": None}, {"ws": p + 8}, {"nbytes": 64}):
        assert norm(**kw) == L.E_WORKSPACE, kw
    space = lambda *sizes: lib.ctmr_gradients_workspace_bytes(len(sizes), (ctypes.c_int64 * len(sizes))(*sizes))
    assert space() == 64 and space(0, 0) == 64 and space(4096) == 80 and space(4097, 1) == 64 + 32
    assert space(1 << 30) == 64 + 2048 * 8 and space(-1) == L.E_INVALID and space(1 << 41) == L.E_UNSUPPORTED
    one = lambda kind, v: (kind * 1)(v)
    clip = lambda ptr=p, out=p, ws=p, nbytes=1 << 20, size=5, most=1.0: lib.ctmr_clip_gradients(
        1, one(ctypes.c_void_p, ptr), one(ctypes.c_int64, size), one(ctypes.c_int32, 0), most, out, ws, nbytes, None)
    for size in (5, 1 << 30):  # both forms
        assert clip(ptr=p + 2, size=size) == clip(out=None, size=size) == clip(most=0.0, size=size) == L.E_INVALID
        assert clip(nbytes=64, size=size) == clip(ws=None, size=size) == L.E_WORKSPACE
    assert clip(size=-1) == L.E_INVALID and clip(size=1 << 41) == L.E_UNSUPPORTED
    scale = lambda ptr=p, factor=p, size=5: lib.ctmr_scale_tensors(1, one(ctypes.c_void_p, ptr), one(ctypes.c_int64, size),
                                                                  one(ctypes.c_int32, 0), factor, None)
    assert scale(factor=None) == L.E_INVALID and scale(ptr=p + 2) == L.E_INVALID and scale(size=-1) == L.E_INVALID
    assert lib.ctmr_scale_tensors(0, None, None, None, p, None) == L.OK

    def adamw(desc={}, elem=1, start=0, master_start=0, m=p, v=p, master=p, steps=p, ws=p, nbytes=1 << 20):
        d = L.AdamwDesc(**({"lr": 1e-3, "beta1": 0.9, "beta2": 0.99, "eps": 1e-8, "scale": 1.0, "most": 1.0} | desc))
        return lib.ctmr_adamw(ctypes.byref(d), 1, one(ctypes.c_void_p, p), one(ctypes.c_void_p, p), one(ctypes.c_int64, 9),
                              one(ctypes.c_int32, elem), one(ctypes.c_int64, start), one(ctypes.c_int64, master_start), m, v,
                              master, steps, None, None, ws, nbytes, None)

    for kw in ({"desc": {"beta1": 1.0}}, {"desc": {"beta2": -0.1}}, {"desc": {"eps": -1.0}}, {"desc": {"lr": -1.0}},
               {"desc": {"decay": -1.0}}, {"desc": {"most": 0.0}}, {"desc": {"scale": math.nan}}, {"elem": 4}, {"start": 2},
               {"start": -4}, {"master_start": 1}, {"m": None}, {"v": None}, {"master": None}, {"steps": None}, {"m": p + 4},
               {"master": p + 8}):
        assert adamw(**kw) == L.E_INVALID, kw
    assert adamw(nbytes=16) == L.E_WORKSPACE and adamw(ws=p + 4) == L.E_WORKSPACE
    assert lib.ctmr_adamw(None, 0, None, None, None, None, None, None, p, p, p, p, None, None, p, 64, None) == L.E_INVALID


@pytest.mark.filterwarnings("error:Accessing the data pointer")
def test_lists_trace(ctmr):
    from torch._subclasses.fake_tensor import FakeTensorMode

    f = ctmr.differentiable
    with FakeTensorMode():
        make = lambda *s, dtype=torch.float32: torch.empty(*s, device="cuda", dtype=dtype)
        grads = [make(3, 4), make(5, dtype=torch.bfloat16), None]
        assert f.gradient_norm(grads).shape == () and f.clip_gradients(grads, 1.0).dtype == torch.float32
        o = f.AdamW(grads[:2], max_norm=1.0)
        assert o.step([make(3, 4), make(5, dtype=torch.bfloat16)]).shape == () and o.master.shape == (64,)


@pytest.mark.filterwarnings("ignore:Sparse CSR")
def test_layouts_without_strides_are_refused(ctmr):
    for call in _calls(ctmr.differentiable).values():
        with pytest.raises(ValueError, match="dense"):
            call([torch.eye(3).to_sparse_csr()])
