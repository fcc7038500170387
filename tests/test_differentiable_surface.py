"""CPU tests of the differentiable operators: what they refuse, their host checks, registration and tracing."""

from __future__ import annotations

import ctypes
import gc

import pytest
import torch


def _norm(f, x=(2, 5, 8), w=8, b=8, xt=torch.float32, wt=torch.float32, bt=torch.float32, groups=2, eps=1e-6):
    return f.group_norm(torch.zeros(x, dtype=xt), torch.zeros(w, dtype=wt), torch.zeros(b, dtype=bt), num_groups=groups,
                        eps=eps)


@pytest.mark.parametrize(
    ("kw", "message"),
    [({"x": (8,)}, "x must be"), ({"xt": torch.float64}, "float32, bfloat16 or float16"),
     ({"groups": 3}, "not divisible"), ({"groups": 0}, "not divisible"), ({"w": 7}, "weight must be"),
     ({"b": 9}, "bias must be"), ({"wt": torch.bfloat16}, "weight must be"), ({"eps": -1.0}, "eps"),
     ({"eps": float("nan")}, "eps"), ({"xt": torch.bfloat16, "wt": torch.bfloat16}, "differ in type"),
     ({}, "on the GPU")])
def test_group_norm_refuses(ctmr, kw, message):
    with pytest.raises(ValueError, match=message):
        _norm(ctmr.differentiable, **kw)


def _rotary(f, q=(2, 4, 6, 32), k=(2, 2, 6, 32), qt=torch.float32, kt=torch.float32, pos=(6, 2), pt=torch.int32,
            sections=(8, 8), base=10000.0):
    return f.rotary(torch.zeros(q, dtype=qt), None if k is None else torch.zeros(k, dtype=kt),
                    torch.zeros(pos, dtype=pt), sections=sections, base=base)


@pytest.mark.parametrize(
    ("kw", "message"),
    [({"q": (4, 6, 32)}, "q must be 4-D"), ({"qt": torch.int32}, "float32, bfloat16"), ({"kt": torch.float16}, "k is"),
     ({"k": (2, 2, 7, 32)}, "differ in more"), ({"k": (1, 2, 6, 32)}, "differ in more"), ({"sections": ()}, "sections"),
     ({"sections": (7, 8)}, "even"), ({"sections": (32, 2)}, "do not fit"), ({"sections": (2,) * 5}, "one to four"),
     ({"sections": (0, 8)}, "even"), ({"base": 0.0}, "base"), ({"base": float("inf")}, "base"),
     ({"pt": torch.float64}, "positions"), ({"pos": (6, 3)}, "positions"), ({"pos": (3, 6, 2)}, "positions"),
     ({"q": (2, 4, 6, 514), "k": None}, "at most 512"), ({}, "on the GPU")])
def test_rotary_refuses(ctmr, kw, message):
    with pytest.raises(ValueError, match=message):
        _rotary(ctmr.differentiable, **kw)


def test_norm_host_checks(ctmr, native_loaded):
    L, p = ctmr._lib, 4096
    space = native_loaded.ctmr_norm_workspace_bytes
    assert space(2, 64, 64, 8, 0, 0) == 0 and space(2, 64, 64, 8, 0, 1) == 2 * 64 * 16
    assert space(1, 64, 64, 8, 0, 1) == 0 and space(1, 100000, 64, 8, 1, 0) > 0
    assert space(0, 1, 8, 2, 0, 0) == L.E_INVALID and space(1, 1, 8, 3, 0, 0) == L.E_INVALID
    assert space(1, 1, 8, 2, 3, 0) == L.E_INVALID and space(1, 1 << 41, 8, 2, 0, 0) == L.E_UNSUPPORTED
    fwd = lambda **kw: native_loaded.ctmr_norm_forward(
        kw.get("n", 1), kw.get("s", 16), 8, 2, 1e-6, kw.get("elem", 0), kw.get("x", p), kw.get("ptype", 0), p, p, 1,
        kw.get("y", p), kw.get("saved", p), kw.get("ws", p), kw.get("bytes", 0), None)
    for kw, code in (({"x": None}, L.E_INVALID), ({"y": None}, L.E_INVALID), ({"saved": None}, L.E_INVALID),
                     ({"saved": p + 4}, L.E_INVALID), ({"elem": 5}, L.E_INVALID), ({"ptype": -1}, L.E_INVALID),
                     ({"n": 70000}, L.E_UNSUPPORTED), ({"s": 100000}, L.E_WORKSPACE),
                     ({"s": 100000, "ws": p + 8, "bytes": 1 << 30}, L.E_WORKSPACE),
                     ({"s": 100000, "ws": None, "bytes": 1 << 30}, L.E_WORKSPACE)):
        assert fwd(**kw) == code, kw
    bwd = lambda **kw: native_loaded.ctmr_norm_backward(
        1, kw.get("s", 16), 8, 2, 0, p, kw.get("dy", p), 0, p, p, 1, p, kw.get("dx", None), kw.get("dw", None),
        kw.get("db", None), p, kw.get("bytes", 0), None)
    assert bwd() == L.OK  # nothing wanted, nothing launched
    assert bwd(dy=None) == L.E_INVALID and bwd(dw=p) == L.E_INVALID and bwd(s=100000, dx=p) == L.E_WORKSPACE


def test_rotary_host_checks(ctmr, native_loaded):
    L, p = ctmr._lib, 4096
    turns = (ctypes.c_double * 256)()

    def call(q=p, out=p, k=p, pos=p, turns=turns, **kw):
        d = L.RotaryDesc(1, 4, 2, 1, 32, 2, (ctypes.c_int32 * 4)(8, 8), 0, 0, 0, 0, 0)
        for name, value in kw.items():
            setattr(d, name, (ctypes.c_int32 * 4)(*value) if name == "widths" else value)
        return native_loaded.ctmr_rotary(ctypes.byref(d), q, k, pos, turns, out, p, None)

    assert native_loaded.ctmr_rotary(None, p, p, p, turns, p, p, None) == L.E_INVALID
    for kw in ({"q": None}, {"k": None}, {"pos": None}, {"turns": None}, {"out": None}, {"n": 0}, {"l": 0}, {"axes": 5},
               {"axes": 0}, {"elem": 3}, {"position_type": 3}, {"head_dim": 31}, {"widths": (7, 8)}, {"widths": (8, 0)},
               {"widths": (24, 10)}, {"q_heads": 0}, {"k_heads": -1}):
        assert call(**kw) == L.E_INVALID, kw
    assert call(n=70000) == L.E_UNSUPPORTED and call(head_dim=514) == L.E_UNSUPPORTED


def test_a_leaf_of_a_living_eager_graph_is_refused_in_a_capture(ctmr, monkeypatch):
    f = ctmr.differentiable
    state = {"capturing": False}
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    leaf, other = torch.zeros(3, requires_grad=True), torch.zeros(3, requires_grad=True)
    token = f._graph_token(leaf, None, leaf * 2)
    assert f._graph_token(leaf.detach()) is None
    state["capturing"] = True
    assert f._graph_token(other) is None and f._graph_token(leaf * 2) is None
    with pytest.raises(RuntimeError, match="outside this capture"):
        f._graph_token(other, leaf)
    with pytest.raises(RuntimeError, match="both"):
        f._check_capture(False)
    f._check_capture(True)
    with pytest.raises(RuntimeError, match="outside this capture"):
        f._graph_token(leaf[None])
    del token
    gc.collect()
    assert f._graph_token(leaf) is None


def test_registered_operators_trace(ctmr):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(2, 5, 8, device="cuda", dtype=torch.bfloat16)
        w = torch.empty(8, device="cuda")
        y, saved = torch.ops.ctmr.norm_forward(x, w, w, 2, 1e-6, True)
        assert y.shape == x.shape and y.dtype == x.dtype and saved.shape == (2, 2, 4)
        dx, dw, db = torch.ops.ctmr.norm_backward(x, y, w, w, saved, True, True, False)
        assert dx.shape == x.shape and dw.shape == db.shape == (0,)
        q = torch.empty(2, 4, 6, 32, device="cuda")
        out, k_out = torch.ops.ctmr.rotary(q, None, torch.empty(6, 2, device="cuda", dtype=torch.int32), [8, 8], 1e4,
                                           False)
        assert out.shape == q.shape and out.transpose(1, 2).is_contiguous() and k_out.shape == (0,)


def _attention(f, q=(2, 4, 6, 32), k=(2, 2, 7, 32), v=None, qt=torch.float32, kt=torch.float32, scale=1.0, **kw):
    return f.attention(torch.zeros(q, dtype=qt), torch.zeros(k, dtype=kt), torch.zeros(v or k, dtype=kt), scale=scale, **kw)


@pytest.mark.parametrize(
    ("kw", "message"),
    [({"q": (4, 6, 32)}, "q must be 4-D"), ({"qt": torch.float64}, "float32, bfloat16"),
     ({"kt": torch.bfloat16}, "k is"), ({"k": (1, 2, 7, 32)}, "do not fit"), ({"k": (2, 2, 7, 16)}, "do not fit"),
     ({"v": (2, 2, 8, 32)}, "do not fit"), ({"k": (2, 3, 7, 32)}, "not a multiple"),
     ({"k": (2, 0, 7, 32)}, "not a multiple"), ({"q": (2, 4, 6, 36), "k": (2, 2, 7, 36)}, "multiple of 8"),
     ({"q": (2, 4, 6, 136), "k": (2, 2, 7, 136)}, "up to 128"), ({"scale": 0.0}, "scale"), ({"scale": -1.0}, "scale"),
     ({"scale": float("inf")}, "scale"), ({"softcap": -1.0}, "softcap"), ({"slopes": torch.zeros(3)}, "slopes"),
     ({"slopes": torch.zeros(4, dtype=torch.float64)}, "slopes"), ({"slopes": [0.0] * 4}, "slopes"),
     ({"slopes": torch.zeros(4, requires_grad=True)}, "no gradient"), ({"prefix": torch.zeros(3).int()}, "prefix"),
     ({"prefix": torch.zeros(2)}, "prefix"), ({}, "on the GPU")])
def test_attention_refuses(ctmr, kw, message):
    with pytest.raises(ValueError, match=message):
        _attention(ctmr.differentiable, **kw)


@pytest.mark.parametrize(
    ("ids", "key_ids", "message"),
    [(torch.zeros(2, 3), None, "int32"), (torch.zeros(2, 3).long(), None, "int32"), (torch.zeros(3).int(), None, "int32"),
     (torch.zeros(2, 0).int(), None, "empty"), (torch.zeros(2, 3).int(), torch.zeros(1, 3).int(), "differ"),
     ([[0]], None, "int32"), (torch.zeros(2, 3).int(), None, "on the GPU")])
def test_documents_refuse(ctmr, ids, key_ids, message):
    with pytest.raises(ValueError, match=message):
        ctmr.differentiable.Documents(ids, key_ids)


def _attention_desc(L, **kw):
    d = L.MaskedAttentionDesc(1, 200, 300, 4, 2, 32, 0, 0, 0, 1.0, 0.0, 0, (25600, 32, 128), (19200, 32, 64),
                              (19200, 32, 64), (25600, 32, 128))
    for name, value in kw.items():
        setattr(d, name, (ctypes.c_int64 * 3)(*value) if name.endswith("strides") else value)
    return d


def test_attention_host_checks(ctmr, native_loaded):
    L, p = ctmr._lib, 4096
    space = lambda **kw: native_loaded.ctmr_masked_attention_workspace_bytes(ctypes.byref(_attention_desc(L, **kw)))
    assert native_loaded.ctmr_masked_attention_workspace_bytes(None) == L.E_INVALID
    for kw in ({"n": 0}, {"lq": 0}, {"lk": 0}, {"q_heads": 3}, {"k_heads": 0}, {"elem": 3}, {"scale": 0.0},
               {"scale": float("nan")}, {"softcap": -1.0}, {"softcap": float("inf")}, {"q_strides": (25600, 32, 130)},
               {"k_strides": (-4, 32, 64)}, {"v_strides": (19200, 33, 64)},
               {"k_strides": (19200, 32, 24)}, {"q_strides": (0, 0, 0)}):
        assert space(**kw) == L.E_INVALID, kw
    for kw in ({"head_dim": 36}, {"head_dim": 136}, {"lq": 1 << 29}, {"k_strides": (0, 0, 1 << 22)},
               {"n": 1 << 20, "q_heads": 1 << 10, "k_heads": 1}):
        assert space(**kw) == L.E_UNSUPPORTED, kw
    # splits: 8 query blocks of 5 key tiles make one part, one token of 16384 keys the most of its 256 tiles
    assert space() == 4 * 0
    assert space(lq=1, lk=16384) == 64 * 4 * (32 + 2) * 4
    assert space(lq=1, lk=16384, n=64) == 2 * 64 * 4 * (32 + 2) * 4

    def call(q=p, plan=None, out=p, ws=p, nbytes=0, **kw):
        return native_loaded.ctmr_masked_attention(ctypes.byref(_attention_desc(L, **kw)), q, p, p, None, None, plan, out,
                                                   None, None, ws, nbytes, None)

    assert call(q=None) == L.E_INVALID and call(out=None) == L.E_INVALID and call(q=p + 8) == L.E_INVALID
    assert call(plan=p + 4) == L.E_INVALID and call(out_strides=(25600, 32, 130)) == L.E_INVALID
    assert call(lq=1, lk=16384, nbytes=100) == L.E_WORKSPACE
    assert call(lq=1, lk=16384, ws=p + 4, nbytes=1 << 30) == L.E_WORKSPACE

    strides = (ctypes.c_int64 * 3)(25600, 32, 128)

    def back(q=p, out=p, lse=p, dout=p, s=strides, dq=None, dq_s=strides, dk=None, ws=p, nbytes=1 << 20, **kw):
        return native_loaded.ctmr_masked_attention_backward(
            ctypes.byref(_attention_desc(L, **kw)), q, p, p, None, None, None, out, None, lse, dout, s, dq, dq_s, dk, strides,
            None, None, ws, nbytes, None)

    assert back() == L.OK  # nothing wanted, nothing launched
    bad = (ctypes.c_int64 * 3)(25600, 32, 126)
    for kw in ({"q": None}, {"out": None}, {"lse": None}, {"dout": None}, {"s": None}, {"dq": p, "dq_s": None},
               {"dout": p + 8}, {"dq": p + 8}, {"s": bad}, {"dq": p, "dq_s": bad}, {"out_strides": (25600, 32, 130)}):
        assert back(**kw) == L.E_INVALID, kw
    assert back(elem=L.ELEM_F16) == L.OK and back(nbytes=100, dq=p) == L.E_WORKSPACE
    assert back(ws=None, dq=p) == L.E_WORKSPACE

    docs = native_loaded.ctmr_documents_bytes
    assert docs(2, 100, 65) == 2 * (128 * 4 + 128 * 4 + 2 * 16 + 2 * 16 + 4 * 48 + 3 * 48 + 4 + 4)
    assert docs(0, 1, 1) == L.E_INVALID and docs(70000, 1, 1) == L.E_UNSUPPORTED
    assert native_loaded.ctmr_documents(2, 100, 65, p, p, p, 10, None) == L.E_WORKSPACE
    assert native_loaded.ctmr_documents(2, 100, 65, None, p, p, 1 << 20, None) == L.E_INVALID


def test_attention_traces(ctmr):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        q, k = (torch.empty(2, h, 6, 32, device="cuda", dtype=torch.bfloat16) for h in (4, 2))
        out, rest, lse = torch.ops.ctmr.masked_attention(q, k, k, None, None, None, 1.0, 0.0, False, 0, True)
        assert out.shape == q.shape and out.transpose(1, 2).is_contiguous() and lse.shape == (2, 4, 6)
        assert rest.shape == out.shape and rest.stride() == out.stride()
        dq, dk, dv = torch.ops.ctmr.masked_attention_backward(q, k, k, None, None, None, out, rest, lse, out, 1.0, 0.0,
                                                              False, 0, True, False)
        assert dq.shape == q.shape and dk.shape == dv.shape == (0,)
        plan = torch.ops.ctmr.documents(*(torch.empty(2, l, device="cuda", dtype=torch.int32) for l in (100, 65)))
        assert plan.dtype == torch.uint8 and plan.numel() == ctmr._lib.lib().ctmr_documents_bytes(2, 100, 65)


def _block_weights(c=64, dtype=torch.float32):
    w = {f"attn.{n}.weight": torch.zeros(c, c, dtype=dtype) for n in ("to_q", "to_k", "to_v", "out_proj")}
    w |= {f"attn.{n}.bias": torch.zeros(c, dtype=dtype) for n in ("to_q", "to_k", "to_v", "out_proj")}
    return w | {"norm.weight": torch.ones(c), "norm.bias": torch.zeros(c)}


def test_packed_volumes(ctmr):
    f = ctmr.differentiable
    one = f.PackedVolumes([(2, 3, 1)], "cpu")
    assert one.documents is None and one.lengths == (6,) and one.positions.dtype == torch.int32
    assert one.positions.tolist() == [[0, 0, 0], [0, 1, 0], [0, 2, 0], [1, 0, 0], [1, 1, 0], [1, 2, 0]]
    for shapes in ((), [(1, 2)], [(2, 0, 1)]):
        with pytest.raises(ValueError, match="shapes must be"):
            f.PackedVolumes(shapes, "cpu")
    with pytest.raises(ValueError, match="on the GPU"):
        f.PackedVolumes([(1, 1, 2), (1, 1, 1)], "cpu")


@pytest.mark.parametrize(
    ("kw", "message"),
    [({"tokens": torch.zeros(5, 64)}, "tokens must be 3-D"), ({"heads": 3}, "not divisible"), ({"heads": 0}, "not divisible"),
     ({"positions": torch.zeros(5, 3)}, "go together"), ({"sections": (8, 12, 12)}, "go together"),
     ({"weights": _block_weights(dtype=torch.bfloat16)}, "to_q.weight is"), ({}, "on the GPU")])
def test_self_attention_tokens_refuses(ctmr, kw, message):
    kw = {"tokens": torch.zeros(1, 5, 64), "weights": _block_weights(), "heads": 2, "scale": 1.0, "include_fc": True} | kw
    with pytest.raises(ValueError, match=message):
        ctmr.differentiable.self_attention_tokens(kw.pop("tokens"), kw.pop("weights"), **kw)


@pytest.mark.parametrize(
    ("volumes", "kw", "message"),
    [([], {}, "one or more"), ([(2, 3, 64)], {}, "one or more"), ([(1, 2, 3, 64), (1, 2, 3, 32)], {}, "differ in channels"),
     ([(1, 2, 3, 64)], {"num_head_channels": 24}, "divisible"), ([(1, 2, 3, 64)], {"num_head_channels": 0}, "divisible"),
     ([(1, 2, 3, 64)], {"packed": (1, 3, 2)}, "packed is for"), ([(1, 2, 3, 64)], {}, "on the GPU")])
def test_spatial_attention_volumes_refuses(ctmr, volumes, kw, message):
    if "packed" in kw:
        kw = kw | {"packed": ctmr.differentiable.PackedVolumes([kw["packed"]], "cpu")}
    kw = {"num_groups": 16, "eps": 1e-6, "num_head_channels": 32, "include_fc": True} | kw
    with pytest.raises(ValueError, match=message):
        ctmr.maisi.spatial_attention_volumes([torch.zeros(s) for s in volumes], _block_weights(), **kw)


def test_leaves_behind_other_operators_are_held(ctmr, monkeypatch):
    f = ctmr.differentiable
    state = {"capturing": False}
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    weight = torch.zeros(3, requires_grad=True)
    out = f._hold(weight * 2, f._graph_token(weight))
    later = out + 1
    del out  # the graph lives on in what was made of it
    gc.collect()
    state["capturing"] = True
    with pytest.raises(RuntimeError, match="outside this capture"):
        f._graph_token(weight)
    del later
    gc.collect()
    assert f._graph_token(weight) is None


def test_calls_that_no_launch_can_take_are_refused(ctmr, native_loaded):
    L, p, f = ctmr._lib, 4096, ctmr.differentiable
    space = lambda **kw: native_loaded.ctmr_masked_attention_workspace_bytes(ctypes.byref(_attention_desc(L, **kw)))
    # 2^23 blocks of 64 rows are the most: their workgroups, two parts each, stay below 2^32 threads
    assert space(n=1 << 19, lq=64, lk=64, q_heads=16, k_heads=16) >= 0
    assert space(n=1 << 19, lq=65, lk=64, q_heads=16, k_heads=16) == L.E_UNSUPPORTED
    assert space(softcap=1e-38, scale=1.0) == L.E_INVALID and space(softcap=1e-20, scale=1.0) >= 0
    with pytest.raises(ValueError, match="too small"):
        _attention(f, softcap=1e-38)
    with pytest.raises(ValueError, match="no heads"):
        _rotary(f, q=(2, 0, 6, 32))
    d = L.RotaryDesc(1, (1 << 31) - 1, 1, 0, 512, 1, (ctypes.c_int32 * 4)(512), 0, 0, 0, 0, 0)
    assert native_loaded.ctmr_rotary(ctypes.byref(d), p, None, p, (ctypes.c_double * 256)(), p, None, None) == L.E_UNSUPPORTED


def test_volumes_are_not_laid_out_inside_a_capture(ctmr, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before a graph is captured"):
        ctmr.differentiable.PackedVolumes([(1, 2, 3)], "cpu")
