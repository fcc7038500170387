"""CPU tests of the position bias: the buckets, its formulas against differences, refusals, host checks, tracing."""

from __future__ import annotations

import ctypes
import math

import position_bias_oracle as oracle
import pytest
import torch


@pytest.mark.parametrize("num_buckets", [4, 6, 8, 10, 16, 32, 64])
@pytest.mark.parametrize("max_distance", [20, 64, 100, 128])
def test_buckets(ctmr, num_buckets, max_distance):
    bucket = ctmr.differentiable.distance_bucket
    got = [bucket(x, num_buckets, max_distance) for x in range(-200, 201)]
    assert got == [oracle.bucket(x, num_buckets, max_distance) for x in range(-200, 201)]
    n = num_buckets // 2
    for sign in (got[200::-1], [b - n for b in got[201:]]):
        assert sign == sorted(sign) and sign[-1] == n - 1 and min(sign) >= 0
    assert got[200] == 0 and bucket(1, num_buckets, max_distance) == n + 1
    assert bucket(max_distance, num_buckets, max_distance) == num_buckets - 1


def test_borders_are_in_the_upper_bucket(ctmr):
    # 16 buckets a sign, 8 of single distances; 8 (128 / 8)^(1 / 4) = 16 is where the eleventh begins
    bucket = ctmr.differentiable.distance_bucket
    assert [bucket(-x, 32, 128) for x in (7, 8, 11, 12, 15, 16, 22, 23, 90, 91)] == [7, 8, 8, 9, 9, 10, 10, 11, 14, 15]


def test_formulas_against_differences():
    """The oracle's gradients are those of its values."""
    torch.manual_seed(0)
    extents, num_buckets = (3, 4), 8
    places = torch.stack([torch.randint(0, e, (12,)) for e in extents], -1)
    which = oracle.numbers(places, places, extents, num_buckets, 5)
    q, k, v, dout = (torch.randn(1, h, 12, 8, dtype=torch.float64) for h in (4, 2, 2, 4))
    table = torch.randn(2, num_buckets, 4, dtype=torch.float64)
    mask = torch.rand(1, 12, 12) < 0.7
    mask[:, 3] = False
    args = dict(scale=0.4, softcap=2.0, mask=mask)
    value = lambda *t: float((oracle.attention(*t, which, **args)[0][0] * dout).sum())
    tensors = [q, k, v, table]
    grads = [g for g, _ in oracle.attention(*tensors, which, **args, dout=dout)[1:]]
    h = 1e-5
    for i, g in enumerate(grads):
        way = torch.randn_like(tensors[i])
        moved = lambda sign: value(*(t + sign * h * way if n == i else t for n, t in enumerate(tensors)))
        # the third derivative's share is h^2, rounding's 2^-52 of a value of about 10 over h
        assert abs((moved(1) - moved(-1)) / (2 * h) - float((g * way).sum())) < 1e-7


def _buckets(f, shape=(6, 2), kshape=None, dtype=torch.int32, **kw):
    return f.PositionBuckets(torch.zeros(shape, dtype=dtype), None if kshape is None else torch.zeros(kshape, dtype=torch.int32),
                             **({"extents": (3, 4)} | kw))


@pytest.mark.parametrize(
    ("kw", "message"),
    [({"extents": ()}, "extents"), ({"extents": (3, 0)}, "extents"), ({"extents": (100, 29)}, "at most 128"),
     ({"extents": (1,) * 5}, "one to four"), ({"num_buckets": 5}, "num_buckets"), ({"num_buckets": 2}, "num_buckets"),
     ({"num_buckets": 514}, "num_buckets"), ({"num_buckets": 32, "max_distance": 8}, "max_distance"),
     ({"max_distance": 1 << 31}, "max_distance"), ({"dtype": torch.int64}, "positions must be"),
     ({"shape": (6, 3)}, "positions must be"), ({"shape": (12,)}, "positions must be"), ({"shape": (0, 2)}, "empty"),
     ({"kshape": (5, 3)}, "key_positions must be"), ({"kshape": (0, 2)}, "empty"),
     ({"shape": (2, 6, 2), "kshape": (3, 6, 2)}, "differ in device or batch"), ({}, "on the GPU")])
def test_position_buckets_refuse(ctmr, kw, message):
    with pytest.raises(ValueError, match=message):
        _buckets(ctmr.differentiable, **kw)


def test_places_that_are_no_tensor_are_refused(ctmr):
    with pytest.raises(ValueError, match="positions must be"):
        ctmr.differentiable.PositionBuckets([[0, 0]], extents=(3, 4))


class _Plan:
    """Buckets without a GPU behind them."""

    extents, num_buckets, items, shape, device = (3, 4), 8, (1, 1), (6, 6), torch.device("cpu")


@pytest.mark.parametrize(
    ("kw", "message"),
    [({"position_bias": None}, "go together"), ({"buckets": None}, "go together"),
     ({"position_bias": torch.zeros(2, 8, 3)}, "position_bias must be"), ({"position_bias": torch.zeros(2, 6, 4)}, "position_bias"),
     ({"position_bias": torch.zeros(2, 8, 4, dtype=torch.float16)}, "position_bias must be"), ({"lq": 5}, "buckets are for"),
     ({"items": (3, 1)}, "buckets are for"), ({"items": (1, 3)}, "buckets are for"), ({"items": (2, 1)}, "on the GPU"),
     ({}, "on the GPU")])
def test_attention_refuses(ctmr, kw, message):
    plan = _Plan()
    plan.items = kw.pop("items", (1, 1))
    q, k = torch.zeros(2, 4, kw.pop("lq", 6), 16), torch.zeros(2, 2, 6, 16)
    args = {"position_bias": torch.zeros(2, 8, 4), "buckets": plan} | kw
    with pytest.raises(ValueError, match=message):
        ctmr.differentiable.attention(q, k, k, scale=1.0, **args)


def test_forward_mode_is_refused(ctmr):
    q, table = torch.zeros(1, 4, 6, 16), torch.zeros(2, 8, 4)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        ctmr.differentiable.attention(q, q, q, scale=1.0, buckets=_Plan(),
                                      position_bias=torch.autograd.forward_ad.make_dual(table, table))


def _desc(L, lq=6, lk=6, qi=1, ki=1, same=1, axes=2, extents=(3, 4, 0, 0), rows=16, elem=0):
    return L.BucketsDesc(lq, lk, qi, ki, same, axes, extents, rows, elem)


def test_host_checks(ctmr, native_loaded):
    L, lib, p = ctmr._lib, native_loaded, 4096
    space = lambda **kw: lib.ctmr_buckets_bytes(ctypes.byref(_desc(L, **kw)))
    # 256 rows of the table, four times 64 words, six one-hot rows of 48 columns (576 bytes) or 96, in pieces of 256 bytes
    assert space() == 1024 + 4 * 256 + 768 and space(same=0) == space()
    assert space(extents=(60, 5, 0, 0)) == 1024 + 4 * 256 + 1280 and space(lq=65, same=0) == space() + 2 * 256
    assert space(same=0, ki=3) == 1024 + 2 * 256 + 2 * 768 + 1792
    assert lib.ctmr_buckets_bytes(None) == L.E_INVALID
    for kw in ({"lq": 0, "lk": 0}, {"qi": 0, "ki": 0}, {"axes": 0}, {"axes": 5}, {"extents": (3, 0, 0, 0)}, {"rows": 0},
               {"rows": 65537}, {"lk": 5}, {"qi": 2}, {"extents": (129, 1, 0, 0)}):
        assert space(**kw) == L.E_INVALID, kw
    assert space(extents=(100, 29, 0, 0)) == L.E_UNSUPPORTED and space(lq=1 << 29, lk=1 << 29) == L.E_UNSUPPORTED
    rows = (ctypes.c_int32 * 12)(*range(12))

    def make(places=p, keys=None, rows=rows, plan=p, nbytes=1 << 20, **kw):
        return lib.ctmr_buckets(ctypes.byref(_desc(L, **kw)), places, keys, rows, plan, nbytes, None)

    assert make(places=None) == L.E_INVALID and make(same=0) == L.E_INVALID and make(rows=None) == L.E_INVALID
    assert make(plan=None) == L.E_INVALID and make(plan=p + 8) == L.E_WORKSPACE and make(nbytes=100) == L.E_WORKSPACE
    assert make(rows=(ctypes.c_int32 * 12)(*[16] * 12)) == L.E_INVALID
    assert make(rows=(ctypes.c_int32 * 12)(*[-1] * 12)) == L.E_INVALID
    strides = (4 * 6 * 16, 16, 4 * 16)
    d = L.MaskedAttentionDesc(1, 6, 6, 4, 4, 16, 0, 0, 0, 1.0, 0.0, 0, strides, strides, strides, strides)

    def forward(q=p, plan=p, table=p, out=p, **kw):
        return lib.ctmr_biased_attention(ctypes.byref(d), ctypes.byref(_desc(L, **kw)), q, p, p, None, None, None, plan, table, 0,
                                         out, None, None, None, 0, None)

    def backward(q=p, plan=p, table=p, dout=p, nbytes=1 << 20, wanted=(p, p, p, p), **kw):
        s = (ctypes.c_int64 * 3)(*strides)
        return lib.ctmr_biased_attention_backward(
            ctypes.byref(d), ctypes.byref(_desc(L, **kw)), q, p, p, None, None, None, plan, table, p, None, p, dout, s,
            wanted[0], s, wanted[1], s, wanted[2], s, wanted[3], p, nbytes, None)

    for call in (forward, backward):
        for kw in ({"q": None}, {"plan": None}, {"plan": p + 4}, {"table": None}, {"lq": 5}, {"lk": 7}, {"qi": 2}, {"ki": 2},
                   {"elem": 3}, {"axes": 0}):
            assert call(**kw) == L.E_INVALID, kw
    assert forward(out=None) == L.E_INVALID and backward(dout=None) == L.E_INVALID and backward(nbytes=64) == L.E_WORKSPACE
    assert backward(wanted=(None,) * 4) == L.OK  # nothing wanted, nothing launched
    need = lib.ctmr_biased_attention_backward_workspace_bytes
    plain = lib.ctmr_masked_attention_backward_workspace_bytes(ctypes.byref(d))
    assert need(ctypes.byref(d), 0) == plain + 4 * 256 * 4 and need(ctypes.byref(d), 1) == plain + 2 * 4 * 256 * 4
    assert need(None, 0) == L.E_INVALID


def test_volumes_have_buckets(ctmr):
    f = ctmr.differentiable
    for shape, message in (((2, 3, 4), "on the GPU"), ((2, 3, 124), "at most 128")):
        with pytest.raises(ValueError, match=message):
            f.PackedVolumes([shape], "cpu").buckets()


@pytest.mark.parametrize(("scale", "softcap", "good"), [(1e-7, 0.0, False), (1e-7, 1.0, True), (1.0, 1e-7, False), (1e-5, 0.0, True)])
def test_scores_too_small_for_a_bias_are_refused(ctmr, native_loaded, scale, softcap, good):
    L, p, q = ctmr._lib, 4096, torch.zeros(1, 4, 6, 16)
    with pytest.raises(ValueError, match="on the GPU" if good else "too small for a position bias"):
        ctmr.differentiable.attention(q, q, q, scale=scale, softcap=softcap, position_bias=torch.zeros(2, 8, 4), buckets=_Plan())
    strides = (4 * 6 * 16, 16, 4 * 16)
    d = L.MaskedAttentionDesc(1, 6, 6, 4, 4, 16, 0, 0, 0, scale, softcap, 0, strides, strides, strides, strides)
    if not good:
        assert native_loaded.ctmr_biased_attention(ctypes.byref(d), ctypes.byref(_desc(L)), p, p, p, None, None, None, p, p, 0,
                                                   p, None, None, None, 0, None) == L.E_UNSUPPORTED


@pytest.mark.filterwarnings("error:Accessing the data pointer")
@pytest.mark.parametrize("tracked", [False, True])
def test_bias_traces(ctmr, monkeypatch, tracked):
    from torch._subclasses.fake_tensor import FakeTensorMode

    f = ctmr.differentiable
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    with FakeTensorMode():
        make = lambda *s, dtype=torch.bfloat16: torch.empty(*s, device="cuda", dtype=dtype)
        q, k = (make(2, 6, h, 32).transpose(1, 2).requires_grad_(tracked) for h in (4, 2))
        plan = f.PositionBuckets(make(6, 3, dtype=torch.int32), extents=(2, 3, 4), num_buckets=8)
        table = make(3, 8, 4, dtype=torch.float32).requires_grad_(tracked)
        out = f.attention(q, k, k, scale=0.2, position_bias=table, buckets=plan)
        assert out.shape == q.shape and out.dtype == q.dtype and out.transpose(1, 2).is_contiguous()
        grads = torch.ops.ctmr.biased_attention_backward(q, k, k, None, None, None, plan.plan, table, out, out,
                                                         make(2, 4, 6, dtype=torch.float32), out, [1, 1, 1, 2, 3, 4], 0.2, 0.0,
                                                         False, 0, True, False, True)
        assert [tuple(t.shape) for t in grads] == [(2, 4, 6, 32), (0,), (0,), (3, 8, 4)]
        weights = {f"attn.{n}.{p}": make(*((64, 64) if p == "weight" else (64,)))
                   for n in ("to_q", "to_k", "to_v", "out_proj") for p in ("weight", "bias")}
        tokens = make(1, 6, 64).requires_grad_(tracked)
        with pytest.raises(KeyError, match="position_bias"):
            f.self_attention_tokens(tokens, weights, heads=4, scale=1.0, include_fc=True, buckets=plan)
        weights["attn.position_bias"] = table
        assert f.self_attention_tokens(tokens, weights, heads=4, scale=1.0, include_fc=True, buckets=plan).shape == tokens.shape
