"""CPU tests of the differentiable operators' guards: caps, forward-mode tangents, leaves in captures, threads, tracing."""

from __future__ import annotations

import ctypes
import sys
import threading

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


@pytest.fixture
def capture(ctmr, monkeypatch):
    """Sets whether a capture is under way."""
    state = {"on": False}
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["on"])
    return lambda on: state.update(on=on)


def _made(f, kind):
    """A leaf, and what an operator's own preparation makes of it before autograd sees it."""
    big = torch.zeros(4, 6, 8, 16)
    if kind == "a slice":
        leaf = big[0:2].requires_grad_()
        return leaf, leaf
    if kind == "a transposed leaf":
        leaf = big.transpose(1, 2).requires_grad_()
        return leaf, leaf.contiguous()
    if kind == "a strided leaf, norm":
        leaf = big[..., ::2].requires_grad_()
        return leaf, leaf.contiguous()
    if kind == "heads, rotary":
        leaf = big.transpose(2, 3).requires_grad_()
        assert not leaf.is_contiguous()
        return leaf, f._heads(leaf)
    if kind == "heads, attention":
        leaf = torch.zeros(4 * 6 * 8 * 16 + 1)[1:].view(4, 6, 8, 16).requires_grad_()
        made = f._attention_heads(leaf)
        assert made is not leaf
        return leaf, made
    leaf = big.requires_grad_()
    return leaf, {"a view": leaf.flatten(0, 1), "views of views": leaf[1:].transpose(0, 1)[2].unbind(0)[1],
                  "a cast": leaf.to(torch.bfloat16), "a cast view": leaf.to(torch.float16)[1].transpose(0, 1).contiguous()}[kind]


@pytest.mark.parametrize("kind", ["a slice", "a transposed leaf", "a strided leaf, norm", "heads, rotary", "heads, attention",
                                  "a view", "views of views", "a cast", "a cast view"])
def test_leaves_behind_copies_casts_and_views_are_held(ctmr, capture, kind):
    f = ctmr.differentiable
    leaf, made = _made(f, kind)
    token = f._graph_token(made)
    assert token is not None
    capture(True)
    for t in (leaf, made, leaf.reshape(-1), leaf.to(torch.bfloat16)):
        with pytest.raises(RuntimeError, match="outside this capture"):
            f._graph_token(t)
    assert f._graph_token(torch.zeros(2, requires_grad=True), leaf.detach()) is None
    del token
    assert f._graph_token(leaf) is None


def test_a_held_leaf_is_found_whichever_way_it_was_recorded(ctmr, capture):
    f = ctmr.differentiable
    leaf = torch.zeros(3, 4).requires_grad_()
    token = f._graph_token(leaf)
    capture(True)
    with pytest.raises(RuntimeError, match="outside this capture"):
        f._graph_token(leaf.T.contiguous().half())
    del token


def _calls(f, dtype=torch.float32):
    """Each operator as a function of one of its tensors, and that tensor."""
    x, w = torch.zeros(2, 5, 8, dtype=dtype), torch.ones(8, dtype=dtype)
    q, k = torch.zeros(2, 4, 6, 16, dtype=dtype), torch.zeros(2, 2, 6, 16, dtype=dtype)
    at = torch.zeros(6, 1)
    norm = lambda x, w, b: f.group_norm(x, w, b, num_groups=2, eps=1e-6)
    turn = lambda q, k, at: f.rotary(q, k, at, sections=(16,))[0]
    att = lambda q, k, v, s=None: f.attention(q, k, v, scale=1.0, slopes=s)
    return {"norm x": (lambda t: norm(t, w, w), x), "norm weight": (lambda t: norm(x, t, w), w),
            "norm bias": (lambda t: norm(x, w, t), w), "rotary q": (lambda t: turn(t, k, at), q),
            "rotary k": (lambda t: turn(q, t, at), k), "rotary positions": (lambda t: turn(q, k, t), at),
            "attention q": (lambda t: att(t, k, k), q), "attention k": (lambda t: att(q, t, k), k),
            "attention v": (lambda t: att(q, k, t), k), "attention slopes": (lambda t: att(q, k, k, t), torch.zeros(4))}


NAMES = ["norm x", "norm weight", "norm bias", "rotary q", "rotary k", "rotary positions", "attention q", "attention k",
         "attention v", "attention slopes"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("tracked", [False, True])
def test_forward_mode_is_refused(ctmr, name, tracked):
    """A tangent would vanish without a word: the kernels have reverse-mode gradients only."""
    call, t = _calls(ctmr.differentiable)[name]
    t.requires_grad_(tracked and name != "attention slopes")
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)))
        with pytest.raises(ValueError, match="on the GPU"):  # no tangent: as outside
            call(t)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(call, (t.detach(),), (torch.ones_like(t),))


def test_forward_mode_through_the_block_is_refused(ctmr):
    c = 16
    w = {f"attn.{n}.{p}": torch.zeros(*((c, c) if p == "weight" else (c,)))
         for n in ("to_q", "to_k", "to_v", "out_proj") for p in ("weight", "bias")}
    call = lambda t: ctmr.differentiable.self_attention_tokens(t, w, heads=2, scale=1.0, include_fc=True)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(call, (torch.zeros(1, 5, c),), (torch.ones(1, 5, c),))


def test_a_capture_while_other_threads_record(ctmr, monkeypatch):
    """The living graphs are walked while others come and go in threads of their own."""
    f, main = ctmr.differentiable, threading.get_ident()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: threading.get_ident() == main)
    stop, failures = threading.Event(), []

    def record():
        try:
            leaf = torch.zeros(2, requires_grad=True)
            kept = []
            while not stop.is_set():
                kept.append(f._graph_token(leaf))
                if len(kept) > 200:
                    kept.clear()
        except Exception as error:
            failures.append(error)

    threads = [threading.Thread(target=record) for _ in range(4)]
    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        for t in threads:
            t.start()
        leaf = torch.zeros(2, requires_grad=True)
        for _ in range(1500):
            assert f._graph_token(leaf) is None
    finally:
        sys.setswitchinterval(interval)
        stop.set()
        for t in threads:
            t.join()
    assert not failures


@pytest.mark.filterwarnings("error:Accessing the data pointer")
@pytest.mark.parametrize("tracked", [False, True])
def test_public_operators_trace(ctmr, monkeypatch, tracked):
    """On fake tensors: shapes, types and strides without an address being read."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    f = ctmr.differentiable
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    with FakeTensorMode():
        make = lambda *s, dtype=torch.bfloat16: torch.empty(*s, device="cuda", dtype=dtype)
        q, k = (make(2, 6, h, 32).transpose(1, 2).requires_grad_(tracked) for h in (4, 2))
        odd = make(2 * 2 * 6 * 32 + 1)[1:].view(2, 2, 6, 32)  # copied: its address is no multiple of 16 bytes
        ids = make(2, 6, dtype=torch.int32)
        for v in (k, odd, make(2, 2, 6, 64)[..., ::2]):
            out = f.attention(q, k, v, scale=0.2, documents=f.Documents(ids))
            assert out.shape == q.shape and out.dtype == q.dtype and out.transpose(1, 2).is_contiguous()
        turned = f.rotary(q, k, make(6, 2, dtype=torch.int32), sections=(8, 8))
        assert [t.shape for t in turned] == [q.shape, k.shape]
        x, w = make(2, 5, 8).requires_grad_(tracked), make(8, dtype=torch.float32)
        assert f.group_norm(x, w, w, num_groups=2, eps=1e-6).shape == x.shape
        weights = {f"attn.{n}.{p}": make(*((64, 64) if p == "weight" else (64,)))
                   for n in ("to_q", "to_k", "to_v", "out_proj") for p in ("weight", "bias")}
        tokens = make(1, 5, 64).requires_grad_(tracked)
        assert f.self_attention_tokens(tokens, weights, heads=2, scale=1.0, include_fc=True).shape == tokens.shape


def test_sizes_past_32_bits_are_refused(ctmr):
    """Sizes that would come out small in the descriptors' 32 bits: 2^32 + 64 rows are not 64."""
    f, big = ctmr.differentiable, 2 ** 32 + 64
    wide = lambda *s: torch.zeros(1).expand(*s)
    row = torch.zeros(1, 1, 64, 8)
    calls = [lambda: f.attention(wide(1, 1, big, 8), row, row, scale=1.0),
             lambda: f.attention(row, wide(1, 1, big, 8), wide(1, 1, big, 8), scale=1.0),
             lambda: f.attention(wide(big, 1, 1, 8), wide(big, 1, 1, 8), wide(big, 1, 1, 8), scale=1.0),
             lambda: f.attention(wide(1, big, 1, 8), row[:, :, :1], row[:, :, :1], scale=1.0),
             lambda: f.rotary(wide(1, 1, big, 8), None, wide(big, 1), sections=(8,)),
             lambda: f.rotary(wide(big, 1, 1, 8), None, wide(1, 1), sections=(8,)),
             lambda: f.rotary(wide(1, big, 1, 8), wide(1, big, 1, 8), wide(1, 1), sections=(8,)),
             lambda: f.group_norm(wide(big, 1, 8), torch.zeros(8), torch.zeros(8), num_groups=2, eps=1e-6),
             lambda: f.group_norm(wide(1, 1, big), wide(big), wide(big), num_groups=1, eps=1e-6),
             lambda: f.Documents(torch.zeros(1, dtype=torch.int32).expand(1, big)),
             lambda: f.Documents(torch.zeros(1, 64, dtype=torch.int32), torch.zeros(1, dtype=torch.int32).expand(1, big))]
    for call in calls:
        with pytest.raises(ValueError, match="2\\^31"):
            call()
