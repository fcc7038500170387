"""CPU tests of what is derived of weights that a recorded graph writes."""

from __future__ import annotations

import gc
import threading

import pytest
import torch


@pytest.fixture
def captured(ctmr, monkeypatch):
    """Notes the writes of a call as if it were recorded."""
    def note(tensors, capturing=True):
        with monkeypatch.context() as m:
            m.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
            ctmr.ops._note_writes(tensors)
    yield note
    ctmr.ops._rewritten.clear()


def _derived(ff, cache, lock, *sources):
    return ff.cached_derived(cache, lock, tuple(map(id, sources)), sources, lambda: sum(t.double() for t in sources))


def test_what_replays_write_is_derived_anew(ctmr, captured):
    ff, cache, lock = ctmr.fast_fp32, {}, threading.RLock()
    row, other = torch.zeros(8), torch.ones(4)
    w = row[:4]
    first = _derived(ff, cache, lock, w, other)
    assert _derived(ff, cache, lock, w, other) is first
    captured([row[4:]], capturing=False)  # outside a capture a call raises the version instead
    assert _derived(ff, cache, lock, w, other) is first
    captured([row[:2].detach()])  # another view of the same memory
    torch.from_numpy(row.numpy()).fill_(2.0)  # as a replay writes: no version shows it
    assert w._version == 0 and bool((_derived(ff, cache, lock, w, other) == 3).all())
    torch.from_numpy(row.numpy()).fill_(5.0)
    assert bool((_derived(ff, cache, lock, w, other) == 6).all())
    assert _derived(ff, {}, lock, other) is not None and bool((_derived(ff, {}, lock, other) == 1).all())


def test_kept_again_once_settled(ctmr, captured):
    ff, lock = ctmr.fast_fp32, threading.RLock()
    w, cache = torch.zeros(4), {}
    ff.register_cache(cache, lock)
    try:
        _derived(ff, cache, lock, w)
        captured([w])
        torch.from_numpy(w.numpy()).fill_(2.0)
        ff.settle_weights([w])
        kept = _derived(ff, cache, lock, w)
        assert bool((kept == 2).all()) and _derived(ff, cache, lock, w) is kept
        captured([w])
        assert _derived(ff, cache, lock, w) is not kept
    finally:
        ff._caches.remove((cache, lock))


def test_steps_of_inference_tensors_are_noticed(ctmr, monkeypatch):
    """They have no version; a step marks them instead."""
    f, ff, lock = ctmr.differentiable, ctmr.fast_fp32, threading.RLock()
    monkeypatch.setattr(f, "_on_gpu", lambda t, name: None)
    monkeypatch.setattr(f, "_stream_of", lambda t: None)
    with torch.inference_mode():
        w = torch.zeros(4)
        monkeypatch.setattr(f.ops, "adamw", lambda *a: w.add_(1))
    other, cache = torch.zeros(4), {}
    o = f.AdamW([w, other])
    kept = _derived(ff, cache, lock, w)
    assert _derived(ff, cache, lock, w) is kept
    try:
        with torch.inference_mode():
            o.step([torch.zeros(4), torch.zeros(4)])
        assert bool((_derived(ff, cache, lock, w) == 1).all())
        assert _derived(ff, cache, lock, other) is _derived(ff, cache, lock, other)
    finally:
        ctmr.ops._rewritten.clear()


def test_marks_end_with_their_memory(ctmr, captured):
    t = torch.zeros(4)
    captured([t, t.view(2, 2)])
    view = t[1:]
    del t
    gc.collect()
    assert ctmr.ops._is_rewritten(view) and len(ctmr.ops._rewritten) == 1
    del view
    gc.collect()
    assert not ctmr.ops._rewritten
