"""The differentiable operators where offsets pass 32 bits, with very many batch items, and on two streams at once."""

from __future__ import annotations

import attention_oracle as oracle
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lq", [1, 200])
def test_attention_to_the_end_of_a_long_cache(ctmr, dev, lq):
    """8 heads of 128 over 2.2 million keys, 2^31 values and more: only the last 1000 keys are of the rows' document."""
    f, (h, d, lk, tail) = ctmr.differentiable, (8, 128, 2_200_000, 1000)
    g = torch.Generator(device=dev).manual_seed(1)
    q, dout = (torch.randn(1, lq, 2 * h, d, device=dev, generator=g).bfloat16().transpose(1, 2) for _ in range(2))
    k, v = (torch.full((1, lk, h, d), 3.0, device=dev, dtype=torch.bfloat16).transpose(1, 2) for _ in range(2))
    assert k.numel() > 2 ** 31
    for t in (k, v):
        t[:, :, -tail:] = torch.randn(1, h, tail, d, device=dev, generator=g)
    key_ids = torch.zeros(1, lk, device=dev, dtype=torch.int32)
    key_ids[:, -tail:] = 1
    documents = f.Documents(torch.ones(1, lq, device=dev, dtype=torch.int32), key_ids)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = f.attention(*leaves, scale=d ** -0.5, documents=documents)
    dq, dk, dv = torch.autograd.grad(out, leaves, dout)
    want = oracle.attention(q, k[:, :, -tail:], v[:, :, -tail:], scale=d ** -0.5, dout=dout)
    for got, w, name in zip((out.detach(), dq, dk[:, :, -tail:], dv[:, :, -tail:]), want, ("out", "dq", "dk", "dv")):
        oracle.check(got, w, name)
    for t in (dk, dv):
        assert not bool(t[:, :, :-tail].any())


def test_norm_of_more_than_2_31_values(ctmr, dev):
    """A volume that repeats has its part's statistics: each repeat gives the part's output and gradient."""
    f, c, rows, times = ctmr.differentiable, 64, 1 << 20, 33
    g = torch.Generator(device=dev).manual_seed(2)
    part, grad = (torch.randn(1, rows, c, device=dev, generator=g).bfloat16() for _ in range(2))
    w, b = (torch.randn(c, device=dev, generator=g) for _ in range(2))
    results = []
    for n in (1, times):
        x = part.repeat(1, n, 1).requires_grad_()
        y = f.group_norm(x, w, b, num_groups=32, eps=1e-6, apply_silu=True)
        dx, = torch.autograd.grad(y, x, grad.repeat(1, n, 1))
        results.append((y.detach(), dx))
        del x
    assert results[1][0].numel() > 2 ** 31
    for one, all_ in zip(*results):
        first, last = all_[:, :rows], all_[:, -rows:]
        assert torch.equal(first, last)
        # statistics that differ by fp32 roundings, 2^-23 of values up to 8, may move a value to bf16's next: a step
        step = 2.0 ** -7 * one.float().abs() + 2.0 ** -20
        assert bool(((first.float() - one.float()).abs() <= step).all())


def test_rotary_past_2_31_values(ctmr, dev):
    f, (h, l, d) = ctmr.differentiable, (32, 530_000, 128)
    q = torch.empty(1, l, h, d, device=dev, dtype=torch.bfloat16).transpose(1, 2)
    assert q.numel() > 2 ** 31
    q[:, :, :100] = q[:, :, -100:] = torch.randn(1, h, 100, d, device=dev)
    positions = torch.randint(0, 4096, (l, 2), device=dev, dtype=torch.int32)
    positions[-100:] = positions[:100]
    out, _ = f.rotary(q, None, positions, sections=(64, 64))
    assert torch.equal(out[:, :, -100:], out[:, :, :100])
    assert torch.equal(out[:, :, :100], f.rotary(q[:, :, :100], None, positions[:100], sections=(64, 64))[0])


def test_many_batch_items(ctmr, dev):
    n = 70_000
    g = torch.Generator(device=dev).manual_seed(3)
    q, k, v, dout = (torch.randn(n, 1, l, 8, device=dev, generator=g) for l in (1, 3, 3, 1))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = ctmr.differentiable.attention(*leaves, scale=0.3)
    got = [out.detach(), *torch.autograd.grad(out, leaves, dout)]
    for t, w in zip(got, oracle.attention(q, k, v, scale=0.3, dout=dout)):
        oracle.check(t, w)
    with pytest.raises(RuntimeError):  # the norm's and the plans' grids end at 65535 items
        ctmr.differentiable.group_norm(torch.zeros(n, 1, 8, device=dev), torch.ones(8, device=dev), torch.zeros(8, device=dev),
                                       num_groups=2, eps=1e-6)


def test_two_streams_at_once(ctmr, dev):
    """Two training passes in flight together give what each gives alone."""
    f = ctmr.differentiable

    def work(seed):
        g = torch.Generator(device=dev).manual_seed(seed)
        x, dy = (torch.randn(1, 3000, 96, device=dev, generator=g).bfloat16() for _ in range(2))
        return x, dy, torch.randn(3000, 3, device=dev, generator=g), torch.ones(96, device=dev), torch.zeros(96, device=dev)

    def run(x, dy, positions, w, b):
        leaf = x.detach().requires_grad_()
        y = f.group_norm(leaf, w, b, num_groups=8, eps=1e-6, apply_silu=True)
        q = y.unflatten(-1, (3, 32)).transpose(1, 2)
        q, k = f.rotary(q, q, positions, sections=(8, 12, 12))
        out = f.attention(q, k, q, scale=0.2, prefix=700).transpose(1, 2).flatten(2)
        return out.detach(), torch.autograd.grad(out, leaf, dy)[0]

    inputs = [work(s) for s in range(2)]
    want = [run(*i) for i in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, i in zip(streams, inputs):
            with torch.cuda.stream(s):
                got.append(run(*i))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
