"""``differentiable.rotary`` and its gradients against 64 bits: sections, types, strides, far positions."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _exact(t, positions, sections, base, way):
    parts = list(torch.split(t.double(), [*sections, t.shape[-1] - sum(sections)], dim=-1))
    if positions.dim() == 2:
        positions = positions[None]
    for a, w in enumerate(sections):
        turn = base ** (torch.arange(0, w, 2, device=t.device, dtype=torch.float64) / -w)
        angle = (way * positions[:, :, a, None].double() * turn)[:, None]
        p, q = parts[a].chunk(2, -1)
        parts[a] = torch.cat([p * angle.cos() - q * angle.sin(), p * angle.sin() + q * angle.cos()], -1)
    return torch.cat(parts, -1)


def _size(t, sections):
    """|p| + |q| of each value's pair, zero where the head passes."""
    parts = list(torch.split(t.double().abs(), [*sections, t.shape[-1] - sum(sections)], dim=-1))
    for a in range(len(sections)):
        p, q = parts[a].chunk(2, -1)
        parts[a] = torch.cat([p + q, p + q], -1)
    parts[-1] = torch.zeros_like(parts[-1])
    return torch.cat(parts, -1)


def _check(got, t, positions, sections, base=10000.0, way=1.0):
    want = _exact(t, positions, sections, base, way)
    # the part of a turn rounds by 2^-26, 2 pi of it an angle's error; sine and cosine to 2 steps of 2^-24; two
    # products and a sum round by 2^-24 each
    err = (2 * math.pi * 2.0 ** -26 + 5 * 2.0 ** -24) * _size(t, sections)
    tol = torch.finfo(t.dtype).eps / 2 * want.abs() + err
    if t.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    assert got.dtype == t.dtype and got.shape == t.shape
    assert bool(((got.double() - want).abs() <= tol).all())


# (b, hq, hk, l, d, sections): vectors of 8, 4, 2 and 1; a rest that passes; one axis over the whole head; one token
CASES = [(1, 8, 8, 256, 32, (8, 12, 12)), (2, 6, 2, 77, 64, (16, 24, 24)), (1, 4, 1, 1, 128, (32, 48, 48)),
         (3, 2, 2, 33, 80, (20, 20, 20)), (1, 3, 3, 130, 18, (6, 4)), (2, 2, 1, 50, 64, (64,)), (1, 1, 1, 9, 2, (2,)),
         (1, 2, 2, 65, 96, (32, 16, 16, 32)), (1, 1, 1, 40, 512, (512,)), (2, 5, 0, 21, 24, (8, 8)),
         (1, 32, 8, 4099, 128, (32, 48, 48))]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_values_and_gradients(ctmr, dev, case, dtype):
    b, hq, hk, l, d, sections = case
    g = torch.Generator(device=dev).manual_seed(1)
    r = lambda h: torch.randn(b, l, h, d, device=dev, generator=g).to(dtype).transpose(1, 2)
    pos = torch.randint(-50, 4096, (b, l, len(sections)), device=dev, generator=g)
    for kind, positions in ((torch.int32, pos.int()), (torch.int64, pos[0]), (torch.float32, pos.float() + 0.25)):
        q, k = r(hq).requires_grad_(), r(hk).requires_grad_() if hk else None
        out, k_out = ctmr.differentiable.rotary(q, k, positions, sections=sections)
        assert out.transpose(1, 2).is_contiguous()
        _check(out.detach(), q.detach(), positions, sections)
        dq = r(hq)
        if hk:
            _check(k_out.detach(), k.detach(), positions, sections)
            dk = r(hk).contiguous()
            gq, gk = torch.autograd.grad((out, k_out), (q, k), (dq, dk))
            _check(gk, dk, positions, sections, way=-1.0)
        else:
            assert k_out is None
            gq, = torch.autograd.grad(out, q, dq)
        _check(gq, dq, positions, sections, way=-1.0)


def test_far_positions_and_base(ctmr, dev):
    q = torch.randn(1, 2, 64, 32, device=dev)
    pos = (torch.arange(64, device=dev) * 310_003)[:, None]  # 2e7: an fp32 angle would be off by 1
    _check(ctmr.differentiable.rotary(q, None, pos, sections=(32,), base=500.0)[0], q, pos, (32,), base=500.0)


def test_strided_heads_and_odd_addresses(ctmr, dev):
    f, pos = ctmr.differentiable, torch.arange(60, device=dev).reshape(20, 3)
    fused = torch.randn(2, 20, 3 * 64 + 1, device=dev).to(torch.bfloat16)
    for at in (0, 1):  # columns of a fused projection, at an address that no vector divides
        q, k = (fused[..., at + o:at + o + 64].unflatten(-1, (2, 32)).transpose(1, 2) for o in (0, 64))
        for got, t in zip(f.rotary(q, k, pos, sections=(8, 12, 12)), (q, k)):
            _check(got, t, pos, (8, 12, 12))
    wide = torch.randn(1, 1, 20, 32, device=dev).expand(2, 4, 20, 32)
    _check(f.rotary(wide, None, pos, sections=(8, 12, 12))[0], wide, pos, (8, 12, 12))
    back = torch.randn(2, 2, 32, 20, device=dev).transpose(2, 3)
    _check(f.rotary(back, None, pos, sections=(8, 12, 12))[0], back, pos, (8, 12, 12))


def test_passing_values_keep_their_bits(ctmr, dev):
    q = torch.randn(1, 2, 10, 48, device=dev).to(torch.bfloat16)
    q[0, 0, 3, 40], q[0, 1, 5, 32] = math.inf, math.nan
    out = ctmr.differentiable.rotary(q, None, torch.arange(10, device=dev)[:, None], sections=(32,))[0]
    assert torch.equal(out[..., 32:].contiguous().view(torch.int16), q[..., 32:].contiguous().view(torch.int16))
    assert bool(out[..., :32].isfinite().all())


def test_differences(ctmr, dev):
    q, u, dy = (torch.randn(1, 3, 17, 32, device=dev) for _ in range(3))
    pos = torch.arange(51, device=dev).reshape(17, 3)
    run = lambda t: ctmr.differentiable.rotary(t, None, pos, sections=(8, 12, 12))[0]
    leaf = q.clone().requires_grad_()
    g, = torch.autograd.grad(run(leaf), leaf, dy)
    slope = float(((run(q + u) - run(q - u)).double() * dy.double()).sum()) / 2
    # linear in q: only rounding, some 2^-24 of each of 1632 values
    assert abs(slope - float((g.double() * u.double()).sum())) <= 1e-5 * float(u.norm() * dy.norm())


def test_streams_and_graph(ctmr, dev):
    f = ctmr.differentiable
    make = lambda: [torch.randn(1, 300, 4, 32, device=dev).to(torch.bfloat16).transpose(1, 2) for _ in range(4)]
    pos = torch.arange(900, device=dev).reshape(300, 3)

    def step(q, k, dq, dk):
        q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
        out = f.rotary(q, k, pos, sections=(8, 12, 12))
        return [t.detach() for t in (*out, *torch.autograd.grad(out, (q, k), (dq, dk)))]

    static = make()
    want = step(*static)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step(*static)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for _ in range(3):
        fresh = make()
        for s, t in zip(static, fresh):
            s.copy_(t)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, step(*fresh)))


def test_empty(ctmr, dev):
    pos = torch.zeros(0, 1, device=dev, dtype=torch.int32)
    q = torch.empty(2, 3, 0, 8, device=dev, requires_grad=True)
    out, _ = ctmr.differentiable.rotary(q, None, pos, sections=(8,))
    assert out.shape == q.shape and torch.autograd.grad(out, q, torch.empty_like(out))[0].shape == q.shape
