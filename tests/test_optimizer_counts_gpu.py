"""``AdamW`` with parameters that some steps leave out: each one's bias corrections go by its own steps."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of fp32
RATE = 1e-2


def _list(dev, sizes, seed, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [scale * torch.randn(*s, device=dev, generator=g) for s in sizes]


def _pattern(count, steps, seed):
    """Which parameters have a gradient in each step; the first always has one, the second from the last step on only."""
    g = torch.Generator().manual_seed(seed)
    return [[i == 0 or (i != 1 and float(torch.rand((), generator=g)) < 0.6) or (i == 1 and t == steps - 1)
             for i in range(count)] for t in range(steps)]


def _inside(ours, theirs, steps):
    for a, b in zip(ours, theirs):
        # each step has at most some twelve half steps of what it moves, five rates at most (a gradient that stands out moves
        # (1 - b1) / (1 - b2)^(1/2) = 3.2 of them), and one of the value, below the start's and what the steps moved
        bound = steps * (12 * U * 5 * RATE + U * (b.abs() + steps * 5 * RATE))
        assert bool(((a.detach().double() - b.detach()).abs() <= bound).all())


@pytest.mark.parametrize("count", [3, 81, 2100])
def test_late_gradients_agree_with_the_library_optimizer(ctmr, dev, count):
    """None for several steps, then a gradient; lists of more absent parameters than a launch takes."""
    steps = 12 if count < 1000 else 3
    sizes = [(1 + (37 * i) % 50,) for i in range(count - 1)] + [(5001,)]
    ours = _list(dev, sizes, 0, scale=0.1)
    theirs = [torch.nn.Parameter(t.double()) for t in ours]
    o = ctmr.differentiable.AdamW(ours, lr=RATE, weight_decay=0.05, max_norm=1.0)
    r = torch.optim.AdamW(theirs, lr=RATE, weight_decay=0.05, foreach=False)
    for t, given in enumerate(_pattern(count, steps, count)):
        grads = [g if use else None for g, use in zip(_list(dev, sizes, t + 1), given)]
        o.step(grads)
        for p, g in zip(theirs, grads):
            p.grad = None if g is None else g.double()
        torch.nn.utils.clip_grad_norm_(theirs, 1.0)
        r.step()
    _inside(ours, theirs, steps)
    assert int(o.steps) == steps and int(o.missed[0]) == 0 and int(o.missed[1]) == steps - 1
    own = torch.tensor([int(r.state[p]["step"]) if p in r.state else 0 for p in theirs], device=dev)
    assert torch.equal(o.steps - o.missed, own)


def test_the_first_gradient_moves_by_the_rate(ctmr, dev):
    late, other = torch.zeros(100, device=dev), torch.zeros(10, device=dev, dtype=torch.bfloat16)
    o = ctmr.differentiable.AdamW([other, late], lr=RATE, weight_decay=0.0)
    for _ in range(200):
        o.step([torch.ones_like(other), None])
    o.step([torch.ones_like(other), torch.full_like(late, -3.0)])
    # m / (1 - b1) = g and v / (1 - b2) = g^2 at its first step: the rate, to eps / 3 and some half steps
    assert bool(((late - RATE).abs() <= RATE * (1e-8 / 3 + 12 * U)).all())


def test_skipped_steps_are_nobodys(ctmr, dev):
    params = _list(dev, [(70,), (50,)], 0)
    o = ctmr.differentiable.AdamW(params, skip_non_finite=True)
    bad = torch.full((70,), math.inf, device=dev)
    for g in (bad, torch.ones(70, device=dev), bad, torch.ones(70, device=dev)):
        o.step([g, None])
    assert int(o.steps) == 2 and o.missed.tolist() == [0, 2]


def test_captured_steps_that_leave_parameters_out(ctmr, dev):
    sizes = [(3001,), (64,), (5,), (0,)]
    grads = _list(dev, sizes, 1)
    make = lambda: (p := _list(dev, sizes, 0), ctmr.differentiable.AdamW(p, lr=RATE))
    eager, o = make()
    for i in range(4):
        o.step([grads[0], grads[1] if i % 2 else None, None, grads[3]])
        o.step(grads)
    params, c = make()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph, second in zip(graphs, (None, grads[1])):
        with torch.cuda.graph(graph):
            c.step([grads[0], second, None, grads[3]])
            c.step(grads)
    for i in range(4):
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        make()[1].step(grads)
    for a, b in zip((*eager, *o.state_dict().values()), (*params, *c.state_dict().values())):
        assert torch.equal(a, b)
    assert c.missed.tolist() == [0, 2, 4, 0]


def test_states_move_to_another_optimizer(ctmr, dev):
    sizes = [(300,), (40,)]
    params, grads = _list(dev, sizes, 0), _list(dev, sizes, 1)
    o = ctmr.differentiable.AdamW(params, lr=RATE)
    for _ in range(3):
        o.step([grads[0], None])
    copies = [p.clone() for p in params]
    other = ctmr.differentiable.AdamW(copies, lr=RATE)
    other.load_state_dict(o.state_dict())
    for opt in (o, other):
        opt.step(grads)
    assert all(torch.equal(a, b) for a, b in zip(params, copies)) and other.missed.tolist() == [0, 3]
