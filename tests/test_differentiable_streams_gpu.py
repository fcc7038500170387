"""What a caller keeps for many calls (documents, packed volumes) used on another stream than its own: the memory stays
as it is until that stream's work is done, also where the caller lets go of it first."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _while_another_stream_is_busy(make, use, bytes_of):
    """``use(make())`` behind 50 ms of other work on a second stream; what was made is dropped and its size allocated and
    filled on the first stream meanwhile.  Returns the result and whether the new memory was the old."""
    side = torch.cuda.Stream()
    kept = make()
    at, size = bytes_of(kept).data_ptr(), bytes_of(kept).numel() * bytes_of(kept).element_size()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
        result = use(kept)
    del kept
    fresh = [torch.empty(size, dtype=torch.uint8, device="cuda").fill_(255) for _ in range(3)]
    reused = any(t.data_ptr() == at for t in fresh)
    torch.cuda.synchronize()
    return result, reused


def test_documents(ctmr, dev):
    f = ctmr.differentiable
    g = torch.Generator(device=dev).manual_seed(0)
    q, k, v = (torch.randn(1, 2, 3000, 32, device=dev, generator=g) for _ in range(3))
    ids = (torch.arange(3000, device=dev) // 700).int()[None]
    make = lambda: f.Documents(ids)
    use = lambda documents: f.attention(q, k, v, scale=0.2, documents=documents)
    want = use(make())
    torch.cuda.synchronize()
    got, reused = _while_another_stream_is_busy(make, use, lambda documents: documents.plan)
    assert not reused and torch.equal(got, want)


def test_packed_volumes(ctmr, dev):
    shapes, c = [(9, 8, 7), (3, 5, 6)], 64
    g = torch.Generator(device=dev).manual_seed(1)
    volumes = [torch.randn(*s, c, device=dev, generator=g) for s in shapes]
    w = {f"attn.{n}.{p}": torch.randn(*((c, c) if p == "weight" else (c,)), device=dev, generator=g) / 8
         for n in ("to_q", "to_k", "to_v", "out_proj") for p in ("weight", "bias")}
    w |= {"norm.weight": torch.ones(c, device=dev), "norm.bias": torch.zeros(c, device=dev)}
    make = lambda: ctmr.differentiable.PackedVolumes(shapes, dev)
    use = lambda packed: ctmr.maisi.spatial_attention_volumes(volumes, w, num_groups=16, eps=1e-6, num_head_channels=32,
                                                              include_fc=True, packed=packed, sections=(8, 12, 12))
    want = use(make())
    torch.cuda.synchronize()
    for part in (lambda packed: packed.positions, lambda packed: packed.documents.plan):
        got, reused = _while_another_stream_is_busy(make, use, part)
        assert not reused and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("kind", ["a slice", "a cast", "a strided leaf"])
def test_a_refused_capture_leaves_the_process_sound(ctmr, dev, kind):
    """The call is refused before it records anything; once the eager graph is gone the same capture works."""
    f = ctmr.differentiable
    g = torch.Generator(device=dev).manual_seed(2)
    big = torch.randn(4, 60, 64, device=dev, generator=g)
    leaf = {"a slice": big[1:3], "a cast": big, "a strided leaf": big[..., ::2]}[kind].requires_grad_()
    w, b = torch.ones(leaf.shape[-1], device=dev), torch.zeros(leaf.shape[-1], device=dev)
    dout = torch.randn(leaf.shape, device=dev, generator=g)

    def step():
        x = leaf.to(torch.bfloat16) if kind == "a cast" else leaf
        y = f.group_norm(x, w, b, num_groups=4, eps=1e-6, apply_silu=True)
        return y, torch.autograd.grad(y, leaf, dout.to(y.dtype))[0]

    kept, want = step()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="outside this capture"):
        with torch.cuda.graph(graph):
            step()
    del kept
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, grad = step()
    for _ in range(3):
        grad.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, want)
