"""Operators of the networks' attention blocks with gradients (reverse mode), on fp32, bf16 and fp16 tensors.

The reference is inference only; these are what fine-tuning its attention blocks (``attention.py``) needs beside the
fp32 surface of ``fast_fp32``, whose convolutions have no gradients:

* ``group_norm``  channels-last group norm + SiLU
* ``rotary``      rotary positions over one to four axes (depth, height, width) for q and k
* ``attention``   attention with grouped heads, a tanh cap, a distance bias, documents and a prefix
* ``Documents``   which tokens of a batch belong together (volumes of different sizes in one row, padding)
* ``PackedVolumes``  the documents and voxel positions of several volumes in one row
* ``self_attention_tokens``  projections, rotary positions and attention of tokens
  (``maisi.spatial_attention_volumes`` is the networks' block over it)
"""

from __future__ import annotations

import math
import weakref
from collections.abc import Mapping, Sequence
from typing import Optional, Union

import torch
import torch.nn.functional as F
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import ops

# Autograd graphs recorded outside any capture that hold leaves, by their identity (see _graph_token).  A plain dictionary:
# its single operations, and the list of its values, are whole whatever other threads and the collector do meanwhile.
_eager_graphs: dict[int, "weakref.ref[_EagerGraph]"] = {}


class _EagerGraph:
    """The leaves of one recorded call; lives as long as the call's autograd node."""

    __slots__ = ("leaves", "__weakref__")

    def __init__(self, leaves: list[Tensor]):
        self.leaves = [weakref.ref(t) for t in leaves]
        key = id(self)
        _eager_graphs[key] = weakref.ref(self, lambda _, graphs=_eager_graphs: graphs.pop(key, None))


def _leaf(t: Tensor) -> Optional[Tensor]:
    """The leaf that ``t`` is, or is made of by operators of one input: views, copies, casts."""
    if t.is_leaf:
        return t
    node = t.grad_fn
    while node is not None and node.name() != "torch::autograd::AccumulateGrad":
        inputs = node.next_functions
        node = inputs[0][0] if len(inputs) == 1 else None
    return None if node is None else node.variable


def _graph_token(*tensors: Optional[Tensor]) -> Optional[_EagerGraph]:
    """What an autograd node keeps while it lives: a mark on the leaves of a call made outside a capture.

    A leaf has one gradient accumulator for all graphs that hold it, bound to the stream of the first.  A
    backward pass captured into a HIP graph while an eager graph of the same leaf lives would make the
    capture wait for a stream outside it, which ends the process; such a call is refused here.  Leaves count
    that these operators were given, or a view, copy or cast of.

    Raises:
        RuntimeError: in a capture, if a leaf belongs to a living graph recorded outside it."""
    leaves = [_leaf(t) for t in tensors if t is not None and t.requires_grad]
    leaves = [t for t in leaves if t is not None]
    if not leaves:
        return None
    if not torch.cuda.is_current_stream_capturing():
        return _EagerGraph(leaves)
    for graph in list(_eager_graphs.values()):
        token = graph()
        for ref in () if token is None else token.leaves:
            held = ref()
            if held is not None and any(held is t for t in leaves):
                raise RuntimeError("an autograd graph recorded outside this capture still holds one of its leaves; "
                                   "drop that graph (its outputs and losses) before capturing, or capture a detached "
                                   "copy of the leaf")
    return None


def _hold(out: Tensor, token: Optional[_EagerGraph]) -> Tensor:
    """``out``, whose graph keeps ``token`` while it lives: for calls whose leaves reach autograd through other
    operators than these."""
    if token is not None and out.grad_fn is not None:
        out.grad_fn.metadata["ctmr.leaves"] = token
    return out


def _check_capture(captured: bool) -> None:
    """Refuses a backward pass in another capture state than its forward pass."""
    if torch.cuda.is_current_stream_capturing() != captured:
        raise RuntimeError("forward and backward must both be inside a graph capture or both outside")


def _activation(t, name: str, ndim: Optional[int] = None) -> Tensor:
    if not isinstance(t, Tensor):
        raise ValueError(f"{name} must be a torch.Tensor")
    if ndim is not None and t.dim() != ndim:
        raise ValueError(f"{name} must be {ndim}-D; got shape {tuple(t.shape)}")
    if t.dtype not in ops.ELEMENTS:
        raise ValueError(f"{name} must be float32, bfloat16 or float16; got {t.dtype}")
    return t


def _sizes(*sizes: int) -> None:
    """Refuses sizes that the descriptors' 32 bits would cut short."""
    if max(sizes) >= 1 << 31:
        raise ValueError(f"sizes must be below 2^31; got {sizes}")


def _no_tangents(*tensors: Optional[Tensor]) -> None:
    """Refuses dual tensors, whose tangents no kernel carries on."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                              for t in tensors):
        raise NotImplementedError("there are no forward-mode derivatives of this operator; use reverse mode")


def _on_gpu(t: Tensor, name: str) -> None:
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be on the GPU (there is no CPU path); got {t.device}")


def _like(t, like: Tensor, name: str, ndim: Optional[int] = None) -> Tensor:
    _activation(t, name, ndim)
    if t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} is {t.dtype} on {t.device}; expected {like.dtype} on {like.device}")
    return t


# ---------------------------------------------------------------------------
# group norm
# ---------------------------------------------------------------------------
class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, silu):
        y, saved = ops.norm_forward(x, weight, bias, groups, eps, silu)
        ctx.save_for_backward(x, weight, bias, saved)
        ctx.silu = silu
        ctx.token, ctx.captured = _graph_token(x, weight, bias), torch.cuda.is_current_stream_capturing()
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _check_capture(ctx.captured)
        x, weight, bias, saved = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        dx, dw, db = ops.norm_backward(x, dy.contiguous(), weight, bias, saved, ctx.silu, want_x, want_w or want_b)
        return dx if want_x else None, dw if want_w else None, db if want_b else None, None, None, None


def group_norm(x: Tensor, weight: Tensor, bias: Tensor, *, num_groups: int, eps: float,
               apply_silu: bool = False) -> Tensor:
    """Group norm, and SiLU with ``apply_silu``, of channels-last ``x`` ``(N, ..., C)``; differentiable.

    ``x`` is fp32, bf16 or fp16 (a copy is made where it is not contiguous); ``weight`` and ``bias`` ``(C,)``
    are fp32 or ``x``'s type.  Statistics are over each batch item's voxels and ``C / num_groups`` channels, with the
    biased variance.  Their sums, and the gradients', are fp64, but for 32 voxels of a channel at a time in fp32 (of
    differences to one of the values; again in fp64 where squares leave fp32's range).  The output has ``x``'s type, the
    gradients their inputs' types.

    Raises:
        ValueError: on other types, devices or shapes, channels that the groups do not divide, or an ``eps``
            that is negative or not finite.
        NotImplementedError: on forward-mode (dual) tensors."""
    _activation(x, "x")
    if x.dim() < 2:
        raise ValueError(f"x must be (N, ..., C); got shape {tuple(x.shape)}")
    c, groups, eps = int(x.shape[-1]), int(num_groups), float(eps)
    if groups < 1 or c < 1 or c % groups:
        raise ValueError(f"{c} channels are not divisible by {num_groups} groups")
    if not (math.isfinite(eps) and eps >= 0.0):
        raise ValueError(f"eps must be finite and not negative; got {eps}")
    for t, name in ((weight, "weight"), (bias, "bias")):
        _activation(t, name, 1)
        if int(t.shape[0]) != c or t.device != x.device or t.dtype not in (torch.float32, x.dtype):
            raise ValueError(f"{name} must be ({c},) in float32 or {x.dtype} on {x.device}; got "
                             f"{tuple(t.shape)} {t.dtype} on {t.device}")
    if weight.dtype != bias.dtype:
        raise ValueError(f"weight and bias differ in type: {weight.dtype} and {bias.dtype}")
    _sizes(int(x.shape[0]), c)
    _no_tangents(x, weight, bias)
    _on_gpu(x, "x")
    x, weight, bias = x.contiguous(), weight.contiguous(), bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or bias.requires_grad):
        return _GroupNorm.apply(x, weight, bias, groups, eps, bool(apply_silu))
    return ops.norm_forward(x, weight, bias, groups, eps, bool(apply_silu))[0]


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------
def _heads(t: Tensor) -> Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, sections, base):
        out, k_out = ops.rotary(q, k, positions, sections, base, False)
        ctx.save_for_backward(positions)
        ctx.sections, ctx.base, ctx.with_k = sections, base, k is not None
        ctx.token, ctx.captured = _graph_token(q, k), torch.cuda.is_current_stream_capturing()
        return out, (k_out if k is not None else None)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        _check_capture(ctx.captured)
        positions, = ctx.saved_tensors
        if not ctx.with_k:
            dk = None
        dq, dk_out = ops.rotary(_heads(dq), None if dk is None else _heads(dk), positions, ctx.sections, ctx.base, True)
        return dq, (dk_out if ctx.with_k else None), None, None, None


def rotary(q: Tensor, k: Optional[Tensor], positions: Tensor, *, sections: Sequence[int],
           base: float = 10000.0) -> tuple[Tensor, Optional[Tensor]]:
    """Rotary positions of ``(B, H, L, D)`` heads over one to four axes; differentiable in ``q`` and ``k``.

    ``positions`` ``(L, A)`` or ``(B, L, A)`` (int32, int64 or fp32; fractions are allowed) holds a token's place on
    each axis, such as a voxel's (depth, height, width).  The first ``sum(sections)`` values of a head are a
    section per axis; value ``i`` of a section of width ``w`` and value ``i + w / 2`` turn by ``position * base **
    (-2 i / w)``; the rest of the head passes.  ``k`` may have fewer heads than ``q``, or be None.  Angles are
    computed in 64 bits.  The outputs have the inputs' type and lie as ``(B, L, H, D)`` in memory.

    Raises:
        ValueError: on other types, devices or shapes, sections that are odd, not positive, wider than the head
            or not one for each axis, or a base that is not positive and finite.
        NotImplementedError: on forward-mode (dual) tensors."""
    _activation(q, "q", 4)
    b, hq, l, d = (int(v) for v in q.shape)
    if hq < 1:
        raise ValueError("q has no heads")
    if k is not None:
        _like(k, q, "k", 4)
        if int(k.shape[0]) != b or int(k.shape[2]) != l or int(k.shape[3]) != d:
            raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} differ in more than their heads")
    sections = tuple(int(w) for w in sections)
    if not 1 <= len(sections) <= 4 or any(w < 2 or w % 2 for w in sections):
        raise ValueError(f"sections must be one to four positive even widths; got {sections}")
    if d % 2 or sum(sections) > d or d > 2 * ops._lib.ROTARY_MAX_PAIRS:
        raise ValueError(f"sections {sections} do not fit heads of {d} values (even, at most 512)")
    base = float(base)
    if not (math.isfinite(base) and base > 0.0):
        raise ValueError(f"base must be positive and finite; got {base}")
    if not isinstance(positions, Tensor) or positions.dtype not in ops.POSITION_TYPES or positions.device != q.device:
        raise ValueError("positions must be an int32, int64 or float32 tensor on q's device")
    if tuple(positions.shape) not in ((l, len(sections)), (1, l, len(sections)), (b, l, len(sections))):
        raise ValueError(f"positions must be ({l}, {len(sections)}) or ({b}, {l}, {len(sections)}); got "
                         f"{tuple(positions.shape)}")
    _sizes(b, hq, l)
    _no_tangents(q, k, positions)
    _on_gpu(q, "q")
    positions = positions.detach().contiguous()
    q, k = _heads(q), None if k is None else _heads(k)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _Rotary.apply(q, k, positions, sections, base)
    out, k_out = ops.rotary(q, k, positions, sections, base, False)
    return out, (None if k is None else k_out)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _stream_of(t: Tensor) -> Optional[int]:
    """The stream that ``t`` is being made on; None on the host and where calls are traced."""
    return ops._raw_stream(t.device) if t.is_cuda and type(t) is Tensor else None


def _used(t: Tensor, made: Optional[int]) -> Tensor:
    """``t``, which was made on the stream ``made``: its memory stays until the current stream's work so far and the
    call to come are done, also if its owner is gone before.  (A captured graph's user keeps the owner.)"""
    if made is not None and ops._raw_stream(t.device) != made and not torch.cuda.is_current_stream_capturing():
        t.record_stream(torch.cuda.current_stream(t.device))
    return t


class Documents:
    """Which query rows and keys belong together, laid out once for every ``attention`` of a batch.

    ``ids`` ``(B, Lq)`` int32 holds each query row's document, ``key_ids`` ``(B, Lk)`` each key's (the same rows
    if left out).  A row sees the keys of its own document; negative ids are padding, which sees and is seen by
    nothing.  Ids may come in any order, but only rows of a document that lie side by side let the kernels skip
    the rest.  The ids are copied: changing the tensors afterwards changes nothing here.  Like a tensor, the documents are
    made on the current stream, which other streams wait for, and outlive the graphs that captured them.

    Raises:
        ValueError: on ids that are not (B, L) int32 tensors of one device and batch on the GPU, or empty."""

    def __init__(self, ids: Tensor, key_ids: Optional[Tensor] = None):
        key_ids = ids if key_ids is None else key_ids
        for t, name in ((ids, "ids"), (key_ids, "key_ids")):
            if not isinstance(t, Tensor) or t.dtype != torch.int32 or t.dim() != 2:
                raise ValueError(f"{name} must be a (B, L) int32 tensor")
            if t.numel() == 0:
                raise ValueError(f"{name} is empty: {tuple(t.shape)}")
        if ids.device != key_ids.device or ids.shape[0] != key_ids.shape[0]:
            raise ValueError("ids and key_ids differ in device or batch")
        _sizes(*ids.shape, *key_ids.shape)
        _on_gpu(ids, "ids")
        self.shape = (int(ids.shape[0]), int(ids.shape[1]), int(key_ids.shape[1]))
        self.plan = ops.documents(ids.contiguous(), key_ids.contiguous())
        self._stream = _stream_of(self.plan)

    @property
    def device(self) -> torch.device:
        return self.plan.device


def _address(t: Tensor) -> int:
    """Where ``t`` starts; what is traced has no address, and memory of its own starts on a multiple of 16 bytes."""
    if type(t) in (Tensor, torch.nn.Parameter) and not torch.compiler.is_compiling():
        return t.data_ptr()
    return t.storage_offset() * t.element_size()


def _attention_heads(t: Tensor) -> Tensor:
    """``t`` with a unit last stride and 16-byte aligned rows that do not overlap, in a stride that the kernels address."""
    size = t.element_size()
    if t.stride(3) == 1 and _address(t) % 16 == 0:
        strides = ops._head_strides(t)
        if (all(s * size % 16 == 0 for s in strides) and strides[2] * size <= 1 << 23
                and (t.shape[2] <= 1 or strides[2] >= t.shape[3])):
            return t
    return t.contiguous() if not t.is_contiguous() else t.clone(memory_format=torch.contiguous_format)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, slopes, prefixes, plan, scale, softcap, prefixed, prefix):
        out, rest, lse = ops.masked_attention(q, k, v, slopes, prefixes, plan, scale, softcap, prefixed, prefix, True)
        ctx.save_for_backward(q, k, v, slopes, prefixes, plan, out, rest, lse)
        ctx.args = (scale, softcap, prefixed, prefix)
        ctx.token, ctx.captured = _graph_token(q, k, v), torch.cuda.is_current_stream_capturing()
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        _check_capture(ctx.captured)
        want_q, want_k, want_v = ctx.needs_input_grad[:3]
        dq, dk, dv = ops.masked_attention_backward(*ctx.saved_tensors, _attention_heads(dout), *ctx.args, want_q,
                                                   want_k or want_v)
        return (dq if want_q else None, dk if want_k else None, dv if want_v else None, *(None,) * 7)


def attention(q: Tensor, k: Tensor, v: Tensor, *, scale: float, softcap: float = 0.0, slopes: Optional[Tensor] = None,
              prefix: Union[int, Tensor, None] = None, documents: Optional[Documents] = None) -> Tensor:
    """Masked attention of ``(B, H, L, D)`` heads; differentiable in ``q``, ``k`` and ``v``.

    ``q`` has ``Hq`` heads and ``Lq`` rows, ``k`` and ``v`` ``Hk`` heads and ``Lk`` keys, ``Hq`` a multiple of
    ``Hk`` (query head ``h`` reads key head ``h // (Hq // Hk)``); ``D`` is a multiple of 8 up to 128.  With
    ``p_i = i + Lk - Lq`` the place of row ``i`` among the keys:

    * ``softcap`` > 0 caps the scores ``s = scale * q.k`` as ``softcap * tanh(s / softcap)``;
    * ``slopes`` ``(Hq,)`` fp32 subtract ``slopes[h] * |p_i - j|`` (no gradient);
    * ``prefix``, an int or a ``(B,)`` int32 tensor, hides key ``j`` from row ``i`` unless ``j <= p_i`` or ``j <
      prefix`` (0: each row sees the keys up to its own place; None: every key);
    * ``documents`` hides the keys of other documents and padding (``Documents``).

    A row that sees no key gives zeros and gets no gradient.  What masked places hold has no effect, NaN included.
    Scores are fp32: their size (the distance's too) is expected below some 2^20, where the weights still have digits.
    Statistics and sums are fp32; the softmax weights, and in the gradients those of the scores, are rounded to the
    inputs' type for their products (in fp16 raised by powers of two that keep them in its range).  The output has
    ``q``'s type and lies as ``(B, Lq, Hq, D)`` in memory, so merging the heads is a view.

    Raises:
        ValueError: on other types, devices or shapes, a scale that is not positive and finite, a cap that is
            negative or too small or large beside it, or slopes that need a gradient.
        NotImplementedError: on forward-mode (dual) tensors."""
    _activation(q, "q", 4)
    _like(k, q, "k", 4)
    _like(v, q, "v", 4)
    b, hq, lq, d = (int(s) for s in q.shape)
    hk, lk = int(k.shape[1]), int(k.shape[2])
    if k.shape != v.shape or int(k.shape[0]) != b or int(k.shape[3]) != d:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit each other")
    if hk < 1 or hq < 1 or hq % hk:
        raise ValueError(f"{hq} query heads are not a multiple of {hk} key heads")
    _sizes(b, hq, lq, lk)
    if d < 8 or d % 8 or d > 128:
        raise ValueError(f"head width must be a multiple of 8 up to 128; got {d}")
    scale, softcap = float(scale), float(softcap)
    if not (math.isfinite(scale) and scale > 0.0) or not (math.isfinite(softcap) and softcap >= 0.0):
        raise ValueError(f"scale must be positive, softcap not negative, both finite; got {scale} and {softcap}")
    if softcap > 0.0 and not scale / softcap < 1e30:
        raise ValueError(f"softcap {softcap} is too small for a scale of {scale}")
    if softcap > 1e30 or (softcap > 0.0 and scale / softcap < 1e-30):
        raise ValueError(f"softcap {softcap} is too large for a scale of {scale}")
    if slopes is not None:
        if not isinstance(slopes, Tensor) or slopes.dtype != torch.float32 or tuple(slopes.shape) != (hq,) or (
                slopes.device != q.device):
            raise ValueError(f"slopes must be a ({hq},) float32 tensor on {q.device}")
        if slopes.requires_grad and torch.is_grad_enabled():
            raise ValueError("slopes have no gradient; pass them detached")
        slopes = slopes.contiguous()
    prefixes, value = None, 0
    if isinstance(prefix, Tensor):
        if prefix.dtype != torch.int32 or tuple(prefix.shape) != (b,) or prefix.device != q.device:
            raise ValueError(f"prefix must be an int or a ({b},) int32 tensor on {q.device}")
        prefixes = prefix.contiguous()
    elif prefix is not None:
        value = max(0, min(int(prefix), lk))
    if documents is not None and (documents.shape != (b, lq, lk) or documents.device != q.device):
        raise ValueError(f"documents are for {documents.shape} rows on {documents.device}; got {(b, lq, lk)} on "
                         f"{q.device}")
    needs = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    _no_tangents(q, k, v, slopes)
    _on_gpu(q, "q")
    q, k, v = _attention_heads(q), _attention_heads(k), _attention_heads(v)
    plan = None if documents is None else _used(documents.plan, documents._stream)
    if needs:
        return _Attention.apply(q, k, v, slopes, prefixes, plan, scale, softcap, prefix is not None, value)
    return ops.masked_attention(q, k, v, slopes, prefixes, plan, scale, softcap, prefix is not None, value, False)[0]


# ---------------------------------------------------------------------------
# the networks' attention over these operators
# ---------------------------------------------------------------------------
class PackedVolumes:
    """Volumes of different sizes as one row of tokens, voxel after voxel in (depth, height, width) order.

    ``shapes`` are the volumes' (D, H, W).  ``positions`` ``(L, 3)`` int32 are the voxels' places for ``rotary``,
    ``documents`` keeps the volumes apart in ``attention`` (None for a single volume, which needs no mask) and
    ``lengths`` are the volumes' voxel counts.  Laid out once for every block that works on the batch.

    Raises:
        ValueError: on no volumes, or a shape that is not three positive sizes.
        RuntimeError: inside a graph capture (it copies from the host)."""

    def __init__(self, shapes: Sequence[Sequence[int]], device: Union[torch.device, str, int] = "cuda"):
        self.shapes = tuple(tuple(int(s) for s in shape) for shape in shapes)
        if not self.shapes or any(len(s) != 3 or min(s) < 1 for s in self.shapes):
            raise ValueError(f"shapes must be one or more (D, H, W) of positive sizes; got {self.shapes}")
        self.lengths = tuple(d * h * w for d, h, w in self.shapes)
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("volumes are laid out before a graph is captured, not inside the capture")
        grids = [torch.stack(torch.meshgrid(*(torch.arange(s, dtype=torch.int32) for s in shape), indexing="ij"),
                             dim=-1).reshape(-1, 3) for shape in self.shapes]
        self.positions = torch.cat(grids).to(device)
        self._stream = _stream_of(self.positions)
        self.documents = None
        if len(self.shapes) > 1:
            ids = torch.repeat_interleave(torch.arange(len(self.shapes), dtype=torch.int32), torch.tensor(self.lengths))
            self.documents = Documents(ids[None].to(self.positions.device))


def self_attention_tokens(tokens: Tensor, weights: Mapping[str, Tensor], *, heads: int, scale: float, include_fc: bool,
                          documents: Optional[Documents] = None, positions: Optional[Tensor] = None,
                          sections: Optional[Sequence[int]] = None, base: float = 10000.0, prefix: str = "attn",
                          qkv_bias: bool = True) -> Tensor:
    """Q/K/V projections, rotary positions, self-attention and optional ``out_proj`` on ``(B, L, C)`` tokens;
    differentiable in the tokens and the weights.

    Takes the weights of ``fast_fp32.self_attention_tokens`` in the tokens' type.  ``documents`` keeps tokens apart;
    ``positions`` with ``sections`` (see ``rotary``) turns q and k, and is left out for attention without positions.

    Raises:
        ValueError: on tokens that are not (B, L, C), heads that do not divide C, positions without sections or the
            reverse, and what ``rotary`` and ``attention`` refuse."""
    _activation(tokens, "tokens", 3)
    n, length, c = (int(s) for s in tokens.shape)
    heads = int(heads)
    if heads < 1 or c < 1 or c % heads:
        raise ValueError(f"{c} channels are not divisible by {heads} heads")
    if (positions is None) != (sections is None):
        raise ValueError("positions and sections go together")
    names = [f"{prefix}.to_{m}" for m in ("q", "k", "v")]
    used = [weights[f"{m}.{part}"] for m in [*names, *([f"{prefix}.out_proj"] if include_fc else [])]
            for part in (("weight", "bias") if qkv_bias or m.endswith("out_proj") else ("weight",))]
    token = _graph_token(tokens, *used) if torch.is_grad_enabled() and tokens.is_cuda else None
    w = torch.cat([_like(weights[f"{m}.weight"], tokens, f"{m}.weight", 2) for m in names])
    b = torch.cat([_like(weights[f"{m}.bias"], tokens, f"{m}.bias", 1) for m in names]) if qkv_bias else None
    # (B, L, 3, H, D): q, k and v are strided views of the one product
    q, k, v = F.linear(tokens, w, b).reshape(n, length, 3, heads, c // heads).permute(2, 0, 3, 1, 4).unbind(0)
    if positions is not None:
        q, k = rotary(q, k, positions, sections=sections, base=base)
    merged = attention(q, k, v, scale=scale, documents=documents).transpose(1, 2).reshape(n, length, c)
    if include_fc:
        merged = F.linear(merged, _like(weights[f"{prefix}.out_proj.weight"], tokens, f"{prefix}.out_proj.weight", 2),
                          _like(weights[f"{prefix}.out_proj.bias"], tokens, f"{prefix}.out_proj.bias", 1))
    return _hold(merged, token)
