"""Masked attention with a position bias, and its gradients, in 64 bits, densely from the formulas, with a bound on what
the kernels' roundings can add to each output (counted as in ``attention_oracle``)."""

from __future__ import annotations

import math
from fractions import Fraction

import torch

U = 2.0 ** -24  # half a step of fp32


def bucket(distance, num_buckets, max_distance):
    """With the borders as whole numbers' powers, compared exactly."""
    n, x = num_buckets // 2, abs(distance)
    e = n // 2
    b = x
    if x >= e:
        ratio, base = Fraction(x, e) ** (n - e), Fraction(max_distance, e)
        b = e + max(s for s in range(0, n - e) if s == 0 or base ** s <= ratio)
    return b + (n if distance > 0 else 0)


def numbers(places, key_places, extents, num_buckets, max_distance):
    """Buckets of every pair on each axis, (items, lq, lk, axes)."""
    far = torch.tensor(extents, device=places.device)
    lay = lambda t: torch.minimum((t[None] if t.dim() == 2 else t).long().clamp(min=0), far - 1)
    x = lay(key_places)[:, None] - lay(places)[:, :, None]
    out = torch.empty_like(x)
    for a, e in enumerate(extents):
        of = torch.tensor([bucket(d, num_buckets, max_distance) for d in range(1 - e, e)], device=places.device)
        out[..., a] = of[x[..., a] + e - 1]
    return out


def attention(q, k, v, table, which, *, scale, softcap=0.0, slopes=None, mask=None, dout=None):
    """``[(value, bound)]`` of out and, with ``dout``, of dq, dk, dv and the table's gradient.  ``which``: ``numbers``;
    ``mask`` (B, Lq, Lk)."""
    kind, table_kind = q.dtype, table.dtype
    u = torch.finfo(kind).eps / 2
    half = kind != torch.float32
    parts = 2.0 ** -18 if half else 2.0 ** -27  # what two or three bf16 parts leave of a value
    tiny = 2.0 ** -25 if kind == torch.float16 else 0.0
    q, k, v, table = (t.detach().double() for t in (q, k, v, table))
    b, hq, lq, d = q.shape
    hk, lk = k.shape[1], k.shape[2]
    group = hq // hk
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    if mask is None:
        mask = torch.ones(b, lq, lk, dtype=torch.bool, device=q.device)
    mask = mask[:, None]
    clean = lambda t, rows: torch.where(rows[:, None, :, None], t, 0.0)  # what nothing sees does not count
    q, k, v = clean(q, mask.any(-1)[:, 0]), clean(k, mask.any(-2)[:, 0]), clean(v, mask.any(-2)[:, 0])
    raw = scale * (q @ k.transpose(2, 3))
    es = 6 * math.sqrt(d) * U * scale * (q.abs() @ k.abs().transpose(2, 3)) + 6 * U * raw.abs()
    s, factor = raw, None
    if softcap > 0:
        t = torch.tanh(raw / softcap)
        s, factor = softcap * t, 1 - t * t
        es = es + softcap * (4 * U if not half else 4e-7) * (1 if half else t.abs())
    for a in range(table.shape[0]):
        add = table[a].t()[:, which[..., a]].transpose(0, 1)  # (items, hq, lq, lk)
        s = s + add
        # the parts, the units (a quotient and a product), and the sums' roundings at the scores' size
        es = es + add.abs() * (parts + 8 * U) + 4 * U * s.abs()
    if slopes is not None:
        j, p = torch.arange(lk, device=q.device), torch.arange(lq, device=q.device)[:, None] + (lk - lq)
        bias = slopes.double().reshape(1, -1, 1, 1) * (p - j).abs()
        s, es = s - bias, es + 3 * U * bias
    es = es + 4 * U * (s.abs() + 16)
    s = torch.where(mask, s, -torch.inf)
    es = torch.where(s > -torch.inf, es, 0.0)
    top = s.amax(-1, keepdim=True).clamp(min=-1e300)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total.clamp(min=1e-300), 0.0)
    ep = p * (es + (p * es).sum(-1, keepdim=True) + 6 * math.sqrt(lk) * U)
    out = p @ v
    eo = (ep + u * p + tiny * 2.0 ** -6 * mask) @ v.abs() + u * out.abs() + tiny
    result = [(out, eo)]
    if dout is None:
        return result
    g = clean(dout.detach().double(), mask.any(-1)[:, 0])
    dp = g @ v.transpose(2, 3)
    delta = (g * out).sum(-1, keepdim=True)
    size = g.abs() @ v.abs().transpose(2, 3)
    # delta comes from the output and, of 16 bits, what its rounding left, itself rounded; the weights have twice their bits
    e_out = (ep + u * u * p + tiny * 2.0 ** -6 * mask) @ v.abs() + (u * u if half else u) * out.abs() + tiny * u
    e_inner = 6 * math.sqrt(d) * U * size + (g.abs() * e_out).sum(-1, keepdim=True) + 4 * U * (dp.abs() + delta.abs())
    db = p * (dp - delta)
    edb = ep * (dp - delta).abs() + p * e_inner
    ds, eds = db, edb
    if factor is not None:
        ds = db * factor
        eds = edb * factor.abs() + db.abs() * (2 * es / softcap + 8e-7)
    eds = eds + u * ds.abs()
    if tiny:
        eds = eds + mask * (2.0 ** -39 * 2 * d * float(g.abs().max()) * float(v.abs().max()))
    dq = scale * (ds @ k)
    edq = scale * ((eds + 6 * math.sqrt(lk) * U * ds.abs()) @ k.abs()) + u * dq.abs() + tiny
    shared = lambda t: t.reshape(b, hk, group, lk, d).sum(2)
    rows = 6 * math.sqrt(lq * group) * U
    dk = shared(scale * (ds.transpose(2, 3) @ q))
    edk = shared(scale * ((eds + rows * ds.abs()).transpose(2, 3) @ q.abs())) + u * dk.abs() + tiny
    dv = shared(p.transpose(2, 3) @ g)
    edv = shared((ep + u * p + rows * p + tiny * 2.0 ** -15 * mask).transpose(2, 3) @ g.abs()) + u * dv.abs() + tiny
    dt, edt = torch.zeros_like(table), torch.zeros_like(table)
    # parts, and fp32 sums over a row's keys and 128 rows
    edb = edb + db.abs() * (parts + 6 * (math.sqrt(lk) + 12) * U)
    for a in range(table.shape[0]):
        for n in range(table.shape[1]):
            pairs = (which[..., a] == n)[:, None]
            dt[a, n] = torch.where(pairs, db, 0.0).sum((0, 2, 3))
            edt[a, n] = torch.where(pairs, edb, 0.0).sum((0, 2, 3))
    tu = torch.finfo(table_kind).eps / 2
    edt = edt + (tu + 2.0 ** -40) * dt.abs() + (2.0 ** -25 if table_kind == torch.float16 else 2.0 ** -134)
    return result + [(dq, edq), (dk, edk), (dv, edv), (dt, edt)]
