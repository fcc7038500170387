"""The masked attention and its gradients in 64 bits, densely from the formulas, with a bound on what the kernels'
roundings can add to each output."""

from __future__ import annotations

import math

import torch

U = 2.0 ** -24  # half a step of fp32


def visible(b, lq, lk, device, ids=None, key_ids=None, prefix=None):
    mask = torch.ones(b, lq, lk, dtype=torch.bool, device=device)
    if ids is not None:
        key_ids = ids if key_ids is None else key_ids
        mask &= (ids[:, :, None] == key_ids[:, None, :]) & (ids[:, :, None] >= 0)
    if prefix is not None:
        j, p = torch.arange(lk, device=device), torch.arange(lq, device=device)[:, None] + (lk - lq)
        first = torch.as_tensor(prefix, device=device).reshape(-1, 1, 1)
        mask &= (j <= p)[None] | (j < first)
    return mask


def attention(q, k, v, *, scale, softcap=0.0, slopes=None, mask=None, dout=None):
    """``[(value, bound)]`` of out and, with ``dout``, of dq, dk and dv.  ``mask`` (B, Lq, Lk).

    The bounds count: fp32 sums of n terms as 6 sqrt(n) half steps (errors of either sign) of the terms' sizes; each
    softmax weight and each ds rounded by half a step of the type; out and the gradients rounded once."""
    kind = q.dtype
    u = torch.finfo(kind).eps / 2
    tiny = 2.0 ** -25 if kind == torch.float16 else 0.0
    q, k, v = (t.detach().double() for t in (q, k, v))
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
        es = es + softcap * (4 * U if kind == torch.float32 else 4e-7) * (1 if kind != torch.float32 else t.abs())
    if slopes is not None:
        j, p = torch.arange(lk, device=q.device), torch.arange(lq, device=q.device)[:, None] + (lk - lq)
        bias = slopes.double().reshape(1, -1, 1, 1) * (p - j).abs()
        s, es = s - bias, es + 3 * U * bias
    # the exponent's base-2 argument is rounded at its own size, the maximum's share is common to a row
    es = es + 4 * U * (s.abs() + 16)
    s = torch.where(mask, s, -torch.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-1e300)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total.clamp(min=1e-300), 0.0)
    es = torch.where(mask, es, 0.0)
    ep = p * (es + (p * es).sum(-1, keepdim=True) + 6 * math.sqrt(lk) * U)  # of a weight, its rounding aside
    out = p @ v
    eo = (ep + u * p + tiny * 2.0 ** -6 * mask) @ v.abs() + u * out.abs() + tiny
    result = [(out, eo)]
    if dout is None:
        return result
    g = clean(dout.detach().double(), mask.any(-1)[:, 0])
    dp = g @ v.transpose(2, 3)
    delta = (g * out).sum(-1, keepdim=True)
    inner = (dp - delta) * (1 if factor is None else factor)
    ds = p * inner
    size = g.abs() @ v.abs().transpose(2, 3)
    e_inner = 6 * math.sqrt(d) * U * size + (g.abs() * eo).sum(-1, keepdim=True) + 4 * U * (dp.abs() + delta.abs())
    if factor is not None:
        e_inner = e_inner + (dp - delta).abs() * (2 * es / softcap + 8e-7)
    eds = ep * inner.abs() + p * e_inner + u * ds.abs()
    if tiny:
        # ds is raised to below 2^15 by a bound of twice d max |g| max |v|, p by 2^15: half a step of the least
        # values, 2^-25, is 2^-39 of the bound (a power of two above it aside), and 2^-40 of p
        eds = eds + mask * (2.0 ** -39 * 2 * d * float(g.abs().max()) * float(v.abs().max()))
    dq = scale * (ds @ k)
    edq = scale * ((eds + 6 * math.sqrt(lk) * U * ds.abs()) @ k.abs()) + u * dq.abs() + tiny
    shared = lambda t: t.reshape(b, hk, group, lk, d).sum(2)
    rows = 6 * math.sqrt(lq * group) * U
    dk = shared(scale * (ds.transpose(2, 3) @ q))
    edk = shared(scale * ((eds + rows * ds.abs()).transpose(2, 3) @ q.abs())) + u * dk.abs() + tiny
    dv = shared(p.transpose(2, 3) @ g)
    edv = shared((ep + u * p + rows * p + tiny * 2.0 ** -15 * mask).transpose(2, 3) @ g.abs()) + u * dv.abs() + tiny
    return result + [(dq, edq), (dk, edk), (dv, edv)]


def check(got, want, name=""):
    value, bound = want
    err = (got.double() - value).abs()
    bad = ~(err <= bound + 1e-30)
    assert not bool(bad.any()), (name, int(bad.sum()), float((err / (bound + 1e-30)).nan_to_num(1e9).max()),
                                 bad.nonzero()[0].tolist())
