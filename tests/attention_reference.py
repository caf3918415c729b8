"""Attention over a paged cache and the append to it, from the definitions in 64 bits, with bounds of what 16-bit results may
be off by."""
import math

import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def gather(pages, table_row, n):
    """Rows 0 .. n - 1 of a sequence: [kv_heads, n, head_dim] in 64 bits."""
    page = pages.shape[2]
    pos = torch.arange(n, device=pages.device)
    return pages[table_row.long()[pos // page], :, pos % page].double().transpose(0, 1)


def attention(q, k_pages, v_pages, table, lens, cu, scale=None):
    """(out, bound) in 64 bits for every row of q; rows of no sequence are NaN.

    The bound, with u the half step of the type and e = 2^-24 that of fp32: the result is rounded once (u |o|); every
    exp(x - max) is rounded to the type before it multiplies its value (u relative, and at most half the smallest subnormal;
    it may be taken against a maximum that is up to 2^8 too small, which leaves the relative error as it is); a score is a
    sum of D products in fp32, off by (D + 2) e sum |q k| scale, which counts twice, in the weight and in their sum; sums
    over n keys are off by n e relative, twice; the exponential itself by 2^-22, and by |x - max| e for the rounding of its argument
    (counted with the scores: |x - max| is below twice their largest sum of magnitudes).  A type's overflow is not in it."""
    T, H, D = q.shape
    Hkv = k_pages.shape[1]
    group = H // Hkv
    scale = D ** -0.5 if scale is None else scale
    u, e = half_step(q.dtype), 2.0 ** -24
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[q.dtype]
    out = torch.full((T, H, D), math.nan, dtype=torch.float64, device=q.device)
    bound = torch.full_like(out, math.nan)
    cu = list(range(T + 1)) if cu is None else cu.tolist()
    for b, length in enumerate(lens.tolist()):
        t0, t1 = cu[b], cu[b + 1]
        n = t1 - t0
        if n == 0:
            continue
        if length == 0:
            out[t0:t1], bound[t0:t1] = 0.0, 0.0
            continue
        k = gather(k_pages, table[b], length).repeat_interleave(group, 0)
        v = gather(v_pages, table[b], length).repeat_interleave(group, 0)
        qb = q[t0:t1].double().transpose(0, 1)
        last = length - n + torch.arange(n, device=q.device)
        hidden = torch.arange(length, device=q.device)[None, :] > last[:, None]
        x = (qb @ k.transpose(1, 2) * scale).masked_fill(hidden, -math.inf)
        mass = (qb.abs() @ k.abs().transpose(1, 2) * abs(scale)).masked_fill(hidden, 0.0).amax(-1, keepdim=True)
        top = x.amax(-1, keepdim=True)
        p = torch.where(hidden, 0.0, torch.exp(x - torch.where(top == -math.inf, 0.0, top)))
        l = p.sum(-1, keepdim=True)
        vz = torch.where(torch.isfinite(v), v, 0.0)  # (a hidden value's infinity is no part of a sum)
        o = torch.where(l > 0, p @ vz / l, 0.0)
        a = torch.where(l > 0, p @ vz.abs() / l, 0.0)
        vmax = vz.abs().amax(dim=(1, 2), keepdim=True)
        rel = u + 2 * (D + 4) * e * mass + 2 * length * e + 2.0 ** -21
        out[t0:t1] = o.transpose(0, 1)
        bound[t0:t1] = (u * o.abs() + rel * a + torch.where(l > 0, length * tiny * vmax, 0.0) + tiny).transpose(0, 1)
    return out, bound


def check_attention(got, want, bound):
    """Rows of a sequence are within the bound; the number of values compared."""
    rows = ~torch.isnan(want)
    assert not torch.isnan(got[rows]).any()
    off = (got.double() - want).abs()[rows] - bound[rows]
    assert off.numel() == 0 or float(off.max()) <= 0.0, f"off by {float(off.max())} more than the bound of {float(bound[rows].max())}"
    return off.numel()


def append(qkv, H, Hkv, D, lens, cu, freqs, interleaved):
    """(q, k, v, positions, sequences, bound) of the rows that belong to a sequence, in 64 bits; the bound (before the rounding
    to the type) is for a rotation in fp32 with sines and cosines that are off by 2^-23."""
    T = qkv.shape[0]
    cu = list(range(T + 1)) if cu is None else cu.tolist()
    seq = torch.full((T,), -1, dtype=torch.long)
    pos = torch.zeros((T,), dtype=torch.long)
    for b, length in enumerate(lens.tolist()):
        n = cu[b + 1] - cu[b]
        seq[cu[b]:cu[b + 1]] = b
        pos[cu[b]:cu[b + 1]] = torch.arange(length - n, length)
    seq, pos = seq.to(qkv.device), pos.to(qkv.device)
    x = qkv.double().view(T, H + 2 * Hkv, D)
    y = x.clone()
    bound = torch.zeros_like(x)
    if freqs is not None:
        angle = pos.double()[:, None, None] * freqs
        c, s = angle.cos(), angle.sin()
        part = x[:, :H + Hkv]
        a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :D // 2], part[..., D // 2:])
        ra, rb, off = a * c - b * s, a * s + b * c, (a.abs() + b.abs()) * 2.0 ** -21
        if interleaved:
            y[:, :H + Hkv] = torch.stack((ra, rb), -1).flatten(-2)
            bound[:, :H + Hkv] = torch.stack((off, off), -1).flatten(-2)
        else:
            y[:, :H + Hkv] = torch.cat((ra, rb), -1)
            bound[:, :H + Hkv] = torch.cat((off, off), -1)
    return y, bound, pos, seq
