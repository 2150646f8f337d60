"""Float64 oracle of rotary positions and of latent attention, in numpy."""

from __future__ import annotations

import numpy as np

from .serving_ref import causal_reads, tree_reads


def rotate(x, positions, freqs, first=0, interleaved=False, inverse=False, scale=1.0):
    """x (T, H, D): of each row the 2 * len(freqs) values from `first` on turned."""
    x = np.array(x, np.float64)
    half = len(freqs)
    angle = np.asarray(positions, np.float64)[:, None] * np.asarray(freqs, np.float64)
    c, s = scale * np.cos(angle)[:, None], (-scale if inverse else scale) * np.sin(angle)[:, None]
    if interleaved:
        ia, ib = first + 2 * np.arange(half), first + 2 * np.arange(half) + 1
    else:
        ia, ib = first + np.arange(half), first + half + np.arange(half)
    a, b = x[..., ia].copy(), x[..., ib].copy()
    x[..., ia], x[..., ib] = a * c - b * s, a * s + b * c
    return x


def rotate_bound(x, y, positions, freqs, eps, subnormal, first=0, interleaved=False, scale=1.0):
    """A bound on the error of y = rotate(x):

    * the angle's rest, at most half a turn, is rounded to fp32: 2^-26 of a turn, 2 pi
      2^-26 radians;
    * sine and cosine of it are within 2^-24 (0.88 of it, over every fp32 value up to half
      a turn, on the card);
    * the scale as an argument, its product, the product with x and the sum of two such round
      once each: 4 times 2^-24.  So far 3.92e-7, less than 2^-21 = 4.77e-7, of |a| + |b|;
    * in 64 bits 1 / 2 pi, its product with f, that with n and the oracle's n f are rounded,
      2^-53 of the angle each: 2^-51 |n f|;
    * the result is rounded to half a step."""
    half = len(freqs)
    e = scale * (2.0**-21 + 2.0**-51 * np.abs(np.asarray(positions, np.float64)[:, None] * freqs))[:, None]
    x, out = np.abs(np.asarray(x, np.float64)), np.zeros(np.shape(x))
    if interleaved:
        ia, ib = first + 2 * np.arange(half), first + 2 * np.arange(half) + 1
    else:
        ia, ib = first + np.arange(half), first + half + np.arange(half)
    part = e * (x[..., ia] + x[..., ib])
    out[..., ia], out[..., ib] = part, part
    turned = out > 0
    return np.where(turned, eps / 2 * np.abs(y) + (1 + eps) * out + subnormal, 0.0)


def rms(c, weight, eps):
    c = np.asarray(c, np.float64)
    return c / np.sqrt((c * c).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)


def attend(q, k, v, reads, sm_scale):
    """q (Lq, H, DK), k (Lk, H or 1, DK), v (Lk, H or 1, DV), reads (Lq, Lk): o (Lq, H,
    DV), lse (H, Lq), the same average of |v|, the largest sum of |q||k| behind a score.
    Finite inputs; rows that read nothing give zeros and -inf."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    Lq, H, _ = q.shape
    o, mag = np.zeros((Lq, H, v.shape[2])), np.zeros((Lq, H, v.shape[2]))
    lse, spread = np.full((H, Lq), -np.inf), 0.0
    for h in range(H):
        kk, vv = k[:, h if k.shape[1] > 1 else 0], v[:, h if v.shape[1] > 1 else 0]
        if not len(kk) or not Lq:
            continue
        s = np.where(reads, q[:, h] @ kk.T * sm_scale, -np.inf)
        top = s.max(1, keepdims=True)
        w = np.exp(s - np.where(np.isneginf(top), 0, top))
        z = w.sum(1, keepdims=True)
        some = z[:, 0] > 0
        z[~some] = 1
        o[:, h], mag[:, h] = w @ vv / z, w @ np.abs(vv) / z
        lse[h, some] = top[some, 0] + np.log(z[some, 0])
        spread = max(spread, (np.abs(q[:, h]) @ np.abs(kk).T).max() * sm_scale)
    return o, lse, mag, spread


def packed(q, k, v, k_rope, cu_q, cu_k, causal, sm_scale):
    """The expanded form: rows of no sequence are NaN."""
    T, HQ, _ = q.shape
    group = HQ // k.shape[1]
    o, mag, lse, spread = np.full((T, HQ, v.shape[2]), np.nan), np.full((T, HQ, v.shape[2]), np.nan), np.full((HQ, T), np.nan), 0.0
    keys = np.concatenate([k, np.broadcast_to(k_rope[:, None], k.shape[:2] + k_rope.shape[1:])], -1)
    for b in range(len(cu_q) - 1):
        r, c = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
        reads = causal_reads(cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b], causal)
        o[r], lse[:, r], mag[r], sp = attend(q[r], np.repeat(keys[c], group, 1) if group > 1 or HQ > 1 else keys[c],
                                             np.repeat(v[c], group, 1) if group > 1 or HQ > 1 else v[c], reads, sm_scale)
        spread = max(spread, sp)
    return o, lse, mag, spread


def paged(q, cache, table, lengths, cu_q, mask, sm_scale, rank=512):
    """The absorbed form over cache (blocks, size, 576); mask (T, words) uint64 or None.
    Rows of no request are NaN."""
    T, H, _ = q.shape
    size = cache.shape[1]
    o, mag, lse, spread = np.full((T, H, rank), np.nan), np.full((T, H, rank), np.nan), np.full((H, T), np.nan), 0.0
    for b in range(len(cu_q) - 1):
        r = slice(cu_q[b], cu_q[b + 1])
        n, context = cu_q[b + 1] - cu_q[b], max(int(lengths[b]), 0)
        reads = tree_reads(None if mask is None else mask[r], context, n)
        at = np.arange(min(context + n, table.shape[1] * size))
        page = table[b][at // size]
        rows = np.where(((page >= 0) & (page < len(cache)))[:, None], cache[np.clip(page, 0, len(cache) - 1), at % size], 0)
        o[r], lse[:, r], mag[r], sp = attend(q[r], rows[:, None], rows[:, None, :rank], reads[:, :len(at)], sm_scale)
        spread = max(spread, sp)
    return o, lse, mag, spread
