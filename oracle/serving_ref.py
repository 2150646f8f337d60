"""Float64 oracle of the packed and the paged attention, and of the cache's
bookkeeping: plain loops over requests, heads and tokens, in numpy."""

from __future__ import annotations

import numpy as np


def masked_attention(q, k, v, reads, sm_scale):
    """One head: q (Lq, D), k and v (Lk, D), reads (Lq, Lk) bool.

    Returns o, lse, and what an error bound needs: the same average of |v|, and
    the largest sum of |q||k| products behind a score.  Rows that read nothing
    give zeros and -inf.  Values that a row does not read never enter it."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    o, mag = np.zeros((len(q), v.shape[1])), np.zeros((len(q), v.shape[1]))
    lse = np.full(len(q), -np.inf)
    for i in range(len(q)):
        at = np.flatnonzero(reads[i])
        if not len(at):
            continue
        s = k[at] @ q[i] * sm_scale
        top = s.max()
        if top == -np.inf:
            continue
        w = np.exp(s - top)
        o[i] = w @ v[at] / w.sum()
        mag[i] = w @ np.abs(v[at]) / w.sum()
        lse[i] = top + np.log(w.sum())
    spread = (np.abs(np.nan_to_num(q)) @ np.abs(np.nan_to_num(k)).T).max(initial=0.0) * sm_scale
    return o, lse, mag, spread


def causal_reads(lq, lk, causal=True):
    if not causal:
        return np.ones((lq, lk), bool)
    return np.arange(lk)[None, :] <= np.arange(lq)[:, None] + lk - lq


def tree_reads(mask, context, nodes):
    """(nodes, context + nodes): all of the context, and the nodes whose bit is
    set (mask: (nodes, words) uint64, or None for a chain)."""
    reads = np.ones((nodes, context + nodes), bool)
    for i in range(nodes):
        for j in range(nodes):
            if mask is None:
                reads[i, context + j] = j <= i
            else:
                reads[i, context + j] = j < 64 * mask.shape[1] and bool((int(mask[i, j // 64]) >> (j % 64)) & 1)
    return reads


def packed_attention(q, k, v, cu_q, cu_k, reads_of, sm_scale):
    """q (T, HQ, D), k and v (TK, HK, D); reads_of(b) gives sequence b's mask.
    Returns o (T, HQ, D), lse (HQ, T), |v| averages and the largest spread; rows
    of no sequence are NaN."""
    T, HQ, D = q.shape
    group = HQ // k.shape[1]
    o, mag = np.full((T, HQ, D), np.nan), np.full((T, HQ, D), np.nan)
    lse, spread = np.full((HQ, T), np.nan), 0.0
    for b in range(len(cu_q) - 1):
        r, c = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
        for h in range(HQ):
            o[r, h], lse[h, r], mag[r, h], sp = masked_attention(q[r, h], k[c, h // group], v[c, h // group],
                                                                 reads_of(b), sm_scale)
            spread = max(spread, sp)
    return o, lse, mag, spread


def tolerances(o, lse, mag, spread, dtype_eps, longest, D, vmax, subnormal):
    """Bounds on |o - o_ref| and |lse - lse_ref|, from the arithmetic:

    * a score is D exact products summed in fp32: off by at most D 2^-24 spread,
      and 2^-22 more for the scale, the exponent's argument and the exponential;
    * sums over the keys are fp32: longest 2^-24 relative;
    * each weight is rounded to the 16-bit type before its product with v: half a
      step of the average of |v|, and `subnormal` per key below the type's normal
      range.  Weights are 2^(score - m), m the row's largest score or (the lazy
      maximum) at most 8 below it: the largest weight is at least 1, but for the
      rounding of its exponent, and so is the sum that divides.  Parts of a row are
      scaled to the largest of their m, by factors of at most 1;
    * the output is rounded once more: half a step of its value.
    """
    h = dtype_eps / 2
    e = D * 2.0**-24 * spread + 2.0**-22 * (1 + spread) + longest * 2.0**-24
    to = h * np.abs(o) * (1 + h) + (h + 3 * e) * mag + (1 + 2 * e) * longest * subnormal * vmax + 1e-7
    tl = 2 * e + 2.0**-23 * np.abs(lse) + 1e-7
    return to, tl


def slots(lengths, counts, table, free, start, size, T):
    """Block tables and slot maps, one token at a time."""
    table = np.array(table)
    width = table.shape[1] if table.ndim == 2 else 0
    cu, out, pos, taken = [0], np.full(T, -1, np.int64), np.zeros(T, np.int64), 0
    for b, (n0, n) in enumerate(zip(lengths, counts)):
        n0, n = max(int(n0), 0), max(int(n), 0)
        have = -(-n0 // size)
        for i in range(n):
            p, t = n0 + i, cu[-1] + i
            j = p // size
            if j >= have and p % size == 0 and j < width:
                f = start + taken
                if t < T:
                    table[b, j] = free[f] if f < len(free) else -1
                taken += 1
            if t < T:
                pos[t] = p
                if j < width and table[b, j] >= 0:
                    out[t] = int(table[b, j]) * size + p % size
        cu.append(cu[-1] + n)
    return np.array(cu, np.int32), out, pos, taken, table
