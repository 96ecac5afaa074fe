"""CPU restatement of the paged key-value cache operators (numpy, float64).

The reference has no such cache (its attention keeps a ring of the window,
model/layers/csa.py:172-206): the definitions are those of include/llmyb.h.
"""
from __future__ import annotations

import numpy as np


def positions(cu_q, lengths, n_tokens: int):
    """(sequence, position) of every packed token; sequence -1 behind cu_q[-1]."""
    seq = np.full(n_tokens, -1, dtype=np.int64)
    pos = np.full(n_tokens, -1, dtype=np.int64)
    for b in range(len(lengths)):
        i = np.arange(cu_q[b], cu_q[b + 1])
        seq[i] = b
        pos[i] = lengths[b] - cu_q[b + 1] + i
    return seq, pos


def norm_rotate(x, weight, eps, pos, inv_freq, interleaved):
    """x [N, H, D]: RMS norm per head, then rotation by pos * inv_freq."""
    x = np.asarray(x, dtype=np.float64).copy()
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    if inv_freq is not None and len(inv_freq):
        half = len(inv_freq)
        t = np.asarray(pos, np.float64)[:, None] * np.asarray(inv_freq, np.float64)
        cos, sin = np.cos(t)[:, None, :], np.sin(t)[:, None, :]
        i = np.arange(half)
        ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        a, b = x[..., ia].copy(), x[..., ib].copy()
        x[..., ia] = a * cos - b * sin
        x[..., ib] = b * cos + a * sin
    return x


def gather(pages, table_row, length):
    """[length, H, D] rows of one sequence from pages [P, H, page_size, D]."""
    size = pages.shape[2]
    p = np.arange(length)
    return pages[table_row[p // size], :, p % size]


def attention(q, k_pages, v_pages, table, lengths, cu_q, *, scale, softcap=0.0, window=0,
              slopes=None, prefix=None):
    """Packed tokens q [N, Hq, D] over the pages.  Returns out [N, Hq, D], the
    same with |v| in place of v (the scale of the weights' rounding) and the
    log-sum-exp [N, Hq]; rows of no sequence are NaN."""
    q = np.asarray(q, dtype=np.float64)
    n, hq, d = q.shape
    hkv = k_pages.shape[1]
    out, mag = np.full((2, n, hq, d), np.nan)
    lse = np.full((n, hq), np.nan)
    for b in range(len(lengths)):
        rows = np.arange(cu_q[b], cu_q[b + 1])
        length = int(lengths[b])
        out[rows], mag[rows], lse[rows] = 0.0, 0.0, -np.inf
        if length == 0 or len(rows) == 0:
            continue
        k = gather(np.asarray(k_pages, np.float64), table[b], length)
        v = gather(np.asarray(v_pages, np.float64), table[b], length)
        i = (length - len(rows) + np.arange(len(rows)))[:, None]
        j = np.arange(length)[None, :]
        seen = j <= i
        if window:
            seen = seen & (i - j < window)
        if prefix is not None:
            seen = seen | (j < prefix[b])
        seen = seen & (i >= 0)
        for h in range(hq):
            s = q[rows, h] @ k[:, h // (hq // hkv)].T * scale
            if softcap:
                s = softcap * np.tanh(s / softcap)
            if slopes is not None:
                s = s - float(slopes[h]) * np.abs(i - j)
            s = np.where(seen, s, -np.inf)
            top = np.where(seen.any(1), s.max(1), 0.0)
            p = np.where(seen, np.exp(s - top[:, None]), 0.0)
            total = p.sum(1)
            some = total > 0
            w = p[some] / total[some][:, None]
            out[rows[some], h] = w @ v[:, h // (hq // hkv)]
            mag[rows[some], h] = w @ np.abs(v[:, h // (hq // hkv)])
            lse[rows[some], h] = top[some] + np.log(total[some])
    return out, mag, lse
