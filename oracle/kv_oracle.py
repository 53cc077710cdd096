"""Paged key-value cache operators in 64 bits (numpy): the checker of the CUDA kernels, never on a product path."""
from __future__ import annotations

import numpy as np


def rows_of(table, page, seq, idx, pages):
    """(page, slot) of each token, or None where it has no place."""
    got = []
    for b, t in zip(seq, idx):
        p = int(table[b][t // page]) if t >= 0 and t // page < len(table[b]) else -1
        got.append((p, int(t) % page) if 0 <= p < pages else None)
    return got


def rotate(x, cos, sin, rot, pairs):
    """x [n, heads, dim] rotated by cos, sin [n, rot / 2]; also sum |terms| of every element, for error bounds."""
    x = x.astype(np.float64)
    y, mag = x.copy(), np.abs(x)
    if rot:
        first = np.arange(rot // 2) if pairs == "halves" else np.arange(0, rot, 2)
        second = first + (rot // 2 if pairs == "halves" else 1)
        a, b = x[..., first], x[..., second]
        c, s = cos[:, None].astype(np.float64), sin[:, None].astype(np.float64)
        y[..., first], y[..., second] = a * c - b * s, b * c + a * s
        mag[..., first] = np.abs(a * c) + np.abs(b * s)
        mag[..., second] = np.abs(b * c) + np.abs(a * s)
    return y, mag


def attend(q, k, v, table, lens, scale, fill=None):
    """q [B, hq, d], k and v [pages, heads, page, d] (values), table [B, wide].  Returns out, lse, and for error bounds
    sum p |v| [B, hq, d], sum |v| [B, hq, d], scale * max sum |q k| [B, hq]."""
    B, hq, d = q.shape
    pages, heads, page, _ = k.shape
    g = hq // heads
    out, pv, av = (np.zeros((B, hq, d)) for _ in range(3))
    lse, mag = np.full((B, hq), -np.inf), np.zeros((B, hq))
    for b in range(B):
        at = []
        for t in range(min(int(lens[b]), len(table[b]) * page)):
            p, s = int(table[b][t // page]), t % page
            if 0 <= p < pages and (fill is None or s < fill[p]):
                at.append((p, s))
        if not at:
            continue
        p, s = np.array(at).T
        for h in range(hq):
            kk, vv, qq = k[p, h // g, s].astype(np.float64), v[p, h // g, s].astype(np.float64), q[b, h].astype(np.float64)
            with np.errstate(invalid="ignore", over="ignore"):
                sc = kk @ qq * scale
                m = sc.max()
                w = np.exp(sc - (m if m != -np.inf else 0.0))
                tot = w.sum()
                if tot == 0.0:      # every score is -infinity: nothing has any weight
                    continue
                out[b, h] = (w @ vv) / tot
                lse[b, h] = m + np.log(tot)
                pv[b, h], av[b, h] = (w @ np.abs(vv)) / tot, np.abs(vv).sum(0) / tot
                mag[b, h] = scale * (np.abs(kk) @ np.abs(qq)).max()
    return out, lse, pv, av, mag
