"""Trees of drafted tokens in 64 bits (numpy): the oracle of the CUDA kernels, never on a product path."""
from __future__ import annotations

import numpy as np


def norm(x, weight, eps):
    """Heads x [..., dim] over their root mean square, times weight."""
    x = x.astype(np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)


def sees(parents):
    """[nodes, nodes]: the nodes that each node sees (itself and its ancestors; a parent that does not come before its node
    is none)."""
    n = len(parents)
    m = np.eye(n, dtype=bool)
    for i, p in enumerate(parents):
        if 0 <= p < i:
            m[i] |= m[p]
    return m


def attend_tree(q, k, v, table, lens, parents, counts, scale, fill=None):
    """q [B, nodes, hq, d], k and v [pages, heads, page, d] (values), parents [B, nodes].  Returns out, lse, and for error
    bounds sum p |v|, |scale| * max sum |q k|."""
    B, nodes, hq, d = q.shape
    pages, heads, page, _ = k.shape
    g = hq // heads
    out, pv = np.zeros((B, nodes, hq, d)), np.zeros((B, nodes, hq, d))
    lse, mag = np.full((B, nodes, hq), -np.inf), np.zeros((B, nodes, hq))
    for b in range(B):
        room = len(table[b]) * page
        n = min(max(int(lens[b]), 0), room)
        count = nodes if counts is None else min(max(int(counts[b]), 0), nodes)
        m = sees(parents[b][:count])
        t = np.arange(min(n + count, room))
        p = np.asarray(table[b])[t // page]
        s = t % page
        ok = (p >= 0) & (p < pages)
        if fill is not None:
            ok &= s < np.asarray(fill)[np.where(ok, p, 0)]
        t, p, s = t[ok], p[ok], s[ok]
        vis = np.concatenate([np.ones((count, (t < n).sum()), bool), m[:, t[t >= n] - n]], 1)
        for h in range(heads):
            kk, vv = k[p, h, s].astype(np.float64), v[p, h, s].astype(np.float64)
            qq = q[b, :count, h * g:(h + 1) * g].astype(np.float64)
            for i in range(count):
                K, V = kk[vis[i]], vv[vis[i]]
                if not len(K):
                    continue
                with np.errstate(invalid="ignore", over="ignore"):
                    sc = qq[i] @ K.T * scale
                    top = sc.max(1, keepdims=True)
                    w = np.exp(sc - np.where(top == -np.inf, 0.0, top))
                    tot = w.sum(1, keepdims=True)
                    at = slice(h * g, (h + 1) * g)
                    safe = np.where(tot == 0, 1, tot)
                    out[b, i, at] = np.where(tot == 0, 0, (w @ V) / safe)
                    pv[b, i, at] = (w @ np.abs(V)) / safe
                    lse[b, i, at] = np.where(tot == 0, -np.inf, top + np.log(safe))[:, 0]
                    mag[b, i, at] = abs(scale) * (np.abs(qq[i]) @ np.abs(K).T).max(1)
    return out, lse, pv, mag


def verify(target, parents, tokens, u, draft=None, counts=None):
    """The path, the number of nodes taken and the next token of each sequence (arrays as drafts.verify takes them, parents
    [B, nodes])."""
    B, rows, vocab = target.shape
    nodes = rows - 1
    clean = lambda x: np.where((x > 0) & np.isfinite(x), x, 0.0).astype(np.float64)  # noqa: E731
    path, kept, token = np.full((B, nodes), -1, np.int32), np.zeros(B, np.int32), np.zeros(B, np.int32)
    for b in range(B):
        count = nodes if counts is None else min(max(int(counts[b]), 0), nodes)
        last, r, m = -1, clean(target[b, 0]), 1.0
        for i in range(count):
            x = int(tokens[b, i])
            if parents[b][i] != last or last >= i or not 0 <= x < vocab:
                continue
            q = clean(draft[b, last + 1]) if draft is not None else (np.arange(vocab) == x).astype(np.float64)
            if float(u[b, i]) * m * q[x] < r[x]:
                path[b, kept[b]] = i
                kept[b] += 1
                last, r, m = i, clean(target[b, i + 1]), 1.0
                continue
            rest = np.maximum(r - m * q, 0.0) if draft is not None else np.where(q > 0, 0.0, r)
            if rest.sum() > 0:
                r, m = rest, rest.sum()
        upto = np.cumsum(r)
        over = np.flatnonzero(upto > float(u[b, nodes]) * upto[-1])
        some = np.flatnonzero(r)
        token[b] = over[0] if len(over) else some[-1] if len(some) else -1
    return path, kept, token


def compact(rows, table, lens, path, page):
    """rows [pages, heads, page, ...] with each path's rows behind one another."""
    got = rows.copy()
    for b in range(len(path)):
        for n, x in enumerate(path[b]):
            if x < 0:
                break
            src, dst = int(lens[b]) + int(x), int(lens[b]) + n
            p, q = table[b][src // page], table[b][dst // page]
            if p >= 0 and q >= 0:
                got[q, :, dst % page] = rows[p, :, src % page]
    return got
