"""The paged key-value cache's operators and the rotary positions, restated in float64 numpy with plain loops.

Heads are (B, H, T, D) float64 arrays; a pool is k (pages, kv heads, page, D) and v (pages, kv heads, D, page) of values
(an e4m3 pool: the codes' values, with the scales given apart).
"""

from __future__ import annotations

import numpy as np


def rotary_angles(cos, sin, positions):
    """Rows of the tables for (B, T) positions; outside the tables NaN."""
    rows = cos.shape[0]
    ok = (positions >= 0) & (positions < rows)
    at = np.where(ok, positions, 0)
    nan = np.where(ok, 0.0, np.nan)[..., None]
    return cos[at] + nan, sin[at] + nan


def rotary(x, cos, sin, positions, layout, inverse=False):
    """(y, size): x (B, H, T, D) turned, and |a c| + |b s| (|b c| + |a s|) of each value, what its rounding errors go by."""
    c, s = rotary_angles(cos.astype(np.float64), sin.astype(np.float64), positions)
    c, s = c[:, None], (-s if inverse else s)[:, None]
    half = cos.shape[1]
    y, size = x.copy(), np.abs(x)
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if layout == "interleaved" else (i, i + half)
        ci, si = c[..., i], s[..., i]
        y[..., a], y[..., b] = x[..., a] * ci - x[..., b] * si, x[..., b] * ci + x[..., a] * si
        size[..., a] = np.abs(x[..., a] * ci) + np.abs(x[..., b] * si)
        size[..., b] = np.abs(x[..., b] * ci) + np.abs(x[..., a] * si)
    return y, size


def head_norm(x, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)


def new_positions(lens, counts, T):
    """(positions (B, T), live (B, T)) of the new tokens."""
    cnt = np.maximum(counts, 0)
    pos = (np.maximum(lens, 0) - cnt)[:, None] + np.arange(T)
    return pos, (np.arange(T) < cnt[:, None]) & (pos >= 0)


def page_of(tables, b, pos, page, pages):
    """The page of a position, or -1."""
    e = pos // page
    if pos < 0 or e >= tables.shape[1]:
        return -1
    return int(tables[b, e]) if 0 <= tables[b, e] < pages else -1


def attention(q, k, v, tables, lens, counts, window, scale, k_scale=None, v_scale=None):
    """(out, lse, size, slack): out (B, H, T, D), the log-sum-exp (B, H, T), sum_j p_j |v_j| / sum_j p_j of each value, and a
    bound on the relative error of a weight p_j computed in fp32 from fp32 products (B, H, T, 1)."""
    B, H, T, D = q.shape
    pages, KV, page, _ = k.shape
    ks = np.ones(KV) if k_scale is None else k_scale.astype(np.float64)
    vs = np.ones(KV) if v_scale is None else v_scale.astype(np.float64)
    out, lse, size, slack = np.zeros((B, H, T, D)), np.full((B, H, T), -np.inf), np.zeros((B, H, T, D)), np.zeros((B, H, T, 1))
    pos, live = new_positions(lens, counts, T)
    for b in range(B):
        for t in range(T):
            i = int(pos[b, t])
            if not live[b, t] or window <= 0:
                continue
            if i >= tables.shape[1] * page:
                out[b, :, t], lse[b, :, t] = np.nan, np.nan
                continue
            keys = np.arange(max(0, i - window + 1), i + 1)
            ids = np.array([page_of(tables, b, j * page, page, pages) for j in range(keys[0] // page, keys[-1] // page + 1)])
            ids = ids[keys // page - keys[0] // page]
            if (ids < 0).any():
                out[b, :, t], lse[b, :, t] = np.nan, np.nan
                continue
            kk, vv = k[ids, :, keys % page], v[ids, :, :, keys % page]        # (n, KV, D)
            for h in range(H):
                g = h // (H // KV)
                x = kk[:, g] @ q[b, h, t] * scale * ks[g]
                m = x.max()
                p = np.exp(x - m)
                out[b, h, t] = p @ vv[:, g] / p.sum() * vs[g]
                size[b, h, t] = p @ np.abs(vv[:, g]) / p.sum() * abs(vs[g])
                lse[b, h, t] = m + np.log(p.sum())
                dots = np.abs(kk[:, g]) @ np.abs(q[b, h, t]) * abs(scale * ks[g])
                slack[b, h, t] = (D + 8) * 2.0 ** -24 * dots.max() * 2 + (len(keys) + 32) * 2.0 ** -24
    return out, lse, size, slack


def reserve(tables, lens, refs, counts, page, window=None):
    tables, lens, refs = tables.copy(), lens.copy(), refs.copy()
    S, M = tables.shape
    P = len(refs)
    tables[(tables < 0) | (tables >= P)] = -1
    if window:
        for s in range(S):
            for j in range(M):
                if tables[s, j] >= 0 and (j + 1) * page <= lens[s] - window + 1:
                    refs[tables[s, j]] -= 1
                    tables[s, j] = -1
    granted, wants, total = np.zeros(S, np.int32), [], 0
    for s in range(S):
        c = int(counts[s])
        fits = c > 0 and lens[s] >= 0 and int(lens[s]) + c <= M * page
        want = [j for j in range(M) if fits and (j + 1) * page > lens[s] and j * page < lens[s] + c and tables[s, j] < 0]
        wants.append((fits, want))
    free = [p for p in range(P) if refs[p] == 0]
    for s, (fits, want) in enumerate(wants):
        first, total = total, total + len(want)
        if not fits or (want and total > len(free)):
            continue
        for j, p in zip(want, free[first:total]):
            tables[s, j] = p
            refs[p] = 1
        lens[s] += counts[s]
        granted[s] = counts[s]
    return tables, lens, refs, granted


def reorder(k, v, tables, lens, refs, parents, page):
    """k, v (L, pages, ..) are changed in place."""
    S, M = tables.shape
    P = len(refs)
    tables = np.where((tables < 0) | (tables >= P), -1, tables)
    old_k, old_v = k.copy(), v.copy()
    new, new_lens, refs, copies = np.full((S, M), -1, np.int32), np.zeros(S, np.int32), refs.copy(), []
    for p in tables.reshape(-1):
        if p >= 0:
            refs[p] -= 1
    for s in range(S):
        r = int(parents[s])
        if not 0 <= r < S:
            continue
        children = [c for c in range(S) if parents[c] == r]
        n = max(0, int(lens[r]))
        new_lens[s] = n
        full = n // page
        if s == (r if r in children else children[0]):
            new[s] = tables[r]
        else:
            new[s, :full] = tables[r, :full]
            if n % page and full < M and tables[r, full] >= 0:
                copies.append((s, full, int(tables[r, full]), n % page))
        for p in new[s]:
            if p >= 0:
                refs[p] += 1
    free = [p for p in range(P) if refs[p] == 0]
    for (s, j, src, used), dst in zip(copies, free + [None] * len(copies)):
        if dst is None:
            for p in new[s]:
                if p >= 0:
                    refs[p] -= 1
            new[s], new_lens[s] = -1, 0
            continue
        new[s, j] = dst
        refs[dst] = 1
        k[:, dst, :, :used] = old_k[:, src, :, :used]
        v[:, dst, :, :, :used] = old_v[:, src, :, :, :used]
    return new, new_lens, refs


def compact(k, v, tables, refs):
    """k, v (L, pages, ..) are changed in place."""
    P = len(refs)
    n = int((refs != 0).sum())
    movers, holes = [p for p in range(n, P) if refs[p]], [p for p in range(n) if not refs[p]]
    to = {p: p for p in range(P) if refs[p]}
    refs = refs.copy()
    for src, dst in zip(movers, holes):
        to[src] = dst
        k[:, dst], v[:, dst] = k[:, src], v[:, src]
        refs[dst], refs[src] = refs[src], 0
    return np.array([[to.get(int(p), -1) for p in row] for row in tables], np.int32), refs, n
