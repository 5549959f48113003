"""The operators of a drafted decoding step from their definitions, in 64 bits on the CPU."""
from __future__ import annotations

import math

import numpy as np

E4M3 = np.array([(-1.0 if c & 0x80 else 1.0) * ((c & 7) * 2.0 ** -9 if not c >> 3 & 15 else (8 + (c & 7)) * 2.0 ** ((c >> 3 & 15) - 10))
                 if c & 0x7f != 0x7f else math.nan for c in range(256)])


def rope(x, pos, inv_freq, layout, scale):
    """x f64 [rows, vectors, seg]; the rotated vectors, not rounded."""
    half = x.shape[-1] // 2
    t = np.remainder(pos.astype(np.longdouble)[:, None] * inv_freq.astype(np.longdouble), 2 * np.pi * np.longdouble(1) + np.longdouble(2.4492935982947064e-16))
    c, s = scale * np.cos(t).astype(np.float64)[:, None], scale * np.sin(t).astype(np.float64)[:, None]
    a, b = (x[..., :half], x[..., half:]) if layout == "half" else (x[..., 0::2], x[..., 1::2])
    u, v = a * c - b * s, a * s + b * c
    return np.stack((u, v), -1).reshape(x.shape) if layout == "adjacent" else np.concatenate((u, v), -1)


def tree_rows(table, page, n_pages, n, rows, tree_pos, t):
    """Pool rows of the n prefix entries and the t nodes of one sequence; -1 where the block table maps nothing."""
    token = [int(rows[j]) if rows is not None else j for j in range(n)] + [tree_pos + j for j in range(t)]
    out = []
    for k in token:
        p = int(table[k // page]) if 0 <= k < len(table) * page else -1
        out.append(p * page + k % page if 0 <= p < n_pages else -1)
    return np.array(out, dtype=np.int64)


def tree_attend(q, codes, scale, pool_rows, n, masks, softmax_scale, kvl, unit=0.0):
    """q f64 [T, H, W]; codes u8 and scale of the pool; returns out f64 [T, H, kvl], lse [T, H], and for a query whose entries are off
    by independent relative errors of deviation ``unit``: the deviations of out and lse by it, and of out by weights off the same way;
    and sum p |L|, which bounds what weights off by a relative error do. With weights times row scales as multiples of a step, an entry
    is off by sum |code| times the step at most, by the root of sum code^2 on the whole: both for a step of the largest such weight."""
    T, H, W = q.shape
    live = pool_rows >= 0
    k = E4M3[codes[pool_rows.clip(0)]] * scale[pool_rows.clip(0)].astype(np.float64)[:, None]
    out, lse = np.zeros((T, H, kvl)), np.full((T, H), -np.inf)
    weight, by_score, by_weight, step, by_step = (np.zeros((T, H, kvl)) for _ in range(5))
    lse_by, s_row = np.zeros((T, H)), scale[pool_rows.clip(0)].astype(np.float64)
    for j in range(T):
        sees = live & np.array([i < n or bool(int(masks[j]) >> (i - n) & 1) for i in range(len(pool_rows))], dtype=bool)
        if not sees.any():
            continue
        ks, v = k[sees], k[sees][:, :kvl]
        s = q[j] @ ks.T * softmax_scale
        top = s.max(1, keepdims=True)
        p = np.exp(s - top)
        lse[j] = top[:, 0] + np.log(p.sum(1))
        p /= p.sum(1, keepdims=True)
        out[j], weight[j] = p @ v, p @ np.abs(v)
        var = (unit * softmax_scale) ** 2 * (q[j] ** 2 @ (ks ** 2).T) * p ** 2       # of p times a score's error
        by_score[j] = np.sqrt(np.maximum(var @ v ** 2 - 2 * out[j] * (var @ v) + out[j] ** 2 * var.sum(1, keepdims=True), 0))
        by_weight[j] = unit * np.sqrt(p ** 2 @ v ** 2)
        lse_by[j] = np.sqrt(var.sum(1))
        top_p, c = (p * s_row[sees]).max(1, keepdims=True), v / np.where(s_row[sees] > 0, s_row[sees], 1.0)[:, None]
        step[j], by_step[j] = top_p * np.abs(c).sum(0), top_p * np.sqrt((c ** 2).sum(0))
    return out, lse, by_score, lse_by, by_weight, weight, step, by_step


def clean(x):
    with np.errstate(invalid="ignore"):
        return np.where((x > 0) & (x < np.inf), x, 0.0).astype(np.float64)


def verify(parent, token, target, draft, u, u_next, max_path):
    """One sequence: parent, token, u of its nodes, target and draft rows [T, vocab]. Returns (path, next token)."""
    T = len(parent)
    if not T:
        return [], -1
    vocab, path = target.shape[1], [0]
    r, hit = clean(target[0]), True
    while hit and len(path) < max_path:
        cur, hit = path[-1], False
        r = clean(target[cur])
        q = None if draft is None else clean(draft[cur])
        for j in (j for j in range(1, T) if parent[j] == cur and parent[j] < j):
            x = int(token[j])
            known = 0 <= x < vocab
            qx, rx = (1.0 if draft is None else q[x] if known else 0.0), r[x] if known else 0.0
            if float(u[j]) * qx < rx:
                path.append(j)
                hit = True
                break
            if draft is None:
                r = r.copy()
                if known:
                    r[x] = 0.0
            else:
                r = np.maximum(r - q, 0.0)
            z = r.sum()
            r = r / z if z > 0 else np.zeros_like(r)
    if hit:
        r = clean(target[path[-1]])
    if not r.sum() > 0:
        r = clean(target[path[-1]])
    alive = np.nonzero(r > 0)[0]
    if not len(alive):
        return path, -1
    over = np.nonzero((np.cumsum(r) > float(u_next) * r.sum()) & (r > 0))[0]
    return path, int(over[0]) if len(over) else int(alive[-1])


def commit(pools, table, page, n_pages, tree_pos, path):
    """In place on arrays [pool rows, ...]; False (and nothing moved) if the path is unsound or its rows are not mapped."""
    rows = []
    for k, j in enumerate(path):
        if j < k or j >= 64 or (k and j <= path[k - 1]):
            return False
        src, dst = tree_rows(table, page, n_pages, 0, None, tree_pos + j, 1)[0], tree_rows(table, page, n_pages, 0, None, tree_pos + k, 1)[0]
        if src < 0 or dst < 0:
            return False
        rows.append((src, dst))
    for a in pools:
        was = [a[s].copy() for s, _ in rows]
        for (_, d), w in zip(rows, was):
            a[d] = w
    return True
