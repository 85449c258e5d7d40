"""The 8-bit paged cache's operators written out plainly: page maps in Python integers, appends and attention in
64-bit floats from the definitions, one page, head and row at a time."""
from __future__ import annotations

import numpy as np

from aihost_b200 import ROPE_INTERLEAVED, ROPE_NEOX


def page_map(page_rows, n_pages, max_pages, max_tokens, seq_len, n_new, free_pages, free_count, table):
    """(table, kv_len, row_start, slots, positions, free_count, refused)"""
    table = [list(r) for r in table]
    need = [-(-(c + n) // page_rows) + c // -page_rows for c, n in zip(seq_len, n_new)]
    refused = (any(n < 0 or c < 0 or c + n > max_pages * page_rows for c, n in zip(seq_len, n_new)) or
               sum(n_new) > max_tokens or not 0 <= free_count <= n_pages or sum(need) > free_count)
    if refused:
        return table, list(seq_len), [0] * (len(seq_len) + 1), [-1] * max_tokens, [0] * max_tokens, free_count, True
    slots, pos, start, kv = [], [], [0], []
    for b, (c, n) in enumerate(zip(seq_len, n_new)):
        have = -(-c // page_rows)
        for p in range(have, -(-(c + n) // page_rows)):
            free_count -= 1
            table[b][p] = free_pages[free_count]
        for t in range(c, c + n):
            slots.append(table[b][t // page_rows] * page_rows + t % page_rows)
            pos.append(t)
        start.append(start[-1] + n)
        kv.append(c + n)
    spare = max_tokens - len(slots)
    return table, kv, start, slots + [-1] * spare, pos + [0] * spare, free_count, False


def freqs(theta, d):
    f = np.float32
    return np.array([f(1) / f(float(theta) ** float(f(2 * i) / f(d))) for i in range(d // 2)], dtype=np.float32)


def rotate(x, pos, theta, mode):
    """x [n, heads, d] float64 rotated at pos [n]; the angle is the fp32 product of position and frequency."""
    d = x.shape[-1]
    ang = (np.asarray(pos, dtype=np.float32)[:, None] * freqs(theta, d)).astype(np.float64)[:, None, :]
    c, s = np.cos(ang), np.sin(ang)
    out = np.array(x, dtype=np.float64)
    if mode == ROPE_INTERLEAVED:
        a, b = x[..., 0::2], x[..., 1::2]
        out[..., 0::2], out[..., 1::2] = a * c - b * s, a * s + b * c
    elif mode == ROPE_NEOX:
        a, b = x[..., :d // 2], x[..., d // 2:]
        out[..., :d // 2], out[..., d // 2:] = a * c - b * s, a * s + b * c
    return out


def append(x, slots, page_rows, pool, scale):
    """Stores x [n, heads, d] (float64) into copies of pool (int8) and scale (fp32): (target, exact, scale). target is
    what every stored value should be rounded from, in units of its page's scale; exact is target rounded."""
    target, scale = pool.astype(np.float64), scale.astype(np.float64)
    t = 0
    while t < len(slots):
        if slots[t] < 0:
            t += 1
            continue
        page, row = divmod(int(slots[t]), page_rows)
        n = 1
        while t + n < len(slots) and row + n < page_rows and slots[t + n] == slots[t] + n:
            n += 1
        rows = x[t:t + n].transpose(1, 0, 2)  # [heads, n, d]
        had = np.zeros_like(scale[page]) if row == 0 else scale[page]
        need = np.where(np.isfinite(rows).all(axis=(1, 2)), np.abs(rows).max(axis=(1, 2)) / 127.0, np.nan)
        now = np.where(np.isnan(had) | np.isnan(need), np.nan, np.maximum(had, need))
        safe = np.where(now > 0, now, 1.0)[:, None, None]
        ok = ~np.isnan(now)
        target[page, ok, :row] *= np.where(now > had, had / safe[:, 0, 0], 1.0)[ok, None, None]
        target[page, :, row:row + n] = np.where(now[:, None, None] > 0, rows / safe, 0.0)
        scale[page] = now
        t += n
    return target, scale


def attend(q, row_start, kv_len, table, page_rows, k_pool, v_pool, k_scale, v_scale, scale, cap=0.0, theta=1.0, mode=None,
           prefix=None, first=None, slopes=None):
    """(out, weight, size): out [n, Hq, d]; weight = sum_j p_j |v_j| of every element; size [n, Hq] = the largest
    scale * sum_d |q_d k_jd| of a visible row j. All float64."""
    n, Hq, d = q.shape
    H = k_pool.shape[1]
    G = Hq // H
    out, weight, size = np.zeros((n, Hq, d)), np.zeros((n, Hq, d)), np.zeros((n, Hq))
    for b in range(len(kv_len)):
        t0, t1, L = row_start[b], row_start[b + 1], int(kv_len[b])
        if t1 == t0:
            continue
        pages = table[b][:-(-L // page_rows)]
        pos = np.arange(L - (t1 - t0), L)
        qb = rotate(q[t0:t1].astype(np.float64), pos, theta, mode)
        for h in range(H):
            k = (k_pool[pages, h].astype(np.float64) * k_scale[pages, h, None, None].astype(np.float64)).reshape(-1, d)[:L]
            v = (v_pool[pages, h].astype(np.float64) * v_scale[pages, h, None, None].astype(np.float64)).reshape(-1, d)[:L]
            for i, p in enumerate(pos):
                end = max(p + 1, min(int(prefix[b]), L) if prefix is not None else 0)
                lo = max(int(first[t0 + i]), 0) if first is not None else 0
                if lo >= end:
                    continue
                j = np.arange(lo, end)
                for g in range(h * G, h * G + G):
                    s = scale * (k[lo:end] @ qb[i, g])
                    size[t0 + i, g] = scale * (np.abs(k[lo:end]) @ np.abs(qb[i, g])).max()
                    if cap:
                        s = cap * np.tanh(s / cap)
                    if slopes is not None:
                        s = s - float(slopes[g]) * np.abs(p - j)
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    out[t0 + i, g] = w @ v[lo:end]
                    weight[t0 + i, g] = w @ np.abs(v[lo:end])
    return out, weight, size
