"""Paged cache operators in numpy: exact integers for the bookkeeping, float64 for the attention."""

from __future__ import annotations

import numpy as np


def reserve(lens, new_lens, table, free_pages, free_count, page, max_tokens, prefix_len=0):
    """(status, table, kv_lens, q_start, slots, positions, free_count); slots and positions hold the used rows only."""
    lens, new = np.asarray(lens, np.int64), np.asarray(new_lens, np.int64)
    table = np.array(table)
    fail = (table, lens, np.zeros(len(lens) + 1, np.int64), np.zeros(0, np.int64), np.zeros(0, np.int64), free_count)
    status = 0
    if (lens < 0).any() or (new < 0).any():
        status |= 8
    good = (lens >= 0) & (new >= 0)
    if (lens + new > table.shape[1] * page).any():
        status |= 2
    need = np.where(good, -(-(lens + new) // page) + (-lens // page), 0)
    if need.sum() > free_count:
        status |= 1
    if np.where(good, new, 0).sum() > max_tokens:
        status |= 4
    if not 0 <= free_count <= len(free_pages):
        status |= 16
    if status:
        return (status, *fail)
    slots, positions = [], []
    for b, (n0, n) in enumerate(zip(lens, new)):
        for blk in range(-(-n0 // page), -(-(n0 + n) // page)):
            free_count -= 1
            table[b, blk] = free_pages[free_count]
        for i in range(n0, n0 + n):
            slots.append(int(table[b, i // page]) * page + i % page)
            positions.append(prefix_len + i)
    return 0, table, lens + new, np.concatenate([[0], np.cumsum(new)]), np.array(slots, np.int64), np.array(positions, np.int64), free_count


def truncate(lens, keep, table, free_pages, free_count, page):
    """(status, lens, free_pages, free_count)."""
    lens = np.asarray(lens, np.int64)
    free_pages = np.array(free_pages)
    kept = np.minimum(np.maximum(keep, 0), np.maximum(lens, 0))
    status = 8 if (lens < 0).any() else 0
    if (lens > table.shape[1] * page).any():
        status |= 2
    bad = (lens < 0) | (lens > table.shape[1] * page)
    back = np.where(bad, 0, -(-lens // page) + (-kept // page)).sum()
    if not 0 <= free_count <= len(free_pages):
        status |= 16
    elif free_count + back > len(free_pages):
        status |= 1
    if status:
        return status, lens, free_pages, free_count
    for b in range(len(lens)):
        for blk in range(-(-kept[b] // page), -(-lens[b] // page)):
            free_pages[free_count] = table[b, blk]
            free_count += 1
    return 0, kept, free_pages, free_count


def rotate(x, positions, cos, sin):
    """x [T, heads, hd] at `positions`; cos, sin [max_pos, hd / 2]."""
    half = x.shape[-1] // 2
    c, s = cos[positions][:, None].astype(np.float64), sin[positions][:, None].astype(np.float64)
    a, b = x[..., :half], x[..., half:]
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


def attention(q, k_pages, v_pages, q_start, kv_lens, table, prefix_table, prefix_len, Hq, scale):
    """out [rows, Hq, hd] float64, and per output a bound's parts: sum_j w_j |v_j|, the row's largest
    scale * sum |q| |k| over its keys, its number of keys, and sum_j |v_j| / sum_j exp(s_j - max)."""
    n_pages, Hkv, page, hd = k_pages.shape
    rows = int(q_start[-1])
    G = Hq // Hkv
    q = np.asarray(q, np.float64).reshape(-1, Hq, hd)
    out = np.zeros((rows, Hq, hd))
    mass, dot, keys, tail = np.zeros_like(out), np.zeros((rows, Hq)), np.zeros((rows, Hq)), np.zeros_like(out)

    def gather(pool, ids, n):
        got, there = np.zeros((Hkv, n, hd)), np.zeros(n, bool)
        for i in range(n):
            pid = ids[i // page]
            if 0 <= pid < n_pages:
                got[:, i], there[i] = pool[pid, :, i % page], True
        return got, there

    kp, tp = gather(k_pages, prefix_table, prefix_len)
    vp, _ = gather(v_pages, prefix_table, prefix_len)
    for b in range(len(kv_lens)):
        lo, hi = int(q_start[b]), int(q_start[b + 1])
        if hi == lo:
            continue
        L = int(kv_lens[b])
        ks, ts = gather(k_pages, table[b], L)
        vs, _ = gather(v_pages, table[b], L)
        for i in range(hi - lo):
            n = max(0, min(L, L - (hi - lo) + i + 1))
            there = np.concatenate([tp, ts[:n]])
            if not there.any():
                continue
            k = np.concatenate([kp, ks[:, :n]], 1)[:, there]
            v = np.concatenate([vp, vs[:, :n]], 1)[:, there]
            for h in range(Hq):
                s = scale * (k[h // G] @ q[lo + i, h])
                w = np.exp(s - s.max())
                out[lo + i, h] = w @ v[h // G] / w.sum()
                mass[lo + i, h] = w @ np.abs(v[h // G]) / w.sum()
                tail[lo + i, h] = np.abs(v[h // G]).sum(0) / w.sum()
                dot[lo + i, h] = scale * (np.abs(k[h // G]) @ np.abs(q[lo + i, h])).max()
                keys[lo + i, h] = len(s)
    return out, mass, dot, keys, tail
