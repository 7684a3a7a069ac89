"""The paged cache in 8 or 4 bits in numpy: groups quantised in float64, blocks of 16 tokens taken apart byte by byte."""

from __future__ import annotations

import numpy as np


def floor16(x):
    """The largest fp16 value that is not above x (float64), past the range as fp16 rounds downwards."""
    x = np.asarray(x, np.float64)
    with np.errstate(over="ignore"):
        h = x.astype(np.float16)
        h = np.where(h.astype(np.float64) > x, np.nextafter(h, np.float16(-np.inf)), h)
    return h.astype(np.float16)


def quantise(x, bits, group):
    """x [..., hd] float32 -> codes [..., hd] int, scales and biases [..., hd / group] fp16."""
    x = np.asarray(x, np.float64)
    x = x.reshape(*x.shape[:-1], -1, group)
    most = 2**bits - 1
    b = floor16(x.min(-1))
    s = -floor16(-(x.max(-1) - b.astype(np.float64)) / most)
    over = (s.astype(np.float64) * most + b.astype(np.float64) > 65504) & (x.max(-1) <= 65504)  # fp16 holds the group: the scale below
    s = np.where(over, np.nextafter(s, np.float16(0)), s)
    c = np.zeros(x.shape, np.int64)
    some = s > 0
    c[some] = np.clip(np.rint((x - b.astype(np.float64)[..., None])[some] / s.astype(np.float64)[..., None][some]), 0, most)
    return c.reshape(*x.shape[:-2], -1), s.astype(np.float16), b


def value(codes, s, b):
    """s c + b in float64."""
    c = codes.reshape(*s.shape, -1).astype(np.float64)
    return (c * s.astype(np.float64)[..., None] + b.astype(np.float64)[..., None]).reshape(codes.shape)


def block_bytes(hd, bits, group):
    return 16 * 2 * (hd * bits // 8 + 4 * (hd // group))


def place(side, tok, d, hd, bits, group):
    """(byte, shift) of dim d of token tok of a block: side 0 is K, 1 is V."""
    row, g, r = hd * bits // 8, d // group, d % group
    if side == 0:  # four threads, each a quarter of every group
        t, dims = r // (group // 4), g * (group // 4) + r % (group // 4)
        byte, shift = dims * bits // 8, dims * bits % 8
        if row == 128:
            half, byte = byte // 16, byte % 16
            return tok * row + (half ^ (tok & 1)) * 64 + t * 16 + byte, shift
        return tok * row + t * (row // 4) + byte, shift
    t, dims = r // (group // 8), g * (group // 8) + r % (group // 8)  # eight threads
    byte, shift = dims * bits // 8, dims * bits % 8
    byte = byte // 2 * 4 + (tok & 1) * 2 + byte % 2
    pair = tok >> 1
    at = 16 * row + pair * 2 * row
    if row == 32:
        return at + (t ^ (4 if pair & 2 else 0)) * 8 + byte, shift
    return at + byte // 16 * 128 + (t ^ (2 * (pair & 3))) * 16 + byte % 16, shift


def meta_place(side, tok, g, hd, bits, group):
    n = hd // group
    return 32 * (hd * bits // 8) + side * 64 * n + (tok * n + g) * 4


def put(data, slot, page, side, codes, s, b, bits, group):
    """Codes [Hkv, hd], scales and biases [Hkv, n] into a slot of data [pages, Hkv, bytes]."""
    Hkv, hd = codes.shape
    pid, off = divmod(int(slot), page)
    at, tok = off // 16 * block_bytes(hd, bits, group), off % 16
    for h in range(Hkv):
        for d in range(hd):
            byte, shift = place(side, tok, d, hd, bits, group)
            old = int(data[pid, h, at + byte])
            mask = (2**bits - 1) << shift
            data[pid, h, at + byte] = (old & ~mask & 255) | (int(codes[h, d]) << shift)
        for g in range(hd // group):
            m = at + meta_place(side, tok, g, hd, bits, group)
            data[pid, h, m:m + 4] = np.array([s[h, g], b[h, g]], np.float16).view(np.uint8)


def take(data, hd, page, bits, group):
    """The whole pool: per side codes [pages, Hkv, page, hd], scales and biases [pages, Hkv, page, n]."""
    n_pages, Hkv, _ = data.shape
    n, size = hd // group, block_bytes(hd, bits, group)
    blocks = data.reshape(n_pages, Hkv, page // 16, size)
    out = []
    for side in (0, 1):
        codes = np.zeros((n_pages, Hkv, page // 16, 16, hd), np.int64)
        meta = np.zeros((n_pages, Hkv, page // 16, 16, n, 4), np.uint8)
        for tok in range(16):
            for d in range(hd):
                byte, shift = place(side, tok, d, hd, bits, group)
                codes[..., tok, d] = (blocks[..., byte] >> shift) & (2**bits - 1)
            for g in range(n):
                m = meta_place(side, tok, g, hd, bits, group)
                meta[..., tok, g, :] = blocks[..., m:m + 4]
        sb = meta.view(np.float16).reshape(n_pages, Hkv, page, n, 2)
        out.append((codes.reshape(n_pages, Hkv, page, hd), sb[..., 0], sb[..., 1]))
    return out


def values(data, hd, page, bits, group):
    """k and v [pages, Hkv, page, hd] in float64."""
    return [value(*x) for x in take(data, hd, page, bits, group)]


def fill(k, v, bits, group):
    """k, v [pages, Hkv, page, hd] -> data [pages, Hkv, bytes]."""
    n_pages, Hkv, page, hd = k.shape
    n, size = hd // group, block_bytes(hd, bits, group)
    data = np.zeros((n_pages, Hkv, page // 16, size), np.uint8)
    for side, x in ((0, k), (1, v)):
        codes, s, b = quantise(x, bits, group)
        codes = codes.reshape(n_pages, Hkv, page // 16, 16, hd)
        meta = np.stack([s, b], -1).astype(np.float16).view(np.uint8).reshape(n_pages, Hkv, page // 16, 16, n, 4)
        for tok in range(16):
            for d in range(hd):
                byte, shift = place(side, tok, d, hd, bits, group)
                data[..., byte] |= (codes[..., tok, d] << shift).astype(np.uint8)
            for g in range(n):
                m = meta_place(side, tok, g, hd, bits, group)
                data[..., m:m + 4] = meta[..., tok, g, :]
    return data.reshape(n_pages, Hkv, -1)


def attention(q, data, q_start, kv_lens, table, prefix_table, prefix_len, Hq, hd, page, bits, group, scale, fp16=None):
    """out [rows, Hq, hd] float64, and per output a bound's parts (as oracle.paged.attention's): sum_j w_j (s c + |b|), the row's
    largest scale * sum |q| (s c + |b|), its number of keys, and max_j (w_j s_j) * sum_j c_j / sum_j w_j.

    fp16: of which tokens s c + b goes through fp16, "none", "prefix" (of 1024 tokens at least, else none) or "all": v, and k in one term for
    rows in whose tile of 256 (token, head) rows all see 1024 keys, in two for the others.  For those tokens the parts hold |k| and |v| in
    place of s c + |b|, and the last one max_j w_j * sum_j |v_j| / sum_j w_j, added to the others'.  Two more parts come with it:
    sqrt(sum_j (w_j (s c + |b|))^2) / sum_j w_j, and the largest scale * sum |q| e of those tokens, e what the two terms may be off a k:
    2^-15 of half its group's range, 2^-11 where the group's middle is further than that from zero, and of all of it next to fp16's
    limits."""
    n_pages, Hkv, _ = data.shape
    (kc, ks, kb), (vc, vs, vb) = take(data, hd, page, bits, group)
    spread = lambda x: np.repeat(x.astype(np.float64), group, -1)  # noqa: E731
    with np.errstate(invalid="ignore", over="ignore"):
        pools = dict(k=value(kc, ks, kb), v=value(vc, vs, vb), ka=value(kc, ks, np.abs(kb)), va=value(vc, vs, np.abs(vb)), c=vc.astype(float),
                     s=spread(vs))
        v16 = pools["v"].astype(np.float16).astype(np.float64)
        pools["k16"] = pools["k"].astype(np.float16).astype(np.float64)
        half = spread(ks) * 2.0 ** (bits - 1)
        middle = np.abs(spread(kb) + half)
        pools["e"] = np.where(middle <= half, 2.0**-15 * half, 2.0**-11 * np.where(middle + half < 30000, half, middle + half))
    through = dict(ka=np.abs(pools["k"]), v=v16, va=np.abs(v16))
    rows, G = int(q_start[-1]), Hq // Hkv
    q = np.asarray(q, np.float64).reshape(-1, Hq, hd)
    out = np.zeros((rows, Hq, hd))
    mass, dot, keys, tail = np.zeros_like(out), np.zeros((rows, Hq)), np.zeros((rows, Hq)), np.zeros_like(out)
    spread_of, split = np.zeros_like(out), np.zeros((rows, Hq))

    def where(ids, n):
        i = np.arange(n)
        pid = np.asarray(ids, np.int64)[i // page] if n else np.zeros(0, np.int64)
        there = (pid >= 0) & (pid < n_pages)
        return pid[there], (i % page)[there], there

    pp, po, _ = where(prefix_table, prefix_len)
    for b in range(len(kv_lens)):
        lo, hi = int(q_start[b]), int(q_start[b + 1])
        L = int(kv_lens[b])
        p1, o1, there = where(table[b], L)
        pid, off = np.concatenate([pp, p1]), np.concatenate([po, o1])
        place_of = np.concatenate([np.full(len(pp), -1), np.flatnonzero(there)])  # a token's place in the request; -1: the prefix
        for h in range(Hkv if hi > lo else 0):
            x = {name: pool[pid, h, off] for name, pool in pools.items()}
            r = np.full(len(pid), fp16 == "all") | ((place_of == -1) if fp16 == "prefix" and prefix_len >= 1024 else False)
            for name, pool in through.items():
                x[name][r] = pool[pid, h, off][r]
            x["s"][r], x["c"][r] = 0.0, 0.0
            heads = slice(h * G, (h + 1) * G)
            for i in range(hi - lo):
                n = int(np.searchsorted(place_of, max(-1, L - (hi - lo) + i), side="right"))  # tokens that the row sees
                if n == 0:
                    continue
                qs = q[lo + i, heads]
                first = (i * G + np.arange(G)) // 256 * 256 // G  # of each head's tile of rows
                deep = prefix_len + np.clip(L - (hi - lo) + first + 1, 0, max(L, 0)) >= 1024
                one = r[:n] & (deep[:, None] if fp16 == "all" else np.full((G, 1), True))
                sc = scale * np.where(one, qs @ x["k16"][:n].T, qs @ x["k"][:n].T) if one.any() else scale * (qs @ x["k"][:n].T)
                w = np.exp(sc - sc.max(-1, keepdims=True))
                total = w.sum(-1, keepdims=True)
                out[lo + i, heads] = w @ x["v"][:n] / total
                mass[lo + i, heads] = w @ x["va"][:n] / total
                tail[lo + i, heads] = (w * x["s"][:n].max(-1)).max(-1, keepdims=True) * x["c"][:n].sum(0) / total
                dot[lo + i, heads] = scale * (np.abs(qs) @ x["ka"][:n].T).max(-1)
                keys[lo + i, heads] = n
                spread_of[lo + i, heads] = np.sqrt((w * w) @ (x["va"][:n] ** 2)) / total
                if r[:n].any():
                    split[lo + i, heads] = scale * np.where(r[:n] & ~one, np.abs(qs) @ x["e"][:n].T, 0.0).max(-1)
                    tail[lo + i, heads] += (w * r[:n]).max(-1, keepdims=True) * x["va"][:n][r[:n]].sum(0) / total
    return (out, mass, dot, keys, tail) if fp16 is None else (out, mass, dot, keys, tail, spread_of, split)
