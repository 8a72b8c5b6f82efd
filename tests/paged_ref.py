"""Plain forms of the paged-cache operators, for the tests: the tables one request at a time
in Python, the attention in float64."""
from __future__ import annotations

import numpy as np


def extend(past, new, page, table, free, n_free, free_cap, n_tok, pad=-1):
    """(table, n_free, n_kv, cu, slots, pos, seq, bad) of qwfn_paged_extend."""
    table, max_pages = table.copy(), table.shape[1]
    n0 = min(max(n_free, 0), free_cap)
    bad = n0 != n_free
    taken, asked, at = 0, 0, 0
    n_kv, cu = [], [0]
    slots, pos, seq = np.full(n_tok, pad, np.int32), np.full(n_tok, -1, np.int32), np.full(n_tok, -1, np.int32)
    for b, (p_in, f_in) in enumerate(zip(past, new)):
        p, f = max(int(p_in), 0), max(int(f_in), 0)
        bad |= p != p_in or f != f_in
        have, need = -(-p // page), -(-(p + f) // page) - -(-p // page)
        at += f
        fits = p + f <= max_pages * page and at <= n_tok
        if fits:
            asked += need
        served = fits and (need == 0 or asked <= n0)
        if served:
            for i in range(need):
                table[b, have + i] = free[n0 - 1 - taken - i]
            taken += need
        bad |= not served
        for t in range(f):
            i = at - f + t
            if i >= n_tok:
                break
            seq[i] = b
            if served:
                entry = int(table[b, (p + t) // page])
                if entry < 0 or entry * page + (p + t) % page >= 2 ** 31:
                    bad = True
                else:
                    slots[i], pos[i] = entry * page + (p + t) % page, p + t
        n_kv.append(p + f if served else p)
        cu.append(min(at, n_tok))
    return table, n0 - taken, np.array(n_kv, np.int32), np.array(cu, np.int32), slots, pos, seq, bad


def trim(keep, n_kv, page, table, free, n_free, free_cap):
    """(free, n_free, n_kv, bad) of qwfn_paged_trim."""
    free = free.copy()
    n0 = min(max(n_free, 0), free_cap)
    bad = n0 != n_free
    room, given, asked, out = table.shape[1] * page, 0, 0, []
    for b, (k_in, n_in) in enumerate(zip(keep, n_kv)):
        n = min(max(int(n_in), 0), room)
        bad |= n != n_in
        k = min(max(int(k_in), 0), n)
        first, last = -(-k // page), -(-n // page)
        asked += last - first
        if last == first or asked <= free_cap - n0:
            free[n0 + given:n0 + given + last - first] = table[b, first:last]
            given += last - first
            out.append(k)
        else:
            bad = True
            out.append(n)
    return free, n0 + given, np.array(out, np.int32), bad


def requantise(x, variant=1):
    """float32 [..., 32 k] as q8_0 and back, in float64: the query's image."""
    b = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    amax = np.abs(b).max(-1, keepdims=True)
    d = (amax / np.float32(127)).astype(np.float32)
    with np.errstate(divide="ignore"):
        if variant == 1:
            inv = np.where(amax > 0, np.float32(127) / amax, np.float32(0)).astype(np.float32)
        else:
            inv = np.where(d > 0, np.float32(1) / d, np.float32(0)).astype(np.float32)
    v = (b * inv).astype(np.float32)
    q = np.rint(v) if variant == 1 else np.copysign(np.floor(np.abs(v.astype(np.float64)) + 0.5), v)
    return (q.astype(np.float64) * d.astype(np.float16).astype(np.float64)).reshape(x.shape)


def rows_f64(cache, rows, kvh, D):
    """q8_0 rows of a uint8 [n, bytes] cache as float64 [len(rows), kvh, D]."""
    seg = D // 32 * 34
    b = cache[rows][:, :kvh * seg].reshape(len(rows), kvh, D // 32, 34)
    d = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float64)
    return (np.ascontiguousarray(b[..., 2:]).view(np.int8).astype(np.float64) * d).reshape(len(rows), kvh, D)


def attention(q, kc, vc, rows, kvh, scale, variant=1):
    """One request: q float32 [T, nh, D] (its last T tokens), rows its cache rows in order (-1: a masked key).
    Returns the output and the tolerance of a correct float32 implementation, float64 [T, nh, D].

    The tolerance: a score is a sum of D / 32 products rounded once each (2^-24 of the running sum), times
    scale * log2(e) with one rounding, minus the reference M with one more (M is as large as the largest
    score); an exponential is 2^-22 off; P dv enters as 22 bits; the sums over n keys lose 2^-24 a step of
    16 keys; all relative to sum p |v| / sum p. Below that P dv ends with the range of f16: a product is held to
    half of its smallest step, 2^-25, where the largest P dv of the reference M's tile is at least 2^7, so a
    key's value (at most 127 dv) is off by at most 2^-32 of the largest |v| of any key (p <= 1 = sum p)."""
    T, nh, D = q.shape
    rep, n = nh // kvh, len(rows)
    out, tol = np.zeros((T, nh, D)), np.zeros((T, nh, D))
    rows = np.asarray(rows)
    live = rows >= 0
    k, v = (rows_f64(c, np.where(live, rows, 0), kvh, D) for c in (kc, vc))
    qd = requantise(q, variant)
    for t in range(T):
        see = live & (np.arange(n) <= n - T + t)
        if not see.any():
            continue
        for h in range(nh):
            ks, vs = k[see, h // rep], v[see, h // rep]
            prod = (ks * qd[t, h]).reshape(len(ks), -1, 32).sum(-1)
            s, mag = prod.sum(-1) * scale, np.abs(prod).sum(-1).max() * abs(scale)
            p = np.exp(s - s.max())
            out[t, h] = p @ vs / p.sum()
            eps = 2 * (D // 32 + 4) * 2.0 ** -24 * mag + 2.0 ** -20 + (len(ks) // 16 + 16) * 2.0 ** -24
            tol[t, h] = 2 * eps * (p @ np.abs(vs)) / p.sum() + len(ks) * 2.0 ** -32 * np.abs(vs).max() + 1e-30
    return out, tol
