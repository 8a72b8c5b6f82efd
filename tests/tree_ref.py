"""Plain forms of shared pages and of drafted trees, for the tests: the tables one request at a time in Python, the
attention and the recurrence in float64."""
from __future__ import annotations

import numpy as np

import paged_ref as R


def _clip(x, top):
    return min(max(int(x), 0), top)


def fork(src, n_tok, n_kv, page, table, shared, free, n_free, cap, states=None):
    """(table, shared, n_free, n_kv, moves, state_moves, bad) of qwfn_paged_fork."""
    B, cols = table.shape
    table, shared, pages = table.copy(), shared.copy(), len(shared)
    n0 = _clip(n_free, cap)
    room = cols * page
    bad = n0 != n_free or any(_clip(n, room) != n for n in n_kv)
    old = [_clip(n, room) for n in n_kv]
    out, moves, smoves, asked, given = list(old), np.zeros((B, 3), np.int32), np.zeros((B, 3), np.int32), 0, 0
    start = table.copy()
    for b in range(B):
        f = int(src[b])
        if f < 0:
            continue
        ok = f < B and src[f] < 0 and old[b] == 0
        n = 0
        if ok:
            n = old[f] if n_tok is None else int(n_tok[b])
            ok = 0 <= n <= old[f]
        full, rest = (n // page, n % page) if ok else (0, 0)
        asked += rest > 0
        if not ok or (rest and asked > n0):
            bad = True
            continue
        out[b] = n
        for c in range(full):
            p = int(start[f, c])
            table[b, c] = p
            if 0 <= p < pages:
                shared[p] += 1
            else:
                bad = True
        if rest:
            fresh, given = int(free[n0 - asked]), given + 1
            table[b, full] = fresh
            p = int(start[f, full])
            if 0 <= p < pages and 0 <= fresh < pages:
                moves[b] = p * page, fresh * page, rest
            else:
                bad = True
        if n == old[f]:
            s, d = (f, b) if states is None else (int(states[f]), int(states[b]))
            if s >= 0 and d >= 0:
                smoves[b] = s, d, 1
    return table, shared, n0 - given, np.array(out, np.int32), moves, smoves, bad


def release(keep, n_kv, page, table, shared, free, n_free, cap):
    """(free, n_free, n_kv, shared, bad) of qwfn_paged_release."""
    free, pages, room = free.copy(), len(shared), table.shape[1] * page
    n0 = _clip(n_free, cap)
    bad = n0 != n_free or bool((shared < 0).any())
    count = np.maximum(shared, 0).astype(np.int64)
    gone, out = np.zeros(pages, np.int64), []
    for b, (k_in, n_in) in enumerate(zip(keep, n_kv)):
        n = _clip(n_in, room)
        bad |= n != n_in
        k = _clip(k_in, n)
        first, last = -(-k // page), -(-n // page)
        if k < n and k % page:
            p = int(table[b, first - 1])
            if 0 <= p < pages and shared[p] > 0:
                bad, k, first = True, n, last
        out.append(k)
        for c in range(first, last):
            p = int(table[b, c])
            if 0 <= p < pages:
                gone[p] += 1
            else:
                bad = True
    bad |= bool((gone > count + 1).any())
    for p in np.nonzero(gone > count)[0]:
        if n0 < cap:
            free[n0] = p
            n0 += 1
        else:
            bad = True
    left = np.where(gone > count, 0, count - gone).astype(np.int32)
    return free, n0, np.array(out, np.int32), left, bad


def compact(n_kv, page, table, shared, free, n_free, cap):
    """(table, shared, free, n_free, map, moves, bad) of qwfn_paged_compact; free: what is on the stack."""
    pages, room = len(shared), table.shape[1] * page
    n0 = _clip(n_free, cap)
    stack = [int(p) for p in free[:n0]]
    dead = {p for p in stack if 0 <= p < pages}
    bad = n0 != n_free or len(dead) != len(stack)
    live = pages - len(dead)
    src = [p for p in range(live, pages) if p not in dead]
    dst = [p for p in range(live) if p in dead]
    new = {p: p for p in range(pages) if p not in dead}
    new.update(zip(src, dst))
    out = np.zeros(pages, np.int32)
    for p, q in new.items():
        out[q] = shared[p]
    table = table.copy()
    for b, n_in in enumerate(n_kv):
        n = _clip(n_in, room)
        bad |= n != n_in
        for c in range(-(-n // page)):
            if int(table[b, c]) in new:
                table[b, c] = new[int(table[b, c])]
            else:
                bad = True
    stack = np.arange(pages - 1, live - 1, -1, dtype=np.int32)
    moves = np.array([(s * page, d * page, page) for s, d in zip(src, dst)], np.int32).reshape(-1, 3)
    return table, out, stack, pages - live, np.array([new.get(p, -1) for p in range(pages)], np.int32), moves, bad


def masks(parents, n_tree=None, n_past=None):
    """(masks uint64, positions int32, bad) of qwfn_tree_masks."""
    B, T = parents.shape
    m, pos, bad = np.zeros((B, T), np.uint64), np.full((B, T), -1, np.int32), False
    for b in range(B):
        n = T if n_tree is None else _clip(n_tree[b], T)
        bad |= n_tree is not None and n != n_tree[b]
        depth = []
        for t in range(n):
            p = int(parents[b, t])
            if p < -1 or p >= t:
                bad, p = True, -1
            m[b, t] = np.uint64(1 << t) | (m[b, p] if p >= 0 else np.uint64(0))
            depth.append(depth[p] + 1 if p >= 0 else 0)
            pos[b, t] = depth[t] + (0 if n_past is None else n_past[b])
    return m, pos, bad


def nodes_of(word, n):
    return [j for j in range(n) if int(word) >> j & 1]


def accept(caches, page, table, n_kv, m, leaf, n_tree=None):
    """(caches, n_keep, cu, path, bad) of qwfn_paged_accept."""
    B, T = m.shape
    caches, bad, keep, cu, path = [c.copy() for c in caches], False, [], [0], []
    pages = len(caches[0]) // page if caches else 0

    def row(b, token):
        p = int(table[b, token // page])
        return p * page + token % page if 0 <= p < pages else None

    for b in range(B):
        n = _clip(n_kv[b], table.shape[1] * page)
        nt = min(T, n) if n_tree is None else _clip(n_tree[b], min(T, n))
        bad |= n != n_kv[b] or (n_tree is not None and nt != n_tree[b]) or not -1 <= leaf[b] < nt
        nodes = nodes_of(m[b, leaf[b]], nt) if 0 <= leaf[b] < nt else []
        keep.append(n - nt + len(nodes))
        cu.append(cu[-1] + len(nodes))
        path += [b * T + t for t in nodes]
        for i, t in enumerate(nodes):
            s, d = row(b, n - nt + t), row(b, n - nt + i)
            if caches:
                bad |= s is None or d is None
            for c in caches:
                if s is not None and d is not None:
                    c[d] = c[s]
    path += [0] * (B * T - len(path))
    return caches, np.array(keep, np.int32), np.array(cu, np.int32), np.array(path, np.int32), bad


def attention(q, kc, vc, rows, kvh, scale, base, words, variant=1, terms=2):
    """One request's tree: q float32 [T, nh, D], rows its cache rows in order (-1: a masked key), the first `base` of them the
    context; node t sees the context and the nodes in words[t] (None: no node, its output is 0). Returns the output and the
    tolerance of a correct float32 implementation, float64 [T, nh, D].

    The tolerance is paged_ref.attention's: scores 2^-24 a block, exponentials 2^-22, sums 2^-24 a step. P and V enter the second
    product as pairs of f16 (each 2^-22 off, and 2^-22 for the product of the two small halves: 3 2^-22 < 2^-20 with the
    exponential's), below the range of f16 at most 2^-32 of the largest |v| of any key, as there. terms = 1 (bf16 results): as one
    f16 each, 2^-11 (cut off) and 2^-12 of sum p |v| more."""
    T, nh, D = q.shape
    rep, n = nh // kvh, len(rows)
    out, tol = np.zeros((T, nh, D)), np.zeros((T, nh, D))
    rows = np.asarray(rows, np.int64)
    live = rows >= 0
    k, v = (R.rows_f64(c, np.where(live, rows, 0), kvh, D) for c in (kc, vc))
    qd = R.requantise(q, variant)
    for t in range(T):
        if words[t] is None:
            continue
        see = live.copy()
        for j in range(base, n):
            see[j] &= bool(int(words[t]) >> (j - base) & 1)
        if not see.any():
            continue
        for h in range(nh):
            ks, vs = k[see, h // rep], v[see, h // rep]
            prod = (ks * qd[t, h]).reshape(len(ks), -1, 32).sum(-1)
            s, mag = prod.sum(-1) * scale, np.abs(prod).sum(-1).max() * abs(scale)
            p = np.exp(s - s.max())
            out[t, h] = p @ vs / p.sum()
            eps = 2 * (D // 32 + 4) * 2.0 ** -24 * mag + 2.0 ** -20 + (len(ks) // 16 + 16) * 2.0 ** -24
            eps = 2 * eps + (2.0 ** -11 + 2.0 ** -12 if terms == 1 else 0)
            tol[t, h] = eps * (p @ np.abs(vs)) / p.sum() + len(ks) * 2.0 ** -32 * np.abs(vs).max() + 1e-30
    return out, tol


def linear(q, k, v, g, state, words, scale):
    """One request and value head: q, k float64 [T, dk], v [T, dv], g [T], state [dk, dv]; node t sees words[t] (None: no node).
    Returns the outputs by the formula and their tolerance, float64 [T, dv].

    The tolerance: products of 24-bit values round once (2^-24), sums of dk and of T terms 2^-24 a term at most in any order, the
    decays' exponentials 2^-22 and the F32 cast of an exponent of size |G| log2(e) 2^-24 |G| 1.5; relative to the sums of the
    absolute values."""
    T, dk = q.shape
    out, tol = np.zeros((T, v.shape[1])), np.zeros((T, v.shape[1]))
    g = np.maximum(g, -1000 * np.log(2.0))
    sees = [nodes_of(w, T) if w is not None else [] for w in words]
    G = np.array([sum(g[j] for j in s) for s in sees])
    for t in range(T):
        if words[t] is None:
            continue
        e = np.exp(G[t])
        out[t] = e * (q[t] @ state)
        mag = e * (np.abs(q[t]) @ np.abs(state)) * (1 + 1.5 * abs(G[t]) / max(dk, 1))
        for j in sees[t]:
            d = np.exp(G[t] - G[j])
            out[t] += d * (q[t] @ k[j]) * v[j]
            mag += d * (np.abs(q[t]) @ np.abs(k[j])) * np.abs(v[j]) * (1 + 1.5 * abs(G[t] - G[j]) / max(dk, 1))
        tol[t] = (dk + T + 16) * 2.0 ** -24 * mag + 1e-38
    return out * scale, tol * abs(scale)
