"""Shared pages on the GPU: forks, releases, compaction and the copies of their rows against a loop in Python."""
import numpy as np
import pytest
import torch

import tree_ref as R
from gpu_util import dev, host, say

pytestmark = pytest.mark.gpu


def ws_of(n):
    return torch.full((max(int(n), 16),), 0x5A, dtype=torch.uint8, device="cuda")


def i32(x):
    return dev(np.asarray(x, np.int32))


def blank(*n):
    return torch.full(n, -99, dtype=torch.int32, device="cuda")


class Pool:
    """Requests in families with common first pages; pages in random order, the others on the stack."""

    def __init__(self, seed, B, page, max_pages, family=1, spare=20):
        rng = np.random.default_rng(seed)
        self.page = page
        self.n_kv = rng.integers(0, max_pages * page + 1, B).astype(np.int32)
        have = -(-self.n_kv // page)
        pages = int(have.sum()) + spare
        ids = rng.permutation(pages).astype(np.int32)
        self.table = np.full((B, max_pages + 1), -7, np.int32)
        at = 0
        for b in range(B):
            f = b // family * family
            common = int(rng.integers(0, min(self.n_kv[b], self.n_kv[f]) // page + 1)) if b != f else 0
            self.table[b, :common] = self.table[f, :common]
            self.table[b, common:have[b]] = ids[at:at + have[b] - common]
            at += have[b] - common
        held = np.bincount(np.concatenate([self.table[b, :have[b]] for b in range(B)]), minlength=pages)
        self.shared = np.maximum(held - 1, 0).astype(np.int32)
        unused = rng.permutation(np.nonzero(held == 0)[0]).astype(np.int32)
        self.n_free = len(unused)
        self.free = np.full(pages + 3, -1, np.int32)
        self.free[:self.n_free] = unused


# ---------------------------------------------------------------- fork

def check_fork(K, src, n_tok, n_kv, page, table, shared, free, n_free, in_place=False, states=None):
    B, cap = len(src), len(free)
    tab, kv, sh, nf = i32(table), i32(n_kv), i32(shared), i32([n_free])
    kvo, sho, nfo = (kv, sh, nf) if in_place else (blank(B), blank(len(shared)), blank(1))
    moves, smoves = blank(B + 1, 3), blank(B + 1, 3)
    K.device_status()
    K.paged_fork(i32(src), kv, page, tab, sh, i32(free), nf, nfo, kvo, sho, moves[:B], n_tok=None if n_tok is None else i32(n_tok),
                 states=None if states is None else i32(states), state_moves=smoves[:B], ws=ws_of(K.paged_workspace_size(B)))
    flags = K.device_status()
    ref = R.fork(src, n_tok, n_kv, page, table, shared, free, n_free, cap, states)
    got = [host(x) for x in (tab, sho, nfo, kvo, moves[:B], smoves[:B])]
    for name, a, b in zip(("table", "shared", "n_free", "n_kv", "moves", "state_moves"), got, ref):
        assert np.array_equal(a, np.asarray(b).reshape(a.shape)), name
    assert (host(moves)[B] == -99).all() and (host(smoves)[B] == -99).all()
    assert flags == (K.DEVERR_PAGES if ref[-1] else 0)
    return ref


@pytest.mark.parametrize("in_place", [False, True])
def test_fork_against_loop(gpu, in_place):
    for seed in range(30):
        rng = np.random.default_rng(seed)
        B, page = int(rng.choice([2, 3, 17, 64, 65, 300, 1025, 1300])), int(rng.choice([1, 2, 16, 33]))
        p = Pool(seed, B, page, int(rng.integers(1, 40)))
        src = np.full(B, -1, np.int32)
        kids = rng.permutation(B)[:int(rng.integers(0, B))]
        olds = np.setdiff1d(np.arange(B), kids)
        src[kids] = rng.choice(olds, len(kids))
        p.n_kv[kids] = 0
        tok = np.where(src >= 0, (p.n_kv[src] * rng.choice([0, 0.3, 1, 1], B)).astype(np.int32), 0)
        say(f"fork seed {seed}: B={B} page={page} forks={len(kids)} in_place={in_place}")
        need = int((tok % page > 0)[src >= 0].sum())
        n_free = min(p.n_free, need if seed % 3 else need // 2)
        states = rng.permutation(B + 5)[:B] - 2 if seed % 2 else None
        check_fork(gpu, src, None if seed % 5 == 4 else tok, p.n_kv, page, p.table, p.shared, p.free, n_free, in_place, states)


@pytest.mark.parametrize("in_place", [False, True])
def test_fork_refused_requests(gpu, in_place):
    say(f"fork: chains, held rows, lengths, broken tables, in_place={in_place}")
    table = np.arange(60, dtype=np.int32).reshape(6, 10)
    shared, free = np.zeros(70, np.int32), np.arange(60, 70, dtype=np.int32)
    n = [35, 0, 0, 20, 0, 0]
    for src, tok, n_kv, n_free in [
            ([-1, 0, 1, -1, 0, 3], None, n, 10),                  # 2 from 1, which is forked itself
            ([-1, 0, 2, 3, 6, 99], None, n, 10),                  # itself, a row that is held, none
            ([-1, 0, 0, 0, 0, 3], [0, 36, -1, 5, 35, 20], n, 10),
            ([-1, 0, 0, 0, 3, 3], [0, 33, 32, 5, 16, 17], n, 1),  # one page for three
            ([-1, 0, 0, -1, 3, 0], [0, 0, 16, 0, 0, 35], n, 0),
            ([-1, 0, -1, -1, 3, -5], None, [-4, 0, 0, 900, 0, -1], 10),
            ([-1, 0, -1, -1, -1, -1], None, n, -1), ([-1, 0, -1, -1, -1, -1], None, n, 99)]:
        check_fork(gpu, src, tok, n_kv, 16, table, shared, free, n_free, in_place)
    broken = table.copy()
    broken[0, 0], broken[3, 1] = -1, 70
    check_fork(gpu, [-1, 0, -1, -1, 3, 0], None, n, 16, broken, shared, free, 10, in_place)
    check_fork(gpu, [-1, 0], None, [35, 0], 16, table[:2], shared, np.array([3, 70], np.int32), 2, in_place)
    check_fork(gpu, [-1], None, [35], 16, table[:1], shared, free, 10, in_place)


# ---------------------------------------------------------------- release

def check_release(K, keep, n_kv, page, table, shared, free, n_free, in_place=False):
    B, cap = len(n_kv), len(free)
    kv, sh, nf, fr = i32(n_kv), i32(shared), i32([n_free]), i32(list(free) + [-55])
    kvo, sho, nfo = (kv, sh, nf) if in_place else (blank(B), blank(len(shared)), blank(1))
    tab = i32(table)
    K.device_status()
    K.paged_release(i32(keep), kv, page, tab, sh, fr[:cap], nf, nfo, kvo, sho,
                    ws=ws_of(K.paged_release_workspace_size(B, len(shared))))
    flags = K.device_status()
    ref = R.release(keep, n_kv, page, table, shared, free, n_free, cap)
    got = [host(x) for x in (fr[:cap], nfo, kvo, sho)]
    for name, a, b in zip(("free", "n_free", "n_kv", "shared"), got, ref):
        assert np.array_equal(a, np.asarray(b).reshape(a.shape)), name
    assert host(fr)[cap] == -55 and np.array_equal(host(tab), table)
    assert flags == (K.DEVERR_PAGES if ref[-1] else 0)
    return ref


@pytest.mark.parametrize("in_place", [False, True])
def test_release_against_loop(gpu, in_place):
    for seed in range(30):
        rng = np.random.default_rng(100 + seed)
        B, page = int(rng.choice([1, 2, 63, 64, 65, 300, 1025])), int(rng.choice([1, 2, 16, 33]))
        p = Pool(seed, B, page, int(rng.integers(1, 60)), family=int(rng.choice([1, 2, 5])))
        keep = np.where(rng.random(B) < 0.4, 0, p.n_kv - rng.integers(-2, 2 * page + 3, B))
        say(f"release seed {seed}: B={B} page={page} pages={len(p.shared)} in_place={in_place}")
        check_release(gpu, keep, p.n_kv, page, p.table, p.shared, p.free, p.n_free, in_place)


@pytest.mark.parametrize("in_place", [False, True])
def test_release_of_bad_tables(gpu, in_place):
    say(f"release: lengths, stack, counts and entries out of range, in_place={in_place}")
    table = np.arange(24, dtype=np.int32).reshape(3, 8)
    zero, free = np.zeros(24, np.int32), np.full(26, -1, np.int32)
    check_release(gpu, [-1, 5, 100], [10, -3, 40], 4, table, zero, free, 0, in_place)
    check_release(gpu, [0, 0, 0], [8, 8, 8], 4, table, zero, free, -2, in_place)
    check_release(gpu, [0, 0, 0], [8, 8, 8], 4, table, zero, free, 99, in_place)
    check_release(gpu, [0, 0, 0], [32, 32, 32], 4, table, zero, free, 7, in_place)       # more pages than the stack has room for
    bad = table.copy()
    bad[0, 1], bad[1, 0], bad[2, 2] = -1, 24, 16
    check_release(gpu, [0, 0, 0], [32, 32, 32], 4, bad, zero, free, 0, in_place)         # one twice, two outside
    counts = zero.copy()
    counts[[0, 1, 2]] = -1, 3, 1
    check_release(gpu, [0, 9, 32], [32, 32, 32], 4, table, counts, free, 0, in_place)
    check_release(gpu, [6, 4, 9], [8, 5, 9], 4, table, counts, free, 0, in_place)        # page 1 is held by others: kept whole
    check_release(gpu, [4, 8, 3], [8, 8, 8], 4, table, counts, free, 0, in_place)


def test_release_of_a_large_pool(gpu):
    """More pages than one workgroup of the last launch takes."""
    for seed, B in ((1, 400), (2, 37)):
        p = Pool(seed, B, 1, 900, family=3, spare=12345)
        say(f"release: {len(p.shared)} pages, {B} requests")
        rng = np.random.default_rng(seed)
        check_release(gpu, np.where(rng.random(B) < 0.5, 0, p.n_kv - 1), p.n_kv, 1, p.table, p.shared, p.free, p.n_free)


# ---------------------------------------------------------------- compact

def check_compact(K, n_kv, page, table, shared, free, n_free, in_place=False):
    B, pages, cap = len(n_kv), len(shared), len(free)
    tab, sh, fr, nf = i32(table), i32(shared), i32(free), i32([n_free])
    tabo, sho, fro, nfo = (tab, sh, fr, nf) if in_place else (tab.clone(), blank(pages), blank(cap), blank(1))
    pmap, moves, n_moves = blank(pages), blank((pages + 1) // 2 + 1, 3), blank(1)
    K.device_status()
    K.paged_compact(i32(n_kv), page, tab, sh, fr, nf, tabo, sho, fro, nfo, pmap, moves, n_moves,
                    ws=ws_of(K.paged_compact_workspace_size(pages)))
    flags = K.device_status()
    t, s, stack, n, m, mv, bad = R.compact(n_kv, page, table, shared, free, n_free, cap)
    assert host(nfo)[0] == n and host(n_moves)[0] == len(mv)
    assert np.array_equal(host(pmap), m) and np.array_equal(host(tabo), t) and np.array_equal(host(sho), s)
    assert np.array_equal(host(fro)[:n], stack) and np.array_equal(host(moves)[:len(mv)], mv)
    assert (host(moves)[len(mv):] == -99).all()
    assert (host(fro)[n:] == (np.asarray(free)[n:] if in_place else -99)).all()
    assert flags == (K.DEVERR_PAGES if bad else 0)
    return t, s, stack, n, m, mv


@pytest.mark.parametrize("in_place", [False, True])
def test_compact_against_loop(gpu, in_place):
    for seed in range(30):
        rng = np.random.default_rng(200 + seed)
        B, page = int(rng.choice([1, 2, 63, 300, 700])), int(rng.choice([1, 2, 16, 33]))
        p = Pool(seed, B, page, int(rng.integers(1, 60)), family=int(rng.choice([1, 3])), spare=int(rng.choice([0, 1, 31, 500, 20000])))
        say(f"compact seed {seed}: B={B} page={page} pages={len(p.shared)} free={p.n_free} in_place={in_place}")
        check_compact(gpu, p.n_kv, page, p.table, p.shared, p.free, p.n_free, in_place)


@pytest.mark.parametrize("in_place", [False, True])
def test_compact_edges(gpu, in_place):
    say(f"compact: full, empty and broken pools, in_place={in_place}")
    one = np.zeros((1, 4), np.int32)
    z = lambda n: np.zeros(n, np.int32)  # noqa: E731
    check_compact(gpu, [0], 16, one, z(1), z(1), 1, in_place)
    check_compact(gpu, [3], 16, one, z(1), z(1), 0, in_place)
    for n in (31, 32, 33, 64):                                    # nothing live; all of it; only the last page
        check_compact(gpu, [0], 16, one, z(n), np.arange(n, dtype=np.int32), n, in_place)
        check_compact(gpu, [0], 16, one, np.arange(n, dtype=np.int32), z(n), 0, in_place)
        check_compact(gpu, [16], 16, np.full((1, 4), n - 1, np.int32), np.arange(n, dtype=np.int32), np.arange(n, dtype=np.int32), n - 1,
                      in_place)
    free = np.array([3, 3, 40, -1, 7, 0] + [0] * 30, np.int32)    # twice, outside
    table = np.array([[1, 2, 35, 7], [-3, 99, 5, 36]], np.int32)  # 7 is on the stack, -3, 99 and 36 are none
    check_compact(gpu, [64, 64], 16, table, np.arange(36, dtype=np.int32), free, 6, in_place)
    check_compact(gpu, [-1, 900], 16, table, np.arange(36, dtype=np.int32), free, 5, in_place)
    check_compact(gpu, [20, 0], 16, table, np.arange(36, dtype=np.int32), free, -4, in_place)
    check_compact(gpu, [20, 0], 16, np.abs(table) % 36, np.arange(36, dtype=np.int32), np.arange(36, dtype=np.int32), 99, in_place)


# ---------------------------------------------------------------- copies

def rows_copied(c, moves, limit, max_rows):
    """(rows after the moves, whether one was left out)."""
    out, bad = c.copy(), False
    for s, d, n in np.asarray(moves).tolist():
        if n == 0:
            continue
        if not 0 < n <= max_rows or s < 0 or d < 0 or s + n > limit or d + n > limit:
            bad = True
            continue
        out[d:d + n] = c[s:s + n]
    return out, bad


@pytest.mark.parametrize("row,dtype,pad", [(544, torch.uint8, 0), (544, torch.uint8, 32), (68, torch.uint8, 0), (34, torch.uint8, 0),
                                           (102, torch.uint8, 4), (272, torch.uint8, 2), (5, torch.float32, 0), (300, torch.bfloat16, 0),
                                           (3, torch.float16, 1), (64, torch.int32, 0)])
def test_copy_rows(gpu, row, dtype, pad):
    rng = np.random.default_rng(row)
    limit = 700
    moves = np.array([(0, 100, 16), (16, 116, 1), (0, 0, 0), (-5, 3, 0), (40, 140, 7), (50, limit - 16, 16), (640, 200, 16)], np.int32)
    many = np.array([(300 + 2 * i, 301 + 2 * i, 1) for i in range(90)], np.int32)
    for n_caches, mv, max_rows in [(1, moves, 16), (3, moves[:1], 16), (65, moves, 16), (2, many, 1), (2, many, 40)]:
        say(f"copy: rows of {row} {dtype}, {n_caches} tensors, {len(mv)} moves of at most {max_rows}")
        bufs = [torch.from_numpy(rng.integers(0, 256, (limit + 1, (row + pad) * torch.empty(0, dtype=dtype).element_size()), np.uint8)).cuda()
                for _ in range(n_caches)]
        before = [host(x) for x in bufs]
        caches = [x[:limit].view(dtype)[:, :row] for x in bufs]
        gpu.device_status()
        gpu.paged_copy(gpu.cache_list(caches), i32(mv), max_rows)
        assert gpu.device_status() == 0
        width = row * caches[0].element_size()
        for x, y in zip(bufs, before):
            want = y.copy()
            want[:limit, :width] = rows_copied(y[:limit, :width], mv, limit, max_rows)[0]
            assert np.array_equal(host(x), want)


def test_copy_bad_moves_and_counts(gpu):
    say("copy: rows and counts out of range")
    rng = np.random.default_rng(3)
    y = rng.integers(0, 256, (100, 272), np.uint8)
    moves = np.array([(0, 50, 4), (-1, 60, 4), (10, 97, 4), (97, 60, 4), (20, 64, -3), (20, 70, 9), (30, 80, 8), (2 ** 31 - 1, 5, 2)], np.int32)
    for count, flagged in ((None, True), (1, False), (0, False), (8, True), (-2, True), (99, True)):
        x = dev(y)
        gpu.device_status()
        gpu.paged_copy([x], i32(moves), 8, n_moves=None if count is None else i32([count]))
        assert gpu.device_status() == (gpu.DEVERR_SET_ROWS_INDEX if flagged else 0)
        n = 8 if count is None else min(max(count, 0), 8)
        assert np.array_equal(host(x), rows_copied(y, moves[:n], 100, 8)[0])
    x = dev(y)
    gpu.paged_copy([], i32(moves), 8)
    gpu.paged_copy([x], i32(moves[:0]), 8)
    assert np.array_equal(host(x), y)


def test_copy_past_4_gib(gpu):
    """Rows on both sides of 2^32 bytes of one tensor, and a row of several MB."""
    say("copy: a tensor of 4.3 GB")
    n = (1 << 32) // 1088 + 3000
    x = torch.zeros((n, 1088), dtype=torch.uint8, device="cuda")
    x[5:9] = torch.arange(4, dtype=torch.uint8, device="cuda")[:, None] + 1
    x[n - 2:] = 9
    gpu.paged_copy([x], i32([(5, n - 100, 4), (n - 2, 40, 2)]), 16)
    torch.cuda.synchronize()
    assert [int(x[n - 100 + i].max()) for i in range(4)] == [1, 2, 3, 4] and int(x[40:42].min()) == 9
    assert int(x.sum(dtype=torch.int64)) == 1088 * (2 * 10 + 4 * 9)
    del x
    s = torch.randn((6, 48, 128, 128), device="cuda")
    want = s.clone()
    want[4] = s[1]
    gpu.paged_copy([s], i32([(1, 4, 1)]), 1)
    assert torch.equal(s, want)


# ---------------------------------------------------------------- together

def test_serving_with_forks(gpu):
    """Prompts, their forks, steps of all, releases and a compaction: every request always reads the rows that it wrote or took
    over. The whole runs in a captured graph too."""
    K, page, B, cols, pages, L = gpu, 4, 6, 12, 60, 3
    rng = np.random.default_rng(11)
    say("shared pages: extend, fork, copy, release, compact")
    caches = [torch.zeros((pages * page, 34), dtype=torch.uint8, device="cuda") for _ in range(L)]
    lst = K.cache_list(caches)
    table, shared = blank(B, cols), torch.zeros(pages, dtype=torch.int32, device="cuda")
    free, n_free = i32(rng.permutation(pages)), i32([pages])
    n_kv = torch.zeros(B, dtype=torch.int32, device="cuda")
    ws = ws_of(K.paged_release_workspace_size(B, pages) + K.paged_compact_workspace_size(pages))
    mine = [[] for _ in range(B)]
    stamp = [0]

    def extend(new):
        n_tok = int(sum(new))
        cu, slots = blank(B + 1), blank(n_tok)
        K.paged_extend(n_kv, i32(new), page, table, free, n_free, n_free, n_kv, cu, slots, ws=ws)
        rows = host(slots)
        assert (rows >= 0).all()
        i = 0
        for b in range(B):
            for _ in range(new[b]):
                stamp[0] += 1
                mine[b].append(stamp[0])
                for j, c in enumerate(caches):
                    c[int(rows[i])] = (stamp[0] * 3 + j) % 251
                i += 1

    def verify():
        t, n, s = host(table), host(n_kv), host(shared)
        held = np.zeros(pages, int)
        for b in range(B):
            assert n[b] == len(mine[b])
            for p in t[b, :-(-n[b] // page)]:
                held[p] += 1
            for j, c in enumerate(caches):
                rows = [t[b, i // page] * page + i % page for i in range(n[b])]
                assert host(c)[rows, 0].tolist() == [(x * 3 + j) % 251 for x in mine[b]]
        assert np.array_equal(np.maximum(held - 1, 0), s)
        stack = host(free)[:int(n_free)]
        assert sorted(stack) == np.nonzero(held == 0)[0].tolist()

    def fork(src, tok=None):
        moves = blank(B, 3)
        K.paged_fork(i32(src), n_kv, page, table, shared, free, n_free, n_free, n_kv, shared, moves,
                     n_tok=None if tok is None else i32(tok), ws=ws)
        K.paged_copy(lst, moves, page)
        for b, f in enumerate(src):
            if f >= 0:
                mine[b] = list(mine[f] if tok is None else mine[f][:tok[b]])

    def release(keep):
        K.paged_release(i32(keep), n_kv, page, table, shared, free, n_free, n_free, n_kv, shared, ws=ws)
        for b in range(B):
            mine[b] = mine[b][:keep[b]]

    def compact():
        pmap, moves, n_moves = blank(pages), blank(pages // 2, 3), blank(1)
        K.paged_compact(n_kv, page, table, shared, free, n_free, table, shared, free, n_free, pmap, moves, n_moves, ws=ws)
        K.paged_copy(lst, moves, page, n_moves=n_moves)

    K.device_status()
    extend([13, 0, 0, 8, 0, 0]); verify()
    fork([-1, 0, 0, -1, 3, -1], [0, 13, 9, 0, 8, 0]); verify()
    extend([1, 2, 3, 4, 5, 6]); verify()
    release([13, 15, 0, 8, 9, 6]); verify()
    compact(); verify()
    fork([-1, -1, 1, -1, -1, -1]); verify()
    extend([3, 3, 3, 3, 3, 3]); verify()
    release([0, 18, 15, 0, 0, 0]); verify()
    compact(); verify()
    release([0, 0, 0, 0, 0, 0]); verify()
    assert K.device_status() == 0 and int(n_free) == pages and int(shared.sum()) == 0


def test_captured_and_replayed(gpu):
    """Fork, copy, release and compaction in one graph, replayed over new inputs with eager work between, two graphs with a
    workspace each."""
    K, page, B = gpu, 4, 40
    say("shared pages: captured and replayed")
    pools = [Pool(s, B, page, 9, family=4, spare=90) for s in (1, 2, 3)]
    pages = max(len(p.shared) for p in pools)

    def pad(p):
        q = Pool.__new__(Pool)
        extra = np.arange(len(p.shared), pages, dtype=np.int32)
        q.page, q.n_kv, q.table = page, p.n_kv.copy(), p.table
        q.n_kv[::4] = 0
        q.shared = np.concatenate([p.shared, np.zeros(pages - len(p.shared), np.int32)])
        q.n_free = p.n_free + len(extra)
        q.free = np.concatenate([p.free[:p.n_free], extra, np.full(pages - q.n_free + 2, -1, np.int32)])
        return q

    pools = [pad(p) for p in pools]
    src = np.full(B, -1, np.int32)
    src[::4] = np.arange(B)[1::4]
    graphs = []
    for keep_off in (0, 5):
        b = dict(table=blank(B, pools[0].table.shape[1]), n_kv=blank(B), shared=blank(pages), free=blank(len(pools[0].free)), n_free=blank(1))
        t = dict(n_kv2=blank(B), shared2=blank(pages), nf2=blank(1), moves=blank(B, 3), nf3=blank(1), n_kv3=blank(B), shared3=blank(pages),
                 pmap=blank(pages), cm=blank((pages + 1) // 2, 3), nm=blank(1))
        cache = torch.randint(0, 256, (pages * page, 34), dtype=torch.uint8, device="cuda")
        keep, sd, lst = blank(B), i32(src), K.cache_list([cache])
        ws = [ws_of(n) for n in (K.paged_workspace_size(B), K.paged_release_workspace_size(B, pages), K.paged_compact_workspace_size(pages))]

        def calls():
            K.paged_fork(sd, b["n_kv"], page, b["table"], b["shared"], b["free"], b["n_free"], t["nf2"], t["n_kv2"], t["shared2"],
                         t["moves"], ws=ws[0])
            K.paged_copy(lst, t["moves"], page)
            K.paged_release(keep, t["n_kv2"], page, b["table"], t["shared2"], b["free"], t["nf2"], t["nf3"], t["n_kv3"], t["shared3"],
                            ws=ws[1])
            K.paged_compact(t["n_kv3"], page, b["table"], t["shared3"], b["free"], t["nf3"], b["table"], t["shared3"], b["free"],
                            t["nf3"], t["pmap"], t["cm"], t["nm"], ws=ws[2])
            K.paged_copy(lst, t["cm"], page, n_moves=t["nm"])

        def load(p):
            for k in ("table", "n_kv", "shared", "free"):
                b[k].copy_(i32(getattr(p, k)))
            b["n_free"].copy_(i32([p.n_free]))
            keep.copy_(i32(np.maximum(p.n_kv - keep_off, 0)))

        load(pools[0])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            calls()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            calls()
        graphs.append((g, b, t, cache, load, keep, (sd, lst, ws)))
    for p in pools + pools[:1]:
        for g, b, t, cache, load, keep, _ in graphs:
            load(p)
            start, k = host(cache).copy(), host(keep)
            g.replay()
            torch.cuda.synchronize()
            tab, sh, nf, nkv, mv, _, _ = R.fork(src, None, p.n_kv, page, p.table, p.shared, p.free, p.n_free, len(p.free))
            c = rows_copied(start, mv, len(start), page)[0]
            free, nf, nkv, sh, _ = R.release(k, nkv, page, tab, sh, p.free, nf, len(p.free))
            tab, sh, stack, nf, _, mv, _ = R.compact(nkv, page, tab, sh, free, nf, len(p.free))
            c = rows_copied(c, mv, len(c), page)[0]
            assert np.array_equal(host(cache), c) and np.array_equal(host(b["table"]), tab)
            assert np.array_equal(host(t["shared3"]), sh) and int(t["nf3"]) == nf
            assert np.array_equal(host(b["free"])[:nf], stack) and np.array_equal(host(t["n_kv3"]), nkv)
            torch.cuda.synchronize()
    K.device_status()


def test_on_another_stream(gpu):
    say("shared pages: on a side stream, behind work of that stream")
    p = Pool(5, 64, 16, 9, family=2)
    side = torch.cuda.Stream()
    B, pages = 64, len(p.shared)
    args = [i32(x) for x in (np.zeros(B), p.n_kv, p.table, p.shared, p.free, [p.n_free])]
    out = [blank(1), blank(B), blank(pages)]
    ws = ws_of(gpu.paged_release_workspace_size(B, pages))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(5):
            big = big @ big * 1e-3
        args[0].fill_(3)
        gpu.paged_release(args[0], args[1], 16, args[2], args[3], args[4], args[5], *out, ws=ws)
    torch.cuda.synchronize()
    ref = R.release(np.full(B, 3), p.n_kv, 16, p.table, p.shared, p.free, p.n_free, len(p.free))
    assert np.array_equal(host(args[4]), ref[0]) and np.array_equal(host(out[2]), ref[3]) and np.array_equal(host(out[1]), ref[2])
    gpu.device_status()
