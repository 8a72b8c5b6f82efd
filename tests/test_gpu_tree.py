"""Trees of drafted tokens on the GPU: masks, accepted paths, attention over pages and linear attention of the nodes against
loops and float64, and a verify step of all of them."""
import numpy as np
import pytest
import torch

import paged_ref as P
import tree_ref as R
from gpu_util import dev, host, say
from test_gpu_paged import HALF_STEP, Case, pool, ws_of

pytestmark = pytest.mark.gpu


def i32(x):
    return dev(np.asarray(x, np.int32))


def blank(*n):
    return torch.full(n, -99, dtype=torch.int32, device="cuda")


def words(m):
    return dev(np.asarray(m, np.uint64).view(np.int64))


def random_parents(rng, B, T, kind=None):
    """Chains, stars, bushes, forests."""
    out = np.zeros((B, T), np.int32)
    for b in range(B):
        k = kind or ("chain", "star", "bush", "bush", "forest")[int(rng.integers(0, 5))]
        for t in range(T):
            out[b, t] = {"chain": t - 1, "star": -1 if t == 0 else 0, "bush": -1 if t == 0 else int(rng.integers(max(0, t - 9), t)),
                         "forest": int(rng.integers(-1, t)) if t else -1}[k]
    return out


# ---------------------------------------------------------------- masks

def check_masks(K, parents, n_tree=None, n_past=None):
    B, T = parents.shape
    m, pos = torch.full((B + 1, T), 77, dtype=torch.int64, device="cuda"), blank(B + 1, T)
    K.device_status()
    K.tree_masks(i32(parents), m[:B], n_tree=None if n_tree is None else i32(n_tree),
                 n_past=None if n_past is None else i32(n_past), pos=pos[:B])
    flags = K.device_status()
    ref, rp, bad = R.masks(parents, n_tree, n_past)
    assert np.array_equal(host(m)[:B].view(np.uint64), ref) and np.array_equal(host(pos)[:B], rp)
    assert (host(m)[B] == 77).all() and (host(pos)[B] == -99).all() and flags == (K.DEVERR_PAGES if bad else 0)


@pytest.mark.parametrize("T", [1, 2, 3, 15, 16, 31, 32, 33, 63, 64])
def test_masks(gpu, T):
    say(f"tree masks: T={T}")
    rng = np.random.default_rng(T)
    for kind in ("chain", "star", "bush", "forest"):
        check_masks(gpu, random_parents(rng, 5, T, kind))
    B = 70
    check_masks(gpu, random_parents(rng, B, T), rng.integers(0, T + 1, B), rng.integers(0, 1 << 20, B))
    par = rng.integers(-3, T + 2, (B, T)).astype(np.int32)                   # parents that are none
    check_masks(gpu, par, rng.integers(-2, T + 3, B))


# ---------------------------------------------------------------- accepted paths

def check_accept(K, caches, page, table, n_kv, m, leaf, n_tree=None, lists=True):
    B, T = m.shape
    cd = [dev(c) for c in caches]
    keep, cu, path = blank(B + 1), blank(B + 2), blank(B * T + 1)
    K.device_status()
    K.paged_accept(K.cache_list(cd), page, i32(table), i32(n_kv), words(m), i32(leaf), keep[:B],
                   n_tree=None if n_tree is None else i32(n_tree), cu_path=cu[:B + 1] if lists else None,
                   path=path[:B * T] if lists else None)
    flags = K.device_status()
    rc, rk, rcu, rp, bad = R.accept(caches, page, table, n_kv, m, leaf, n_tree)
    assert np.array_equal(host(keep)[:B], rk) and host(keep)[B] == -99
    if lists:
        assert np.array_equal(host(cu)[:B + 1], rcu) and np.array_equal(host(path)[:B * T], rp)
    assert host(cu)[-1] == -99 and host(path)[-1] == -99
    for a, b in zip(cd, rc):
        assert np.array_equal(host(a), b)
    assert flags == (K.DEVERR_PAGES if bad else 0)


def accept_inputs(rng, B, T, page, row, n_caches, full=False):
    lens = rng.integers(0, 3 * page + 40, B)
    nt = np.full(B, T) if full else rng.integers(0, T + 1, B)
    n_kv = lens + nt
    have = -(-n_kv // page)
    pages = int(have.sum()) + 3
    ids, at = rng.permutation(pages), 0
    table = np.full((B, int(have.max()) + 1), -5, np.int32)
    for b in range(B):
        table[b, :have[b]] = ids[at:at + have[b]]
        at += have[b]
    m, _, _ = R.masks(random_parents(rng, B, T), nt)
    leaf = np.array([rng.integers(-1, n) if n else -1 for n in nt])
    return [rng.integers(0, 256, (pages * page, row), np.uint8) for _ in range(n_caches)], table, n_kv, m, leaf, nt


@pytest.mark.parametrize("B,T,page,row,n_caches", [(1, 1, 16, 544, 1), (1, 8, 16, 544, 24), (3, 64, 7, 34, 2), (5, 33, 1, 102, 3),
                                                   (70, 20, 32, 68, 2), (300, 64, 16, 272, 1), (9, 48, 16, 2176, 64), (6, 9, 4, 544, 0)])
def test_accept(gpu, B, T, page, row, n_caches):
    say(f"accept: B={B} T={T} page={page} rows of {row} in {n_caches} caches")
    rng = np.random.default_rng(B + T)
    for full in (False, True):
        c, table, n_kv, m, leaf, nt = accept_inputs(rng, B, T, page, row, n_caches, full)
        check_accept(gpu, c, page, table, n_kv, m, leaf, nt)
        check_accept(gpu, c, page, table, n_kv, m, leaf, nt, lists=False)
        if full:
            check_accept(gpu, c, page, table, n_kv, m, leaf)


def test_accept_long_paths_and_bad_inputs(gpu):
    """Paths of every length over rows that overlap their sources; leaves, lengths and pages out of range."""
    say("accept: chains with one node left out, bad inputs")
    rng = np.random.default_rng(5)
    for skip in (0, 1, 7, 8, 9, 62):
        par = np.arange(-1, 63, dtype=np.int32)[None].copy()
        if skip < 63:
            par[0, skip + 1] = skip - 1                                      # node `skip` is off the path
        m, _, _ = R.masks(par)
        table = rng.permutation(20)[None, :9].astype(np.int32)
        for leaf in (skip, skip + 1, 40, 63):
            check_accept(gpu, [rng.integers(0, 256, (20 * 16, 544), np.uint8)], 16, table, [100], m, [leaf])
    c, table, n_kv, m, leaf, nt = accept_inputs(rng, 6, 12, 4, 68, 2, True)
    for bad in (dict(leaf=[12, -2, 99, 3, 5, 0]), dict(n_tree=[-1, 13, 12, 12, 4, 0]), dict(n_kv=[-3, 10 ** 6, 5, 0, 12, 11])):
        a = dict(n_kv=n_kv, leaf=leaf, n_tree=nt)
        a.update(bad)
        a["n_kv"] = np.minimum(a["n_kv"], 10 ** 6)
        if "n_kv" in bad:
            tab = np.abs(table) % (len(c[0]) // 4)
            # a clipped length reads every column: distinct pages, so that no request writes another's rows
            tab = rng.permutation(6 * table.shape[1])[:table.size].reshape(table.shape).astype(np.int32)
            big = [rng.integers(0, 256, (tab.size * 4, 68), np.uint8) for _ in range(2)]
            check_accept(gpu, big, 4, tab, a["n_kv"], m, a["leaf"], a["n_tree"])
        else:
            check_accept(gpu, c, 4, table, a["n_kv"], m, a["leaf"], a["n_tree"])
    torn = table.copy()
    torn[:, :] = np.where(rng.random(table.shape) < 0.4, 10 ** 6, table)
    check_accept(gpu, c, 4, torn, n_kv, m, leaf, nt)


# ---------------------------------------------------------------- attention

class TreeCase(Case):
    """Requests whose last n_tree tokens are a tree."""

    def __init__(self, lens, D, kvh, rep, T, page, n_tree=None, seed=0, kind=None, m=None, **kw):
        super().__init__(lens, D, kvh, rep, T, page, seed=seed, **kw)
        rng = np.random.default_rng(seed + 77)
        B = len(lens)
        self.n_tree = n_tree
        self.nt = [min(T, n) for n in lens] if n_tree is None else list(n_tree)
        self.m = R.masks(random_parents(rng, B, T, kind))[0] if m is None else m       # (bits past a tree's nodes stay set)

    def on_gpu(self, K, ws=True, gate=False, variant=1, q=None, n_kv=None, table=None, stream=None, scale=None, m=None, n_tree=0):
        B = len(self.lens)
        self.kd, self.vd = dev(self.kc), dev(self.vc)
        qd = self.q.cuda() if q is None else q
        nb = (34, self.kd.stride(0), self.D // 32 * 34, self.n_rows * self.kd.stride(0))
        kv, vv = (K.tensor(x.data_ptr(), K.TYPE_Q8_0, (self.D, self.n_rows, self.kvh, 1), nb) for x in (self.kd, self.vd))
        td, nd = dev(self.table if table is None else table), i32(self.lens if n_kv is None else n_kv)
        tree = self.n_tree if n_tree == 0 else n_tree
        buf = torch.full((B * self.T * self.kvh * self.rep * self.D + 64,), 7.0, dtype=self.dtype, device="cuda")
        o = buf[:-64].view(B, self.T, self.kvh * self.rep, self.D)
        qv, ov = K.q_view(qd), K.out_view(o)
        w = ws_of(K.fattn_workspace_size_paged_tree(qv, kv, vv, td, self.page)) if ws else None
        if w is not None:
            w.fill_(0xFF)
        K.flash_attn_ext_paged_tree(qv, kv, vv, td, self.page, nd, words(self.m if m is None else m),
                                    self.scale if scale is None else scale, ov, n_tree=None if tree is None else i32(tree),
                                    gate=self.gate.cuda() if gate else None, variant=variant, ws=w, stream=stream)
        torch.cuda.synchronize()
        assert bool((buf[-64:] == 7.0).all())
        return o

    def reference(self, gate=False, variant=1, rows=None, scale=None, m=None):
        q, out, tol = self.q.float().numpy(), [], []
        m = self.m if m is None else m
        for b, n in enumerate(self.lens):
            w = [int(m[b, t]) if t < self.nt[b] else None for t in range(self.T)]
            x, y = R.attention(q[b], self.kc, self.vc, (rows or self.rows)[b], self.kvh, self.scale if scale is None else scale,
                               n - self.nt[b], w, variant, 1 if self.dtype == torch.bfloat16 else 2)
            out.append(x)
            tol.append(y)
        out, tol = np.stack(out), np.stack(tol)
        if gate:
            s = 1 / (1 + np.exp(-self.gate.float().numpy().astype(np.float64)))
            out, tol = out * s, tol * s + 4 * 2.0 ** -22 * np.abs(out * s)
        return out, tol + HALF_STEP[self.dtype] * (np.abs(out) + tol) + (2.0 ** -25 if self.dtype == torch.float16 else 0)


LENS = [70, 31, 32, 33, 0, 129, 65, 64, 200, 300]


@pytest.mark.parametrize("D,kvh,rep,T,page", [
    (256, 2, 8, 1, 16), (256, 2, 8, 2, 16), (256, 2, 12, 5, 64), (256, 2, 8, 9, 7), (256, 1, 16, 64, 16), (256, 2, 8, 33, 32),
    (256, 1, 1, 64, 1), (256, 1, 3, 43, 100), (128, 8, 4, 16, 16), (128, 2, 7, 37, 5), (128, 1, 16, 64, 33), (128, 1, 2, 64, 16),
    (64, 8, 8, 8, 16), (64, 1, 64, 16, 3), (64, 1, 3, 50, 256), (64, 2, 16, 64, 16)])
def test_attention_shapes(gpu, D, kvh, rep, T, page):
    say(f"tree attention D={D} kvh={kvh} rep={rep} T={T} page={page}")
    rng = np.random.default_rng(T)
    nt = [int(rng.integers(0, min(T, n) + 1)) for n in LENS]
    nt[0], nt[5] = min(T, 70), 0                                             # a whole tree, none
    TreeCase(LENS, D, kvh, rep, T, page, n_tree=nt, seed=D + T).check(gpu)
    TreeCase(LENS[:4], D, kvh, rep, T, page, seed=D).check(gpu)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gate", [False, True])
def test_attention_types_and_gate(gpu, dtype, gate):
    say(f"tree attention {dtype} gate={gate}")
    for D in (256, 128, 64):
        for T, rep in ((4, 4), (40, 6)):
            TreeCase([70, 1, 333, 0, 97], D, 2, rep, T, 16, n_tree=[min(T, 30), 1, T, 0, 3], seed=3, dtype=dtype).check(gpu, gate=gate)


@pytest.mark.parametrize("variant", [0, 1])
def test_attention_rounding_variants(gpu, variant):
    say(f"tree attention variant {variant}")
    for T in (3, 30):
        TreeCase([200, 50], 256, 2, 8, T, 16, seed=4).check(gpu, variant=variant)


@pytest.mark.parametrize("lens,D,kvh,rep,T", [
    ([6001], 256, 2, 8, 20), ([3000, 40, 5000, 3], 256, 2, 4, 24), ([9000, 1], 128, 1, 8, 16), ([1500] * 7, 256, 2, 12, 8),
    ([20000], 64, 1, 4, 12), ([2500, 2500], 256, 1, 16, 64)])
def test_attention_long_and_split(gpu, lens, D, kvh, rep, T):
    say(f"tree attention lens={lens[:4]} D={D} T={T}")
    nt = [min(T, n) for n in lens]
    TreeCase(lens, D, kvh, rep, T, 64, n_tree=nt, seed=5).check(gpu)


def test_attention_many_requests(gpu):
    """More requests than a wave has lanes, trees of every size."""
    for T, rep in ((6, 2), (20, 4)):
        say(f"tree attention: 300 short requests, T={T}")
        rng = np.random.default_rng(6)
        lens = [int(x) for x in rng.integers(0, 90, 300)]
        TreeCase(lens, 128, 1, rep, T, 16, n_tree=[int(rng.integers(0, min(T, n) + 1)) for n in lens], seed=6).check(gpu)


def test_attention_a_chain_is_the_causal_order(gpu):
    """Trees that are chains: the results of the attention without a tree, to rounding."""
    for T in (1, 2, 4):
        say(f"tree attention: chain of {T}")
        c = TreeCase([300, 77, 5], 256, 2, 8, T, 16, seed=12, kind="chain")
        a, b = c.on_gpu(gpu), Case.on_gpu(c, gpu)
        ref, tol = c.reference()
        assert (np.abs(a.cpu().numpy() - ref) <= tol).all() and (np.abs((a - b).cpu().numpy()) <= 2 * tol).all()


def test_attention_any_masks(gpu):
    """Nodes that do not see themselves, see later ones, or nothing: with no context a row of zeros."""
    for T, rep in ((12, 3), (12, 8), (64, 4)):
        say(f"tree attention: masks of any bits, T={T}")
        rng = np.random.default_rng(T)
        lens = [T, T + 40, T + 3, T]
        m = rng.integers(0, 1 << 63, (4, T), np.int64).astype(np.uint64) << np.uint64(1)
        m[0, 0], m[0, T - 1], m[3, :] = 0, 0, 0
        c = TreeCase(lens, 256, 2, rep, T, 16, n_tree=[T, T, T, T], seed=13, m=m)
        o = c.check(gpu)
        assert (o[3] == 0).all() and (o[0, 0] == 0).all() and (o[0, T - 1] == 0).all()


def test_attention_large_scores_and_small_values(gpu):
    for T in (4, 24):
        for q_scale, scale in ((30.0, None), (1e-3, None), (1.0, -0.1), (1.0, 0.0)):
            say(f"tree attention T={T}: q x {q_scale}, scale {scale}")
            TreeCase([300, 77], 256, 2, 8, T, 16, seed=7, q_scale=q_scale).check(gpu, scale=scale)
        for gain in (1e-4, 3e-2, 300.0, 20000.0):
            say(f"tree attention T={T}: V scales x {gain}")
            c = TreeCase([300, 77, 30], 256, 2, 8, T, 16, seed=8)
            used = np.concatenate(c.rows)
            b = c.vc[used].reshape(len(used), -1, 34)
            d = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float32)
            d[::3] *= gain                                              # every third key
            b[..., :2] = d.astype(np.float16).view(np.uint8)
            c.vc[used] = b.reshape(len(used), -1)
            c.check(gpu)


@pytest.mark.parametrize("T", [5, 40])
@pytest.mark.parametrize("kd,vd", [(0x7E, 0x7E), (0x7C, 0x7C), (0x7C, 0x7E), (0x7B, 0x7B)])
def test_attention_unseen_nodes_stay_out(gpu, T, kd, vd):
    """A node whose scales are infinite, NaN or huge: only nodes that see it feel it. Also a block of V alone."""
    say(f"tree attention: scales {kd:x} / {vd:x} in one node, T={T}")
    c = TreeCase([100, 60], 256, 2, 8, T, 16, seed=9)
    ref, tol = c.reference()
    node = 2
    for b, n in enumerate(c.lens):
        r = c.rows[b][n - T + node]
        c.kc[r, 0::34], c.kc[r, 1::34] = 0xFF if kd == 0x7B else 0, kd
        c.vc[r, 0::34], c.vc[r, 1::34] = 0xFF if vd == 0x7B else 0, vd
    o = c.on_gpu(gpu).cpu().numpy()
    sees = (c.m >> np.uint64(node) & np.uint64(1)).astype(bool)
    for b in range(2):
        for t in range(T):
            if not sees[b, t]:
                assert (np.abs(o[b, t] - ref[b, t]) <= tol[b, t]).all(), (b, t)
            elif kd == 0x7E:
                assert np.isnan(o[b, t]).all()
    # one block of V: the other blocks of the nodes that see it are as they were
    c = TreeCase([100, 60], 256, 2, 8, T, 16, seed=9)
    for b, n in enumerate(c.lens):
        r = c.rows[b][n - T + node]
        c.vc[r, 34 * 3], c.vc[r, 34 * 3 + 1] = 0, 0x7E
    o = c.on_gpu(gpu).cpu().numpy()
    for b in range(2):
        for t in range(T):
            d = np.abs(o[b, t] - ref[b, t]) <= tol[b, t]
            hit = np.zeros_like(d)
            if sees[b, t]:
                hit[:8, 96:128] = True                                   # head 0's block 3
                assert np.isnan(o[b, t][:8, 96:128]).all()
            assert d[~hit].all()


def test_attention_bad_pages_and_lengths(gpu):
    for T in (3, 40):
        say(f"tree attention: entries outside the pool, lengths and node counts out of range, T={T}")
        c = TreeCase([100, 70, 64, 90], 256, 2, 8, T, 16, seed=10, extra_cols=0)
        table = c.table.copy()
        table[0, 2], table[1, 0], table[2, 0:4] = -1, c.n_rows // 16, 2 ** 31 - 1
        rows = [r.copy() for r in c.rows]
        rows[0][32:48], rows[1][:16], rows[2][:] = -1, -1, -1
        gpu.device_status()
        o = c.on_gpu(gpu, table=table).cpu().numpy()
        assert gpu.device_status() == gpu.DEVERR_GET_ROWS_INDEX
        ref, tol = c.reference(rows=rows)
        assert (np.abs(o - ref) <= tol).all() and (o[2] == 0).all()
        lens, cols = [100, 70, 64, 90], c.table.shape[1] * 16
        o = c.on_gpu(gpu, n_tree=[T + 1, -1, T, 1000]).cpu().numpy()
        assert gpu.device_status() == gpu.DEVERR_GET_ROWS_INDEX
        c.nt = [T, 0, T, T]
        ref, tol = c.reference()
        assert (np.abs(o - ref) <= tol).all() and (o[1] == 0).all()
        c.lens, c.nt = [-5, 0, 64, 90], [0, 0, T, T]
        c.rows = [c.rows[0][:0], c.rows[1][:0]] + c.rows[2:]
        o = c.on_gpu(gpu, n_kv=[-5, 0, 64, 90]).cpu().numpy()
        assert gpu.device_status() == gpu.DEVERR_GET_ROWS_INDEX
        c.lens = [0, 0, 64, 90]
        ref, tol = c.reference()
        assert (np.abs(o - ref) <= tol).all()
        assert cols >= max(lens)


def test_attention_strides_and_workspaces(gpu):
    """Queries with gaps, padded rows, no workspace, and the same bits whatever the workspace holds."""
    for T in (4, 40):
        say(f"tree attention: strides, T={T}")
        c = TreeCase([100, 33, 90], 256, 2, 8, T, 16, n_tree=[min(T, 30), 2, T], seed=11, pad=32)
        a = c.check(gpu)
        wide = torch.full((3, T, 20, 272), 3.0, device="cuda")
        wide[:, :, 2:18, :256] = c.q.cuda()
        b = c.on_gpu(gpu, q=wide[:, :, 2:18, :256], ws=False)
        assert np.array_equal(a, b.cpu().numpy().astype(np.float64))
        assert torch.equal(b, c.on_gpu(gpu))


def test_attention_captured(gpu):
    """Two graphs of one call with a workspace each, replayed in turn with new lengths, masks and queries, eager calls between."""
    K, T = gpu, 20
    say("tree attention: captured")
    cases = [TreeCase([400, 90, 33], 256, 2, 8, T, 16, n_tree=n, seed=s) for s, n in ((20, [20, 3, 11]), (21, [1, 20, 20]))]
    c = cases[0]
    graphs = []
    for _ in range(2):
        kd, vd, td = dev(c.kc), dev(c.vc), dev(c.table)
        nb = (34, kd.stride(0), 272, c.n_rows * kd.stride(0))
        kv, vv = (K.tensor(x.data_ptr(), K.TYPE_Q8_0, (256, c.n_rows, 2, 1), nb) for x in (kd, vd))
        q, o = c.q.cuda(), torch.zeros((3, T, 16, 256), device="cuda")
        nd, nt, m = i32(c.lens), i32(c.n_tree), words(c.m)
        qv, ov = K.q_view(q), K.out_view(o)
        w = ws_of(K.fattn_workspace_size_paged_tree(qv, kv, vv, td, 16))

        def call():
            K.flash_attn_ext_paged_tree(qv, kv, vv, td, 16, nd, m, c.scale, ov, n_tree=nt, ws=w)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        graphs.append((g, q, o, nd, nt, m, (kd, vd, td, w)))
    for turn in range(4):
        outs = []
        for i, (g, q, o, nd, nt, m, _) in enumerate(graphs):
            x = cases[(turn + i) % 2]
            q.copy_(x.q.cuda()); nt.copy_(i32(x.n_tree)); m.copy_(words(x.m))
            g.replay()
            outs.append((o, x))
        torch.cuda.synchronize()
        for o, x in outs:
            keep = x.kc, x.vc, x.table, x.rows, x.n_rows
            x.kc, x.vc, x.table, x.rows, x.n_rows = c.kc, c.vc, c.table, c.rows, c.n_rows
            assert torch.equal(o, x.on_gpu(K))
            x.kc, x.vc, x.table, x.rows, x.n_rows = keep


# ---------------------------------------------------------------- linear attention

class LinearCase:
    def __init__(self, B, T, kh, vh, dk, dv, n_tree=None, dtype=torch.float32, fixed=False, seed=0, m=None, kind=None):
        rng = np.random.default_rng(seed)
        self.B, self.T, self.kh, self.vh, self.dk, self.dv, self.dtype, self.n_tree = B, T, kh, vh, dk, dv, dtype, n_tree
        self.nt = [T] * B if n_tree is None else [int(x) for x in n_tree]
        draw = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32))  # noqa: E731
        self.q, self.k = (draw(B * T, kh, dk).to(dtype) for _ in range(2))
        self.v = draw(B * T, vh, dv).to(dtype)
        rate = np.exp(rng.random(vh) * 6) * 0.003
        self.g = torch.from_numpy((-rate if fixed else -rng.random((B * T, vh)) * rate).astype(np.float32))
        self.state = draw(B + 2, vh, dk, dv) * 0.5
        self.slots = rng.permutation(B + 2)[:B].astype(np.int32)
        self.m = R.masks(random_parents(rng, B, T, kind))[0] if m is None else m

    def on_gpu(self, K, slots=None, state=True, n_tree=0, g=None, q=None, k=None, v=None):
        out = torch.full((self.B * self.T + 1, self.vh, self.dv), 7.0, dtype=self.dtype, device="cuda")
        tree = self.n_tree if n_tree == 0 else n_tree
        K.linear_attn_tree((self.q if q is None else q).cuda(), (self.k if k is None else k).cuda(),
                           (self.v if v is None else v).cuda(), (self.g if g is None else g).cuda(), words(self.m),
                           self.state.cuda() if state else None, out[:-1], n_tree=None if tree is None else i32(tree),
                           slots=i32(self.slots if slots is None else slots))
        torch.cuda.synchronize()
        assert bool((out[-1] == 7).all())
        return out[:-1].float().cpu().numpy().astype(np.float64).reshape(self.B, self.T, self.vh, self.dv)

    def reference(self, slots=None, state=True, g=None):
        f = lambda x: x.float().numpy().astype(np.float64)  # noqa: E731
        q, k, v = (f(x).reshape(self.B, self.T, -1, x.shape[2]) for x in (self.q, self.k, self.v))
        g = f(self.g if g is None else g)
        g = np.broadcast_to(g, (self.B * self.T, self.vh)).reshape(self.B, self.T, self.vh)
        S = f(self.state)
        slots = self.slots if slots is None else slots
        out, tol = np.zeros((self.B, self.T, self.vh, self.dv)), np.zeros((self.B, self.T, self.vh, self.dv))
        for b in range(self.B):
            w = [int(self.m[b, t]) if t < self.nt[b] else None for t in range(self.T)]
            w = [x if x is None else x & ((1 << self.nt[b]) - 1) for x in w]
            for h in range(self.vh):
                s = S[slots[b], h] if state and 0 <= slots[b] < len(S) else np.zeros((self.dk, self.dv))
                hk = h // (self.vh // self.kh)
                out[b, :, h], tol[b, :, h] = R.linear(q[b, :, hk], k[b, :, hk], v[b, :, h], g[b, :, h], s, w, self.dk ** -0.5)
        return out, tol + HALF_STEP[self.dtype] * (np.abs(out) + tol) + (2.0 ** -25 if self.dtype == torch.float16 else 0)

    def check(self, K, **kw):
        o = self.on_gpu(K, **kw)
        kw.pop("n_tree", None)
        ref, tol = self.reference(**kw)
        worst = np.max(np.abs(o - ref) / np.maximum(tol, 1e-300))
        assert np.isfinite(o).all() and (np.abs(o - ref) <= tol).all(), f"{worst} of the tolerance"
        return o


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 33, 48, 49, 64])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (16, 16), (48, 80), (144, 208), (256, 64), (112, 512)])
def test_linear_shapes(gpu, T, dk, dv):
    say(f"linear tree T={T} dk={dk} dv={dv}")
    rng = np.random.default_rng(T + dk)
    nt = rng.integers(0, T + 1, 4)
    nt[0] = T
    LinearCase(4, T, 1, 3, dk, dv, n_tree=nt, seed=T).check(gpu)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("fixed", [False, True])
def test_linear_types(gpu, dtype, fixed):
    say(f"linear tree {dtype} fixed={fixed}")
    LinearCase(3, 20, 4, 8, 128, 128, n_tree=[20, 7, 0], dtype=dtype, fixed=fixed, seed=2).check(gpu)
    LinearCase(3, 64, 2, 2, 64, 256, dtype=dtype, fixed=fixed, seed=3, kind="chain").check(gpu)


def test_linear_formula_is_the_recurrence(gpu):
    """The formula against the state carried from each node's parent, in float64."""
    c = LinearCase(2, 24, 1, 2, 32, 16, seed=4)
    rng = np.random.default_rng(4 + 1)
    par = random_parents(rng, 2, 24)
    c.m = R.masks(par)[0]
    say("linear tree: against the recurrence")
    o = c.on_gpu(gpu)
    ref, tol = c.reference()
    f = lambda x: x.float().numpy().astype(np.float64)  # noqa: E731
    for b in range(2):
        for h in range(2):
            S = []
            for t in range(24):
                i = b * 24 + t
                before = S[par[b, t]] if par[b, t] >= 0 else f(c.state)[c.slots[b], h]
                S.append(np.exp(f(c.g)[i, h]) * before + np.outer(f(c.k)[i, 0], f(c.v)[i, h]))
                y = f(c.q)[i, 0] @ S[t] * 32 ** -0.5
                assert np.allclose(y, ref[b, t, h], rtol=1e-9, atol=1e-9) and (np.abs(o[b, t, h] - y) <= tol[b, t, h] + 1e-9).all()


def test_linear_slots_masks_and_decays(gpu):
    say("linear tree: slots, left out requests, any masks, strong decays")
    c = LinearCase(5, 18, 2, 4, 64, 48, n_tree=[18, 3, 18, 18, 9], seed=5)
    gpu.device_status()
    slots = np.array([3, -1, -2 - 4, 0, 99], np.int32)
    o = c.on_gpu(gpu, slots=slots)
    assert gpu.device_status() == gpu.DEVERR_SET_ROWS_INDEX
    ref, tol = c.reference(slots=slots)
    ok = np.abs(o - ref) <= tol
    assert ok[[0, 1, 3, 4]].all() and (o[2] == 7).all()
    c.check(gpu, state=False)
    gpu.device_status()
    o = c.on_gpu(gpu, n_tree=[19, -2, 18, 18, 9])
    assert gpu.device_status() == gpu.DEVERR_SET_ROWS_INDEX
    assert (o[1] == 0).all()
    rng = np.random.default_rng(6)
    m = rng.integers(0, 1 << 62, (5, 18), np.int64).astype(np.uint64)
    m[0, 3] = 0
    LinearCase(5, 18, 2, 4, 64, 48, seed=6, m=m).check(gpu)
    g = c.g.clone()
    g[::3] = -float("inf")
    g[1::5] = -200.0
    c.check(gpu, g=g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_unseen_nodes_stay_out(gpu, dtype):
    """Infinities and NaN in one node's q, k, v: only nodes that see it, or itself for q, feel them; nor do rows behind a tree."""
    for what in ("q", "k", "v", "behind"):
        for x in (float("inf"), float("nan")):
            say(f"linear tree: {x} in {what} {dtype}")
            c = LinearCase(2, 33, 2, 4, 64, 64, n_tree=[33, 20], dtype=dtype, seed=8)
            ref, tol = c.reference()
            parts = dict(q=c.q.clone(), k=c.k.clone(), v=c.v.clone())
            node = 4
            for name, t in parts.items():
                if what in (name, "behind"):
                    for b in range(2):
                        t[b * 33 + (node if what != "behind" else 32)] = x
            o = c.on_gpu(gpu, **parts)
            sees = (c.m >> np.uint64(node) & np.uint64(1)).astype(bool)
            for b in range(2):
                for t in range(33):
                    hit = {"q": t == node, "k": sees[b, t], "v": sees[b, t], "behind": b == 0 and t == 32}[what] and t < c.nt[b]
                    if not hit:
                        assert (np.abs(o[b, t] - ref[b, t]) <= tol[b, t]).all(), (what, b, t)
                    elif what != "behind" or dtype == torch.float32:
                        assert not np.isfinite(o[b, t]).all()


def test_linear_strides_and_many_requests(gpu):
    say("linear tree: strided q, k, v and 700 requests")
    c = LinearCase(3, 17, 2, 4, 64, 64, n_tree=[17, 5, 16], seed=9, dtype=torch.float16)
    a = c.check(gpu)
    wide = torch.full((51, 8, 80), 5.0, dtype=torch.float16)
    wide[:, :2, :64], wide[:, 2:4, :64], wide[:, 4:8, 16:80] = c.q, c.k, c.v
    d = wide.cuda()
    out = torch.zeros((51, 4, 64), dtype=torch.float16, device="cuda")
    gpu.linear_attn_tree(d[:, :2, :64], d[:, 2:4, :64], d[:, 4:8, 16:80], c.g.cuda(), words(c.m), c.state.cuda(), out,
                         n_tree=i32(c.n_tree), slots=i32(c.slots))
    assert np.array_equal(out.float().cpu().numpy().reshape(a.shape), a)
    rng = np.random.default_rng(1)
    LinearCase(700, 5, 1, 1, 16, 16, n_tree=rng.integers(0, 6, 700), seed=10).check(gpu)


# ---------------------------------------------------------------- a verify step

def test_verify_step(gpu):
    """Append a tree's rows, attend, run the recurrent layer, accept a path, hand the rest back and bring the state forward: the
    cache and the state are those of the accepted tokens fed one after another."""
    K, B, T, page, kvh, D, nh, vh, dk, dv = gpu, 3, 12, 8, 2, 64, 4, 3, 32, 32
    say("verify step over a tree, in a graph")
    rng = np.random.default_rng(21)
    pages, cols = 80, 20
    kc, vc = (torch.zeros((pages * page, kvh * D // 32 * 34), dtype=torch.uint8, device="cuda") for _ in range(2))
    table, free, n_free = blank(B, cols), i32(rng.permutation(pages)), i32([pages])
    shared = torch.zeros(pages, dtype=torch.int32, device="cuda")
    n_kv = torch.zeros(B, dtype=torch.int32, device="cuda")
    lst = K.cache_list([kc, vc])
    state = torch.zeros((B, vh, dk, dv), device="cuda")
    ws = ws_of(max(K.paged_workspace_size(B), K.paged_release_workspace_size(B, pages)))
    draw = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()  # noqa: E731
    # the prompts
    lens = [30, 1, 17]
    n = sum(lens)
    cu, slots = blank(B + 1), blank(n)
    K.paged_extend(n_kv, i32(lens), page, table, free, n_free, n_free, n_kv, cu, slots, ws=ws)
    K.set_rows_q8_0_kv(kc, draw(n, kvh * D), vc, draw(n, kvh * D), slots)
    x = dict(q=draw(B * T, nh, D), kr=draw(B * T, kvh * D), vr=draw(B * T, kvh * D), lq=draw(B * T, 1, dk), lk=draw(B * T, 1, dk),
             lv=draw(B * T, vh, dv), g=-draw(B * T, vh).abs() * 0.1, parents=i32(random_parents(rng, B, T)), leaf=i32([7, -1, 11]))
    m, pos, keep = torch.zeros((B, T), dtype=torch.int64, device="cuda"), blank(B, T), blank(B)
    cu_p, path, new = blank(B + 1), blank(B * T), i32([T] * B)
    cu_t, slots_t, out = blank(B + 1), blank(B * T), torch.zeros((B, T, nh, D), device="cuda")
    lout, lout2, state2 = (torch.zeros((B * T, vh, dv), device="cuda") for _ in range(2)), None, torch.zeros_like(state)
    lout, lout2 = lout
    kv, vv = (K.cache_attn_view(c, pages * page, kvh, D) for c in (kc, vc))
    qv, ov = K.q_view(x["q"].view(B, T, nh, D)), K.out_view(out)
    aws = ws_of(K.fattn_workspace_size_paged_tree(qv, kv, vv, table, page))
    got = {k: torch.zeros_like(x[k]) for k in ("lq", "lk", "lv", "g")}
    lws = ws_of(K.linear_attn_workspace_size(x["lq"], x["lv"], B, T))
    past = torch.zeros_like(n_kv)

    def step():
        past.copy_(n_kv)
        K.paged_extend(n_kv, new, page, table, free, n_free, n_free, n_kv, cu_t, slots_t, ws=ws)
        K.tree_masks(x["parents"], m, n_past=past, pos=pos)
        K.set_rows_q8_0_kv(kc, x["kr"], vc, x["vr"], slots_t)
        K.flash_attn_ext_paged_tree(qv, kv, vv, table, page, n_kv, m, D ** -0.5, ov, ws=aws)
        K.linear_attn_tree(x["lq"], x["lk"], x["lv"], x["g"], m, state, lout)
        K.paged_accept(lst, page, table, n_kv, m, x["leaf"], keep, cu_path=cu_p, path=path)
        K.paged_release(keep, n_kv, page, table, shared, free, n_free, n_free, n_kv, shared, ws=ws)
        for k in got:
            K.get_rows_i32(x[k].view(B * T, -1).view(torch.uint8), path, got[k].view(B * T, -1).view(torch.uint8))
        K.linear_attn(got["lq"], got["lk"], got["lv"], got["g"], cu_p, T, state, state2, lout2, ws=lws)
        state.copy_(state2)

    mine = [host(kc)[[int(host(table)[b, i // page]) * page + i % page for i in range(lens[b])]] for b in range(B)]
    S = np.zeros((B, vh, dk, dv))
    keep_state = [t.clone() for t in (kc, vc, table, free, n_free, n_kv, shared, state)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for t, k in zip((kc, vc, table, free, n_free, n_kv, shared, state), keep_state):
        t.copy_(k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for turn in range(3):
        for k in ("q", "kr", "vr", "lq", "lk", "lv"):
            x[k].copy_(draw(*x[k].shape))
        x["parents"].copy_(i32(random_parents(rng, B, T)))
        x["leaf"].copy_(i32(rng.integers(-1, T, B)))
        K.device_status()
        before = host(n_kv).copy()
        graph.replay()
        torch.cuda.synchronize()
        assert K.device_status() == 0
        wm, wpos, _ = R.masks(host(x["parents"]), None, before)
        assert np.array_equal(host(m).view(np.uint64), wm) and np.array_equal(host(pos), wpos)
        leaf, tab = host(x["leaf"]), host(table)
        # the rows as the append writes them
        kq = torch.zeros((B * T, kc.shape[1]), dtype=torch.uint8, device="cuda")
        vq = torch.zeros_like(kq)
        K.set_rows_q8_0_kv(kq, x["kr"], vq, x["vr"], i32(np.arange(B * T)))
        for b in range(B):
            nodes = R.nodes_of(wm[b, leaf[b]], T) if leaf[b] >= 0 else []
            mine[b] = np.concatenate([mine[b], host(kq)[np.array([b * T + t for t in nodes], int)]])
            assert host(n_kv)[b] == before[b] + len(nodes) == len(mine[b])
            rows = [int(tab[b, i // page]) * page + i % page for i in range(len(mine[b]))]
            assert np.array_equal(host(kc)[rows], mine[b])
            for h in range(vh):
                for t in nodes:
                    i = b * T + t
                    S[b, h] = np.exp(host(x["g"])[i, h]) * S[b, h] + np.outer(host(x["lk"])[i, 0], host(x["lv"])[i, h])
            assert np.abs(host(state)[b] - S[b]).max() <= 64 * 2.0 ** -24 * max(1, np.abs(S[b]).max()) * (turn + 1)
        # the step's outputs at the accepted leaf are what the accepted chain gives
        for b in range(B):
            if leaf[b] < 0:
                continue
            c = R.nodes_of(wm[b, leaf[b]], T)
            rows = [int(tab[b, i // page]) * page + i % page for i in range(len(mine[b]))]
            ref, tol = P.attention(host(x["q"]).reshape(B, T, nh, D)[b, leaf[b]][None], host(kc), host(vc), rows, kvh, D ** -0.5)
            assert (np.abs(host(out)[b, leaf[b]] - ref[0]) <= tol[0] + 2.0 ** -24 * np.abs(ref[0])).all()
            for h in range(vh):
                y = host(x["lq"])[b * T + c[-1], 0] @ S[b, h] * dk ** -0.5
                assert np.abs(host(lout)[b * T + leaf[b], h] - y).max() <= 1e-4 * max(1, np.abs(y).max())
