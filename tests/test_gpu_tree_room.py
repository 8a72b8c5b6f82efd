"""A verify step over trees for which the pool has no room for every request, captured: with n_tree = n_kv - n_past a request that
is not served keeps its rows, its length and its state, whatever leaf it is given, and the others go on."""
import numpy as np
import pytest
import torch

import tree_ref as R
from gpu_util import dev, host, say
from test_gpu_tree import blank, i32, random_parents, ws_of

pytestmark = pytest.mark.gpu


def test_verify_step_without_room(gpu):
    say("verify step over trees, a pool too small for all")
    K, B, T, page, kvh, D, nh, vh, dk, dv = gpu, 4, 9, 4, 1, 64, 2, 2, 16, 16
    rng = np.random.default_rng(5)
    lens, pages, cols = [10, 3, 14, 1], 16, 12                 # 3 + 1 + 4 + 1 pages held, 7 left for needs of 2, 2, 2 and 2
    kc, vc = (dev(rng.integers(0, 100, (pages * page, 68), np.uint8)) for _ in range(2))
    table, free, n_free = blank(B, cols), i32(rng.permutation(pages)), i32([pages])
    n_kv, past, nt, shared = i32([0] * B), i32([0] * B), i32([0] * B), i32([0] * pages)
    ws = ws_of(max(K.paged_workspace_size(B), K.paged_release_workspace_size(B, pages)))
    K.paged_extend(n_kv, i32(lens), page, table, free, n_free, n_free, n_kv, blank(B + 1), blank(sum(lens)), ws=ws)
    lst = K.cache_list([kc, vc])
    draw = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()  # noqa: E731
    q, out, kr, vr = draw(B, T, nh, D), torch.full((B, T, nh, D), 9.0, device="cuda"), draw(B * T, 64), draw(B * T, 64)
    lq, lk, lv, g = draw(B * T, 1, dk), draw(B * T, 1, dk), draw(B * T, vh, dv), -draw(B * T, vh).abs()
    state, lout = draw(B, vh, dk, dv), torch.full((B * T, vh, dv), 9.0, device="cuda")
    lout2 = torch.zeros_like(lout)
    parents, leaf, new = i32(random_parents(rng, B, T)), i32([T - 1, 4, T - 1, T - 1]), i32([T] * B)
    m, keep, cu_p, path, cu, slots = torch.zeros((B, T), dtype=torch.int64, device="cuda"), blank(B), blank(B + 1), blank(B * T), blank(B + 1), blank(B * T)
    pos = blank(B, T)
    kv, vv = (K.cache_attn_view(c, pages * page, kvh, D) for c in (kc, vc))
    qv, ov = K.q_view(q), K.out_view(out)
    aws = ws_of(K.fattn_workspace_size_paged_tree(qv, kv, vv, table, page))
    lws = ws_of(K.linear_attn_workspace_size(lq, lv, B, T))
    got = {n: torch.zeros_like(t) for n, t in (("q", lq), ("k", lk), ("v", lv), ("g", g))}

    def step():
        past.copy_(n_kv)
        K.paged_extend(n_kv, new, page, table, free, n_free, n_free, n_kv, cu, slots, ws=ws)
        torch.sub(n_kv, past, out=nt)
        K.tree_masks(parents, m, n_tree=nt, n_past=past, pos=pos)
        K.set_rows_q8_0_kv(kc, kr, vc, vr, slots)
        K.flash_attn_ext_paged_tree(qv, kv, vv, table, page, n_kv, m, 0.125, ov, n_tree=nt, ws=aws)
        K.linear_attn_tree(lq, lk, lv, g, m, state, lout, n_tree=nt)
        K.paged_accept(lst, page, table, n_kv, m, leaf, keep, n_tree=nt, cu_path=cu_p, path=path)
        K.paged_release(keep, n_kv, page, table, shared, free, n_free, n_free, n_kv, shared, ws=ws)
        for n, t in (("q", lq), ("k", lk), ("v", lv), ("g", g)):
            K.get_rows_i32(t.view(B * T, -1).view(torch.uint8), path, got[n].view(B * T, -1).view(torch.uint8))
        K.linear_attn(got["q"], got["k"], got["v"], got["g"], cu_p, T, state, state, lout2, ws=lws)

    held = [t.clone() for t in (kc, vc, table, free, n_free, n_kv, state, shared)]

    def restore():
        for t, h in zip((kc, vc, table, free, n_free, n_kv, state, shared), held):
            t.copy_(h)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    restore()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for turn in range(4):
        if turn % 2 == 0:
            restore()                                          # (odd turns: the next step of the same requests)
        parents.copy_(i32(random_parents(rng, B, T)))
        n0, tab, s0 = host(n_kv).copy(), host(table).copy(), host(state).copy()
        rows = [[int(tab[b, j // page]) * page + j % page for j in range(n0[b])] for b in range(B)]
        k0, v0 = host(kc).copy(), host(vc).copy()
        need = -(-(n0 + T) // page) - -(-n0 // page)
        served = np.cumsum(need) <= host(n_free)[0]
        assert served.any() and not served.all()
        K.device_status()
        graph.replay()
        torch.cuda.synchronize()
        flags = K.device_status()
        assert flags & K.DEVERR_PAGES                          # no room, and a leaf of a tree without nodes
        wm, _, _ = R.masks(host(parents), np.where(served, T, 0), n0)
        assert np.array_equal(host(m).view(np.uint64), wm) and host(nt).tolist() == [T if s else 0 for s in served]
        assert (host(pos)[~served] == -1).all()
        for b in range(B):
            n = n0[b] + (len(R.nodes_of(wm[b, host(leaf)[b]], T)) if served[b] else 0)
            assert host(n_kv)[b] == host(keep)[b] == n
            assert np.array_equal(host(kc)[rows[b]], k0[rows[b]]) and np.array_equal(host(vc)[rows[b]], v0[rows[b]])
            assert np.array_equal(host(table)[b, :-(-n0[b] // page)], tab[b, :-(-n0[b] // page)])
            if not served[b]:
                assert np.array_equal(host(state)[b], s0[b])
                assert (host(out)[b] == 0).all() and (host(lout)[b * T:(b + 1) * T] == 0).all()
            else:
                assert not np.array_equal(host(state)[b], s0[b]) and (host(out)[b] != 0).any()
