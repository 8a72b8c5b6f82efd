"""Refusals of the entry points of shared pages and drafted trees, before anything is launched; the plain forms of the tests
against each other; the assembly of their kernels."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import paged_ref as P
import qwfn_kv as K
import tree_ref as R
from test_asm_hazards import HIPCC, PKG, ROOT, _op
from test_paged_cpu import FAKE, GB, paged_views, refused

r = ctypes.byref


def fork(**kw):
    a = dict(src=FAKE, n_tok=None, n_kv=FAKE + GB, n_seq=4, page=16, table=FAKE + 2 * GB, stride=8, cols=8, shared=FAKE + 3 * GB, n_pages=40,
             free=FAKE + 4 * GB, cap=40, n_free=FAKE + 5 * GB, n_free_out=FAKE + 6 * GB, n_kv_out=FAKE + 7 * GB,
             shared_out=FAKE + 8 * GB, moves=FAKE + 9 * GB, states=None, state_moves=None, ws=FAKE + 10 * GB, ws_bytes=1 << 20)
    a.update(kw)
    return K.load().qwfn_paged_fork(*a.values(), None)


def release(**kw):
    a = dict(keep=FAKE, n_kv=FAKE + GB, n_seq=4, page=16, table=FAKE + 2 * GB, stride=8, cols=8, shared=FAKE + 3 * GB, n_pages=40,
             free=FAKE + 4 * GB, cap=40, n_free=FAKE + 5 * GB, n_free_out=FAKE + 6 * GB, n_kv_out=FAKE + 7 * GB,
             shared_out=FAKE + 8 * GB, ws=FAKE + 10 * GB, ws_bytes=1 << 20)
    a.update(kw)
    return K.load().qwfn_paged_release(*a.values(), None)


def compact(**kw):
    a = dict(n_kv=FAKE + GB, n_seq=4, page=16, table=FAKE + 2 * GB, stride=8, cols=8, shared=FAKE + 3 * GB, n_pages=40,
             free=FAKE + 4 * GB, cap=40, n_free=FAKE + 5 * GB, table_out=FAKE + 11 * GB, shared_out=FAKE + 8 * GB,
             free_out=FAKE + 12 * GB, n_free_out=FAKE + 6 * GB, page_map=FAKE + 7 * GB, moves=FAKE + 9 * GB, n_moves=FAKE + 13 * GB,
             ws=FAKE + 10 * GB, ws_bytes=1 << 20)
    a.update(kw)
    return K.load().qwfn_paged_compact(*a.values(), None)


@pytest.mark.parametrize("call", [fork, release, compact])
def test_pool_refusals(call):
    refused(call(n_free=None), K.EINVAL, "NULL")
    refused(call(shared=None), K.EINVAL, "NULL")
    refused(call(table=None), K.EINVAL, "NULL")
    for n in (0, -1, 65537):
        refused(call(n_seq=n), K.EINVAL, "n_seq")
    refused(call(page=0), K.EINVAL, "page_size")
    refused(call(page=1 << 20, cols=1 << 11, stride=1 << 11), K.EINVAL, "2^31")
    refused(call(stride=7), K.EINVAL, "overlap")
    refused(call(cap=-1), K.EINVAL, "free_cap")
    refused(call(n_pages=0), K.EINVAL, "n_pages")
    refused(call(n_pages=1 << 27), K.EINVAL, "n_pages")
    refused(call(ws=None), K.ENOMEM, "ws")
    refused(call(ws_bytes=16), K.ENOMEM, "ws")
    refused(call(ws=FAKE + 10 * GB + 4), K.EALIGN, "16-byte")
    refused(call(shared=FAKE + 3 * GB + 2), K.EALIGN, "shared")
    refused(call(shared_out=FAKE + 3 * GB + 4), K.EINVAL, "shared_out overlaps shared")
    refused(call(n_free_out=FAKE + 2 * GB + 8), K.EINVAL, "overlaps")
    refused(call(ws=FAKE + 8 * GB + 128), K.EINVAL, "ws overlaps shared_out")


def test_pool_refusals_of_each():
    refused(fork(moves=None), K.EINVAL, "NULL")
    refused(fork(moves=FAKE + 3 * GB + 16), K.EINVAL, "moves overlaps shared")
    refused(fork(state_moves=FAKE + 9 * GB + 44), K.EINVAL, "state_moves overlaps moves")
    refused(fork(states=FAKE + 9 * GB + 40), K.EINVAL, "moves overlaps states")
    refused(fork(n_kv_out=FAKE + GB + 4), K.EINVAL, "n_kv_out overlaps n_kv")
    refused(fork(n_kv_out=FAKE), K.EINVAL, "n_kv_out overlaps from")
    refused(release(cap=39), K.EINVAL, "free_cap must be at least n_pages")
    refused(compact(cap=39), K.EINVAL, "free_cap must be at least n_pages")
    refused(release(free=FAKE + 2 * GB + 64), K.EINVAL, "overlaps table")
    refused(compact(table_out=FAKE + 2 * GB + 4), K.EINVAL, "table_out overlaps table")
    refused(compact(free_out=FAKE + 4 * GB + 4), K.EINVAL, "free_out overlaps free_pages")
    refused(compact(page_map=FAKE + 9 * GB + 200), K.EINVAL, "moves overlaps page_map")
    assert K.paged_release_workspace_size(0, 5) == K.paged_release_workspace_size(5, 0) == K.paged_compact_workspace_size(0) == 0
    assert K.paged_release_workspace_size(5, 1000) > K.paged_workspace_size(5) and K.paged_compact_workspace_size(33) > 16


def caches(n=2, kv_dim=512, rows=100, typ=K.TYPE_Q8_0, nb0=34, nb1=544, step=GB, base=FAKE):
    arr = (K.Tensor * max(n, 1))()
    for i in range(n):
        arr[i] = K.tensor(base + i * step, typ, (kv_dim, rows), (nb0, nb1))
    return arr


def copy(c=None, n=2, moves=FAKE + 90 * GB, cap=5, n_moves=None, max_rows=16):
    return K.load().qwfn_paged_copy(c if c is not None else caches(), n, moves, cap, n_moves, max_rows, None)


def accept(c=None, n=2, **kw):
    a = dict(table=FAKE + 80 * GB, stride=8, cols=8, page=16, n_kv=FAKE + 81 * GB, n_tree=None, masks=FAKE + 82 * GB, leaf=FAKE + 83 * GB,
             n_seq=4, T=8, n_keep=FAKE + 84 * GB, cu=FAKE + 85 * GB, path=FAKE + 86 * GB)
    a.update(kw)
    return K.load().qwfn_paged_accept(c if c is not None else caches(), n, *a.values(), None)


@pytest.mark.parametrize("call", [copy, accept])
def test_cache_list_refusals(call):
    refused(call(None, -1), K.EINVAL, "n_caches")
    refused(call(caches(nb0=32)), K.EINVAL, "contiguous")
    refused(call(caches(nb1=510)), K.EINVAL, "overlap")
    refused(call(caches(kv_dim=500)), K.EINVAL, "[ne0, n_rows]")
    refused(call(caches(rows=0)), K.EINVAL, "[ne0, n_rows]")
    refused(call(caches(rows=1 << 31)), K.ENOTSUP, "rows")
    refused(call(caches(typ=7)), K.EINVAL, "f32, f16, bf16, i32 or q8_0")
    refused(call(caches(step=8192)), K.EINVAL, "caches overlap")
    refused(call(caches(nb1=545)), K.EALIGN, "2-byte")
    refused(call(caches(base=FAKE + 1)), K.EALIGN, "2-byte")
    c = caches()
    c[1].ne[1] = 99
    refused(call(c), K.EINVAL, "one type, shape")
    c = caches()
    c[1].data = None
    refused(call(c), K.EINVAL, "NULL")
    c = caches()
    c[1].ne[2] = 2
    refused(call(c), K.EINVAL, "[ne0, n_rows]")


def test_copy_refusals():
    refused(copy(moves=None), K.EINVAL, "moves")
    refused(copy(cap=-1), K.EINVAL, "cap")
    refused(copy(max_rows=0), K.EINVAL, "max_rows")
    refused(copy(max_rows=0x7fffffff), K.ENOTSUP, "max_rows")
    refused(copy(moves=FAKE + 90 * GB + 2), K.EALIGN, "moves")
    refused(copy(n_moves=FAKE + 2), K.EALIGN, "n_moves")
    refused(copy(moves=FAKE + GB + 64), K.EINVAL, "overlaps moves")
    refused(copy(n_moves=FAKE + 540), K.EINVAL, "overlaps n_moves")
    assert copy(n=0) == K.OK and copy(cap=0, moves=None) == K.OK


def test_accept_refusals():
    for name in ("table", "n_kv", "masks", "leaf", "n_keep"):
        refused(accept(**{name: None}), K.EINVAL, "NULL")
    refused(accept(cu=None), K.EINVAL, "path without cu_path")
    for T in (0, 65):
        refused(accept(T=T), K.ENOTSUP, "T must")
    refused(accept(n_seq=0), K.EINVAL, "n_seq")
    refused(accept(page=0), K.EINVAL, "page_size")
    refused(accept(stride=7), K.EINVAL, "overlap")
    refused(accept(masks=FAKE + 82 * GB + 4), K.EALIGN, "masks")
    refused(accept(leaf=FAKE + 83 * GB + 2), K.EALIGN, "leaf")
    refused(accept(n_keep=FAKE + 81 * GB), K.EINVAL, "n_keep overlaps n_kv")
    refused(accept(path=FAKE + 85 * GB + 16), K.EINVAL, "path overlaps cu_path")
    refused(accept(n_keep=FAKE + 100), K.EINVAL, "a cache overlaps n_keep")
    refused(accept(caches(65), 65), K.ENOTSUP, "at most 64")


def masks_call(**kw):
    a = dict(parents=FAKE, n_tree=None, n_past=None, n_seq=4, T=8, masks=FAKE + GB, pos=FAKE + 2 * GB)
    a.update(kw)
    return K.load().qwfn_tree_masks(*a.values(), None)


def test_masks_refusals():
    refused(masks_call(parents=None), K.EINVAL, "NULL")
    refused(masks_call(masks=None), K.EINVAL, "NULL")
    refused(masks_call(n_seq=0), K.EINVAL, "n_seq")
    for T in (0, 65, -3):
        refused(masks_call(T=T), K.ENOTSUP, "T must")
    refused(masks_call(masks=FAKE + GB + 4), K.EALIGN, "masks")
    refused(masks_call(pos=FAKE + 2), K.EALIGN, "pos")
    refused(masks_call(masks=FAKE + 64), K.EINVAL, "masks overlaps parents")
    refused(masks_call(pos=FAKE + GB + 128), K.EINVAL, "pos overlaps masks")


def tree(q, k, o, v=None, table=FAKE, stride=40, cols=40, page=16, n_kv=FAKE, n_tree=None, masks=FAKE + 4 * GB, scale=0.0625, gate=None,
         variant=1, ws=FAKE + 3 * GB, ws_bytes=1 << 30):
    return K.load().qwfn_flash_attn_ext_q8_0_paged_tree(r(q), r(k), r(v or k), table, stride, cols, page, n_kv, n_tree, masks, scale,
                                                        r(gate) if gate else None, r(o), variant, ws, ws_bytes, None)


def test_tree_attention_refusals():
    q, k, o = paged_views(T=64)
    assert K.load().qwfn_fattn_workspace_size_paged_tree(r(q), r(k), r(k), 40, 16) > 0
    assert K.load().qwfn_fattn_workspace_size_paged(r(q), r(k), r(k), 40, 16) == 0
    for D in (32, 96, 512):
        refused(tree(*paged_views(D=D)), K.ENOTSUP, "head size")
    refused(tree(*paged_views(T=65)), K.ENOTSUP, "64 nodes")
    refused(tree(*paged_views(T=64, nh=34)), K.ENOTSUP, "1024 query rows")
    refused(tree(q, k, o, masks=None), K.EINVAL, "masks")
    refused(tree(q, k, o, masks=FAKE + 4 * GB + 4), K.EALIGN, "masks 8")
    refused(tree(q, k, o, n_tree=FAKE + 2), K.EALIGN, "n_tree")
    refused(tree(q, k, o, masks=FAKE + 2 * GB + 64), K.EINVAL, "dst overlaps masks")
    refused(tree(q, k, o, n_tree=FAKE + 3 * GB + 64), K.EINVAL, "ws overlaps n_tree")
    refused(tree(q, k, o, n_kv=None), K.EINVAL, "NULL")
    refused(tree(q, k, o, stride=39), K.EINVAL, "overlap")
    refused(tree(q, k, o, ws_bytes=64), K.ENOMEM, "ws")
    refused(tree(q, k, o, scale=float("nan")), K.EINVAL, "finite")
    refused(tree(q, k, paged_views(T=63)[2]), K.EINVAL, "dst must be contiguous")


def linear(n_seq=3, T=5, kh=2, vh=4, dk=64, dv=32, typ=K.TYPE_F32, **kw):
    es = 4 if typ == K.TYPE_F32 else 2

    def heads(ptr, h, d):
        return K.tensor(ptr, typ, (d, h, n_seq * T), (es, d * es, h * d * es))

    a = dict(q=heads(FAKE, kh, dk), k=heads(FAKE + GB, kh, dk), v=heads(FAKE + 2 * GB, vh, dv), g=FAKE + 3 * GB, g_ts=vh, n_tree=None,
             masks=FAKE + 4 * GB, n_seq=n_seq, T=T, slots=None, n_slots=n_seq, state=FAKE + 5 * GB, scale=1.0,
             dst=heads(FAKE + 6 * GB, vh, dv))
    a.update(kw)
    a = {n: r(x) if isinstance(x, K.Tensor) else x for n, x in a.items()}
    return K.load().qwfn_linear_attn_tree(*a.values(), None)


def test_linear_tree_refusals():
    for name in ("q", "k", "v", "dst", "g", "masks"):
        refused(linear(**{name: None}), K.EINVAL, "NULL")
    refused(linear(typ=K.TYPE_I32), K.EINVAL, "f32, f16 or bf16")
    for T in (0, 65):
        refused(linear(T=T), K.ENOTSUP if T else K.ENOTSUP, "T must")
    refused(linear(n_seq=0), K.EINVAL, "n_seq")
    refused(linear(dk=24), K.ENOTSUP, "multiples of 16")
    refused(linear(dk=272), K.ENOTSUP, "dk at most 256")
    refused(linear(dv=528), K.ENOTSUP, "dv at most 512")
    refused(linear(vh=5), K.EINVAL, "multiple of n_k_heads")
    refused(linear(g_ts=3), K.EINVAL, "g_token_stride")
    refused(linear(n_slots=2), K.EINVAL, "slots")
    refused(linear(scale=float("inf")), K.EINVAL, "finite")
    refused(linear(masks=FAKE + 4 * GB + 4), K.EALIGN, "masks 8")
    refused(linear(state=FAKE + 5 * GB + 8), K.EALIGN, "state")
    refused(linear(state=FAKE + 6 * GB), K.EINVAL, "dst overlaps state")
    refused(linear(masks=FAKE + 6 * GB + 64), K.EINVAL, "dst overlaps masks")
    q = K.tensor(FAKE, K.TYPE_F32, (64, 2, 14), (4, 256, 512))
    refused(linear(q=q), K.EINVAL, "n_seq * T tokens")
    q = K.tensor(FAKE, K.TYPE_F32, (64, 2, 15), (4, 256, 1 << 24))
    refused(linear(q=q), K.ENOTSUP, "2^24")
    refused(linear(n_seq=65535, T=1, kh=1024, vh=1024, dk=16, dv=16), K.ENOTSUP, "too many")


# ---------------------------------------------------------------- the plain forms

def test_tree_attention_of_a_chain_is_causal():
    rng = np.random.default_rng(0)
    c = rng.integers(0, 256, (40, 2, 2, 34), np.uint8)
    c[..., :2] = rng.random((40, 2, 2, 1)).astype(np.float16).view(np.uint8)
    c = c.reshape(40, -1)
    q = rng.standard_normal((4, 4, 64)).astype(np.float32)
    m, pos, _ = R.masks(np.arange(-1, 3, dtype=np.int32)[None], None, [26])
    rows = rng.permutation(40)[:30]
    a, _ = R.attention(q, c, c, rows, 2, 0.125, 26, [int(x) for x in m[0]])
    b, _ = P.attention(q, c, c, rows, 2, 0.125)
    assert np.allclose(a, b) and pos[0].tolist() == [26, 27, 28, 29]


def test_linear_formula_is_the_recurrence():
    rng = np.random.default_rng(1)
    T, dk, dv = 9, 8, 5
    par = np.array([[-1, 0, 0, 1, 2, 2, -1, 6, 3]], np.int32)
    q, k, v, g = rng.standard_normal((T, dk)), rng.standard_normal((T, dk)), rng.standard_normal((T, dv)), -rng.random(T)
    S0 = rng.standard_normal((dk, dv))
    out, _ = R.linear(q, k, v, g, S0, [int(x) for x in R.masks(par)[0][0]], 0.5)
    S = []
    for t in range(T):
        S.append(np.exp(g[t]) * (S[par[0, t]] if par[0, t] >= 0 else S0) + np.outer(k[t], v[t]))
        assert np.allclose(out[t], 0.5 * q[t] @ S[t])


def test_fork_then_release_gives_every_page_back():
    rng = np.random.default_rng(2)
    table = np.full((5, 8), -1, np.int32)
    table[0, :4] = [3, 9, 1, 7]
    free = np.array([0, 2, 4, 5, 6, 8, 10, 11, -1, -1, -1, -1], np.int32)
    shared = np.zeros(12, np.int32)
    table, shared, n, kv, moves, _, bad = R.fork([-1, 0, 0, -1, 0], [0, 14, 8, 0, 3], [15, 0, 0, 0, 0], 4, table, shared, free, 8, 12)
    assert not bad and n == 6 and kv.tolist() == [15, 14, 8, 0, 3] and shared[[3, 9, 1]].tolist() == [2, 2, 1]
    assert moves.tolist() == [[0, 0, 0], [28, 44, 2], [0, 0, 0], [0, 0, 0], [12, 40, 3]]
    f, n, kv, shared, bad = R.release(rng.permutation([0] * 5), kv, 4, table, shared, free, n, 12)
    assert not bad and n == 12 and sorted(f) == list(range(12)) and not shared.any()


# ---------------------------------------------------------------- assembly

@pytest.mark.parametrize("name", ["paged_share"])
def test_no_packed_f32_and_no_scratch(name, tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    out = str(tmp_path / "x.s")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                    "-I", os.path.join(PKG, "csrc"), "-I", os.path.join(ROOT, "include"), "--cuda-device-only", "-S",
                    os.path.join(PKG, "csrc", name + ".hip"), "-o", out], check=True, capture_output=True, timeout=600)
    lines = open(out).read().split("\n")
    assert [x.strip() for x in lines if _op(x) in ("v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32")] == []
    assert {x.split()[-1] for x in lines if ".private_segment_fixed_size:" in x} == {"0"}
