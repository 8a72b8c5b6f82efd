"""The paged cache on the GPU: page tables against a loop in Python, attention over pages against
float64, and a serving step of both with the cache append between them."""
import numpy as np
import pytest
import torch

import paged_ref as R
from gpu_util import dev, host, say

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def ws_of(n):
    return torch.empty(max(int(n), 16), dtype=torch.uint8, device="cuda")


# ---------------------------------------------------------------- tables

def run_extend(K, past, new, page, table, free, n_free, n_tok, in_place=False, pad=-1, cap=None):
    B = len(past)
    d = {k: dev(np.asarray(v, np.int32)) for k, v in dict(past=past, new=new, free=free, n_free=[n_free]).items()}
    tab = dev(np.asarray(table, np.int32))
    full = lambda n: torch.full((n,), -99, dtype=torch.int32, device="cuda")  # noqa: E731
    n_kv, nfo = (d["past"], d["n_free"]) if in_place else (full(B), full(1))
    cu, slots, pos, seq = full(B + 1), full(n_tok + 4), full(n_tok + 4), full(n_tok + 4)
    K.device_status()
    K.paged_extend(d["past"], d["new"], page, tab, d["free"] if cap is None else d["free"][:cap], d["n_free"], nfo, n_kv, cu,
                   slots[:n_tok], pos[:n_tok], seq[:n_tok], pad_slot=pad, ws=ws_of(K.paged_workspace_size(B)))
    flags = K.device_status()
    for x in (slots, pos, seq):
        assert (host(x)[n_tok:] == -99).all()
    return [host(x) for x in (tab, nfo, n_kv, cu, slots[:n_tok], pos[:n_tok], seq[:n_tok])], flags


def check_extend(K, past, new, page, max_pages, n_free, n_tok, seed=0, in_place=False, pad=-1, cap=None, table=None):
    rng = np.random.default_rng(seed)
    B = len(past)
    total = B * max_pages + max(n_free, 0) + 8
    ids = rng.permutation(total).astype(np.int32)
    if table is None:
        table = ids[:B * max_pages].reshape(B, max_pages).copy()
    free = ids[B * max_pages:]
    cap = len(free) if cap is None else cap
    got, flags = run_extend(K, past, new, page, table, free, n_free, n_tok, in_place, pad, cap)
    ref = R.extend(past, new, page, table, free, n_free, cap, n_tok, pad)
    for name, a, b in zip(("table", "n_free", "n_kv", "cu", "slots", "pos", "seq"), got, ref):
        assert np.array_equal(a, np.asarray(b).reshape(a.shape)), name
    assert flags == (K.DEVERR_PAGES if ref[-1] else 0)
    return ref


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("B,page,most_new", [(1, 16, 1), (1, 1, 40), (3, 7, 5), (64, 16, 1), (65, 8, 3), (130, 16, 100),
                                             (1025, 16, 2), (1500, 4, 20)])
def test_extend_against_loop(gpu, B, page, most_new, in_place):
    say(f"extend B={B} page={page} new<={most_new} in_place={in_place}")
    rng = np.random.default_rng(B)
    past, new = rng.integers(0, 6 * page, B), rng.integers(0, most_new + 1, B)
    max_pages = int((past + new).max() // page + 2)
    check_extend(gpu, past, new, page, max_pages, int(new.sum()) + B, int(new.sum()) + 3, in_place=in_place)


def test_extend_pool_runs_out(gpu):
    """Requests past the free pages keep their length; ones that need no page are served behind them."""
    say("extend: pool runs out")
    past, new = [16, 5, 0, 15, 16, 7, 32], [1, 3, 40, 1, 100, 2, 1]
    for n_free in (0, 1, 3, 4, 5, 11, 12, 13, 50):
        ref = check_extend(gpu, past, new, 16, 9, n_free, sum(new) + 2, seed=n_free)
        assert ref[-1] == (n_free < 12)


def test_extend_width_lists_and_bad_lengths(gpu):
    say("extend: width, short lists, negative and huge lengths")
    check_extend(gpu, [30, 31, 0, 33], [2, 2, 33, 0], 16, 2, 20, 60)                  # two do not fit two pages
    check_extend(gpu, [0, 0, 0], [10, 10, 10], 4, 8, 20, 25)                          # the third passes the lists
    check_extend(gpu, [0, 0], [0, 0], 4, 8, 20, 0)                                    # nothing new, no lists
    check_extend(gpu, [-5, 4, 2 ** 31 - 1], [3, -2, 2 ** 31 - 1], 4, 8, 20, 50)
    check_extend(gpu, [0, 3], [5, 5], 4, 8, -3, 50)                                   # a broken stack: n_free below 0
    check_extend(gpu, [0, 3], [5, 5], 4, 8, 900, 50, cap=10)                          # and above its capacity
    check_extend(gpu, [0, 3, 8], [5, 50, 1], 4, 8, 20, 80, pad=77)                    # a row kept for padding
    table = np.full((3, 8), 5, np.int32)
    table[1, 0], table[2, 1] = -4, 2 ** 30                                            # a partly filled page without a row
    check_extend(gpu, [2, 3, 5], [1, 3, 2], 4, 8, 20, 12, table=table)


def test_extend_random_draws(gpu):
    say("extend: 60 random draws")
    for seed in range(60):
        rng = np.random.default_rng(1000 + seed)
        B, page = int(rng.integers(1, 90)), int(rng.choice([1, 2, 3, 16, 33]))
        past, new = rng.integers(0, 5 * page + 1, B), rng.integers(0, int(rng.choice([1, 2, 12, 80])) + 1, B)
        need = sum(-(-(p + f) // page) - -(-p // page) for p, f in zip(past, new))
        max_pages = int((past + new).max() // page + 1)
        check_extend(gpu, past, new, page, max_pages, int(rng.integers(0, need + 3)),
                     max(0, int(new.sum()) + int(rng.integers(-3, 9))), seed=seed, in_place=bool(seed & 1))


def check_trim(K, keep, n_kv, page, max_pages, n_free, cap, seed=0, in_place=False):
    rng = np.random.default_rng(seed)
    B = len(n_kv)
    ids = rng.permutation(B * max_pages + cap + 8).astype(np.int32)
    table, free = ids[:B * max_pages].reshape(B, max_pages), ids[B * max_pages:B * max_pages + cap + 8]
    tab, fr = dev(table), dev(free)
    kv, nf = dev(np.asarray(n_kv, np.int32)), dev(np.asarray([n_free], np.int32))
    out, nfo = (kv, nf) if in_place else (torch.zeros_like(kv), torch.zeros_like(nf))
    K.device_status()
    K.paged_trim(dev(np.asarray(keep, np.int32)), kv, page, tab, fr[:cap], nf, nfo, out, ws=ws_of(K.paged_workspace_size(B)))
    flags = K.device_status()
    f, n, k, bad = R.trim(keep, n_kv, page, table, free[:cap], n_free, cap)
    got = host(fr)
    assert np.array_equal(got[:cap], f) and np.array_equal(got[cap:], free[cap:])
    assert host(nfo)[0] == n and np.array_equal(host(out), k) and np.array_equal(host(tab), table)
    assert flags == (K.DEVERR_PAGES if bad else 0)


@pytest.mark.parametrize("in_place", [False, True])
def test_trim_against_loop(gpu, in_place):
    for seed in range(40):
        rng = np.random.default_rng(seed)
        B, page, max_pages = int(rng.choice([1, 2, 63, 64, 65, 700, 1300])), int(rng.choice([1, 3, 16])), int(rng.integers(1, 90))
        n = rng.integers(0, max_pages * page + 1, B)
        keep = np.where(rng.random(B) < 0.3, 0, n - rng.integers(0, 5, B))
        back = sum(-(-int(a) // page) - -(-max(0, int(k)) // page) for a, k in zip(n, keep))
        cap = back + int(rng.integers(0, 20)) if seed % 3 else max(1, back // 2)
        say(f"trim seed {seed}: B={B} page={page} max_pages={max_pages} back={back} cap={cap}")
        check_trim(gpu, keep, n, page, max_pages, int(rng.integers(0, 3)) if cap > 3 else 0, cap, seed, in_place)


@pytest.mark.parametrize("in_place", [False, True])
def test_tables_on_both_sides_of_a_workgroup(gpu, in_place):
    """1023 to 1025 requests with many and few tokens, and every irregular length, in place and not."""
    for B in (1023, 1024, 1025):
        for most in (3, 40):
            say(f"tables: B={B} new<={most} in_place={in_place}")
            rng = np.random.default_rng(B + most)
            past, new = rng.integers(0, 60, B), rng.integers(0, most + 1, B)
            need = sum(-(-(p + f) // 16) - -(-p // 16) for p, f in zip(past, new))
            for n_free in (need, need // 2):
                check_extend(gpu, past, new, 16, 8, n_free, int(new.sum()) - 5, seed=B, in_place=in_place)
        n = rng.integers(0, 120 * 16 + 1, B)
        keep = np.where(rng.random(B) < 0.3, 0, n - rng.integers(0, 40, B))
        check_trim(gpu, keep, n, 16, 120, 3, 120 * B, B, in_place)
        check_trim(gpu, keep, n, 16, 120, 3, 9 * B, B, in_place)
    check_extend(gpu, [-5, 4, 2 ** 31 - 1], [3, -2, 2 ** 31 - 1], 4, 8, 20, 50, in_place=in_place)
    check_extend(gpu, [0, 3], [5, 5], 4, 8, -3, 50, in_place=in_place)
    check_extend(gpu, [0, 3], [5, 5], 4, 8, 900, 50, cap=10, in_place=in_place)
    check_trim(gpu, [-1, 5, 100], [10, -3, 40], 4, 8, 0, 40, in_place=in_place)
    check_trim(gpu, [0, 0], [8, 8], 4, 8, -2, 40, in_place=in_place)


def test_trim_bad_lengths(gpu):
    say("trim: lengths and stack out of range")
    check_trim(gpu, [-1, 5, 100], [10, -3, 40], 4, 8, 0, 40)
    check_trim(gpu, [0, 0], [8, 8], 4, 8, -2, 40)
    check_trim(gpu, [0, 3], [8, 8], 4, 8, 50, 40)


# ---------------------------------------------------------------- attention

def pool(rng, rows, kvh, D, pad=0, outliers=True):
    """A q8_0 cache uint8 [rows, bytes + pad] of N(0, 1) rows with a few large channels."""
    x = rng.standard_normal((rows, kvh * D)).astype(np.float32)
    if outliers:
        x[:, rng.choice(kvh * D, max(1, D // 64) * kvh, replace=False)] *= 8
    b = x.reshape(rows, -1, 32)
    amax = np.abs(b).max(-1, keepdims=True)
    q = np.rint(b * (np.float32(127) / amax)).astype(np.int8)
    out = np.zeros((rows, b.shape[1], 34), np.uint8)
    out[..., :2] = (amax[..., 0] / np.float32(127)).astype(np.float16)[..., None].view(np.uint8).reshape(rows, -1, 2)
    out[..., 2:] = q.view(np.uint8)
    out = out.reshape(rows, -1)
    return np.concatenate([out, np.full((rows, pad), 0xFF, np.uint8)], 1) if pad else out


class Case:
    """Requests over one pool: pages in random order, every unused row and table entry poisoned."""

    def __init__(self, lens, D, kvh, rep, T, page, seed=0, dtype=torch.float32, pad=0, extra_cols=1, q_scale=1.0):
        rng = np.random.default_rng(seed)
        self.lens, self.D, self.kvh, self.rep, self.T, self.page, self.dtype = lens, D, kvh, rep, T, page, dtype
        B, cols = len(lens), max(1, max(-(-max(n, 0) // page) for n in lens)) + extra_cols
        pages = sum(-(-max(n, 0) // page) for n in lens) + 3
        ids = rng.permutation(pages)
        self.n_rows = pages * page + (1 if page > 1 else 0)         # a torn page at the end
        self.kc, self.vc = (pool(rng, self.n_rows, kvh, D, pad) for _ in range(2))
        self.table = np.full((B, cols), -12345, np.int32)
        used, at = np.zeros(self.n_rows, bool), 0
        self.rows = []
        for b, n in enumerate(lens):
            m = -(-n // page)
            self.table[b, :m] = ids[at:at + m]
            at += m
            self.rows.append(np.array([self.table[b, j // page] * page + j % page for j in range(n)], np.int64))
            used[self.rows[-1]] = True
        for c in (self.kc, self.vc):
            c[~used] = 0xFF                                        # d and quants: NaN and -1
        self.q = torch.from_numpy((rng.standard_normal((B, T, kvh * rep, D)) * q_scale).astype(np.float32)).to(dtype)
        self.gate = torch.from_numpy(rng.standard_normal((B, T, kvh * rep, D)).astype(np.float32)).to(dtype)

    def on_gpu(self, K, ws=True, gate=False, variant=1, q=None, out=None, n_kv=None, table=None, stream=None, scale=None):
        B = len(self.lens)
        self.kd, self.vd = dev(self.kc), dev(self.vc)
        qd = self.q.cuda() if q is None else q
        nb = (34, self.kd.stride(0), self.D // 32 * 34, self.n_rows * self.kd.stride(0))
        kv, vv = (K.tensor(x.data_ptr(), K.TYPE_Q8_0, (self.D, self.n_rows, self.kvh, 1), nb) for x in (self.kd, self.vd))
        td = dev(self.table if table is None else table)
        nd = dev(np.asarray(self.lens if n_kv is None else n_kv, np.int32))
        buf = torch.full((B * self.T * self.kvh * self.rep * self.D + 64,), 7.0, dtype=self.dtype, device="cuda")
        o = buf[:-64].view(B, self.T, self.kvh * self.rep, self.D)
        qv, ov = K.q_view(qd), K.out_view(o)
        w = ws_of(K.fattn_workspace_size_paged(qv, kv, vv, td, self.page)) if ws else None
        gd = self.gate.cuda() if gate else None
        K.flash_attn_ext_paged(qv, kv, vv, td, self.page, nd, self.scale if scale is None else scale, ov, gate=gd,
                               variant=variant, ws=w, stream=stream)
        torch.cuda.synchronize()
        assert bool((buf[-64:] == 7.0).all())
        return o

    @property
    def scale(self):
        return self.D ** -0.5

    def reference(self, gate=False, variant=1, rows=None, scale=None):
        q = self.q.float().numpy()
        both = [R.attention(q[b], self.kc, self.vc, (rows or self.rows)[b], self.kvh, self.scale if scale is None else scale,
                            variant) for b in range(len(self.lens))]
        out, tol = np.stack([x for x, _ in both]), np.stack([y for _, y in both])
        if gate:
            s = 1 / (1 + np.exp(-self.gate.float().numpy().astype(np.float64)))
            out, tol = out * s, tol * s + 4 * 2.0 ** -22 * np.abs(out * s)
        # one rounding to the type (the smallest f16 step for values below its normal range)
        return out, tol + HALF_STEP[self.dtype] * (np.abs(out) + tol) + (2.0 ** -25 if self.dtype == torch.float16 else 0)

    def check(self, K, **kw):
        o = self.on_gpu(K, **kw).float().cpu().numpy().astype(np.float64)
        ref, tol = self.reference(kw.get("gate", False), kw.get("variant", 1), scale=kw.get("scale"))
        worst = np.max(np.abs(o - ref) / np.maximum(tol, 1e-300))
        assert np.isfinite(o).all() and (np.abs(o - ref) <= tol).all(), f"{worst} of the tolerance"
        return o


LENS = [1, 31, 32, 33, 0, 129, 127, 128, 64, 700]


@pytest.mark.parametrize("D,kvh,rep,T,page", [
    (256, 2, 8, 1, 16), (256, 2, 12, 1, 64), (256, 2, 8, 3, 16), (256, 2, 12, 4, 7), (256, 1, 1, 1, 1), (256, 3, 16, 1, 100),
    (128, 8, 4, 1, 16), (128, 2, 7, 2, 5), (128, 1, 17, 3, 33), (64, 8, 8, 1, 16), (64, 1, 64, 1, 3), (64, 5, 1, 5, 256),
    (256, 2, 8, 8, 32)])
def test_attention_shapes(gpu, D, kvh, rep, T, page):
    say(f"paged attention D={D} kvh={kvh} rep={rep} T={T} page={page}")
    Case(LENS, D, kvh, rep, T, page, seed=D + T).check(gpu)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gate", [False, True])
def test_attention_types_and_gate(gpu, dtype, gate):
    say(f"paged attention {dtype} gate={gate}")
    for D in (256, 128, 64):
        Case([40, 1, 333, 0, 97], D, 2, 6, 2, 16, seed=3, dtype=dtype).check(gpu, gate=gate)


@pytest.mark.parametrize("variant", [0, 1])
def test_attention_rounding_variants(gpu, variant):
    say(f"paged attention variant {variant}")
    Case([200, 50], 256, 2, 8, 1, 16, seed=4).check(gpu, variant=variant)


@pytest.mark.parametrize("lens,D,kvh,rep,T", [
    ([9001], 256, 2, 8, 1), ([5000, 40, 9000, 3], 256, 2, 4, 2), ([20000, 1], 128, 1, 8, 1), ([2500] * 7, 256, 2, 12, 3),
    ([33000], 64, 1, 4, 1)])
def test_attention_long_and_split(gpu, lens, D, kvh, rep, T):
    say(f"paged attention lens={lens[:4]} D={D} T={T}")
    Case(lens, D, kvh, rep, T, 64, seed=5).check(gpu)


def test_attention_many_requests(gpu):
    say("paged attention: 900 short requests")
    rng = np.random.default_rng(6)
    Case([int(x) for x in rng.integers(0, 90, 900)], 128, 1, 4, 1, 16, seed=6).check(gpu)


def test_attention_large_scores_and_small_values(gpu):
    """Sharp and flat softmax, V blocks of very different scales, a negative and a zero scale."""
    for q_scale, scale in ((30.0, None), (1e-3, None), (1.0, -0.1), (1.0, 0.0)):
        say(f"paged attention q x {q_scale}, scale {scale}")
        Case([300, 77], 256, 2, 8, 1, 16, seed=7, q_scale=q_scale).check(gpu, scale=scale)
    for gain in (1e-4, 3e-2, 300.0, 20000.0):
        say(f"paged attention: V scales x {gain}")
        c = Case([300, 77, 1], 256, 2, 8, 2, 16, seed=8)
        used = np.concatenate(c.rows)
        b = c.vc[used].reshape(len(used), -1, 34)
        d = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float32)
        d[::3] *= gain                                              # every third key
        b[..., :2] = d.astype(np.float16).view(np.uint8)
        c.vc[used] = b.reshape(len(used), -1)
        c.check(gpu)


@pytest.mark.parametrize("kd,vd", [(0x7E, 0x7E), (0x7C, 0x7C), (0x7C, 0x7E)])
def test_attention_masked_rows_stay_out(gpu, kd, vd):
    """Drafted rows whose scales are infinite (0x7C00) or NaN (0x7E00), unseen by the earlier queries."""
    say(f"paged attention: scales {kd:x} / {vd:x} behind a query")
    c = Case([100, 35, 2], 256, 2, 8, 3, 16, seed=9)
    ref, tol = c.reference()
    for b, n in enumerate(c.lens):
        r = c.rows[b][n - 1]
        c.kc[r, 0::34], c.kc[r, 1::34] = 0x00, kd
        c.vc[r, 0::34], c.vc[r, 1::34] = 0x00, vd
    o = c.on_gpu(gpu).cpu().numpy()
    assert (np.abs(o[:, :2] - ref[:, :2]) <= tol[:, :2]).all()
    if kd == 0x7E:
        assert np.isnan(o[:, 2]).all()


def test_attention_bad_pages_and_lengths(gpu):
    say("paged attention: entries outside the pool, lengths outside the table")
    c = Case([100, 70, 40, 64], 256, 2, 8, 1, 16, seed=10, extra_cols=0)
    table, cols = c.table.copy(), c.table.shape[1]
    table[0, 2], table[1, 0], table[2, 0:3] = -1, c.n_rows // 16, 2 ** 31 - 1
    rows = [r.copy() for r in c.rows]
    rows[0][32:48], rows[1][:16], rows[2][:] = -1, -1, -1
    lens = [100, 70, 40, 64]
    gpu.device_status()
    o = c.on_gpu(gpu, table=table, n_kv=lens).cpu().numpy()
    assert gpu.device_status() == gpu.DEVERR_GET_ROWS_INDEX
    ref, tol = c.reference(rows=rows)
    assert (np.abs(o - ref) <= tol).all() and (o[2] == 0).all()
    # too long and negative
    c = Case([cols * 16, 70], 256, 2, 8, 1, 16, seed=11, extra_cols=0)
    o = c.on_gpu(gpu, n_kv=[c.lens[0] + 1000, -70]).cpu().numpy()
    assert gpu.device_status() == gpu.DEVERR_GET_ROWS_INDEX
    ref, tol = c.reference()
    assert (np.abs(o[0] - ref[0]) <= tol[0]).all() and (o[1] == 0).all()
    c.on_gpu(gpu)
    assert gpu.device_status() == 0


def test_attention_strides_and_library_workspace(gpu):
    """Queries out of a wider projection, padded cache rows, table rows wider than the table; ws NULL."""
    say("paged attention: strides, library workspace")
    c = Case([100, 35, 513], 256, 2, 8, 2, 16, seed=12, pad=32)
    ref, tol = c.reference()
    wide = torch.full((3, 2, 20, 256), 9.0, device="cuda")
    wide[:, :, 2:18] = c.q.cuda()
    o = c.on_gpu(gpu, q=wide[:, :, 2:18], ws=False).cpu().numpy()
    assert (np.abs(o - ref) <= tol).all()
    swapped = c.q.cuda().permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3)
    o2 = c.on_gpu(gpu, q=swapped).cpu().numpy()
    assert np.array_equal(o, o2)


def test_attention_repeats_bit_for_bit(gpu):
    say("paged attention: same bits twice")
    c = Case([5000, 40, 900], 256, 2, 8, 1, 16, seed=13)
    assert torch.equal(c.on_gpu(gpu), c.on_gpu(gpu))


def test_attention_far_rows(gpu):
    """Pages behind 4 GiB of a pool."""
    say("paged attention: rows past 2^32 bytes")
    c = Case([200, 45], 256, 2, 8, 1, 16, seed=14)
    page, far = 16, (2 ** 32 // 544 + 4096) // 16
    rows = (far + 64) * page
    kd, vd = (torch.full((rows, 544), 0xFF, dtype=torch.uint8, device="cuda") for _ in range(2))
    table = c.table.copy()
    for b, n in enumerate(c.lens):
        for j in range(-(-n // page)):
            src = int(c.table[b, j])
            dst = far + src
            table[b, j] = dst
            for d, s in ((kd, c.kc), (vd, c.vc)):
                d[dst * page:(dst + 1) * page] = dev(s[src * page:(src + 1) * page])
    o = torch.empty((2, 1, 16, 256), device="cuda")
    qd, td, nd = c.q.cuda(), dev(table), dev(np.asarray(c.lens, np.int32))
    kv, vv = gpu.cache_attn_view(kd, rows, 2), gpu.cache_attn_view(vd, rows, 2)
    gpu.flash_attn_ext_paged(gpu.q_view(qd), kv, vv, td, page, nd, c.scale, gpu.out_view(o))
    ref, tol = c.reference()
    assert (np.abs(host(o) - ref) <= tol).all()


def test_attention_graphs_with_moving_lengths(gpu):
    """Two captured graphs with workspaces of their own, replayed in turn while lengths and pages change."""
    say("paged attention: graphs")
    K, cases, graphs = gpu, [Case([300, 50, 0], 256, 2, 8, 1, 16, seed=s) for s in (15, 16)], []
    for c in cases:
        t = dict(q=c.q.cuda(), k=dev(c.kc), v=dev(c.vc), table=dev(c.table), n=dev(np.asarray(c.lens, np.int32)))
        t["out"] = torch.zeros((3, 1, 16, 256), device="cuda")
        kv, vv = K.cache_attn_view(t["k"], c.n_rows, 2), K.cache_attn_view(t["v"], c.n_rows, 2)
        qv, ov = K.q_view(t["q"]), K.out_view(t["out"])
        t["ws"] = ws_of(K.fattn_workspace_size_paged(qv, kv, vv, t["table"], 16))
        t["call"] = lambda t=t, qv=qv, kv=kv, vv=vv, ov=ov: K.flash_attn_ext_paged(
            qv, kv, vv, t["table"], 16, t["n"], 1 / 16, ov, ws=t["ws"])
        t["call"]()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            t["call"]()
        graphs.append((g, t))
    for lens in ([300, 50, 0], [17, 0, 0], [299, 49, 0], [0, 0, 0]):
        for (g, t), c in zip(graphs, cases):
            t["n"].copy_(dev(np.asarray(lens, np.int32)))
            t["out"].fill_(5.0)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            got = t["out"].clone()
            ref, tol = c.reference(rows=[r[:n] for r, n in zip(c.rows, lens)])
            assert (np.abs(got.cpu().numpy() - ref) <= tol).all()
            t["call"]()
            torch.cuda.synchronize()
            assert torch.equal(got, t["out"])


def test_attention_random_draws(gpu):
    """Shapes, lengths and page sizes drawn over their ranges."""
    rng = np.random.default_rng(23)
    for i in range(14):
        D, kvh, T = int(rng.choice([64, 128, 256])), int(rng.integers(1, 9)), int(rng.integers(1, 9))
        rep, page = int(rng.integers(1, 64 // T + 1)), int(np.exp(rng.uniform(0, np.log(300))))
        lens = [int(np.exp(rng.uniform(0, np.log(3000)))) - 1 for _ in range(int(np.exp(rng.uniform(0, np.log(24)))))]
        dtype = [torch.float32, torch.float16, torch.bfloat16][i % 3]
        say(f"paged attention draw {i}: D={D} kvh={kvh} rep={rep} T={T} page={page} lens={lens} {dtype}")
        Case(lens, D, kvh, rep, T, page, seed=100 + i, dtype=dtype).check(gpu, gate=bool(i & 1))


def test_attention_gate_in_place(gpu):
    say("paged attention: the gate's tensor is the output")
    K, c = gpu, Case([3000, 0, 70, 5], 128, 2, 6, 2, 16, seed=24)
    want = c.on_gpu(K, gate=True)
    o, q, td, nd = c.gate.cuda(), c.q.cuda(), dev(c.table), dev(np.asarray(c.lens, np.int32))
    kv, vv = K.cache_attn_view(c.kd, c.n_rows, 2, 128), K.cache_attn_view(c.vd, c.n_rows, 2, 128)
    K.flash_attn_ext_paged(K.q_view(q), kv, vv, td, 16, nd, c.scale, K.out_view(o), gate=o)
    torch.cuda.synchronize()
    assert torch.equal(o, want)


def test_calls_on_two_streams_at_once(gpu):
    """Calls under way on two streams, each with its workspaces, beside work on the default one: the bits of calls alone."""
    say("paged attention: two streams")
    K, cases = gpu, [Case([4000, 90, 700], 256, 2, 8, 1, 16, seed=s) for s in (25, 26)]
    want = [c.on_gpu(K) for c in cases]
    streams, runs = [torch.cuda.Stream() for _ in cases], []
    for c in cases:
        q, td, nd = c.q.cuda(), dev(c.table), dev(np.asarray(c.lens, np.int32))
        kv, vv = K.cache_attn_view(c.kd, c.n_rows, 2), K.cache_attn_view(c.vd, c.n_rows, 2)
        o = torch.full_like(q, 3.0)
        runs.append((q, td, nd, kv, vv, o, ws_of(K.fattn_workspace_size_paged(K.q_view(q), kv, vv, td, 16))))
    torch.cuda.synchronize()
    for _ in range(5):
        for st, c, (q, td, nd, kv, vv, o, ws) in zip(streams, cases, runs):
            with torch.cuda.stream(st):
                o.fill_(3.0)
                K.flash_attn_ext_paged(K.q_view(q), kv, vv, td, 16, nd, c.scale, K.out_view(o), ws=ws)
    torch.cuda.synchronize()
    for (*_, o, _), w in zip(runs, want):
        assert torch.equal(o, w)


def test_tables_captured_in_place(gpu):
    """A step's extend and trim in one graph, lengths and stack in place: every replay as the eager calls."""
    say("page tables: captured in place")
    K, B, page = gpu, 70, 16
    i32 = lambda x: dev(np.asarray(x, np.int32))  # noqa: E731
    rng = np.random.default_rng(27)
    start = dict(n_kv=i32(rng.integers(0, 40, B) // page * 0), table=i32(np.full((B, 9), -1)), free=i32(rng.permutation(500)),
                 n_free=i32([500]))
    new, keep = i32([0] * B), i32([0] * B)
    sets = []
    for _ in range(2):
        t = {k: x.clone() for k, x in start.items()}
        t.update(cu=i32([0] * (B + 1)), slots=i32([0] * 900), seq=i32([0] * 900), ws=ws_of(K.paged_workspace_size(B)))
        sets.append(t)

    def step(t):
        K.paged_extend(t["n_kv"], new, page, t["table"], t["free"], t["n_free"], t["n_free"], t["n_kv"], t["cu"], t["slots"],
                       seq=t["seq"], ws=t["ws"])
        K.paged_trim(keep, t["n_kv"], page, t["table"], t["free"], t["n_free"], t["n_free"], t["n_kv"], ws=t["ws"])

    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(sets[0])
    for i in range(6):
        new.copy_(i32(rng.integers(0, 12, B)))
        keep.copy_(i32(rng.integers(0, 60, B) if i % 2 else [1 << 20] * B))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        step(sets[1])
        torch.cuda.synchronize()
        for name in ("n_kv", "table", "n_free", "cu", "slots", "seq", "free"):
            assert torch.equal(sets[0][name], sets[1][name]), (i, name)


def test_wrappers_refuse_tensors_elsewhere(gpu):
    """Host tensors and other types where the calls read device int32, before anything is launched."""
    K, c = gpu, Case([30], 256, 2, 8, 1, 16, seed=28)
    c.on_gpu(K)
    q, td, nd = c.q.cuda(), dev(c.table), dev(np.asarray(c.lens, np.int32))
    kv = K.cache_attn_view(c.kd, c.n_rows, 2)
    call = lambda table=td, n=nd, ws=None: K.flash_attn_ext_paged(  # noqa: E731
        K.q_view(q), kv, kv, table, 16, n, 1 / 16, K.out_view(torch.empty_like(q)), ws=ws)
    for kw in (dict(table=td.cpu()), dict(table=td.long()), dict(n=nd.cpu()), dict(n=nd[:0]), dict(table=td[0]),
               dict(ws=torch.empty(1 << 20, dtype=torch.uint8))):
        with pytest.raises(ValueError):
            call(**kw)
    # the transposed table is one of one page a request: a call like another, its request clipped to that page
    K.device_status()
    call(table=td.t())
    assert K.device_status() == K.DEVERR_GET_ROWS_INDEX
    v = torch.zeros((4, 2, 64), device="cuda")
    s, cu = torch.zeros((1, 2, 64, 64), device="cuda"), dev(np.array([0, 4], np.int32))
    for kw in (dict(q=v.cpu()), dict(g=torch.zeros(2)), dict(cu=cu.long()), dict(s=s.cpu()), dict(g=torch.zeros(3, device="cuda"))):
        a = dict(q=v, g=torch.zeros(2, device="cuda"), cu=cu, s=s)
        a.update(kw)
        with pytest.raises(ValueError):
            K.linear_attn(a["q"], v, v, a["g"], a["cu"], 4, a["s"], a["s"], torch.empty_like(v))


def test_null_workspace_is_refused_in_capture(gpu):
    say("paged attention: ws NULL under capture")
    c = Case([30], 256, 2, 8, 1, 16, seed=17)
    c.on_gpu(gpu)
    q, o, t, n = c.q.cuda(), torch.zeros((1, 1, 16, 256), device="cuda"), dev(c.table), dev(np.asarray(c.lens, np.int32))
    kv, vv = gpu.cache_attn_view(c.kd, c.n_rows, 2), gpu.cache_attn_view(c.vd, c.n_rows, 2)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o.zero_()
        with pytest.raises(gpu.QwfnError) as e:
            gpu.flash_attn_ext_paged(gpu.q_view(q), kv, vv, t, 16, n, 1 / 16, gpu.out_view(o))
    assert e.value.code == gpu.EINVAL


# ---------------------------------------------------------------- a serving loop

def test_serving_steps(gpu):
    """Prompts, decode steps, rejected drafts, ends and new requests: extend, append over the slots, attend, trim; every
    step's attention against float64 over the rows that a host-side list of each request's tokens names, pages never shared
    and never lost."""
    K, rng = gpu, np.random.default_rng(18)
    B, page, n_pages, kvh, rep, D, T = 6, 16, 60, 2, 8, 256, 3
    kc, vc = (torch.full((n_pages * page, 544), 0xFF, dtype=torch.uint8, device="cuda") for _ in range(2))
    table = torch.full((B, 20), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(n_pages, device="cuda").to(torch.int32)
    n_free, n_kv = (torch.tensor([n_pages], dtype=torch.int32, device="cuda"),
                    torch.zeros(B, dtype=torch.int32, device="cuda"))
    ws = ws_of(K.paged_workspace_size(B))
    lens, rows_k, rows_v = [0] * B, [np.zeros((0, 512), np.float32)] * B, [np.zeros((0, 512), np.float32)] * B
    i32 = lambda x: dev(np.asarray(x, np.int32))  # noqa: E731
    K.device_status()
    for step in range(12):
        new = [0 if step and lens[b] == 0 and rng.random() < 0.5 else int(rng.integers(1, 60)) if lens[b] == 0 else 3
               for b in range(B)]
        n = sum(new)
        say(f"serving step {step}: lens {lens} new {new}")
        cu, slots, pos = i32([0] * (B + 1)), i32([0] * (n + 2)), i32([0] * (n + 2))
        K.paged_extend(n_kv, i32(new), page, table, free, n_free, n_free, n_kv, cu, slots[:n], pos[:n], ws=ws)
        k, v = (rng.standard_normal((n, 512)).astype(np.float32) for _ in range(2))
        K.set_rows_q8_0_kv(kc, dev(k), vc, dev(v), slots[:n])
        q = torch.from_numpy(rng.standard_normal((B, T, kvh * rep, D)).astype(np.float32)).cuda()
        out = torch.full_like(q, 3.0)
        K.flash_attn_ext_paged(K.q_view(q), K.cache_attn_view(kc, kc.shape[0], kvh), K.cache_attn_view(vc, vc.shape[0], kvh),
                               table, page, n_kv, 1 / 16, K.out_view(out))
        assert K.device_status() == 0
        at = host(cu)
        for b in range(B):
            rows_k[b], rows_v[b] = (np.concatenate([x, y[at[b]:at[b + 1]]]) for x, y in ((rows_k[b], k), (rows_v[b], v)))
            assert np.array_equal(host(pos)[at[b]:at[b + 1]], np.arange(lens[b], lens[b] + new[b]))
            lens[b] += new[b]
        assert list(host(n_kv)) == lens
        # the same tokens in a contiguous cache of the host's
        o, tab = host(out), host(table)
        held = [int(x) for b in range(B) for x in tab[b, :-(-lens[b] // page)]]
        assert len(set(held)) == len(held) and sorted(held + list(host(free)[:host(n_free)[0]])) == list(range(n_pages))
        for b in range(B):
            pk, pv = (quantised(x) for x in (rows_k[b], rows_v[b]))
            ref, tol = R.attention(q[b].cpu().numpy(), pk, pv, np.arange(lens[b]), kvh, 1 / 16)
            assert (np.abs(o[b] - ref) <= tol + 2.0 ** -24 * np.abs(ref)).all(), (step, b)
        # a request's prompt for the contiguous attention: its rows gathered by their slots
        b = int(np.argmax(lens))
        where = i32([tab[b, j // page] * page + j % page for j in range(lens[b])])
        got = torch.zeros((lens[b], 544), dtype=torch.uint8, device="cuda")
        K.get_rows_i32(kc, where, got)
        assert np.array_equal(host(got), quantised(rows_k[b]))
        # drafts rejected, some requests done
        keep = [0 if rng.random() < 0.15 else max(0, x - int(rng.integers(0, 3))) for x in lens]
        K.paged_trim(i32(keep), n_kv, page, table, free, n_free, n_free, n_kv, ws=ws)
        lens = keep
        rows_k, rows_v = [x[:m] for x, m in zip(rows_k, keep)], [x[:m] for x, m in zip(rows_v, keep)]
        assert list(host(n_kv)) == lens


def quantised(x):
    """float32 [n, 512] rows as q8_0 bytes (the x86 rounding)."""
    b = x.reshape(len(x), 16, 32)
    amax = np.abs(b).max(-1, keepdims=True)
    q = np.rint(b * (np.float32(127) / amax)).astype(np.int8)
    out = np.zeros((len(x), 16, 34), np.uint8)
    out[..., :2] = (amax[..., 0] / np.float32(127)).astype(np.float16)[..., None].view(np.uint8).reshape(len(x), 16, 2)
    out[..., 2:] = q.view(np.uint8)
    return out.reshape(len(x), 544)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("with_states", [False, True])
@pytest.mark.parametrize("B,most_new", [(5, 3), (5, 90), (300, 2), (300, 40), (1024, 40), (1030, 40), (1030, 3)])
def test_extend_state_slots(gpu, B, most_new, with_states, in_place):
    """The slots of a step's recurrent states, by every way the lists are made; all else as without them."""
    say(f"extend: state slots, B={B} new<={most_new} states={with_states} in_place={in_place}")
    K, rng, page = gpu, np.random.default_rng(B + most_new), 16
    past, new = rng.integers(0, 70, B), rng.integers(0, most_new + 1, B)
    past[B // 2], new[B // 3] = -1, -1                     # (as lengths of 0)
    max_pages, n_tok = 8, int(np.maximum(new, 0).sum()) - 2
    free = rng.permutation(4 * B + 9).astype(np.int32)
    n_free = sum(-(-(max(p, 0) + max(f, 0)) // page) - -(-max(p, 0) // page) for p, f in zip(past, new)) * 2 // 3
    states = rng.permutation(B + 3)[:B].astype(np.int32)
    states[rng.random(B) < 0.1] = -1
    states[0] = -4
    i32 = lambda x: dev(np.asarray(x, np.int32))  # noqa: E731
    ids, got = rng.permutation(B * max_pages).reshape(B, max_pages), []
    for slots_too in (False, True):
        d = dict(past=i32(past), table=i32(ids), n_free=i32([n_free]), cu=i32([0] * (B + 1)), slots=i32([0] * n_tok),
                 pos=i32([0] * n_tok), seq=i32([0] * n_tok), state_slots=torch.full((B + 2,), -99, dtype=torch.int32, device="cuda"))
        d["n_kv"], d["nfo"] = (d["past"], d["n_free"]) if in_place else (i32([0] * B), i32([0]))
        kw = dict(state_slots=d["state_slots"][1:B + 1], states=i32(states) if with_states else None) if slots_too else {}
        K.paged_extend(d["past"], i32(new), page, d["table"], i32(free), d["n_free"], d["nfo"], d["n_kv"], d["cu"], d["slots"],
                       pos=d["pos"], seq=d["seq"], ws=ws_of(K.paged_workspace_size(B)), **kw)
        got.append({k: host(x) for k, x in d.items()})
    K.device_status()
    assert all(np.array_equal(got[0][k], got[1][k]) for k in got[0] if k != "state_slots")
    p, f = np.maximum(past, 0), np.maximum(new, 0)
    runs = (got[1]["n_kv"] == p + f) & (f > 0)
    assert 0 < runs.sum() < B and ((got[1]["n_kv"] == p) & (f > 0)).any()
    own = states if with_states else np.arange(B)
    want = np.where(runs | (own < 0), own, -2 - own)
    assert np.array_equal(got[1]["state_slots"], np.concatenate([[-99], want, [-99]]))
