"""Linear attention with a decay per head on the GPU against the recurrence in float64."""
import numpy as np
import pytest
import torch

from gpu_util import dev, host, say

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def reference(q, k, v, g, lens, starts, S0, scale, A0=None):
    """Outputs and final states in float64, and the same recurrence over absolute values (the scale of errors; A0: that
    of a state that an earlier call left, whose error is relative to its A and not to |S0|, which sums may have cancelled)."""
    n, n_k, dk = q.shape
    n_v, dv = v.shape[1:]
    rep = n_v // n_k
    out, mag = np.zeros((n, n_v, dv)), np.zeros((n, n_v, dv))
    S, A = S0.astype(np.float64).copy(), (np.abs(S0) if A0 is None else A0).astype(np.float64)
    for b, (t0, m) in enumerate(zip(starts, lens)):
        for t in range(t0, t0 + m):
            e = np.exp(g[t].astype(np.float64))[:, None, None]
            kt, qt = (np.repeat(x[t].astype(np.float64), rep, axis=0) for x in (k, q))
            kv = kt[:, :, None] * v[t].astype(np.float64)[:, None, :]
            with np.errstate(invalid="ignore"):
                S[b] = S[b] * e + kv
                A[b] = A[b] * e + np.abs(kv)
            out[t] = scale * np.einsum("hr,hrc->hc", qt, S[b])
            mag[t] = abs(scale) * np.einsum("hr,hrc->hc", np.abs(qt), A[b])
    return out, mag, S, A


class Case:
    def __init__(self, lens, n_k, n_v, dk, dv, dtype=torch.float32, seed=0, fixed=False, gap=0, decay=0.2, zero=False):
        rng = np.random.default_rng(seed)
        self.lens, self.dtype, self.fixed, self.zero = lens, dtype, fixed, zero
        self.starts = list(gap + np.concatenate([[0], np.cumsum(lens)[:-1]])) if lens else []
        n = gap + sum(lens) + gap
        t = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to(dtype)  # noqa: E731
        self.q, self.k, self.v = t(n, n_k, dk), t(n, n_k, dk), t(n, n_v, dv)
        self.k = (self.k.float() / dk ** 0.5).to(dtype)
        rate = np.exp(rng.uniform(np.log(1e-3), np.log(decay * 10), n_v))
        self.g = (-rate if fixed else -rng.random((n, n_v)) * rate).astype(np.float32)
        self.cu = np.array([gap] + [gap + int(x) for x in np.cumsum(lens)], np.int32)
        B = len(lens)
        self.slots = rng.permutation(B + 2)[:B].astype(np.int32)
        self.state = rng.standard_normal((B + 2, n_v, dk, dv)).astype(np.float32)
        self.scale = dk ** -0.5

    def on_gpu(self, K, in_place=False, max_len=None, slots=True, q=None, k=None, v=None, cu=None):
        qd, kd, vd = (x.cuda() if y is None else y for x, y in ((self.q, q), (self.k, k), (self.v, v)))
        buf = torch.full((self.v.numel() + 64,), 7.0, dtype=self.dtype, device="cuda")
        o = buf[:-64].view(self.v.shape)
        s_in = dev(self.state)
        s_out = s_in if in_place else torch.full_like(s_in, 5.0)
        B, most = len(self.lens), max(1, max(self.lens)) if max_len is None else max_len
        ws = torch.empty(max(16, K.linear_attn_workspace_size(qd, vd, B, most)), dtype=torch.uint8, device="cuda")
        ws.fill_(0xFF)
        K.linear_attn(qd, kd, vd, dev(self.g), dev(self.cu if cu is None else cu), most, None if self.zero else s_in, s_out, o,
                      slots=dev(self.slots) if slots else None, scale=self.scale, ws=ws)
        torch.cuda.synchronize()
        assert bool((buf[-64:] == 7.0).all())
        return o, s_out

    def reference(self, slots=True):
        at = self.slots if slots else np.arange(len(self.lens))
        S0 = self.state[at] * (0 if self.zero else 1)
        g = np.broadcast_to(self.g, (self.q.shape[0],) + self.g.shape[-1:])
        return reference(self.q.float().numpy(), self.k.float().numpy(), self.v.float().numpy(), g, self.lens, self.starts, S0,
                         self.scale), at

    def bounds(self, ref):
        """Error bounds. The state: a token's decay, product and sum round by 2^-24 each of the running magnitude A
        (decays an exponential, 2^-22), products of 16-bit values split into 24 bits: (3 len + 64) 2^-24 A. The
        output: the state's error through |q|, dk more sums; for 16-bit types the state and the weighted scores
        enter the products rounded to the type once each (half a step of |q| A each), and the output once."""
        out, mag, S, A = ref
        rel = np.zeros((len(mag), 1, 1))
        for t0, m in zip(self.starts, self.lens):
            rel[t0:t0 + m] = (3 * m + 64 + self.q.shape[2]) * 2.0 ** -24
        h = HALF_STEP[self.dtype]
        tol = rel * mag + h * np.abs(out) + (0 if self.dtype == torch.float32 else 2 * h * mag) + \
            (2.0 ** -25 if self.dtype == torch.float16 else 1e-30)
        st = np.array([(3 * m + 64) * 2.0 ** -24 for m in self.lens])[:, None, None, None] * A + 1e-30
        return tol, st

    def check(self, K, **kw):
        o, s = self.on_gpu(K, **kw)
        self.compare(o, s, kw.get("slots", True), kw.get("in_place", False))
        return o, s

    def compare(self, o, s, slots=True, in_place=False):
        ref, at = self.reference(slots)
        tol, st = self.bounds(ref)
        o, s = o.float().cpu().numpy().astype(np.float64), s.cpu().numpy()
        live = np.zeros(len(o), bool)
        for t0, m in zip(self.starts, self.lens):
            live[t0:t0 + m] = True
        err = np.abs(o - ref[0])[live]
        assert (err <= tol[live]).all(), f"out: {np.max(err / tol[live])} of the tolerance"
        assert (o[~live] == 7.0).all()
        for b, m in enumerate(self.lens):
            if m:
                e = np.abs(s[at[b]] - ref[2][b])
                assert (e <= st[b]).all(), f"state {b}: {np.max(e / st[b])} of the tolerance"
        rest = [i for i in range(len(s)) if i not in set(at[np.array(self.lens) > 0])]
        assert np.array_equal(s[rest], self.state[rest] if in_place else np.full_like(s[rest], 5.0))


SINGLE = [1, 0, 2, 1, 3, 8, 1]
LONG = [1, 0, 64, 63, 65, 130, 17, 15, 300]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens", [SINGLE, LONG])
@pytest.mark.parametrize("n_k,n_v,dk,dv", [(2, 6, 128, 128), (2, 2, 64, 64), (1, 3, 16, 16), (1, 2, 96, 80), (1, 1, 256, 48),
                                           (1, 2, 112, 208)])
def test_shapes_and_types(gpu, dtype, lens, n_k, n_v, dk, dv):
    say(f"linear attention {dtype} lens={lens} heads {n_k}/{n_v} dk={dk} dv={dv}")
    Case(lens, n_k, n_v, dk, dv, dtype, seed=dk + dv).check(gpu)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens", [SINGLE, LONG, [600]])
@pytest.mark.parametrize("n_k,n_v,dk,dv", [(1, 2, 240, 112), (1, 1, 256, 256), (1, 1, 144, 400), (2, 2, 48, 128), (1, 2, 160, 32)])
def test_wide_heads(gpu, dtype, lens, n_k, n_v, dk, dv):
    say(f"linear attention {dtype} lens={lens} heads {n_k}/{n_v} dk={dk} dv={dv}")
    Case(lens, n_k, n_v, dk, dv, dtype, seed=dk + dv).check(gpu)


def test_random_draws(gpu):
    """Shapes and lengths drawn over their ranges."""
    rng = np.random.default_rng(31)
    for i in range(18):
        n_k = int(rng.integers(1, 4))
        n_v, dk, dv = n_k * int(rng.integers(1, 4)), 16 * int(rng.integers(1, 17)), 16 * int(rng.integers(1, 17))
        lens = [int(np.exp(rng.uniform(0, np.log(700)))) - 1 for _ in range(int(rng.integers(1, 9)))]
        dtype = [torch.float32, torch.float16, torch.bfloat16][i % 3]
        say(f"linear attention draw {i}: {dtype} heads {n_k}/{n_v} dk={dk} dv={dv} lens={lens}")
        Case(lens, n_k, n_v, dk, dv, dtype, seed=200 + i, fixed=bool(i & 1), gap=i % 3).check(gpu, in_place=bool(i & 2))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens", [[1], [4], [1500], [700, 5, 900], [16], [129]])
def test_lengths(gpu, dtype, lens):
    say(f"linear attention {dtype} lens={lens}")
    Case(lens, 1, 2, 128, 128, dtype, seed=sum(lens), decay=0.05).check(gpu)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("lens", [SINGLE, LONG])
def test_variants_of_a_call(gpu, dtype, lens):
    for kw, case in ((dict(in_place=True), {}), (dict(slots=False), {}), ({}, dict(fixed=True)), ({}, dict(zero=True)),
                     ({}, dict(gap=5))):
        say(f"linear attention {dtype} {kw} {case} lens={lens}")
        Case(lens, 2, 4, 64, 64, dtype, seed=3, **case).check(gpu, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens", [SINGLE, LONG])
def test_max_len_above_the_lengths(gpu, dtype, lens):
    """A larger bound (another path for the same tokens) gives the same results to rounding."""
    say(f"linear attention {dtype}: max_len 5000 for {lens}")
    Case(lens, 1, 2, 128, 128, dtype, seed=4).check(gpu, max_len=5000)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(gpu, dtype):
    """q, k and v as slices of one projection."""
    say(f"linear attention {dtype}: strided")
    for lens in (SINGLE, LONG):
        c = Case(lens, 2, 4, 64, 128, dtype, seed=5)
        n = c.q.shape[0]
        wide = torch.full((n, 2 * 64 + 2 * 64 + 4 * 128 + 32), 3.0, dtype=dtype, device="cuda")
        q, k, v = wide[:, :128].view(n, 2, 64), wide[:, 128:256].view(n, 2, 64), wide[:, 272:272 + 512].view(n, 4, 128)
        for x, y in ((q, c.q), (k, c.k), (v, c.v)):
            x.copy_(y.cuda())
        c.check(gpu, q=q, k=k, v=v)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_decays(gpu, dtype):
    """No decay, decays that leave nothing (0 and below the smallest float), resets in the middle, growth."""
    for lens in ([6, 1], [200, 70]):
        for kind in ("none", "reset", "strong", "far", "growth"):
            say(f"linear attention {dtype}: {kind} decays, lens {lens}")
            c = Case(lens, 1, 2, 64, 64, dtype, seed=6)
            if kind == "none":
                c.g[:] = 0.0
            elif kind == "reset":
                c.g[[0, 3, 5]], c.g[len(c.g) // 2] = -np.inf, -np.inf
            elif kind == "strong":
                c.g[:, 0] = -5.0
                c.g[:, 1] = -60.0
            elif kind == "far":
                c.g[:] = -1e30
            else:
                c.g[:] = 0.02
            c.check(gpu)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_non_finite_tokens_stay_behind(gpu, dtype):
    """A NaN or an infinity at token t: earlier tokens, other columns, heads and sequences are not touched."""
    for lens, at in (([7, 5], 4), ([150, 90], 77), ([150, 90], 0), ([700, 3], 650)):
        for what in ("v", "k", "q", "g"):
            say(f"linear attention {dtype}: non-finite {what} at {at} of {lens}")
            c = Case(lens, 1, 2, 64, 64, dtype, seed=7)
            ref, _ = c.reference()
            tol, _ = c.bounds(ref)
            if what == "v":
                c.v[at, 1, 5] = float("inf")
            elif what == "k":
                c.k[at, 0, 3] = float("nan")
            elif what == "q":
                c.q[at, 0, 3] = float("nan")
            else:
                c.g[at, 1] = float("nan")
            o, s = c.on_gpu(gpu)
            o, s = o.float().cpu().numpy(), s.cpu().numpy()
            hit = np.zeros(o.shape, bool)
            if what == "v":
                hit[at:lens[0], 1, 5] = True
            elif what == "k":
                hit[at:lens[0]] = True
            elif what == "q":
                hit[at] = True
            else:
                hit[at:lens[0], 1] = True
            assert not np.isfinite(o[hit]).any(), "a hit token is not finite"
            assert (np.abs(o - ref[0]) <= tol)[~hit].all()
            s0 = s[c.slots[0]]
            gone = dict(v=~np.isfinite(s0[1, :, 5]).all(), k=np.isnan(s0[:, 3]).all(), q=np.isfinite(s0).all(),
                        g=np.isnan(s0[1]).all())
            gone["v"] = not np.isfinite(s0[1, :, 5]).any()
            assert gone[what] and np.isfinite(s[c.slots[1]]).all()


def test_bad_sequences_and_slots(gpu):
    """Offsets that descend, leave the tokens or pass max_len; slots outside the states."""
    for lens in ([3, 2, 4], [100, 20, 90]):
        say(f"linear attention: bad offsets and slots, lens {lens}")
        c = Case(lens, 1, 2, 64, 64, seed=8)
        n, m = sum(lens), lens[0]
        gpu.device_status()
        ref, _ = c.reference()
        tol, _ = c.bounds(ref)
        # the second pair descends; the third starts earlier and stays inside
        cu = np.array([0, m, m - 1, m - 1 + lens[2]], np.int32)
        o, s = c.on_gpu(gpu, cu=cu)
        assert gpu.device_status() == gpu.DEVERR_SET_ROWS_INDEX
        assert np.array_equal(host(s)[c.slots[1]], np.full_like(host(s)[0], 5.0))
        assert (np.abs(host(o)[:m - 1] - ref[0][:m - 1]) <= tol[:m - 1]).all()
        o, s = c.on_gpu(gpu, cu=np.array([-4, m, m + lens[1], 2 ** 31 - 1], np.int32))
        assert gpu.device_status() == gpu.DEVERR_SET_ROWS_INDEX
        assert (np.abs(host(o) - ref[0]) <= tol).all()
        c.on_gpu(gpu, max_len=max(lens) - 1)
        assert gpu.device_status() == gpu.DEVERR_SET_ROWS_INDEX
        # -1: a state of zeros that is not kept; one outside: the same, reported
        keep = c.slots.copy()
        for bad, flag in ((-1, 0), (5, gpu.DEVERR_SET_ROWS_INDEX), (-7, gpu.DEVERR_SET_ROWS_INDEX)):
            c.slots = keep.copy()
            c.slots[0] = bad
            o, s = c.on_gpu(gpu)
            assert gpu.device_status() == flag
            assert np.array_equal(host(s)[keep[0]], np.full_like(host(s)[0], 5.0))
            z = Case(lens, 1, 2, 64, 64, seed=8)
            z.state[keep[0]] = 0
            zr, _ = z.reference()
            assert (np.abs(host(o) - zr[0]) <= z.bounds(zr)[0]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_many_sequences_in_parts(gpu, dtype):
    """More sequences than a workgroup has threads, most of them short or empty, a few in parts."""
    rng = np.random.default_rng(32)
    lens = [int(x) for x in rng.integers(0, 9, 600)]
    for b in (0, 255, 256, 511, 599):
        lens[b] = int(rng.integers(300, 700))
    say(f"linear attention {dtype}: 600 sequences, {sum(lens)} tokens")
    c = Case(lens, 1, 2, 64, 64, dtype, seed=32)
    assert gpu.linear_attn_workspace_size(c.q, c.v, 600, max(lens)) > 0
    c.check(gpu, in_place=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_in_place_is_the_same_bits(gpu, dtype):
    """More parts than run at once, states updated in place: no part reads what the sequence's last one wrote."""
    K = gpu
    say(f"linear attention {dtype}: in place")
    c = Case([300] * 40, 4, 16, 64, 64, dtype, seed=22)
    a, b = c.on_gpu(K), c.on_gpu(K, in_place=True)
    assert torch.equal(a[0], b[0])
    assert torch.equal(a[1][c.slots.tolist()], b[1][c.slots.tolist()])


def test_descending_offsets_stay_in_the_workspace(gpu):
    """Sequences that share their tokens have more parts together than the workspace has room for."""
    K, n, d, n_v = gpu, 1000, 64, 2
    c = Case([n], 1, n_v, d, d, seed=21)
    cu = dev(np.array([0, n, 0, n, 0, n], np.int32))
    q, k, v, g = c.q.cuda(), c.k.cuda(), c.v.cuda(), dev(c.g)
    s_in = dev(np.repeat(c.state[c.slots], 5, axis=0))
    s_out, o = torch.full_like(s_in, 5.0), torch.full_like(v, 7.0)
    need = K.linear_attn_workspace_size(q, v, 5, n)
    assert need > 0
    ws = torch.full((need + (1 << 20),), 0xA5, dtype=torch.uint8, device="cuda")
    say("linear attention: sequences that share tokens")
    K.device_status()
    K.linear_attn(q, k, v, g, cu, n, s_in, s_out, o, scale=c.scale, ws=ws[:need])
    torch.cuda.synchronize()
    assert K.device_status() == K.DEVERR_SET_ROWS_INDEX
    assert bool((ws[need:] == 0xA5).all())
    ref, _ = c.reference()
    tol, st = c.bounds(ref)
    assert (np.abs(host(s_out)[0] - ref[2][0]) <= st[0]).all()
    assert (host(s_out)[[1, 3]] == 5.0).all()
    assert (np.abs(host(o) - ref[0]) <= tol).all()         # every sequence has the same tokens and the same state


def test_repeats_and_graphs(gpu):
    """The same bits twice; two captured graphs with workspaces of their own, replayed with other lengths."""
    K = gpu
    for lens in ([1, 2, 1], [500, 90, 3]):
        say(f"linear attention: graphs, lens {lens}")
        c = Case(lens, 2, 4, 128, 128, torch.bfloat16, seed=9)
        a, b = c.on_gpu(K), c.on_gpu(K)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        sets = []
        for _ in range(2):
            t = dict(q=c.q.cuda(), k=c.k.cuda(), v=c.v.cuda(), g=dev(c.g), cu=dev(c.cu), s=dev(c.state), slots=dev(c.slots))
            t["o"], t["so"] = torch.zeros_like(t["v"]), torch.zeros_like(t["s"])
            t["ws"] = torch.empty(max(16, K.linear_attn_workspace_size(t["q"], t["v"], 3, max(lens))), dtype=torch.uint8,
                                  device="cuda")
            call = lambda t=t: K.linear_attn(t["q"], t["k"], t["v"], t["g"], t["cu"], max(lens), t["s"], t["so"], t["o"],  # noqa: E731
                                             slots=t["slots"], scale=c.scale, ws=t["ws"])
            call()
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                call()
            sets.append((g, t, call))
        for cu in (c.cu, np.array([0, 0, 1, 1], np.int32), np.array([0, lens[0], lens[0], lens[0] + 1], np.int32)):
            for g, t, call in sets:
                t["cu"].copy_(dev(cu))
                t["o"].fill_(7.0), t["so"].fill_(5.0)
                torch.cuda.synchronize()
                g.replay()
                torch.cuda.synchronize()
                o, so = t["o"].clone(), t["so"].clone()
                z = Case(lens, 2, 4, 128, 128, torch.bfloat16, seed=9)
                z.cu, z.lens, z.starts = cu, list(np.diff(cu)), list(cu[:-1])
                z.compare(o, so)
                t["o"].fill_(7.0), t["so"].fill_(5.0)
                call()
                torch.cuda.synchronize()
                assert torch.equal(o, t["o"]) and torch.equal(so, t["so"])


def test_hybrid_step(gpu):
    """A prompt step and two decode steps of a recurrent layer over the ragged batch that paged_extend lists."""
    K, rng = gpu, np.random.default_rng(10)
    B, n_k, n_v, d = 3, 1, 2, 64
    i32 = lambda x: dev(np.asarray(x, np.int32))  # noqa: E731
    n_kv, table, free, n_free = i32([0] * B), i32(np.full((B, 40), -1)), i32(np.arange(64)), i32([64])
    ws = torch.empty(K.paged_workspace_size(B), dtype=torch.uint8, device="cuda")
    state = [torch.zeros((B, n_v, d, d), device="cuda") for _ in range(2)]
    ref = mag = np.zeros((B, n_v, d, d))
    for step, new in enumerate(([90, 7, 33], [1, 1, 1], [1, 0, 3])):
        say(f"hybrid step {step}: {new}")
        n = sum(new)
        cu, slots = i32([0] * (B + 1)), i32([0] * n)
        K.paged_extend(n_kv, i32(new), 4, table, free, n_free, n_free, n_kv, cu, slots, ws=ws)
        c = Case(new, n_k, n_v, d, d, seed=step)
        out = torch.empty_like(c.v, device="cuda")
        lw = torch.empty(max(16, K.linear_attn_workspace_size(c.q.cuda(), c.v.cuda(), B, max(new))), dtype=torch.uint8, device="cuda")
        state[1].copy_(state[0])
        K.linear_attn(c.q.cuda(), c.k.cuda(), c.v.cuda(), dev(c.g), cu, max(new), state[0], state[1], out, scale=c.scale, ws=lw)
        state.reverse()
        r = reference(c.q.numpy(), c.k.numpy(), c.v.numpy(), c.g, new, list(np.cumsum([0] + new[:-1])), ref, c.scale, mag)
        assert (np.abs(host(out) - r[0]) <= (3 * 100 + 200) * 2.0 ** -24 * r[1] + 1e-30).all()
        ref, mag = r[2], r[3]
        assert (np.abs(host(state[0]) - ref) <= 2 * (3 * 100 + 200) * 2.0 ** -24 * r[3] + 1e-30).all()
    assert K.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens", [LONG, [600, 40], [1500]])
@pytest.mark.parametrize("n_k,n_v,dk,dv", [(1, 3, 128, 128), (2, 2, 64, 64), (1, 2, 256, 48), (1, 1, 256, 256)])
def test_outputs_in_chunks_are_rounded_once(gpu, dtype, lens, n_k, n_v, dk, dv):
    """A 16-bit output differs from the recurrence by its own rounding, an f32 one by the roundings of f32 sums.

    By element: a value x in two bf16 terms is off by 2^-16 |x|, and a product of two such values without its last pair of
    terms by another 2^-16. bf16: the state and the scores are in two terms, all else is exact: 2^-16 of mag. f16: q, k and v
    are exact in two; the state's product 2, the scores' and the weighted scores' together 3: 3 2^-16 of mag.
    In the 2-norm: an error before the rounding of e adds to it as sqrt(r^2 + e^2); e is below 3 2^-16, r of f16 (uniform in a
    step of 2^-10 to 2^-11 of the value) at least 2^-11 / sqrt(12) = 1.4e-4: at most 5 % more. With a term less e is 2^-9.
    f32: 3 roundings a chunk, dk / 16 sums and the split's 6, each 2^-24 / sqrt(3) in the mean: sqrt(3 47 + 16 + 6) / sqrt(3) = 7.4
    steps of 2^-24 at 1500 tokens; 16 allowed. With a term less it is 2^-17."""
    say(f"linear attention in chunks {dtype} lens={lens} heads {n_k}/{n_v} dk={dk} dv={dv}")
    c = Case(lens, n_k, n_v, dk, dv, dtype, seed=dk + dv + 1, decay=0.05)
    o, _ = c.on_gpu(gpu, max_len=max(lens))
    (out, mag, _, _), _ = c.reference()
    o = o.float().cpu().numpy().astype(np.float64)
    err = np.linalg.norm(o - out) / np.linalg.norm(out)
    if dtype == torch.float32:
        assert err <= 2.0 ** -20, err
        return
    once = torch.from_numpy(out).to(dtype).double().numpy()
    assert err <= 1.05 * np.linalg.norm(once - out) / np.linalg.norm(out), err
    h, e = HALF_STEP[dtype], np.zeros((len(mag), 1, 1))
    for t0, m in zip(c.starts, c.lens):
        e[t0:t0 + m] = (3 * m + 64 + dk) * 2.0 ** -24 + (1 if dtype == torch.bfloat16 else 3) * 2.0 ** -16
    tol = h * np.abs(out) + (1 + h) * e * mag + (2.0 ** -25 if dtype == torch.float16 else 1e-30)
    assert (np.abs(o - out) <= tol).all(), np.max(np.abs(o - out) / tol)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,held", [(SINGLE, (1, 3, 4)), (LONG, (0, 1, 5)), ([700, 0, 40, 500], (1, 3)), ([5], (0,)),
                                       ([900], (0,)), ([0, 0], (0, 1))])
@pytest.mark.parametrize("dk,dv", [(64, 64), (112, 208)])
def test_sequences_left_out_keep_their_states(gpu, dtype, lens, held, dk, dv):
    """Slots of -2 - s, for sequences with and without tokens: no output, the state as it was, in the other buffer too."""
    for kw, case in ((dict(), {}), (dict(in_place=True), {}), (dict(), dict(zero=True))):
        say(f"linear attention {dtype}: left out {held} of {lens} {kw} {case} dk={dk} dv={dv}")
        c = Case(lens, 2, 4, dk, dv, dtype, seed=40, **case)
        (out, mag, S, A), at = c.reference()
        tol, st = c.bounds((out, mag, S, A))
        c.slots = c.slots.copy()
        for b in held:
            c.slots[b] = -2 - c.slots[b]
        gpu.device_status()
        o, s = c.on_gpu(gpu, **kw)
        assert gpu.device_status() == 0
        o, s = o.float().cpu().numpy().astype(np.float64), s.cpu().numpy()
        for b, (t0, m) in enumerate(zip(c.starts, c.lens)):
            if b in held:
                assert (o[t0:t0 + m] == 7.0).all()
                assert np.array_equal(s[at[b]], c.state[at[b]] * np.float32(0 if c.zero else 1))
            elif m:
                assert (np.abs(o - out) <= tol)[t0:t0 + m].all()
                assert (np.abs(s[at[b]] - S[b]) <= st[b]).all()
        rest = [i for i in range(len(s)) if i not in set(at)]
        assert np.array_equal(s[rest], c.state[rest] if kw else np.full_like(s[rest], 5.0))


def test_left_out_slots_outside_the_states(gpu):
    """-2 - s of a slot that is not there: a zero state that is not kept, and reported, as another bad slot."""
    for lens in ([3, 1], [60, 40]):
        say(f"linear attention: left-out slots outside, lens {lens}")
        c = Case(lens, 1, 2, 64, 64, seed=41)
        for bad in (-2 - len(c.state), -2 ** 31):
            z = Case(lens, 1, 2, 64, 64, seed=41)
            c.slots[0], z.state[z.slots[0]] = bad, 0
            gpu.device_status()
            o, s = c.on_gpu(gpu)
            assert gpu.device_status() == gpu.DEVERR_SET_ROWS_INDEX
            ref, at = z.reference()
            assert (np.abs(host(o) - ref[0]) <= z.bounds(ref)[0]).all()
            assert np.array_equal(host(s)[at[0]], np.full_like(host(s)[0], 5.0))


@pytest.mark.parametrize("max_len", [1, 700])
def test_no_tokens_at_all(gpu, max_len):
    """An idle step of a batch: empty tensors; states that go on are carried over, the others left alone."""
    K = gpu
    say(f"linear attention: no tokens, max_len {max_len}")
    q, v = (torch.zeros((0, h, 64), device="cuda", dtype=torch.bfloat16) for h in (1, 2))
    g, cu = torch.zeros((0, 2), device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    s_in = torch.randn((5, 2, 64, 64), device="cuda")
    K.device_status()
    for slots, want in ((None, []), ([2, 0, 4], []), ([2, -2, -6], [0, 4]), ([-1, -1, -5], [3])):
        for src in (s_in, None):
            out = torch.full_like(s_in, 5.0)
            ws = torch.empty(16, dtype=torch.uint8, device="cuda")
            K.linear_attn(q, q, v, g, cu, max_len, src, out, torch.empty_like(v), ws=ws,
                          slots=None if slots is None else torch.tensor(slots, dtype=torch.int32, device="cuda"))
            torch.cuda.synchronize()
            ref = torch.full_like(s_in, 5.0)
            ref[want] = s_in[want] if src is not None else 0.0
            assert torch.equal(out, ref)
    same = s_in.clone()
    K.linear_attn(q, q, v, g, cu, max_len, same, same, torch.empty_like(v), slots=torch.tensor([2, -2, -6], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(same, s_in) and K.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("two_buffers", [False, True])
def test_hybrid_steps_of_a_short_pool(gpu, dtype, two_buffers):
    """Steps whose pool has no room for some requests, which come again later, and of idle requests: a layer's states hold the
    tokens of the served steps once each, in place and with two buffers that change places after every step."""
    K, rng = gpu, np.random.default_rng(50)
    B, n_k, n_v, d, page, n_pages = 4, 1, 2, 64, 16, 20
    i32 = lambda x: dev(np.asarray(x, np.int32))  # noqa: E731
    n_kv, table, free, n_free = i32([0] * B), i32(np.full((B, 40), -1)), i32(rng.permutation(n_pages)), i32([n_pages])
    states, state_slots = i32([3, 0, 4, 1]), i32([0] * B)
    at = host(states)
    ws = torch.empty(K.paged_workspace_size(B), dtype=torch.uint8, device="cuda")
    first = torch.full((5, n_v, d, d), float("nan"), device="cuda")           # (slot 2 belongs to nobody)
    first[at.tolist()] = 0.0
    buf = [first, torch.full_like(first, float("nan")) if two_buffers else first]
    ref = mag = np.zeros((B, n_v, d, d))
    lens, n_seen = [0] * B, 0
    refused = []
    #        prompts; the third does not fit      again, others decode       idle ones       room is made   single tokens, one refused
    steps = [([100, 0, 250, 90], None), ([1, 40, 250, 1], None), ([1, 0, 0, 3], [0, 41, 0, 93]), ([0, 1, 130, 0], None),
             ([1, 1, 1, 1], None), ([5, 9, 200, 2], [0, 51, 0, 80]), ([2, 0, 60, 1], None)]
    for step, (new, keep) in enumerate(steps):
        n, longest = sum(new), max(new)
        cu, slots = i32([0] * (B + 1)), i32([0] * n)
        K.paged_extend(n_kv, i32(new), page, table, free, n_free, n_free, n_kv, cu, slots, ws=ws, states=states, state_slots=state_slots)
        after = list(host(n_kv))
        runs = [m if a == x + m else 0 for m, a, x in zip(new, after, lens)]
        refused.append([b for b in range(B) if new[b] != runs[b]])
        say(f"hybrid step {step} {dtype} two_buffers={two_buffers}: lens {lens} new {new} refused {refused[-1]}")
        c = Case(new, n_k, n_v, d, d, dtype, seed=60 + step)
        out = torch.full_like(c.v, 7.0, device="cuda")
        lw = torch.empty(max(16, K.linear_attn_workspace_size(c.q.cuda(), c.v.cuda(), B, longest)), dtype=torch.uint8, device="cuda")
        K.linear_attn(c.q.cuda(), c.k.cuda(), c.v.cuda(), dev(c.g), cu, longest, buf[0], buf[1], out, slots=state_slots, scale=c.scale, ws=lw)
        buf.reverse()
        starts = list(np.cumsum([0] + new[:-1]))
        o = host(out.float())
        r = reference(*(x.float().numpy() for x in (c.q, c.k, c.v)), c.g, runs, starts, ref, c.scale, mag)
        ref, mag, n_seen = r[2], r[3], n_seen + longest
        # the bounds of Case.bounds over all the tokens there were; 16-bit outputs 2 2^-16 of the state's and scores' split
        rel, h = (3 * n_seen + 64 * (step + 1) + d) * 2.0 ** -24, HALF_STEP[dtype]
        for b, (t0, m) in enumerate(zip(starts, new)):
            if runs[b]:
                tol = h * np.abs(r[0]) + (1 + h) * (rel + (0 if dtype == torch.float32 else 2 * 2.0 ** -16)) * r[1] + 1e-30
                assert (np.abs(o - r[0]) <= tol)[t0:t0 + m].all(), (step, b)
            else:
                assert (o[t0:t0 + m] == 7.0).all(), (step, b)
        s = host(buf[0])
        assert (np.abs(s[at] - ref) <= rel * mag + 1e-30).all(), step
        assert np.isnan(s[2]).all()
        lens = after
        if keep is not None:                               # requests end: their cache rows go; their states start anew
            K.paged_trim(i32(keep), n_kv, page, table, free, n_free, n_free, n_kv, ws=ws)
            lens = [min(x, m) for x, m in zip(lens, keep)]
            for b in range(B):
                if keep[b] == 0:
                    buf[0][at[b]] = 0.0
                    ref, mag = ref.copy(), mag.copy()
                    ref[b] = mag[b] = 0.0
            assert list(host(n_kv)) == lens
    assert any(refused) and not all(refused), refused
    assert K.device_status() == K.DEVERR_PAGES
