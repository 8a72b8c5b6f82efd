"""Workloads of the batched-serving operators: page tables, paged attention, linear attention.

listed() names the cases, draw(rng) makes another one of the same ranges, prepare(case,
seed) builds what a serving program holds before the call on the GPU, run(state) is one
pass through an operator, work(case) its compulsory bytes and operations, exact(case,
seed) the results in float64. run computes the operators in plain torch where `own` is
false and calls the library where it is true.

Shapes: 2 KV heads of 256 under 16 query heads (the benchmark's configurations) or 24
(the reference's model), q8_0 rows with N(0, 1) values and 4 outlier channels a head;
48 / 16 value / key heads of 128 in the recurrent layers; page sizes, batches and other
head sizes as serving programs use them.
"""
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _lib():
    path = os.path.join(ROOT, "qwfn-hybrid_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import qwfn_kv
    return qwfn_kv


def listed():
    return [
        # a decode step of a large batch: one new token a request
        dict(name="extend_decode_b256", kind="extend", B=256, lo=64, hi=32768, new_lo=1, new_hi=1, page=16, short=False),
        # prompts of different lengths arriving together while the pool runs out: the last ones are refused
        dict(name="extend_prompts_b24", kind="extend", B=24, lo=0, hi=0, new_lo=300, new_hi=9000, page=64, short=True),
        # rejected drafts of a verify step handed back
        dict(name="trim_drafts_b48", kind="trim", B=48, lo=128, hi=16384, end=0.0, back=3, page=16),
        # a fifth of a large batch finished: their pages return
        dict(name="trim_finished_b512", kind="trim", B=512, lo=128, hi=16384, end=0.2, back=1, page=16),
        # one conversation, a short one: the smallest attention call
        dict(name="paged_T1_b1_613_h24", kind="paged", B=1, lo=613, hi=613, T=1, kvh=2, rep=12, D=256, page=16, type="f32",
             gate=False),
        # a decode step of a ragged batch, half-precision activations, with the layer's output gate
        dict(name="paged_T1_b48_ragged_h16", kind="paged", B=48, lo=400, hi=24000, T=1, kvh=2, rep=8, D=256, page=64,
             type="bf16", gate=True),
        # a verify step (1 + 2 drafts) of a few conversations
        dict(name="paged_T3_b8_12295_h16", kind="paged", B=8, lo=12295, hi=12295, T=3, kvh=2, rep=8, D=256, page=32,
             type="f32", gate=False),
        # two very long contexts (the largest attention call)
        dict(name="paged_T1_b2_131072_h16", kind="paged", B=2, lo=131072, hi=131072, T=1, kvh=2, rep=8, D=256, page=256,
             type="f32", gate=False),
        # a decode step of the recurrent layers: the states are the work
        dict(name="linear_T1_b64", kind="linear", B=64, lo=1, hi=1, kh=16, vh=48, dk=128, dv=128, type="bf16",
             fixed=False),
        # one prompt's chunk
        dict(name="linear_4096_b1", kind="linear", B=1, lo=4096, hi=4096, kh=16, vh=48, dk=128, dv=128, type="bf16",
             fixed=False),
        # a ragged batch of prompts and single tokens, small heads, one constant decay a head
        dict(name="linear_ragged_b16", kind="linear", B=16, lo=1, hi=2500, kh=32, vh=32, dk=64, dv=64, type="f16",
             fixed=True),
        # single precision, as the DeltaNet update next to it
        dict(name="linear_509_b2_f32", kind="linear", B=2, lo=509, hi=509, kh=16, vh=48, dk=128, dv=128, type="f32",
             fixed=False),
    ]


def _log_int(rng, lo, hi):
    if hi <= 1 or lo >= hi:
        return hi
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(hi)))))))


def _ints(lo, hi, n, what):
    """n lengths spread over [lo, hi] by their logarithm, from the case alone."""
    rng = random.Random("%s %d %d %d" % (what, lo, hi, n))
    return [_log_int(rng, lo, hi) for _ in range(n)]


def draw(rng):
    kind = rng.choice(["extend", "trim", "paged", "paged", "paged", "linear", "linear", "linear"])
    page = rng.choice([1, 8, 16, 16, 32, 64, 100, 128, 256])
    if kind == "extend":
        B = _log_int(rng, 1, 512)
        if rng.random() < 0.5:
            hi = _log_int(rng, 256, 32768)
            return dict(kind=kind, B=B, lo=1, hi=hi, new_lo=1, new_hi=rng.randint(1, 4), page=max(page, 8),
                        short=rng.random() < 0.3)
        hi = _log_int(rng, 64, max(64, min(9000, 100000 // B)))
        return dict(kind=kind, B=B, lo=0, hi=_log_int(rng, 1, 2000), new_lo=1, new_hi=hi, page=max(page, 8),
                    short=rng.random() < 0.3)
    if kind == "trim":
        return dict(kind=kind, B=_log_int(rng, 1, 512), lo=1, hi=_log_int(rng, 256, 16384), end=rng.choice([0.0, 0.1, 0.5]),
                    back=rng.randint(0, 4), page=max(page, 8))
    if kind == "paged":
        D, kvh, rep = rng.choice([(256, 2, 8), (256, 2, 12), (256, 1, 16), (256, 4, 6), (128, 8, 4), (128, 2, 7),
                                  (128, 4, 1), (64, 8, 8), (64, 1, 3)])
        T, B = rng.choice([1, 1, 1, 2, 3, 4]), _log_int(rng, 1, 64)
        most = 250000 * 512 // (kvh * D)                 # keys of all requests, as many bytes as the largest case
        hi = _log_int(rng, 100, min(131072, most // B))
        return dict(kind=kind, B=B, lo=rng.choice([1, hi // 8 + 1, hi]), hi=hi, T=T, kvh=kvh, rep=rep, D=D, page=page,
                    type=rng.choice(["f32", "f16", "bf16"]), gate=rng.random() < 0.3)
    kh, vh, dk, dv = rng.choice([(16, 48, 128, 128), (16, 16, 128, 128), (32, 32, 64, 64), (8, 32, 64, 128), (4, 8, 128, 64),
                                 (2, 4, 128, 256)])
    typ = rng.choice(["f32", "f16", "bf16", "bf16"])
    if rng.random() < 0.4:
        return dict(kind=kind, B=_log_int(rng, 1, 64), lo=1, hi=rng.choice([1, 1, 1, 2, 4]), kh=kh, vh=vh, dk=dk, dv=dv,
                    type=typ, fixed=rng.random() < 0.5)
    B = _log_int(rng, 1, 16)
    hi = _log_int(rng, 8, (512 if typ == "f32" else 4096) // B + 64)
    return dict(kind=kind, B=B, lo=rng.choice([1, hi // 4 + 1, hi]), hi=hi, kh=kh, vh=vh, dk=dk, dv=dv, type=typ,
                fixed=rng.random() < 0.5)


# ---------------------------------------------------------------- inputs

def _gen(seed, salt=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + salt)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _rand(g, *shape):
    return torch.rand(shape, generator=g, device="cuda", dtype=torch.float32)


def _perm(g, n):
    return torch.randperm(n, generator=g, device="cuda").to(torch.int32)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _pages(n, page):
    return (n + page - 1) // page


def _quant(x):
    """F32 rows [..., 32 k] as q8_0 blocks (d = amax / 127 in F16, q = x * (127 / amax) rounded half to
    even): (q int8 [..., k, 32], d F16 [..., k])."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    amax = b.abs().amax(dim=-1)
    # quotients rounded once to float32 (a float64 quotient, then float32)
    inv = torch.where(amax > 0, (127.0 / amax.double()).float(), torch.zeros_like(amax))
    return torch.round(b * inv[..., None]).to(torch.int8), (amax.double() / 127.0).float().to(torch.float16)


def _cache(g, rows, kvh, D):
    """q8_0 cache bytes of rows tokens: N(0, 1), 4 channels of each head 8 times larger."""
    out = torch.empty((rows, kvh * D // 32, 34), dtype=torch.uint8, device="cuda")
    gain = torch.ones(kvh * D, device="cuda")
    for h in range(kvh):
        gain[torch.randperm(D, generator=g, device="cuda")[:4] + h * D] = 8.0
    for r in range(0, rows, 1 << 17):
        q, d = _quant(_randn(g, min(1 << 17, rows - r), kvh * D) * gain)
        out[r:r + q.shape[0], :, :2] = d.contiguous().view(torch.uint8).reshape(*d.shape, 2)
        out[r:r + q.shape[0], :, 2:] = q.view(torch.uint8)
    return out.reshape(rows, kvh * D // 32 * 34)


def _tables(case, past, new=None):
    """Sizes that follow from a case's lengths: table columns, pages in use, pages of the pool."""
    page = case["page"]
    cols = max(_pages(p + n, page) for p, n in zip(past, new or [0] * len(past))) + 3
    used = sum(_pages(p, page) for p in past)
    need = sum(_pages(p + n, page) - _pages(p, page) for p, n in zip(past, new or [0] * len(past)))
    return cols, used, need


def _filled_table(g, past, page, cols, pages):
    """A block table whose first ceil(past / page) columns hold distinct pages in random order."""
    have = _i32([_pages(p, page) for p in past])
    perm = _perm(g, pages)
    at = torch.cumsum(have, 0) - have
    j = torch.arange(cols, device="cuda")
    held = j[None, :] < have[:, None]
    idx = torch.where(held, at[:, None] + j[None, :], torch.zeros_like(j)[None, :])
    return torch.where(held, perm[idx.long()], torch.full_like(perm[:1], -7)).contiguous(), perm[int(have.sum()):].contiguous()


def _past_new(case):
    past = _ints(case["lo"], case["hi"], case["B"], "past") if case["hi"] else [0] * case["B"]
    return past, _ints(case["new_lo"], case["new_hi"], case["B"], "new")


def _keeps(case):
    past = _ints(case["lo"], case["hi"], case["B"], "past")
    rng = random.Random("keep %d %d" % (case["B"], case["hi"]))
    return past, [0 if rng.random() < case["end"] else max(0, p - rng.randint(0, case["back"])) for p in past]


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    kind, g, B = case["kind"], _gen(seed), case["B"]
    if kind == "extend":
        past, new = _past_new(case)
        cols, used, need = _tables(case, past, new)
        free = need * 3 // 4 if case["short"] else need + 40
        table, rest = _filled_table(g, past, case["page"], cols, used + free + 8)
        return dict(past=_i32(past), new=_i32(new), table=table, free=rest, n_free=_i32([min(free, rest.numel())]),
                    n_tok=sum(new) + 5)
    if kind == "trim":
        past, keep = _keeps(case)
        cols, used, _ = _tables(case, past)
        table, rest = _filled_table(g, past, case["page"], cols, used + 100)
        free = torch.full((used + 100,), -1, dtype=torch.int32, device="cuda")
        free[:rest.numel()] = rest
        return dict(past=_i32(past), keep=_i32(keep), table=table, free=free, n_free=_i32([rest.numel()]))
    if kind == "paged":
        lens, page, D, typ = _ints(case["lo"], case["hi"], B, "len"), case["page"], case["D"], TYPES[case["type"]]
        cols, used, _ = _tables(case, lens)
        pages = used + 7
        table, _ = _filled_table(g, lens, page, cols, pages)
        nh = case["kvh"] * case["rep"]
        q = _randn(g, B, case["T"], nh, D).to(typ)
        return dict(kc=_cache(g, pages * page, case["kvh"], D), vc=_cache(g, pages * page, case["kvh"], D), table=table,
                    n_kv=_i32(lens), q=q, gate=_randn(g, B, case["T"], nh, D).to(typ) if case["gate"] else None,
                    longest=max(lens))
    lens, typ = _ints(case["lo"], case["hi"], B, "len"), TYPES[case["type"]]
    n, kh, vh, dk, dv = sum(lens), case["kh"], case["vh"], case["dk"], case["dv"]
    q, k = _randn(g, n, kh, dk), _randn(g, n, kh, dk)
    q, k = (x / x.norm(dim=2, keepdim=True) for x in (q, k))
    # log decay: heads with short and with long memory
    rate = torch.exp(_rand(g, vh) * math.log(500.0)) * 0.003
    decay = -rate.contiguous() if case["fixed"] else (-_rand(g, n, vh) * rate).contiguous()
    cu = [0]
    for x in lens:
        cu.append(cu[-1] + x)
    return dict(q=q.to(typ), k=k.to(typ), v=_randn(g, n, vh, dv).to(typ), g=decay, cu=_i32(cu), longest=max(lens),
                state=_randn(g, B + 3, vh, dk, dv) * 0.05, slots=_perm(g, B + 3)[:B].contiguous())


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"], s["kind"] = case, case["kind"]
    B, dev = case["B"], "cuda"
    i32 = lambda n: torch.zeros(max(1, n), dtype=torch.int32, device=dev)  # noqa: E731
    if s["kind"] == "extend":
        s.update(n_free_out=i32(1), n_kv=i32(B), cu=i32(B + 1), slots=i32(s["n_tok"]), pos=i32(s["n_tok"]),
                 seq=i32(s["n_tok"]))
    elif s["kind"] == "trim":
        s.update(n_free_out=i32(1), n_kv=i32(B))
    elif s["kind"] == "paged":
        s["out"] = torch.zeros_like(s["q"])
    else:
        s["out"] = torch.zeros_like(s["v"])
        s["state_out"] = torch.zeros_like(s["state"])
    if own:
        K = _lib()
        K.check(K.load().qwfn_init(0))
        if s["kind"] in ("extend", "trim"):
            n = K.paged_workspace_size(B)
        elif s["kind"] == "paged":
            s["qv"], s["ov"] = K.q_view(s["q"]), K.out_view(s["out"])
            s["kv"], s["vv"] = (K.cache_attn_view(c, c.shape[0], case["kvh"], case["D"]) for c in (s["kc"], s["vc"]))
            n = K.fattn_workspace_size_paged(s["qv"], s["kv"], s["vv"], s["table"], case["page"])
        else:
            n = K.linear_attn_workspace_size(s["q"], s["v"], B, s["longest"])
        s["ws"] = torch.empty(max(256, n), dtype=torch.uint8, device=dev)
    return s


def run(s):
    kind, case = s["kind"], s["case"]
    if own:
        K = _lib()
        if kind == "extend":
            K.paged_extend(s["past"], s["new"], case["page"], s["table"], s["free"], s["n_free"], s["n_free_out"], s["n_kv"],
                           s["cu"], s["slots"], pos=s["pos"], seq=s["seq"], ws=s["ws"])
        elif kind == "trim":
            K.paged_trim(s["keep"], s["past"], case["page"], s["table"], s["free"], s["n_free"], s["n_free_out"], s["n_kv"],
                         ws=s["ws"])
            return dict(free=s["free"], n_free=s["n_free_out"], n_kv=s["n_kv"])
        elif kind == "paged":
            K.flash_attn_ext_paged(s["qv"], s["kv"], s["vv"], s["table"], case["page"], s["n_kv"], case["D"] ** -0.5,
                                   s["ov"], gate=s["gate"], ws=s["ws"])
            return dict(out=s["out"])
        else:
            K.linear_attn(s["q"], s["k"], s["v"], s["g"], s["cu"], s["longest"], s["state"], s["state_out"], s["out"],
                          slots=s["slots"], ws=s["ws"])
            return dict(out=s["out"], state=s["state_out"])
        return dict(table=s["table"], n_free=s["n_free_out"], n_kv=s["n_kv"], cu=s["cu"], slots=s["slots"], pos=s["pos"],
                    seq=s["seq"])
    return dict(extend=_extend, trim=_trim, paged=_paged, linear=_linear)[kind](s, case)


# ---------------------------------------------------------------- the plain forms

def _extend(s, case):
    page, past, new = case["page"], s["past"].long(), s["new"].long()
    cols, n_free = s["table"].shape[1], s["n_free"].long()
    have, total = (past + page - 1) // page, past + new
    fits = total <= cols * page
    need = torch.where(fits, (total + page - 1) // page - have, torch.zeros_like(have))
    cum = torch.cumsum(need, 0)
    served = fits & ((need == 0) | (cum <= n_free))
    need = torch.where(served, need, torch.zeros_like(need))
    j = torch.arange(cols, device="cuda")[None, :]
    taken = (j >= have[:, None]) & (j < (have + need)[:, None])
    at = n_free - 1 - ((cum - need)[:, None] + j - have[:, None])
    at = torch.where(taken, at, torch.zeros_like(at))
    table = torch.where(taken, s["free"][at], s["table"])
    cu = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0)])
    i = torch.arange(s["n_tok"], device="cuda")
    seq = torch.searchsorted(cu[1:].contiguous(), i, right=True)
    live = i < cu[-1]
    b = torch.where(live, seq, torch.zeros_like(seq))
    p = past[b] + i - cu[b]
    has = live & served[b]
    col = torch.where(has, p // page, torch.zeros_like(p))
    slot = table[b, col].long() * page + p % page
    none = torch.full_like(p, -1)
    return dict(table=table, n_free=(n_free - need.sum()).to(torch.int32),
                n_kv=torch.where(served, total, past).to(torch.int32), cu=cu.to(torch.int32),
                slots=torch.where(has, slot, none).to(torch.int32), pos=torch.where(has, p, none).to(torch.int32),
                seq=torch.where(live, seq, none).to(torch.int32))


def _trim(s, case):
    page, past, cols = case["page"], s["past"].long(), s["table"].shape[1]
    keep = torch.minimum(torch.clamp(s["keep"].long(), min=0), past)
    first, last = (keep + page - 1) // page, (past + page - 1) // page
    back = last - first
    off = torch.cumsum(back, 0) - back
    j = torch.arange(cols, device="cuda")[None, :]
    goes = (j >= first[:, None]) & (j < last[:, None])
    at = s["n_free"].long() + off[:, None] + j - first[:, None]
    free = s["free"].clone()
    free[at[goes]] = s["table"][goes]
    return dict(free=free, n_free=(s["n_free"].long() + back.sum()).to(torch.int32), n_kv=keep.to(torch.int32))


def _paged(s, case):
    B, T, kvh, rep, D, page = (case[x] for x in ("B", "T", "kvh", "rep", "D", "page"))
    n = s["longest"]
    j = torch.arange(n, device="cuda")
    held = j[None, :] < s["n_kv"][:, None]
    page_of = s["table"][:, torch.div(j, page, rounding_mode="floor")]
    slot = torch.where(held, page_of * page + j % page, torch.zeros_like(page_of)).long().reshape(-1)

    def values(cache):                                    # [B, kvh, n, D] in f32 (exact: 11 bits times 8)
        rows = cache[slot].reshape(B, n, kvh, D // 32, 34)
        d = rows[..., :2].contiguous().view(torch.float16).float()
        x = (rows[..., 2:].contiguous().view(torch.int8).float() * d).reshape(B, n, kvh, D)
        return x.permute(0, 2, 1, 3).contiguous()

    qi, dq = _quant(s["q"].float())
    q = (qi.float() * dq.float()[..., None]).reshape(B, T, kvh, rep, D)
    q = q.permute(0, 2, 4, 1, 3).reshape(B, kvh, D, T * rep).contiguous()
    sc = torch.matmul(values(s["kc"]), q) * D ** -0.5     # [B, kvh, n, T rep]
    t = torch.arange(T, device="cuda").repeat_interleave(rep)
    seen = j[None, :, None] < (s["n_kv"][:, None, None] - (T - 1) + t[None, None, :])
    sc = torch.where(seen[:, None], sc, torch.full_like(sc[:1, :1, :1, :1], float("-inf")))
    top = sc.amax(dim=2, keepdim=True)
    p = torch.exp(sc - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(dim=2)[..., None]
    out = torch.matmul(p.permute(0, 1, 3, 2).contiguous(), values(s["vc"]))
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    out = out.reshape(B, kvh, T, rep, D).permute(0, 2, 1, 3, 4).reshape(B, T, kvh * rep, D)
    if s["gate"] is not None:
        out = out / (1.0 + torch.exp(-s["gate"].float()))
    return dict(out=out.to(s["q"].dtype).contiguous())


def _linear(s, case):
    B, kh, vh, dk, dv = (case[x] for x in ("B", "kh", "vh", "dk", "dv"))
    n, longest = s["q"].shape[0], s["longest"]
    C = min(64, longest)
    nc = (longest + C - 1) // C
    cu = s["cu"].long()
    at = cu[:-1, None] + torch.arange(nc * C, device="cuda")[None, :]
    held = at < cu[1:, None]
    at = torch.where(held, at, torch.zeros_like(at))

    def chunks(x, rep):                                   # packed tokens -> [B, vh, nc, C, d] in f32, 0 past the end
        x = torch.where(held[..., None, None], x[at].float(), torch.zeros((), device="cuda"))
        x = x.reshape(B, nc, C, x.shape[2], -1).permute(0, 3, 1, 2, 4)
        return x.repeat_interleave(rep, dim=1).contiguous()

    q, k, v = chunks(s["q"], vh // kh), chunks(s["k"], vh // kh), chunks(s["v"], 1)
    g = s["g"].double()
    g = g[None, :].expand(n, vh) if case["fixed"] else g
    g = torch.where(held[..., None], g[at], torch.zeros((), dtype=torch.float64, device="cuda"))
    G = torch.cumsum(g.reshape(B, nc, C, vh).permute(0, 3, 1, 2), dim=3)         # [B, vh, nc, C], within the chunk
    end = torch.cumsum(G[..., -1], dim=2)                                        # to the end of each chunk
    start = end - G[..., -1]
    i, c = torch.arange(C, device="cuda"), torch.arange(nc + 1, device="cuda")
    inner = torch.where(i[:, None] >= i[None, :], G[..., :, None] - G[..., None, :],
                        torch.full((), -math.inf, dtype=torch.float64, device="cuda"))
    p = torch.matmul(q, k.transpose(-1, -2).contiguous()) * torch.exp(inner).float()
    out = torch.matmul(p, v)
    # each chunk's own contribution to the state at its end, then the states before every chunk and after the last
    kw = k * torch.exp(G[..., -1:] - G).float()[..., None]
    own_state = torch.matmul(kw.transpose(-1, -2).contiguous(), v).reshape(B, vh, nc, dk * dv)
    starts = torch.cat([start, end[..., -1:]], dim=2)
    outer = torch.where(c[:, None] > c[None, :nc], starts[..., :, None] - end[..., None, :],
                        torch.full((), -math.inf, dtype=torch.float64, device="cuda"))
    S0 = s["state"][s["slots"].long()].reshape(B, vh, 1, dk * dv)
    S = torch.matmul(torch.exp(outer).float(), own_state) + torch.exp(starts).float()[..., None] * S0
    S = S.reshape(B, vh, nc + 1, dk, dv)
    out = out + torch.matmul(q * torch.exp(G).float()[..., None], S[:, :, :nc].contiguous())
    out = (out * dk ** -0.5).permute(0, 2, 3, 1, 4).reshape(B, nc * C, vh, dv)[held]
    state = s["state_out"].clone()
    state[s["slots"].long()] = S[:, :, nc]
    return dict(out=out.to(s["v"].dtype), state=state)


# ---------------------------------------------------------------- work and exact results

def work(case):
    kind, B = case["kind"], case["B"]
    if kind == "extend":
        past, new = _past_new(case)
        _, _, need = _tables(case, past, new)
        need = need * 3 // 4 if case["short"] else need
        return dict(bytes=16.0 * B + 8 * need + 12 * sum(new), flops=0.0)
    if kind == "trim":
        past, keep = _keeps(case)
        back = sum(_pages(p, case["page"]) - _pages(x, case["page"]) for p, x in zip(past, keep))
        return dict(bytes=12.0 * B + 8 * back, flops=0.0)
    if kind == "paged":
        lens, T, D, kvh = _ints(case["lo"], case["hi"], B, "len"), case["T"], case["D"], case["kvh"]
        rows, es = B * T * kvh * case["rep"], 4 if case["type"] == "f32" else 2
        n = sum(lens)
        return dict(bytes=float(n * kvh * D // 32 * 34 * 2 + 4 * n // case["page"] + rows * D * es * (3 if case["gate"] else 2)),
                    flops=4.0 * n * T * kvh * case["rep"] * D)
    lens, es = _ints(case["lo"], case["hi"], B, "len"), 4 if case["type"] == "f32" else 2
    n, kh, vh, dk, dv = sum(lens), case["kh"], case["vh"], case["dk"], case["dv"]
    return dict(bytes=float(n * es * (2 * kh * dk + 2 * vh * dv) + (4 * vh if case["fixed"] else 4 * n * vh) + 8 * B * vh * dk * dv),
                flops=4.0 * n * vh * dk * dv)


def exact(case, seed):
    """The outputs in float64: softmax attention one request at a time, linear attention one token at a time."""
    kind = case["kind"]
    if kind in ("extend", "trim"):
        return None                                       # whole numbers
    s = _inputs(case, seed)
    B = case["B"]
    if kind == "paged":
        T, kvh, rep, D, page = (case[x] for x in ("T", "kvh", "rep", "D", "page"))
        out = torch.zeros((B, T, kvh * rep, D), dtype=torch.float64, device="cuda")
        # the query's q8_0 image is part of the definition: its scale and its whole numbers in single precision
        x = s["q"].float().reshape(B, T, kvh, rep, D // 32, 32)
        amax = x.abs().amax(-1, keepdim=True)
        inv = (127.0 / amax.double()).float()
        qd = torch.round(x * inv).double() * (amax.double() / 127.0).float().half().double()
        qd = qd.reshape(B, T, kvh, rep, D)
        for b, n in enumerate(s["n_kv"].tolist()):
            key = torch.arange(n, device="cuda")
            rows = s["table"][b].long()[key // page] * page + key % page
            for h in range(kvh):
                def side(cache):
                    seg = cache[rows].reshape(n, kvh, D // 32, 34)[:, h]
                    scale = seg[..., :2].contiguous().view(torch.float16).double()
                    return (seg[..., 2:].contiguous().view(torch.int8).double() * scale).reshape(n, D)
                kd, vd = side(s["kc"]), side(s["vc"])
                for t in range(T):
                    m = n - T + t + 1
                    if m > 0:
                        w = torch.softmax(qd[b, t, h] @ kd[:m].t().contiguous() / math.sqrt(D), dim=-1)
                        out[b, t, h * rep:(h + 1) * rep] = w @ vd[:m]
        if s["gate"] is not None:
            out = out * torch.sigmoid(s["gate"].double())
        return dict(out=out)
    kh, vh, dk = case["kh"], case["vh"], case["dk"]
    lens = torch.diff(s["cu"].long())
    slots = s["slots"].long()
    state = s["state"][slots].double()
    res = torch.zeros(s["v"].shape, dtype=torch.float64, device="cuda")
    for t in range(s["longest"]):
        live = torch.nonzero(t < lens).reshape(-1)
        tok = s["cu"].long()[live] + t
        qt, kt = (s[x][tok].double().repeat_interleave(vh // kh, dim=1) for x in ("q", "k"))
        d = s["g"].double().expand(len(tok), vh) if case["fixed"] else s["g"][tok].double()
        new = state[live] * torch.exp(d)[..., None, None] + kt[..., :, None] * s["v"][tok].double()[..., None, :]
        state[live] = new
        res[tok] = (qt[..., None, :] @ new)[..., 0, :] / math.sqrt(dk)
    full = torch.zeros_like(s["state"], dtype=torch.float64)
    full[slots] = state
    return dict(out=res, state=full)
