"""Workloads of shared pages and of drafted trees: forks, releases and compaction of the paged q8_0 cache, attention and
linear attention of a tree of drafted tokens, and the step that keeps the accepted ones.

listed() names the cases, draw(rng) makes another one of the same ranges, prepare(case, seed) builds what a serving
program holds before the call on the GPU, run(state) is one pass through an operator, work(case) its compulsory bytes and
operations, exact(case, seed) the results in float64. run computes the operators in plain torch where `own` is false and
calls the library where it is true.

Shapes: 2 KV heads of 256 under 16 query heads (the benchmark's configurations) or 24 (the reference's model), 12 attention
layers (24 cache tensors); 48 / 16 value / key heads of 128 in the recurrent layers; page sizes, batches, other head sizes
and draft trees of up to 64 tokens as serving programs use them.
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
        # one prompt answered seven times more: its pages shared, the partly filled one copied in every layer
        dict(name="fork_b8_1237", kind="fork", B=8, forks=7, lo=1237, hi=1237, page=16, row=544, caches=24),
        # a beam search's step, or a batch that starts from cached prefixes: half of the requests from the other half
        dict(name="fork_b256_ragged", kind="fork", B=256, forks=128, lo=64, hi=4096, page=32, row=544, caches=8),
        # a batch of which some requests end, some hand rejected drafts back, all in families with a common prefix
        dict(name="release_b512", kind="release", B=512, family=4, lo=128, hi=16384, end=0.3, back=3, page=16),
        # a pool with holes before it is made smaller: the pages behind the live ones' number move, layer by layer
        dict(name="compact_12000", kind="compact", B=96, pages=12000, live=0.6, page=16, row=544, caches=8),
        # one conversation, 8 drafted tokens: the smallest attention call
        dict(name="tree_T8_b1_701_h24", kind="tree", B=1, lo=701, hi=701, T=8, kvh=2, rep=12, D=256, page=16, type="f32",
             gate=False, full=True),
        # a verify step of a ragged batch with trees of different sizes, half-precision activations, the output gate
        dict(name="tree_T32_b16_ragged_h16", kind="tree", B=16, lo=300, hi=20000, T=32, kvh=2, rep=8, D=256, page=64,
             type="bf16", gate=True, full=False),
        # smaller heads, 16 rows of queries a KV head and node
        dict(name="tree_T24_b4_9001_d128", kind="tree", B=4, lo=9001, hi=9001, T=24, kvh=8, rep=4, D=128, page=16,
             type="f16", gate=False, full=True),
        # large trees over long contexts (the largest attention call)
        dict(name="tree_T64_b8_12295_h16", kind="tree", B=8, lo=12295, hi=12295, T=64, kvh=2, rep=8, D=256, page=32,
             type="f32", gate=False, full=True),
        # after the verify step of one conversation: masks, the accepted path, its rows moved in all layers
        dict(name="accept_T8_b1", kind="accept", B=1, lo=701, hi=701, T=8, page=16, row=544, caches=24, full=True),
        # the same of a batch with larger trees
        dict(name="accept_T48_b64", kind="accept", B=64, lo=64, hi=1500, T=48, page=32, row=544, caches=24, full=False),
        # the recurrent layers of a verify step of one conversation
        dict(name="linear_tree_T12_b1", kind="linear", B=1, T=12, kh=16, vh=48, dk=128, dv=128, type="bf16", fixed=False,
             full=True),
        # and of a batch
        dict(name="linear_tree_T32_b48", kind="linear", B=48, T=32, kh=16, vh=48, dk=128, dv=128, type="bf16", fixed=False,
             full=False),
    ]


def _log_int(rng, lo, hi):
    if lo >= hi:
        return hi
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(hi)))))))


def _ints(lo, hi, n, what):
    """n lengths spread over [lo, hi] by their logarithm, from the case alone."""
    rng = random.Random("%s %d %d %d" % (what, lo, hi, n))
    return [_log_int(rng, lo, hi) for _ in range(n)]


def draw(rng):
    kind = rng.choice(["fork", "release", "compact", "tree", "tree", "tree", "tree", "accept", "linear", "linear"])
    page = rng.choice([8, 16, 16, 32, 64, 100, 128])
    row = rng.choice([544, 544, 1088, 272, 68])
    if kind == "fork":
        B = _log_int(rng, 2, 256)
        return dict(kind=kind, B=B, forks=rng.randint(1, B - 1), lo=1, hi=_log_int(rng, 64, 4096), page=page, row=min(row, 544),
                    caches=rng.randint(1, 8))
    if kind == "release":
        return dict(kind=kind, B=_log_int(rng, 1, 512), family=rng.choice([1, 2, 4, 8]), lo=16, hi=_log_int(rng, 256, 16384),
                    end=rng.choice([0.0, 0.2, 0.6]), back=rng.randint(0, 40), page=page)
    if kind == "compact":
        return dict(kind=kind, B=_log_int(rng, 1, 128), pages=_log_int(rng, 300, 190000 // page), live=rng.uniform(0.1, 0.95),
                    page=page, row=min(row, 544), caches=rng.randint(1, 8))
    if kind == "tree":
        D, kvh, rep = rng.choice([(256, 2, 8), (256, 2, 12), (256, 1, 16), (256, 4, 6), (128, 8, 4), (128, 2, 7),
                                  (128, 4, 1), (64, 8, 8), (64, 1, 3)])
        T, B = _log_int(rng, 2, 64), _log_int(rng, 1, 32)
        most = 8 * 12295 * 64 * 16 * 256 // (T * kvh * rep * D)            # keys, by the largest case's products
        most = min(most, 250000 * 512 // (kvh * D))                         # and bytes
        hi = _log_int(rng, 100, max(100, min(65536, most // B)))
        return dict(kind=kind, B=B, lo=rng.choice([1, hi // 8 + 1, hi]), hi=hi, T=T, kvh=kvh, rep=rep, D=D, page=page,
                    type=rng.choice(["f32", "f16", "bf16"]), gate=rng.random() < 0.3, full=rng.random() < 0.5)
    if kind == "accept":
        return dict(kind=kind, B=_log_int(rng, 1, 64), lo=1, hi=_log_int(rng, 64, 1500), T=_log_int(rng, 2, 64), page=page,
                    row=min(row, 544), caches=rng.randint(1, 24), full=rng.random() < 0.5)
    kh, vh, dk, dv = rng.choice([(16, 48, 128, 128), (16, 16, 128, 128), (32, 32, 64, 64), (8, 32, 64, 128), (4, 8, 128, 64),
                                 (2, 4, 128, 256)])
    T = _log_int(rng, 2, 64)
    return dict(kind=kind, B=_log_int(rng, 1, max(1, 48 * 32 // max(T, 32))), T=T, kh=kh, vh=vh, dk=dk, dv=dv,
                type=rng.choice(["f32", "f16", "bf16", "bf16"]), fixed=rng.random() < 0.4, full=rng.random() < 0.5)


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


def _bytes(g, rows, row, n):
    """n cache tensors of any bytes: what is moved is not looked at."""
    return [torch.randint(0, 256, (rows, row), generator=g, device="cuda", dtype=torch.uint8) for _ in range(n)]


def _trees(case):
    """Each request's parents (-1: the context) and node counts, from the case alone: breadth first, 2 to 5 children a node,
    a few nodes hung elsewhere, where a request has room a second root."""
    rng = random.Random("tree %d %d %d" % (case["B"], case["T"], case.get("hi", 0)))
    par, cnt = [], []
    for _ in range(case["B"]):
        k = rng.randint(2, 5)
        p = [-1] + [(t - 1) // k if rng.random() < 0.8 else rng.randint(max(0, t // 4), t - 1) for t in range(1, case["T"])]
        if case["T"] > 20 and rng.random() < 0.3:
            p[2] = -1
        par.append(p)
        cnt.append(case["T"] if case["full"] else rng.randint(max(1, case["T"] // 4), case["T"]))
    return par, cnt


def _masks(par):
    """Ancestors and self of every node as bits of a signed 64-bit word, and the nodes' depths."""
    masks, depth = [], []
    for p in par:
        m, d = [], []
        for t, q in enumerate(p):
            m.append((1 << t) | (m[q] if q >= 0 else 0))
            d.append(d[q] + 1 if q >= 0 else 0)
        masks.append([x - (1 << 64) if x >> 63 else x for x in m])
        depth.append(d)
    return masks, depth


def _leaves(case, par, cnt):
    """A node a request whose path an engine could have accepted. Only such whose rows move onto rows that no other one is
    moved from, so that a pass can be repeated on the same cache."""
    rng = random.Random("leaf %d %d" % (case["B"], case["T"]))
    out = []
    for p, n in zip(par, cnt):
        fine = [-1]
        for t in range(n):
            path, x = [], t
            while x >= 0:
                path.insert(0, x)
                x = p[x]
            if all(x == i or x >= len(path) for i, x in enumerate(path)):
                fine += [t] * len(path) ** 3               # rather the deep ones
        out.append(rng.choice(fine))
    return out


def _filled(g, lens, page, cols, pages):
    """A block table whose first ceil(length / page) columns hold distinct pages in random order, and the other pages."""
    have = _i32([_pages(n, page) for n in lens])
    perm = _perm(g, pages)
    at = torch.cumsum(have, 0) - have
    j = torch.arange(cols, device="cuda")
    held = j[None, :] < have[:, None]
    idx = torch.where(held, at[:, None] + j[None, :], torch.zeros_like(j)[None, :])
    return torch.where(held, perm[idx.long()], torch.full_like(perm[:1], -7)).contiguous(), perm[int(have.sum()):].contiguous()


def _fork_plan(case):
    """Lengths (0 for the requests that are forked into), parents and how many tokens each fork takes over."""
    rng = random.Random("fork %d %d %d" % (case["B"], case["forks"], case["hi"]))
    B, forks = case["B"], case["forks"]
    kids = set(rng.sample(range(1, B), forks) if forks < B - 1 else range(1, B))
    olds = [b for b in range(B) if b not in kids]
    lens = _ints(case["lo"], case["hi"], B, "len")
    lens = [0 if b in kids else lens[b] for b in range(B)]
    src = [rng.choice(olds) if b in kids else -1 for b in range(B)]
    tok = [0 if f < 0 else lens[f] if rng.random() < 0.7 else rng.randint(0, lens[f]) for f in src]
    return lens, src, tok


def _families(case):
    """Lengths, what each keeps, and the pages that the families share at their start."""
    rng = random.Random("family %d %d %d" % (case["B"], case["family"], case["hi"]))
    B, f, page = case["B"], case["family"], case["page"]
    lens = _ints(case["lo"], case["hi"], B, "len")
    common = []
    for b0 in range(0, B, f):
        n = min(lens[b0:b0 + f]) // page
        common += [rng.randint(0, n) if len(lens[b0:b0 + f]) > 1 else 0] * len(lens[b0:b0 + f])
    keep = [0 if rng.random() < case["end"] else max(0, n - rng.randint(0, case["back"])) for n in lens]
    return lens, keep, common


def _pool(case):
    """Lengths of a pool's requests: `live` of its pages."""
    rng = random.Random("pool %d %d %d" % (case["B"], case["pages"], case["page"]))
    n = max(1, min(case["pages"], int(case["pages"] * case["live"])))
    cuts = sorted(rng.randint(0, n) for _ in range(case["B"] - 1))
    held = [b - a for a, b in zip([0] + cuts, cuts + [n])]
    return [0 if h == 0 else h * case["page"] - rng.randint(0, case["page"] - 1) for h in held]


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    kind, g, B = case["kind"], _gen(seed), case["B"]
    if kind == "fork":
        lens, src, tok = _fork_plan(case)
        page = case["page"]
        used = sum(_pages(n, page) for n in lens)
        fresh = sum(1 for n in tok if n % page)
        pages = used + fresh + 9
        table, free = _filled(g, lens, page, max(_pages(n, page) for n in lens) + 2, pages)
        return dict(n_kv=_i32(lens), src=_i32(src), tok=_i32(tok), table=table, free=free, n_free=_i32([free.numel()]),
                    shared=torch.zeros(pages, dtype=torch.int32, device="cuda"),
                    caches=_bytes(g, pages * page, case["row"], case["caches"]))
    if kind == "release":
        lens, keep, common = _families(case)
        page, f = case["page"], case["family"]
        used = sum(_pages(n, page) for n in lens)
        pages = used + 100
        table, _ = _filled(g, lens, page, max(_pages(n, page) for n in lens) + 2, pages)
        first = _i32([b // f * f for b in range(B)]).long()
        j = torch.arange(table.shape[1], device="cuda")
        table = torch.where(j[None, :] < _i32(common)[:, None], table[first], table).contiguous()
        have = _i32([_pages(n, page) for n in lens])
        held = torch.bincount(table[j[None, :] < have[:, None]].long(), minlength=pages)
        shared = torch.clamp(held - 1, min=0).to(torch.int32)
        unused = torch.nonzero(held == 0).reshape(-1).to(torch.int32)
        free = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        free[:unused.numel()] = unused[torch.randperm(unused.numel(), generator=g, device="cuda")]
        return dict(n_kv=_i32(lens), keep=_i32(keep), table=table, shared=shared, free=free, n_free=_i32([unused.numel()]))
    if kind == "compact":
        lens, page, pages = _pool(case), case["page"], case["pages"]
        table, rest = _filled(g, lens, page, max(_pages(n, page) for n in lens) + 2, pages)
        shared = torch.zeros(pages, dtype=torch.int32, device="cuda")
        live = table[table >= 0].long()
        shared[live] = torch.randint(0, 3, (live.numel(),), generator=g, device="cuda", dtype=torch.int32)
        free = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        free[:rest.numel()] = rest
        return dict(n_kv=_i32(lens), table=table, shared=shared, free=free, n_free=_i32([rest.numel()]),
                    caches=_bytes(g, pages * page, case["row"], case["caches"]))
    par, cnt = _trees(case)
    masks, _ = _masks(par)
    T = case["T"]
    masks = torch.tensor(masks, dtype=torch.int64, device="cuda").reshape(B, T)
    s = dict(parents=_i32(par).reshape(B, T), masks=masks, n_tree=None if case["full"] else _i32(cnt), cnt=cnt)
    if kind in ("tree", "accept"):
        lens = [n + c for n, c in zip(_ints(case["lo"], case["hi"], B, "len"), cnt)]
        page = case["page"]
        pages = sum(_pages(n, page) for n in lens) + 7
        table, _ = _filled(g, lens, page, max(_pages(n, page) for n in lens) + 3, pages)
        s.update(n_kv=_i32(lens), table=table, lens=lens)
        if kind == "accept":
            s.update(leaf=_i32(_leaves(case, par, cnt)), n_past=_i32([n - c for n, c in zip(lens, cnt)]),
                     caches=_bytes(g, pages * page, case["row"], case["caches"]))
            return s
        D, kvh, typ = case["D"], case["kvh"], TYPES[case["type"]]
        nh = kvh * case["rep"]
        s.update(kc=_cache(g, pages * page, kvh, D), vc=_cache(g, pages * page, kvh, D), q=_randn(g, B, T, nh, D).to(typ),
                 gate=_randn(g, B, T, nh, D).to(typ) if case["gate"] else None)
        return s
    kh, vh, dk, dv, typ = case["kh"], case["vh"], case["dk"], case["dv"], TYPES[case["type"]]
    q, k = _randn(g, B * T, kh, dk), _randn(g, B * T, kh, dk)
    q, k = (x / x.norm(dim=2, keepdim=True) for x in (q, k))
    # log decay: heads with short and with long memory
    rate = torch.exp(_rand(g, vh) * math.log(500.0)) * 0.003
    decay = -rate.contiguous() if case["fixed"] else (-_rand(g, B * T, vh) * rate).contiguous()
    s.update(q=q.to(typ), k=k.to(typ), v=_randn(g, B * T, vh, dv).to(typ), g=decay, state=_randn(g, B + 3, vh, dk, dv) * 0.05,
             slots=_perm(g, B + 3)[:B].contiguous())
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"], s["kind"] = case, case["kind"]
    kind, B, dev = case["kind"], case["B"], "cuda"
    i32 = lambda *n: torch.zeros(n, dtype=torch.int32, device=dev)  # noqa: E731
    if kind in ("fork", "release", "compact"):
        s.update(n_free_out=i32(1), shared_out=torch.zeros_like(s["shared"]))
    if kind == "fork":
        s.update(n_kv_out=i32(B), moves=i32(B, 3))
    elif kind == "release":
        s.update(n_kv_out=i32(B), free_out=s["free"].clone())
    elif kind == "compact":
        n = case["pages"]
        s.update(table_out=s["table"].clone(), free_out=torch.full_like(s["free"], -1), page_map=i32(n), moves=i32((n + 1) // 2, 3),
                 n_moves=i32(1))
    elif kind == "accept":
        T = case["T"]
        s.update(masks_out=torch.zeros_like(s["masks"]), pos=i32(B, T), n_keep=i32(B), cu=i32(B + 1), path=i32(B * T))
    elif kind == "tree":
        s["out"] = torch.zeros_like(s["q"])
    else:
        s["out"] = torch.zeros_like(s["v"])
    if own:
        K = _lib()
        K.check(K.load().qwfn_init(0))
        if "caches" in s:
            s["list"] = K.cache_list(s["caches"])
        n = 0
        if kind == "tree":
            s["qv"], s["ov"] = K.q_view(s["q"]), K.out_view(s["out"])
            s["kv"], s["vv"] = (K.cache_attn_view(c, c.shape[0], case["kvh"], case["D"]) for c in (s["kc"], s["vc"]))
            n = K.fattn_workspace_size_paged_tree(s["qv"], s["kv"], s["vv"], s["table"], case["page"])
        elif kind in ("fork", "release"):
            n = K.paged_workspace_size(B) if kind == "fork" else K.paged_release_workspace_size(B, s["shared"].numel())
        elif kind == "compact":
            n = K.paged_compact_workspace_size(case["pages"])
        s["ws"] = torch.empty(max(256, n), dtype=torch.uint8, device=dev)
    return s


def run(s):
    kind, case = s["kind"], s["case"]
    if not own:
        return dict(fork=_fork, release=_release, compact=_compact, tree=_tree, accept=_accept, linear=_linear)[kind](s, case)
    K = _lib()
    if kind == "fork":
        K.paged_fork(s["src"], s["n_kv"], case["page"], s["table"], s["shared"], s["free"], s["n_free"], s["n_free_out"],
                     s["n_kv_out"], s["shared_out"], s["moves"], n_tok=s["tok"], ws=s["ws"])
        K.paged_copy(s["list"], s["moves"], case["page"])
        return dict(table=s["table"], n_free=s["n_free_out"], n_kv=s["n_kv_out"], shared=s["shared_out"], moves=s["moves"],
                    caches=s["caches"])
    if kind == "release":
        K.paged_release(s["keep"], s["n_kv"], case["page"], s["table"], s["shared"], s["free_out"], s["n_free"], s["n_free_out"],
                        s["n_kv_out"], s["shared_out"], ws=s["ws"])
        return dict(free=s["free_out"], n_free=s["n_free_out"], n_kv=s["n_kv_out"], shared=s["shared_out"])
    if kind == "compact":
        K.paged_compact(s["n_kv"], case["page"], s["table"], s["shared"], s["free"], s["n_free"], s["table_out"], s["shared_out"],
                        s["free_out"], s["n_free_out"], s["page_map"], s["moves"], s["n_moves"], ws=s["ws"])
        K.paged_copy(s["list"], s["moves"], case["page"], n_moves=s["n_moves"])
        return dict(table=s["table_out"], shared=s["shared_out"], free=s["free_out"], n_free=s["n_free_out"], map=s["page_map"],
                    n_moves=s["n_moves"], caches=s["caches"])
    if kind == "tree":
        K.flash_attn_ext_paged_tree(s["qv"], s["kv"], s["vv"], s["table"], case["page"], s["n_kv"], s["masks"],
                                    case["D"] ** -0.5, s["ov"], n_tree=s["n_tree"], gate=s["gate"], ws=s["ws"])
        return dict(out=s["out"])
    if kind == "accept":
        K.tree_masks(s["parents"], s["masks_out"], n_tree=s["n_tree"], n_past=s["n_past"], pos=s["pos"])
        K.paged_accept(s["list"], case["page"], s["table"], s["n_kv"], s["masks_out"], s["leaf"], s["n_keep"], n_tree=s["n_tree"],
                       cu_path=s["cu"], path=s["path"])
        return dict(masks=s["masks_out"], pos=s["pos"], n_keep=s["n_keep"], cu=s["cu"], path=s["path"], caches=s["caches"])
    K.linear_attn_tree(s["q"], s["k"], s["v"], s["g"], s["masks"], s["state"], s["out"], n_tree=s["n_tree"], slots=s["slots"])
    return dict(out=s["out"])


# ---------------------------------------------------------------- the plain forms

def _put(caches, src, dst):
    for c in caches:
        c[dst] = c[src]


def _fork(s, case):
    """Request b with src[b] = f >= 0 becomes a copy of f's first tok[b] tokens: whole pages shared, the rest on a new page."""
    page, src, tok, n_kv, table = case["page"], s["src"].long(), s["tok"].long(), s["n_kv"].long(), s["table"]
    kid = src >= 0
    f = torch.where(kid, src, torch.zeros_like(src))
    fits = kid & (n_kv == 0) & (src[f] < 0) & (tok >= 0) & (tok <= n_kv[f])
    full = torch.div(tok, page, rounding_mode="floor")
    rest = tok % page
    need = (fits & (rest > 0)).long()
    served = fits & ((need == 0) | (torch.cumsum(need, 0) <= s["n_free"].long()))
    need = torch.where(served, need, torch.zeros_like(need))
    n_free = s["n_free"].long()
    at = n_free - 1 - (torch.cumsum(need, 0) - need)
    fresh = s["free"][torch.where(need > 0, at, torch.zeros_like(at))].long()
    j = torch.arange(table.shape[1], device="cuda")[None, :]
    takes = served[:, None] & (j < full[:, None])
    rows = table[f]
    shared = s["shared"] + torch.bincount(rows[takes].long(), minlength=s["shared"].numel()).to(torch.int32)
    new = torch.where(takes, rows, table)
    new = torch.where((need > 0)[:, None] & (j == full[:, None]), fresh[:, None].to(torch.int32), new)
    old = rows.gather(1, torch.clamp(full, max=table.shape[1] - 1)[:, None])[:, 0].long()
    moves = torch.stack([old * page, fresh * page, rest], dim=1)
    moves = torch.where((need > 0)[:, None], moves, torch.zeros_like(moves))
    table.copy_(new)
    i = torch.arange(page, device="cuda")[None, :]
    on = i < moves[:, 2:3]
    _put(s["caches"], (moves[:, 0:1] + i)[on], (moves[:, 1:2] + i)[on])
    return dict(table=table, n_free=(n_free - need.sum()).to(torch.int32), n_kv=torch.where(served, tok, n_kv).to(torch.int32),
                shared=shared, moves=moves.to(torch.int32), caches=s["caches"])


def _release(s, case):
    """Request b keeps its first keep[b] tokens; pages behind them that nobody else holds go onto the stack, lowest first."""
    page, n, table = case["page"], s["n_kv"].long(), s["table"]
    keep = torch.minimum(torch.clamp(s["keep"].long(), min=0), n)
    first, last = (keep + page - 1) // page, (n + page - 1) // page
    end = table.gather(1, torch.clamp(first - 1, min=0)[:, None])[:, 0].long()
    inside = (keep < n) & (keep % page != 0) & (s["shared"][torch.clamp(end, min=0)] > 0)
    keep = torch.where(inside, n, keep)
    first = torch.where(inside, last, first)
    j = torch.arange(table.shape[1], device="cuda")[None, :]
    goes = (j >= first[:, None]) & (j < last[:, None])
    back = torch.bincount(table[goes].long(), minlength=s["shared"].numel())
    freed = back > s["shared"]
    pages = torch.nonzero(freed).reshape(-1).to(torch.int32)
    free = s["free"].clone()
    n_free = int(s["n_free"])
    free[n_free:n_free + pages.numel()] = pages
    shared = torch.where(freed, torch.zeros_like(back), s["shared"].long() - back).to(torch.int32)
    return dict(free=free, n_free=s["n_free"] + pages.numel(), n_kv=keep.to(torch.int32), shared=shared)


def _compact(s, case):
    """Live pages (those not on the stack) behind the live pages' number move to the free ones before it, both ascending."""
    page, pages = case["page"], case["pages"]
    dead = torch.zeros(pages, dtype=torch.bool, device="cuda")
    dead[s["free"][:int(s["n_free"])].long()] = True
    n_live = pages - int(dead.sum())
    p = torch.arange(pages, device="cuda")
    src, dst = p[(p >= n_live) & ~dead], p[(p < n_live) & dead]
    m = torch.where(dead, torch.full_like(p, -1), p)
    m[src] = dst
    have = (s["n_kv"].long() + page - 1) // page
    j = torch.arange(s["table"].shape[1], device="cuda")[None, :]
    held = j < have[:, None]
    table = torch.where(held, m[torch.where(held, s["table"], torch.zeros_like(s["table"])).long()].to(torch.int32), s["table"])
    shared = s["shared"].clone()
    shared[dst] = s["shared"][src]
    shared[n_live:] = 0
    free = torch.full_like(s["free"], -1)
    free[:pages - n_live] = torch.arange(pages - 1, n_live - 1, -1, device="cuda").to(torch.int32)
    i = torch.arange(page, device="cuda")[None, :]
    _put(s["caches"], (src[:, None] * page + i).reshape(-1), (dst[:, None] * page + i).reshape(-1))
    return dict(table=table, shared=shared, free=free, n_free=_i32([pages - n_live]), map=m.to(torch.int32),
                n_moves=_i32([src.numel()]), caches=s["caches"])


def _bits(masks, n_tree):
    """[B, T, T]: node t sees node j."""
    B, T = masks.shape
    j = torch.arange(T, device="cuda")
    bits = (masks[:, :, None] >> j[None, None, :] & 1) != 0
    if n_tree is not None:
        bits &= (j[None, None, :] < n_tree[:, None, None]) & (j[None, :, None] < n_tree[:, None, None])
    return bits


def _tree(s, case):
    """Query t of request b: all tokens before the tree, and the nodes of its mask."""
    B, T, kvh, rep, D, page = (case[x] for x in ("B", "T", "kvh", "rep", "D", "page"))
    n = max(s["lens"])
    j = torch.arange(n, device="cuda")
    held = j[None, :] < s["n_kv"][:, None]
    page_of = s["table"][:, torch.div(j, page, rounding_mode="floor")]
    slot = torch.where(held, page_of * page + j % page, torch.zeros_like(page_of)).long().reshape(-1)

    def values(cache):                                    # [B, kvh, n, D] in f32 (exact: 11 bits times 8)
        rows = cache[slot].reshape(B, n, kvh, D // 32, 34)
        d = rows[..., :2].contiguous().view(torch.float16).float()
        x = (rows[..., 2:].contiguous().view(torch.int8).float() * d).reshape(B, n, kvh, D)
        return x.permute(0, 2, 1, 3).contiguous()

    n_tree = _i32(s["cnt"]).long()
    base = s["n_kv"].long() - n_tree
    bits = _bits(s["masks"], n_tree)
    node = j[None, :] - base[:, None]                     # [B, n]
    at = torch.clamp(node, 0, T - 1)[:, None, :].expand(B, T, n)
    seen = (node[:, None, :] < 0) | (bits.gather(2, at) & (node[:, None, :] >= 0))
    seen = seen & held[:, None, :] & (torch.arange(T, device="cuda")[None, :, None] < n_tree[:, None, None])    # [B, T, n]
    seen = seen.permute(0, 2, 1)[..., None].expand(B, n, T, rep).reshape(B, 1, n, T * rep)

    qi, dq = _quant(s["q"].float())
    q = (qi.float() * dq.float()[..., None]).reshape(B, T, kvh, rep, D)
    q = q.permute(0, 2, 4, 1, 3).reshape(B, kvh, D, T * rep).contiguous()
    sc = torch.matmul(values(s["kc"]), q) * D ** -0.5     # [B, kvh, n, T rep]
    sc = torch.where(seen, sc, torch.full_like(sc[:1, :1, :1, :1], float("-inf")))
    top = sc.amax(dim=2, keepdim=True)
    p = torch.exp(sc - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(dim=2)[..., None]
    out = torch.matmul(p.permute(0, 1, 3, 2).contiguous(), values(s["vc"]))
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    out = out.reshape(B, kvh, T, rep, D).permute(0, 2, 1, 3, 4).reshape(B, T, kvh * rep, D)
    if s["gate"] is not None:
        out = out / (1.0 + torch.exp(-s["gate"].float()))
    return dict(out=out.to(s["q"].dtype).contiguous())


def _accept(s, case):
    """Masks and positions of the trees; the accepted path's rows moved to the front of the tree's, in every cache."""
    B, T, page = case["B"], case["T"], case["page"]
    cnt = _i32(s["cnt"]).long()
    t = torch.arange(T, device="cuda")
    par = s["parents"].long()
    live = t[None, :] < cnt[:, None]
    masks, depth, up = (torch.ones_like(par) << t[None, :]), torch.zeros_like(par), par
    for _ in range(T):                                    # one ancestor further up
        has = up >= 0
        if not bool(has.any()):
            break
        masks = torch.where(has, masks | (torch.ones_like(par) << torch.clamp(up, min=0)), masks)
        depth = depth + has.long()
        up = torch.where(has, par.gather(1, torch.clamp(up, min=0)), up)
    masks = torch.where(live, masks, torch.zeros_like(masks))
    pos = torch.where(live, s["n_past"].long()[:, None] + depth, torch.full_like(depth, -1))
    leaf = s["leaf"].long()
    path = masks.gather(1, torch.clamp(leaf, min=0)[:, None])
    on = (path >> t[None, :] & 1 != 0) & (leaf[:, None] >= 0) & live
    rank = torch.cumsum(on.long(), 1) - 1
    count = on.long().sum(1)
    base = s["n_kv"].long() - cnt
    b = torch.arange(B, device="cuda")[:, None].expand(B, T)

    def slot(token):
        return s["table"].long()[b, torch.div(token, page, rounding_mode="floor")] * page + token % page

    src, dst = slot(base[:, None] + t[None, :]), slot(torch.clamp(base[:, None] + rank, min=0))
    _put(s["caches"], src[on], dst[on])
    cu = torch.cat([torch.zeros_like(count[:1]), torch.cumsum(count, 0)])
    full = torch.zeros(B * T, dtype=torch.int64, device="cuda")
    full[(cu[:-1, None] + rank)[on]] = (b * T + t[None, :])[on]
    return dict(masks=masks, pos=pos.to(torch.int32), n_keep=(base + count).to(torch.int32), cu=cu.to(torch.int32),
                path=full.to(torch.int32), caches=s["caches"])


def _linear(s, case):
    """o_t = scale (e^{G_t} S^T q_t + sum over the nodes j on t's path of e^{G_t - G_j} (q_t . k_j) v_j), G_t = the sum of g
    along the path."""
    B, T, kh, vh, dk, dv = (case[x] for x in ("B", "T", "kh", "vh", "dk", "dv"))
    bits = _bits(s["masks"], s["n_tree"])

    def heads(x, rep):                                    # [B T, h, d] -> [B, vh, T, d] in f32
        return x.reshape(B, T, x.shape[1], -1).permute(0, 2, 1, 3).float().repeat_interleave(rep, dim=1).contiguous()

    q, k, v = heads(s["q"], vh // kh), heads(s["k"], vh // kh), heads(s["v"], 1)
    g = s["g"].double()
    g = g[None, :].expand(B * T, vh) if case["fixed"] else g
    g = g.reshape(B, T, vh).permute(0, 2, 1)
    G = torch.matmul(bits.double()[:, None], g[..., None])[..., 0]              # [B, vh, T]
    decay = torch.where(bits[:, None], G[..., :, None] - G[..., None, :],
                        torch.full((), -math.inf, dtype=torch.float64, device="cuda"))
    p = torch.matmul(q, k.transpose(-1, -2).contiguous()) * torch.exp(decay).float()
    out = torch.matmul(p, v) + torch.exp(G).float()[..., None] * torch.matmul(q, s["state"][s["slots"].long()])
    live = torch.arange(T, device="cuda")[None, :] < _i32(s["cnt"])[:, None]
    out = torch.where(live[:, None, :, None], out * dk ** -0.5, torch.zeros((), device="cuda"))
    return dict(out=out.permute(0, 2, 1, 3).reshape(B * T, vh, dv).to(s["v"].dtype).contiguous())


# ---------------------------------------------------------------- work and exact results

def work(case):
    kind, B = case["kind"], case["B"]
    if kind == "fork":
        _, src, tok = _fork_plan(case)
        page = case["page"]
        cols, rows = sum(n // page for n in tok), sum(n % page for n in tok)
        return dict(bytes=16.0 * B + 16 * cols + 2 * rows * case["row"] * case["caches"], flops=0.0)
    if kind == "release":
        lens, keep, common = _families(case)
        back = sum(_pages(n, case["page"]) - _pages(x, case["page"]) for n, x in zip(lens, keep))
        return dict(bytes=12.0 * B + 16 * back, flops=0.0)
    if kind == "compact":
        lens, pages = _pool(case), case["pages"]
        n_live = sum(_pages(n, case["page"]) for n in lens)
        moved = n_live * (pages - n_live) // pages        # on average: a live page lies behind with this chance
        return dict(bytes=8.0 * n_live + 16 * pages + 2.0 * moved * case["page"] * case["row"] * case["caches"], flops=0.0)
    par, cnt = _trees(case)
    T = case["T"]
    if kind == "accept":
        masks, _ = _masks(par)
        rows = sum(sum(1 for i, t in enumerate(j for j in range(T) if m[x] >> j & 1) if t != i)
                   for m, x in zip(masks, _leaves(case, par, cnt)) if x >= 0)
        return dict(bytes=20.0 * B * T + 2.0 * rows * case["row"] * case["caches"], flops=0.0)
    if kind == "tree":
        D, kvh, rep = case["D"], case["kvh"], case["rep"]
        lens, es = _ints(case["lo"], case["hi"], B, "len"), 4 if case["type"] == "f32" else 2
        n = sum(lens) + sum(cnt)
        pairs = sum((a + c) * c for a, c in zip(lens, cnt))
        return dict(bytes=float(n * kvh * D // 32 * 34 * 2 + 4 * n // case["page"] + 8 * B * T +
                                (sum(cnt) * (2 if case["gate"] else 1) + B * T) * kvh * rep * D * es),
                    flops=4.0 * pairs * kvh * rep * D)
    kh, vh, dk, dv = case["kh"], case["vh"], case["dk"], case["dv"]
    n, es = sum(cnt), 4 if case["type"] == "f32" else 2
    masks, _ = _masks(par)
    pairs = sum(bin(x & (1 << 64) - 1).count("1") for m, c in zip(masks, cnt) for x in m[:c])
    return dict(bytes=float(es * (n * (2 * kh * dk + vh * dv) + B * T * vh * dv) + (4 * vh if case["fixed"] else 4 * n * vh) +
                            4 * B * vh * dk * dv),
                flops=2.0 * n * vh * dk * dv + 2.0 * pairs * vh * (dk + dv))


def exact(case, seed):
    """The outputs in float64: attention one request and KV head at a time, linear attention by its recurrence from each
    node's parent."""
    kind = case["kind"]
    if kind in ("fork", "release", "compact", "accept"):
        return None                                       # whole numbers
    s = _inputs(case, seed)
    B, T = case["B"], case["T"]
    par, cnt = _trees(case)
    if kind == "tree":
        kvh, rep, D, page = (case[x] for x in ("kvh", "rep", "D", "page"))
        out = torch.zeros((B, T, kvh * rep, D), dtype=torch.float64, device="cuda")
        # the query's q8_0 image is part of the definition: its scale and its whole numbers in single precision
        x = s["q"].float().reshape(B, T, kvh, rep, D // 32, 32)
        amax = x.abs().amax(-1, keepdim=True)
        inv = (127.0 / amax.double()).float()
        qd = torch.round(x * inv).double() * (amax.double() / 127.0).float().half().double()
        qd = qd.reshape(B, T, kvh, rep, D)
        for b, n in enumerate(s["lens"]):
            base, c = n - cnt[b], cnt[b]
            key = torch.arange(n, device="cuda")
            rows = s["table"][b].long()[key // page] * page + key % page
            hide = torch.zeros((c, n), dtype=torch.bool, device="cuda")
            sees = [set() for _ in range(c)]
            for t in range(c):
                sees[t] = {t} | (sees[par[b][t]] if par[b][t] >= 0 else set())
            hide[:, base:] = torch.tensor([[j not in sees[t] for j in range(c)] for t in range(c)], device="cuda")
            for h in range(kvh):
                def side(cache):
                    seg = cache[rows].reshape(n, kvh, D // 32, 34)[:, h]
                    scale = seg[..., :2].contiguous().view(torch.float16).double()
                    return (seg[..., 2:].contiguous().view(torch.int8).double() * scale).reshape(n, D)
                kd, vd = side(s["kc"]), side(s["vc"])
                for r in range(rep):
                    w = (qd[b, :c, h, r] @ kd.t().contiguous() / math.sqrt(D)).masked_fill(hide, -math.inf)
                    out[b, :c, h * rep + r] = torch.softmax(w, dim=-1) @ vd
        if s["gate"] is not None:
            out = out * torch.sigmoid(s["gate"].double())
        return dict(out=out)
    kh, vh, dk, dv = case["kh"], case["vh"], case["dk"], case["dv"]
    out = torch.zeros((B, T, vh, dv), dtype=torch.float64, device="cuda")
    q, k = (s[x].double().reshape(B, T, kh, dk).repeat_interleave(vh // kh, dim=2) for x in ("q", "k"))
    v = s["v"].double().reshape(B, T, vh, dv)
    g = s["g"].double().expand(B * T, vh).reshape(B, T, vh)
    start = s["state"][s["slots"].long()].double()
    for b in range(B):
        states = []
        for t in range(cnt[b]):
            before = states[par[b][t]] if par[b][t] >= 0 else start[b]
            states.append(before * torch.exp(g[b, t])[:, None, None] + k[b, t][:, :, None] * v[b, t][:, None, :])
            out[b, t] = (q[b, t][:, None, :] @ states[t])[:, 0] / math.sqrt(dk)
    return dict(out=out.reshape(B * T, vh, dv))
