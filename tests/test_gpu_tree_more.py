"""Linear attention of a tree in a captured graph, every type, and releases of more pages a request than a wave has lanes."""
import numpy as np
import pytest
import torch

import tree_ref as R
from gpu_util import dev, host, say
from test_gpu_tree import i32, random_parents, words

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,dk,dv", [(5, 64, 32), (32, 128, 128), (64, 256, 192)])
def test_linear_captured(gpu, dtype, T, dk, dv):
    """Replays with new inputs, eager calls between: the bits of the eager call."""
    say(f"linear attention of a tree, captured: {dtype} T={T} dk={dk} dv={dv}")
    K, B, kh, vh = gpu, 3, 2, 4
    rng = np.random.default_rng(T)
    draw = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()  # noqa: E731
    q, k, v = draw(B * T, kh, dk).to(dtype), draw(B * T, kh, dk).to(dtype), draw(B * T, vh, dv).to(dtype)
    g, state, nt = -draw(B * T, vh).abs() * 0.1, draw(B + 1, vh, dk, dv), i32([T, T // 2, 0])
    m, slots = words(R.masks(random_parents(rng, B, T))[0]), i32([2, 0, 3])
    out, ref = torch.zeros_like(v), torch.zeros_like(v)

    def call(o):
        K.linear_attn_tree(q, k, v, g, m, state, o, n_tree=nt, slots=slots)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(out)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for turn in range(4):
        q.copy_(draw(*q.shape).to(dtype))
        state.copy_(draw(*state.shape))
        nt.copy_(i32(rng.integers(0, T + 1, B)))
        graph.replay()
        call(ref)
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and bool(torch.isfinite(ref.float()).all())


@pytest.mark.parametrize("cols", [63, 64, 65, 511, 512, 513, 1100])
def test_release_of_long_requests(gpu, cols):
    """Requests of `cols` pages, each page held by one, two or three of them; entries outside the pool between."""
    say(f"release: requests of {cols} pages")
    K, page = gpu, 2
    rng = np.random.default_rng(cols)
    B, pages = 4, 3 * cols + 40
    ids = rng.permutation(pages)[:2 * cols + 1]
    table = np.full((B, cols + 2), -7, np.int32)
    table[0, :cols], table[1, :cols] = ids[:cols], ids[:cols]                # the same pages
    table[2, :cols] = np.concatenate([ids[:cols // 2], ids[cols:cols + cols - cols // 2]])
    table[3, :1] = ids[2 * cols]
    n_kv = np.array([cols * page, cols * page, cols * page - 1, 1], np.int32)
    holders = np.bincount(np.concatenate([table[b, :-(-n_kv[b] // page)] for b in range(B)]), minlength=pages)
    shared = np.maximum(holders - 1, 0).astype(np.int32)
    on_stack = np.array([p for p in range(pages) if holders[p] == 0], np.int32)
    free = np.full(pages, -1, np.int32)
    free[:len(on_stack)] = on_stack
    for keep in ([0, n_kv[1], 0, 1], [0, 0, 0, 0], [page, 0, n_kv[2], 0]):
        for torn in (False, True):
            tab = table.copy()
            if torn:
                tab[0, cols // 3], tab[0, cols - 1] = pages, -1
            f, n = dev(free.copy()), i32([len(on_stack)])
            kv, sh, tb = dev(n_kv.copy()), dev(shared.copy()), dev(tab)
            ws = torch.full((K.paged_release_workspace_size(B, pages),), 255, dtype=torch.uint8, device="cuda")
            K.device_status()
            K.paged_release(i32(keep), kv, page, tb, sh, f, n, n, kv, sh, ws=ws)
            flags = K.device_status()
            rf, rn, rkv, rsh, bad = R.release(np.array(keep), n_kv, page, tab, shared, free, len(on_stack), pages)
            assert np.array_equal(host(f)[:rn], rf[:rn]) and host(n)[0] == rn
            assert np.array_equal(host(kv), rkv) and np.array_equal(host(sh), rsh)
            assert flags == (K.DEVERR_PAGES if bad else 0)
