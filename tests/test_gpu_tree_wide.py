"""The attention tests of test_gpu_tree with page tables so wide that the calls take the kernel of 128 or 256 query rows a workgroup."""
import pytest
import torch

import test_gpu_tree as G

pytestmark = pytest.mark.gpu


class WideCase(G.TreeCase):
    def __init__(self, lens, D, kvh, rep, T, page, extra_cols=1, **kw):
        tiles = -(-48 * 512 // (len(lens) * -(-T * rep // 16) * kvh)) + 1       # of 32 keys a request: 48 for each of 512 workgroups
        super().__init__(lens, D, kvh, rep, T, page, extra_cols=max(extra_cols, -(-tiles * 32 // page)), **kw)


@pytest.fixture(autouse=True)
def wide(monkeypatch):
    monkeypatch.setattr(G, "TreeCase", WideCase)


@pytest.mark.parametrize("D,kvh,rep,T,page", [
    (256, 2, 8, 9, 7), (256, 1, 3, 22, 1), (256, 2, 8, 16, 32), (256, 2, 8, 17, 100), (256, 1, 8, 32, 16), (256, 2, 8, 33, 32),
    (256, 1, 8, 64, 16), (256, 3, 12, 64, 5), (128, 8, 4, 24, 16), (128, 2, 7, 37, 5), (128, 1, 2, 64, 16), (128, 2, 8, 64, 33),
    (64, 1, 3, 50, 256), (64, 2, 8, 31, 3), (64, 3, 5, 17, 9), (64, 1, 8, 64, 16)])
def test_shapes(gpu, D, kvh, rep, T, page):
    G.test_attention_shapes(gpu, D, kvh, rep, T, page)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gate", [False, True])
def test_types_and_gate(gpu, dtype, gate):
    G.test_attention_types_and_gate(gpu, dtype, gate)


@pytest.mark.parametrize("variant", [0, 1])
def test_rounding_variants(gpu, variant):
    G.test_attention_rounding_variants(gpu, variant)


@pytest.mark.parametrize("lens,D,kvh,rep,T", [
    ([6001], 256, 2, 8, 20), ([3000, 40, 5000, 3], 256, 2, 4, 24), ([9000, 1], 128, 1, 8, 32), ([1500] * 7, 256, 2, 12, 8),
    ([20000], 64, 1, 4, 40), ([2500, 2500], 256, 2, 8, 48)])
def test_long_and_split(gpu, lens, D, kvh, rep, T):
    G.test_attention_long_and_split(gpu, lens, D, kvh, rep, T)


def test_many_requests(gpu):
    G.test_attention_many_requests(gpu)


def test_any_masks(gpu):
    G.test_attention_any_masks(gpu)


def test_large_scores_and_small_values(gpu):
    G.test_attention_large_scores_and_small_values(gpu)


@pytest.mark.parametrize("kd,vd", [(0x7E, 0x7E), (0x7C, 0x7C), (0x7C, 0x7E), (0x7B, 0x7B)])
def test_unseen_nodes_stay_out(gpu, kd, vd):
    G.test_attention_unseen_nodes_stay_out(gpu, 40, kd, vd)


def test_bad_pages_and_lengths(gpu):
    G.test_attention_bad_pages_and_lengths(gpu)


def test_strides_and_workspaces(gpu):
    G.test_attention_strides_and_workspaces(gpu)


def test_captured(gpu):
    G.test_attention_captured(gpu)


def test_two_streams_at_once(gpu):
    """Calls on two streams with a workspace each, several in flight: the bits of calls one after another."""
    G.say("tree attention: two streams")
    K = gpu
    cases = [WideCase([900, 40, 1300], 256, 2, 8, 24, 16, n_tree=[24, 3, 20], seed=31), WideCase([1500, 7], 128, 2, 6, 32, 16, seed=32)]
    want = [c.on_gpu(K) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    outs = []
    for c, st in zip(cases, streams):
        nb = (34, c.kd.stride(0), c.D // 32 * 34, c.n_rows * c.kd.stride(0))
        kv, vv = (K.tensor(x.data_ptr(), K.TYPE_Q8_0, (c.D, c.n_rows, c.kvh, 1), nb) for x in (c.kd, c.vd))
        q, td, nd, m = c.q.cuda(), G.dev(c.table), G.i32(c.lens), G.words(c.m)
        nt = None if c.n_tree is None else G.i32(c.n_tree)
        o = torch.zeros((8,) + tuple(want[len(outs)].shape), device="cuda")
        qv = K.q_view(q)
        w = G.ws_of(K.fattn_workspace_size_paged_tree(qv, kv, vv, td, c.page))
        outs.append((o, (q, td, nd, m, nt, w, kv, vv, qv, c)))
    torch.cuda.synchronize()
    for i in range(8):
        for (o, (q, td, nd, m, nt, w, kv, vv, qv, c)), st in zip(outs, streams):
            K.flash_attn_ext_paged_tree(qv, kv, vv, td, c.page, nd, m, c.scale, K.out_view(o[i]), n_tree=nt, ws=w, stream=st)
    torch.cuda.synchronize()
    for (o, _), x in zip(outs, want):
        for i in range(8):
            assert torch.equal(o[i], x)
