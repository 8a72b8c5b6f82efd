"""Rows that are 0 because their query sees nothing, or is no node of its tree: what their gate holds does not matter, whichever
kernel takes the call and wherever its runs are cut."""
import numpy as np
import pytest
import torch

from gpu_util import say
from test_gpu_paged import Case
from test_gpu_tree import TreeCase
from test_gpu_tree_wide import WideCase

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def check(K, c, least):
    """The bits of a call with finite gates where the gates of the rows that are 0 are NaN or infinite; at least `least` such rows."""
    ref, _ = c.reference()
    zero = (ref == 0).all((2, 3))
    assert int(zero.sum()) >= least and not zero.all()
    want = c.check(K, gate=True)
    assert (want[zero] == 0).all()
    for x in (float("nan"), float("inf"), float("-inf")):
        c.gate[torch.from_numpy(zero)] = x
        assert np.array_equal(c.on_gpu(K, gate=True).float().cpu().numpy(), want)


def blind(c, *nodes):
    """Masks without a bit for nodes of requests that are all tree."""
    for b, t in nodes:
        assert c.lens[b] == c.nt[b]
        c.m[b, t] = 0
    return c


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("make", [TreeCase, WideCase])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_tree_rows_without_a_node(gpu, D, make, dtype):
    """Requests inside a run, without a node, without a key; nodes that see nothing."""
    say(f"gates of rows of 0: {make.__name__} D={D} {dtype}")
    for T, rep in ((4, 4), (24, 6)):
        c = make([70, T, 333, 0, 97], D, 2, rep, T, 16, n_tree=[T - 1, T, 2, 0, 0], seed=D + T, dtype=dtype)
        check(gpu, blind(c, (1, 0), (1, T - 1)), 1 + 2 + (T - 2) + 2 * T)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("make", [TreeCase, WideCase])
def test_tree_rows_of_split_requests(gpu, make, dtype):
    """Requests of many runs (their parts joined by a second launch), and many of a few tiles each, some of them cut."""
    say(f"gates of rows of 0 in parts: {make.__name__} {dtype}")
    check(gpu, make([5000], 256, 2, 8, 12, 64, n_tree=[7], seed=1, dtype=dtype), 5)
    check(gpu, make([2000, 30, 3000], 128, 2, 6, 20, 64, n_tree=[20, 3, 11], seed=2, dtype=dtype), 17 + 9)
    c = make([64] * 40, 64, 1, 2, 64, 16, n_tree=[64] * 40, seed=3, dtype=dtype)
    check(gpu, blind(c, *[(b, b) for b in range(40)]), 40)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_before_the_first_token(gpu, dtype):
    """The attention without a tree: queries before a request's first token, requests of length 0, cut and uncut."""
    say(f"gates of rows of 0: no tree, {dtype}")
    for D in (64, 128, 256):
        check(gpu, Case([3, 1, 0, 700], D, 2, 4, 4, 16, seed=D, dtype=dtype), 1 + 3 + 4)
    check(gpu, Case([60] * 40, 64, 1, 1, 64, 16, seed=4, dtype=dtype), 160)
