"""The attention of a tree with bf16 queries: F32 softmax and accumulation and one rounding, as with the other types."""
import numpy as np
import pytest
import torch

from gpu_util import say
from test_gpu_paged import HALF_STEP
from test_gpu_tree import TreeCase
from test_gpu_tree_wide import WideCase

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("make", [TreeCase, WideCase])
@pytest.mark.parametrize("D,lens,T,rep,n_tree", [
    (256, [70, 30, 97, 40], 30, 6, [30, 9, 1, 22]), (128, [70, 30, 97, 40], 24, 4, [24, 9, 2, 0]), (64, [70, 24, 97, 40], 24, 3, None),
    (256, [2500], 24, 8, [20]), (256, [1200, 40, 900], 13, 7, None)])
def test_one_rounding(gpu, make, D, lens, T, rep, n_tree):
    """Within the tolerance of an F32 implementation (tree_ref.attention, two terms) and half a bf16 step of the value; few keys and
    peaked weights, so that many values are small beside the sum of their terms."""
    say(f"tree attention bf16: {make.__name__} D={D} lens={lens} T={T} rep={rep}")
    c = make(lens, D, 2, rep, T, 16, n_tree=n_tree, seed=D + T, dtype=torch.bfloat16, q_scale=3.0)
    o = c.on_gpu(gpu).float().cpu().numpy().astype(np.float64)
    c.dtype = torch.float32                                # (the queries are bf16 values still)
    ref, tol = c.reference()
    tol += HALF_STEP[torch.bfloat16] * (np.abs(ref) + tol)
    assert np.isfinite(o).all() and (np.abs(o - ref) <= tol).all(), np.max(np.abs(o - ref) / np.maximum(tol, 1e-300))
    # and next to the same queries as F32, both within the tolerance of F32 of the value: one rounding of what those give
    c.q = c.q.float()
    f = c.on_gpu(gpu).cpu().numpy().astype(np.float64)
    _, tol = c.reference()
    near = np.abs(f) + 2 * tol
    assert (np.abs(o - f) <= 2 * tol + HALF_STEP[torch.bfloat16] * near).all()
