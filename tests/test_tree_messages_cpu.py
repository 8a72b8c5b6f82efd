"""What calls of trees and cache lists say when they refuse (CPU)."""
import pytest
import torch

import qwfn_kv as K
from test_paged_cpu import paged_views, refused
from test_tree_cpu import r, tree


def test_small_workspaces_name_their_size_function():
    q, k, o = paged_views(T=64)
    need = K.load().qwfn_fattn_workspace_size_paged_tree(r(q), r(k), r(k), 40, 16)
    refused(tree(q, k, o, ws_bytes=need - 1), K.ENOMEM, "qwfn_fattn_workspace_size_paged_tree")
    q, k, o = paged_views()
    rc = K.load().qwfn_flash_attn_ext_q8_0_paged(r(q), r(k), r(k), 1 << 40, 40, 40, 16, 1 << 40, 0.0625, None, r(o), 1, 3 << 40, 64, None)
    refused(rc, K.ENOMEM, "qwfn_fattn_workspace_size_paged")
    assert "paged_tree" not in K.load().qwfn_last_error().decode()


def test_cache_lists_without_rows():
    for bad in (torch.empty((0, 34), dtype=torch.uint8), torch.zeros(34, dtype=torch.uint8), torch.zeros((5, 68), dtype=torch.uint8)[:, ::2]):
        with pytest.raises(ValueError, match="contiguous rows"):
            K.cache_list([torch.zeros((5, 34), dtype=torch.uint8), bad])
