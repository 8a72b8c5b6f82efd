"""The checks of test_asm_lds_dma on the attention of trees of many query rows (CPU)."""
import os
import subprocess

import pytest

from test_asm_hazards import HIPCC, PKG, ROOT
from test_asm_lds_dma import test_m0_and_scc, test_m0_is_read_a_wait_state_after_its_write, test_no_packed_f32  # noqa: F401


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    out = str(tmp_path_factory.mktemp("asm") / "paged_tree.s")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "-I", os.path.join(PKG, "csrc"), "-I", os.path.join(ROOT, "include"),
                    "--cuda-device-only", "-S", os.path.join(PKG, "csrc", "paged_tree.hip"), "-o", out],
                   check=True, capture_output=True, timeout=600)
    return open(out).read().split("\n")
