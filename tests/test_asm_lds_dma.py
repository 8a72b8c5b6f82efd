"""The checks of test_asm_hazards on the paged and the linear attention, whose LDS DMA sets M0 in inline asm too (CPU)."""
import os
import subprocess

import pytest

from test_asm_hazards import HIPCC, PKG, ROOT, _op, asm_blocks, scc_carried_across


@pytest.fixture(scope="module", params=["paged_attn", "linear_attn"])
def asm(request, tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    out = str(tmp_path_factory.mktemp("asm") / (request.param + ".s"))
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "-I", os.path.join(PKG, "csrc"), "-I", os.path.join(ROOT, "include"),
                    "--cuda-device-only", "-S", os.path.join(PKG, "csrc", request.param + ".hip"), "-o", out],
                   check=True, capture_output=True, timeout=600)
    return open(out).read().split("\n")


def dma_blocks(lines):
    """The instructions of each inline-asm block that sets M0."""
    blocks = [[l.split(";")[0].strip() for l in lines[a + 1:b] if _op(l)] for a, b in asm_blocks(lines)]
    return [b for b in blocks if any("m0" in l for l in b)]


def short_of_a_wait(blocks):
    """Blocks whose LDS DMA does not stand one instruction behind the write of M0."""
    return [b for b in blocks if len(b) != 3 or not b[0].startswith("s_mov_b32 m0,") or "_load_lds_" not in b[2]]


def test_m0_and_scc(asm):
    assert scc_carried_across(asm, asm_blocks(asm)) == []
    inside = set()
    for a, b in asm_blocks(asm):
        inside.update(range(a, b + 1))
    assert [l.strip() for i, l in enumerate(asm) if i not in inside and _op(l) and "m0" in l.split(";")[0]] == []


def test_m0_is_read_a_wait_state_after_its_write(asm):
    blocks = dma_blocks(asm)
    assert len(blocks) > 20 and short_of_a_wait(blocks) == []


def test_no_packed_f32(asm):
    assert [l.strip() for l in asm if _op(l) in ("v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32")] == []


def test_the_scan_finds_a_missing_wait():
    lines = ["\t;;#ASMSTART", "\ts_mov_b32 m0, s3", "\tglobal_load_lds_dwordx4 v1, s[4:5]", "\t;;#ASMEND"]
    assert len(short_of_a_wait(dma_blocks(lines))) == 1
    lines.insert(2, "\ts_nop 0")
    assert short_of_a_wait(dma_blocks(lines)) == []
