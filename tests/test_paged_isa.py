"""ISA checks of the paged kernels (CPU: hipcc cross-compiles, nothing runs): those of
test_isa.py, and one of the compiler's spills.

Where a kernel holds all its registers and spills four of them as one tuple, the compiler can
put some of the four into accumulation registers and the rest into scratch memory, and then
leave one of them out when it reads the tuple back: the f32 queries of one row in 32 once came
back with another row's cosines (head_dim 256, bf16).  So no kernel may spill to both: the
compiler marks the first kind "Reload Reuse".
"""
import os
import subprocess

import pytest

from test_isa import CSRC, FLAGS, _hipcc, lds_read_hazards, mfma_result_hazards

SOURCES = ["pages.hip", "paged.hip"]


def split_spills(text):
    """Kernels that spill registers to accumulation registers and to scratch memory."""
    bad = []
    for body in text.split(".Lfunc_end")[:-1]:
        if "Reload Reuse" in body and "scratch_" in body:
            bad.append(body[:200])
    return bad


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    hipcc = _hipcc()
    if not hipcc:
        pytest.skip("hipcc not available")
    d = tmp_path_factory.mktemp("isa")
    out = {}
    for src in SOURCES:
        path = str(d / (src + ".s"))
        subprocess.run([hipcc, *FLAGS, os.path.join(CSRC, src), "-o", path], check=True,
                       capture_output=True)
        out[src] = open(path).read()
    return out


@pytest.mark.parametrize("src", SOURCES)
def test_lds_reads_waited_before_use(asm, src):
    assert lds_read_hazards(asm[src]) == []


@pytest.mark.parametrize("src", SOURCES)
def test_mfma_results_not_read_early(asm, src):
    assert mfma_result_hazards(asm[src]) == []


@pytest.mark.parametrize("src", SOURCES)
def test_no_kernel_spills_to_two_places(asm, src):
    assert split_spills(asm[src]) == []


def test_the_checker_catches_a_planted_spill():
    one = "k:\n v_accvgpr_write_b32 a195, v19           ;  Reload Reuse\n"
    two = " scratch_store_dword off, v12, off       ; 4-byte Folded Spill\n"
    assert len(split_spills(one + two + ".Lfunc_end0:\n")) == 1
    assert split_spills(one + ".Lfunc_end0:\n" + two + ".Lfunc_end1:\n") == []
