"""ISA checks of the kernels of rotary positions and 8-bit paged caches (CPU: hipcc cross-compiles,
nothing runs): those of test_isa.py and test_paged_isa.py, and that no packed-fp32 instruction is made."""
import os
import subprocess

import pytest

from test_isa import CSRC, FLAGS, _hipcc, lds_read_hazards, mfma_result_hazards
from test_paged_isa import split_spills

SOURCES = ["rope.hip", "paged8.hip"]


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    hipcc = _hipcc()
    if not hipcc:
        pytest.skip("hipcc not available")
    d = tmp_path_factory.mktemp("isa")
    out = {}
    for src in SOURCES:
        path = str(d / (src + ".s"))
        subprocess.run([hipcc, *FLAGS, os.path.join(CSRC, src), "-o", path], check=True, capture_output=True)
        out[src] = open(path).read()
    return out


@pytest.mark.parametrize("src", SOURCES)
def test_waits_spills_and_packed_arithmetic(asm, src):
    assert lds_read_hazards(asm[src]) == []
    assert mfma_result_hazards(asm[src]) == []
    assert split_spills(asm[src]) == []
    for name in ("add", "mul", "fma"):
        assert f"v_pk_{name}_f32" not in asm[src]
