"""Whether a paged kernel spills vector registers to accumulation registers (CPU: nothing runs).

test_paged_isa.py looks for kernels that spill to both places by the compiler's comments.  This says it
without them: the code is the same, instruction for instruction, with such spills forbidden.
"""
import os
import re
import subprocess

import pytest

from test_isa import CSRC, FLAGS, _hipcc

FORBID = ["-mllvm", "-amdgpu-spill-vgpr-to-agpr=false"]


def instructions(path):
    """The kernels' lines without comments, and the spill counts of their descriptions."""
    text = open(path).read()
    code = [re.sub(r"\s*;.*", "", line) for line in text.splitlines()]
    return ([line for line in code if line.startswith("\t") and not line.startswith("\t.")],
            re.findall(r"\.vgpr_spill_count: *(\d+)", text))


@pytest.mark.parametrize("src", ["pages.hip", "paged.hip"])
def test_no_register_is_spilled_to_an_accumulation_register(tmp_path, src):
    hipcc = _hipcc()
    if not hipcc:
        pytest.skip("hipcc not available")
    runs = [subprocess.Popen([hipcc, *FLAGS, *more, os.path.join(CSRC, src), "-o", str(tmp_path / f"{i}.s")],
                             stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
            for i, more in enumerate(([], FORBID))]
    assert [r.wait() for r in runs] == [0, 0]
    (a, spills), (b, forbidden) = (instructions(tmp_path / f"{i}.s") for i in range(2))
    assert len(a) > 1000 and spills and spills == forbidden
    assert a == b
