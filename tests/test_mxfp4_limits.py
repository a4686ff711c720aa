"""CPU check of a bound between two files: the direct kernel (gemm_direct.hpp) has no form for
any K of 4-bit operands, so the packed layout's largest number of panels (mxfp4.hpp) must fit
the forms it has.  The product's source compiles with that number and not with one past the
bound."""
from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LAST = (2 ** 32 - 1) // (64 * 128)  # panels whose 64 rows of codes stay below 2^32 bytes


@pytest.mark.parametrize("panels,compiles", [(None, True), (LAST, True), (LAST + 1, False)])
def test_panels_fit_the_direct_forms(tmp_path, panels, compiles):
    hipcc = "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    for part in ("include", os.path.join("fe2o3_amd", "csrc")):
        shutil.copytree(os.path.join(ROOT, part), tmp_path / part,
                        ignore=shutil.ignore_patterns("*.o", "*.so"))
    csrc = tmp_path / "fe2o3_amd" / "csrc"
    header = csrc / "mxfp4.hpp"
    text, found = re.subn(r"kMaxPanels = \d+;", lambda m: f"kMaxPanels = {panels};" if panels
                          else m.group(), header.read_text())
    assert found == 1
    header.write_text(text)
    r = subprocess.run([hipcc, "--offload-arch=gfx950", "-std=c++17", "--cuda-host-only",
                        "-fsyntax-only", "-I" + str(csrc / "_build"),
                        str(csrc / "gemm_mxfp4.hip")], capture_output=True, text=True)
    assert (r.returncode == 0) == compiles, r.stderr[-2000:]
    assert compiles or "a form that this type lacks" in r.stderr
