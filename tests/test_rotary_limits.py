"""CPU check of the largest tokens that rotary positions take: the refusal is where the header's
macro says, compiled as a C program's.  A size below it fails on the length given."""
from __future__ import annotations

import math
import os
import shutil
import subprocess

import numpy as np
import pytest

from test_rotary_host import LENGTH, ROOT, SHAPE, _call, _rows

SIZES = [(2, 2), (3, 2), (16, 16), (16, 2), (17, 16), (18, 18), (64, 48), (64, 64), (128, 128),
         (128, 36), (256, 64), (4096, 4096), (1 << 20, 4096)]  # head_dim, rotary_dim


@pytest.fixture(scope="module")
def pieces(tmp_path_factory):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    at = tmp_path_factory.mktemp("rotary")
    lines = ['#include <stdio.h>', '#include "fe2o3_mi355x.h"', "int main(void) {"]
    lines += [f'printf("%llu\\n", (unsigned long long)FE2O3_ROTARY_PIECES(1u, {d}u, {r}u));'
              for d, r in SIZES]
    (at / "p.c").write_text("\n".join(lines + ["return 0;", "}"]))
    subprocess.run([cc, "-std=c11", "-I", os.path.join(ROOT, "include"), str(at / "p.c"), "-o",
                    str(at / "p")], check=True)
    got = subprocess.run([str(at / "p")], capture_output=True, text=True, check=True).stdout
    return dict(zip(SIZES, map(int, got.split())))


@pytest.mark.parametrize("head_dim,rotary_dim", SIZES)
def test_largest_token(pieces, head_dim, rotary_dim):
    from fe2o3_amd import _lib
    each = pieces[head_dim, rotary_dim]
    assert each == -(-rotary_dim // 16) + -(-(head_dim - rotary_dim) // 16)
    most = ((1 << 22) - 1) // each  # heads
    size = dict(head_dim=head_dim, rotary_dim=rotary_dim, freq_len=rotary_dim // 2 + 1)
    lib = _lib.lib()
    for heads, want in [(most, LENGTH), (most + 1, SHAPE), (0xFFFFFFFF, SHAPE)]:
        assert _call(lib, q=_rows(heads=heads), **size) == want
        if heads > 1:  # of both arrays together
            assert _call(lib, q=_rows(heads=heads - 1), k=_rows(heads=1), **size) == want
    assert _call(lib, q=_rows(heads=0xFFFFFFFF), k=_rows(heads=0xFFFFFFFF), **size) == SHAPE
    assert _call(lib, q=_rows(heads=0xFFFFFFFF), k=_rows(heads=0xFFFFFFFF), head_dim=0xFFFFFFFF,
                 rotary_dim=2, freq_len=2) == SHAPE


@pytest.mark.parametrize("slow,fast", [(1.0, 32.0), (0.0, 4.0), (2.0, 64.0)])
def test_a_line_in_turns(slow, fast):
    """Between slow_turns and fast_turns a pair's speed is a straight line in its turns, not in
    its number."""
    from fe2o3_amd import kernels
    plain = kernels.rotary_frequencies(128)[0]
    got = kernels.rotary_frequencies(128, factor=8.0, schedule="by_turns", slow_turns=slow,
                                     fast_turns=fast)[0]
    turns = 4096 * plain / (2 * math.pi)
    inner = (turns > slow) & (turns < fast)
    assert inner.sum() > 3
    share = (got - plain / 8) / (plain - plain / 8)  # of the plain speed
    assert np.allclose(share[inner], (turns[inner] - slow) / (fast - slow), rtol=1e-12, atol=1e-12)
    number = np.arange(64)[inner]
    along = (number[-1] - number) / (number[-1] - number[0])
    assert np.abs(share[inner] - along * (share[inner][0] - share[inner][-1])
                  - share[inner][-1]).max() > 0.05
