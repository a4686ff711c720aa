"""CPU checks of the rotary positions: the record's layout, frequency schedules, and every
refusal.  A refused call returns before any HIP call."""
from __future__ import annotations

import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LENGTH, SHAPE, STRIDE, OVERFLOW, NULL, ALIGNMENT = -2, -3, -4, -16, -19, -21
P = 0x10000


@pytest.fixture(scope="module")
def L():
    from fe2o3_amd import _lib
    return _lib.lib()


def _rows(**over):
    from fe2o3_amd import _lib
    a = dict(x=P, x_len=10 * 3 * 64, out=P, out_len=10 * 3 * 64, token_stride=192, head_stride=64,
             out_token_stride=192, out_head_stride=64, heads=3, reserved=0)
    a.update(over)
    return _lib.Fe2o3RotaryRowsV1(*a.values())


def _call(L, q=None, k=None, **over):
    a = dict(positions=P, positions_len=10, freq=P, freq_len=24, dtype=1, tokens=10, head_dim=64,
             rotary_dim=48, flags=0, scale=1.0)
    a.update(over)
    q = _rows() if q is None else q
    return L.fe2o3_rotary(C.byref(q) if q != 0 else None, None if k is None else C.byref(k),
                          *a.values(), None)


def test_record_layout(tmp_path):
    from fe2o3_amd import _lib
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    rec = _lib.Fe2o3RotaryRowsV1
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "fe2o3_mi355x.h"',
             "int main(void) {", 'printf("%zu\\n", sizeof(Fe2o3RotaryRowsV1));']
    expect = [str(C.sizeof(rec))]
    for field, _ in rec._fields_:
        lines.append(f'printf("%zu\\n", offsetof(Fe2o3RotaryRowsV1, {field}));')
        expect.append(str(getattr(rec, field).offset))
    (tmp_path / "r.c").write_text("\n".join(lines + ["return 0;", "}"]))
    subprocess.run([cc, "-std=c11", "-I", os.path.join(ROOT, "include"), str(tmp_path / "r.c"),
                    "-o", str(tmp_path / "r")], check=True)
    got = subprocess.run([str(tmp_path / "r")], capture_output=True, text=True, check=True).stdout
    assert got.split("\n")[:-1] == expect


@pytest.mark.parametrize("over,want", [
    (dict(dtype=2), SHAPE), (dict(flags=4), SHAPE), (dict(rotary_dim=0, freq_len=0), SHAPE),
    (dict(rotary_dim=47), SHAPE), (dict(rotary_dim=66, freq_len=33), SHAPE),
    (dict(head_dim=5000, rotary_dim=4098, freq_len=2049), SHAPE),
    (dict(scale=float("nan")), SHAPE), (dict(scale=float("inf")), SHAPE),
    (dict(tokens=1 << 31, positions_len=1 << 31), SHAPE),
    (dict(head_dim=1 << 30), SHAPE),
    (dict(positions_len=9), LENGTH), (dict(freq_len=23), LENGTH), (dict(freq_len=48), LENGTH),
    (dict(positions=None), NULL), (dict(freq=None), NULL), (dict(positions=P + 2), ALIGNMENT),
    (dict(freq=P + 4), ALIGNMENT),
])
def test_refusals(L, over, want):
    assert _call(L, **over) == want
    assert _call(L, k=_rows(heads=1), **over) == want


ROWS = [
    (dict(heads=0), SHAPE), (dict(head_stride=63), STRIDE), (dict(token_stride=191), STRIDE),
    (dict(out_head_stride=63), STRIDE), (dict(out_token_stride=0), STRIDE),
    (dict(token_stride=1 << 62), OVERFLOW), (dict(out_token_stride=1 << 60), OVERFLOW),
    (dict(x_len=1919), LENGTH), (dict(out_len=1919), LENGTH), (dict(x=None), NULL),
    (dict(out=None), NULL), (dict(x=P + 1), ALIGNMENT), (dict(out=P + 1), ALIGNMENT),
]


@pytest.mark.parametrize("over,want", ROWS)
def test_rows_refused(L, over, want):
    assert _call(L, q=_rows(**over)) == want
    assert _call(L, k=_rows(**over)) == want
    assert _call(L, q=0) == NULL


def test_f32_alignment_and_no_tokens(L):
    assert _call(L, q=_rows(x=P + 2), dtype=0) == ALIGNMENT
    none = _rows(x=None, x_len=0, out=None, out_len=0)
    assert _call(L, q=none, positions=None, positions_len=0, freq=None, tokens=0) == 0


def test_injected_failure(L, monkeypatch):
    monkeypatch.setenv("FE2O3_FAULT_POINT", "fe2o3_rotary")
    assert _call(L) == -23


def test_frequencies():
    from fe2o3_amd import kernels
    f, m = kernels.rotary_frequencies(8, 10000.0)
    assert m == 1.0 and np.allclose(f, [1, 0.1, 0.01, 0.001], rtol=1e-15)
    g, m = kernels.rotary_frequencies(8, 10000.0, factor=4.0)
    assert m == 1.0 and np.array_equal(g, f / 4)
    g, m = kernels.rotary_frequencies(8, 10000.0, factor=4.0, schedule="base")
    assert m == 1.0 and g[0] == 1.0 and np.isclose(g[-1], f[-1] / 4, rtol=1e-14)
    g, m = kernels.rotary_frequencies(64, factor=8.0, schedule="by_turns")
    f = kernels.rotary_frequencies(64)[0]
    turns = 4096 * f / (2 * np.pi)
    assert np.allclose(g[turns >= 32], f[turns >= 32], rtol=1e-15)
    assert np.allclose(g[turns <= 1], f[turns <= 1] / 8, rtol=1e-15)
    assert np.all(np.diff(g) < 0) and np.all(g <= f) and np.all(g >= f / 8)
    assert np.isclose(m, 0.1 * np.log(8.0) + 1.0)
    assert kernels.rotary_frequencies(2, schedule="base", factor=2.0)[0].tolist() == [1.0]
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, base=-1.0),
                dict(rotary_dim=8, factor=0.0), dict(rotary_dim=8, schedule="none"),
                dict(rotary_dim=8, slow_turns=32.0)):
        with pytest.raises(ValueError):
            kernels.rotary_frequencies(**bad)
