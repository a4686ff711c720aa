"""CPU checks of the microscaled 4-bit entry points: sizes, every refusal, and the format's
definition in numpy against the values written out.  A refused call returns before any
HIP call, so the pointers need only not be NULL; no call here passes validation."""
from __future__ import annotations

import os
import shutil
import subprocess

import numpy as np
import pytest

import mxfp4_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LENGTH, SHAPE, STRIDE, OVERFLOW, NULL, ALIGNMENT = -2, -3, -4, -16, -19, -21
P = 0x10000  # an aligned address that nothing reads


@pytest.fixture(scope="module")
def L():
    from fe2o3_amd import _lib
    return _lib.lib()


def test_sizes_match_the_header(tmp_path):
    from fe2o3_amd import kernels
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines, expect = ['#include <stdio.h>', '#include "fe2o3_mi355x.h"', "int main(void) {"], []
    for rows, cols in [(1, 1), (16, 256), (17, 257), (0, 5), (5, 0), (4096, 14336),
                       (0xFFFFFFFF, 16776960)]:
        codes, scales = kernels.mxfp4_shapes(rows, cols)
        lines.append(f'printf("%llu %llu\\n", (unsigned long long)FE2O3_MXFP4_CODE_BYTES({rows}u, '
                     f'{cols}u), (unsigned long long)FE2O3_MXFP4_SCALE_BYTES({rows}u, {cols}u));')
        expect.append(f"{codes[0] * codes[1]} {scales[0] * scales[1] * scales[2]}")
    (tmp_path / "s.c").write_text("\n".join(lines + ["return 0;", "}"]))
    subprocess.run([cc, "-std=c11", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.c"),
                    "-o", str(tmp_path / "s")], check=True)
    got = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout
    assert got.split("\n")[:-1] == expect


def test_the_format():
    """The definition's own corners, so that the reference used elsewhere is checked too."""
    x = np.zeros((1, 32))
    x[0, :16] = [4, 0.25, 0.26, 0.75, 1.25, 1.26, 1.75, 2.5, 2.6, 3.5, 5.0, 5.01, 6, 7.99, -0.25,
                 -7.99]
    byte = ref.scale_bytes(x)
    assert byte.tolist() == [127]  # 7.99 has the exponent of 4
    v = ref.values(ref.codes(x, byte), byte)[0, :16]
    assert v.tolist() == [4, 0, 0.5, 1, 1, 1.5, 2, 2, 3, 4, 4, 6, 6, 6, 0, -6]
    assert np.signbit(v[14])
    for top, want in [(8.0, 128), (2.0 ** -126, 0), (2.0 ** -124, 1), (2.0 ** -149, 0), (0.0, 0),
                      (2.0 ** 127, 252), (np.inf, 255), (np.nan, 255)]:
        x = np.full((1, 32), 0.0)
        x[0, 5] = top
        assert ref.scale_bytes(x).tolist() == [want]
    rng = np.random.default_rng(0)
    x = rng.standard_normal((40, 300)).astype(np.float32)
    q, s = ref.pack(x)
    back = ref.unpack(q, s)
    assert not back[:, 300:].any()
    again = ref.pack(back[:, :300].astype(np.float32))
    assert np.array_equal(ref.unpack(*again), back)  # a packed value is its own nearest


def _quantize(L, entry="fe2o3_quantize_mxfp4", **over):
    a = dict(x=P, x_len=20 * 300, dtype=1, q=P, q_len=20 * 256, scales=P, scales_len=2 * 32 * 8,
             rows=20, cols=300, stride=300)
    a.update(over)
    if entry == "fe2o3_dequantize_mxfp4":
        order = ("q", "q_len", "scales", "scales_len", "x", "x_len", "dtype", "rows", "cols",
                 "stride")
        return getattr(L, entry)(*(a[n] for n in order), None)
    return getattr(L, entry)(*a.values(), None)


@pytest.mark.parametrize("entry", ["fe2o3_quantize_mxfp4", "fe2o3_dequantize_mxfp4"])
@pytest.mark.parametrize("over,want", [
    (dict(dtype=2), SHAPE), (dict(cols=65535 * 256 + 1), SHAPE),
    (dict(rows=0xFFFFFFFF, cols=16 * 256, stride=1 << 20), SHAPE),
    (dict(stride=299), STRIDE), (dict(stride=1 << 63), OVERFLOW),
    (dict(stride=1 << 59), OVERFLOW), (dict(x_len=5999), LENGTH), (dict(stride=301), LENGTH),
    (dict(q_len=5119), LENGTH), (dict(q_len=5121), LENGTH), (dict(scales_len=511), LENGTH),
    (dict(scales_len=320), LENGTH), (dict(x=None), NULL), (dict(q=None), NULL),
    (dict(scales=None), NULL), (dict(x=P + 1), ALIGNMENT), (dict(x=P + 2, dtype=0), ALIGNMENT),
    (dict(q=P + 8), ALIGNMENT), (dict(scales=P + 8), ALIGNMENT),
])
def test_packing_refusals(L, entry, over, want):
    assert _quantize(L, entry, **over) == want


@pytest.mark.parametrize("entry", ["fe2o3_quantize_mxfp4", "fe2o3_dequantize_mxfp4"])
def test_packing_of_nothing(L, entry):
    none = dict(x=None, x_len=0, q=None, q_len=0, scales=None, scales_len=0)
    assert _quantize(L, entry, **none, rows=0) == 0
    assert _quantize(L, entry, **none, cols=0, rows=16) == 0


def _product(L, **over):
    a = dict(a=P, a_len=20 * 256, sa=P, sa_len=2 * 32 * 8, b=P, b_len=40 * 256, sb=P,
             sb_len=2 * 48 * 8, c=P, c_len=800, m=20, n=40, k=300)
    a.update(over)
    return L.fe2o3_gemm_mxfp4_nt(*a.values(), None)


@pytest.mark.parametrize("over,want", [
    (dict(k=65535 * 256 + 1), SHAPE), (dict(a_len=20 * 150), LENGTH), (dict(sa_len=320), LENGTH),
    (dict(b_len=1), LENGTH), (dict(sb_len=1), LENGTH), (dict(c_len=799), LENGTH),
    (dict(a=None), NULL), (dict(sa=None), NULL), (dict(b=None), NULL), (dict(sb=None), NULL),
    (dict(c=None), NULL), (dict(a=P + 8), ALIGNMENT), (dict(sa=P + 8), ALIGNMENT),
    (dict(b=P + 8), ALIGNMENT), (dict(sb=P + 8), ALIGNMENT), (dict(c=P + 1), ALIGNMENT),
])
def test_product_refusals(L, over, want):
    assert _product(L, **over) == want


def test_product_without_outputs(L):
    assert _product(L, m=0, a_len=0, sa_len=0, c_len=0) == 0


def test_injected_failures(L, monkeypatch):
    for entry in ("fe2o3_quantize_mxfp4", "fe2o3_dequantize_mxfp4", "fe2o3_gemm_mxfp4_nt"):
        monkeypatch.setenv("FE2O3_FAULT_POINT", entry)
        call = _product if "gemm" in entry else lambda L: _quantize(L, entry)
        assert call(L) == -23
