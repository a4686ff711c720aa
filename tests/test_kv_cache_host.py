"""CPU checks of the paged key-value cache's entry points: the record's layout,
the page division, and every refusal.  A refused call returns before any HIP
call, so the pointers need only not be NULL; no call here passes validation."""
from __future__ import annotations

import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LENGTH, SHAPE, STRIDE, OVERFLOW, NULL, ALIGNMENT, WORKSPACE = -2, -3, -4, -16, -19, -21, -22
P = 0x10000  # an aligned address that nothing reads
BF16, E4M3 = 0, 1


@pytest.fixture(scope="module")
def L():
    from fe2o3_amd import _lib
    return _lib.lib()


def _cache(fmt=BF16, pages=4, page_size=16, kv_heads=2, head_dim=64, **over):
    from fe2o3_amd import _lib
    row = kv_heads * head_dim
    n = pages * page_size * row
    scales = pages * page_size * kv_heads if fmt == E4M3 else 0
    rec = _lib.Fe2o3KvCacheV1(P, n, P, n, P if scales else None, scales, P if scales else None,
                              scales, page_size * row, row, head_dim, fmt, pages, page_size,
                              kv_heads, head_dim, 0)
    for name, value in over.items():
        setattr(rec, name, value)
    return rec


def _write(L, rec, **over):
    a = dict(k=P, k_len=3 * 128, v=P, v_len=3 * 128, slots=P, slots_len=3, tokens=3,
             token_stride=128, head_stride=64)
    a.update(over)
    return L.fe2o3_kv_cache_write(rec if rec is None else C.byref(rec), *a.values(), None)


def _read(L, rec, **over):
    a = dict(table=P, table_len=2 * 5, starts=P, starts_len=3, k=P, k_len=3 * 128, v=P,
             v_len=3 * 128, seqs=2, table_cols=5, tokens=3, token_stride=128, head_stride=64)
    a.update(over)
    return L.fe2o3_kv_cache_read(rec if rec is None else C.byref(rec), *a.values(), None)


def _decode(L, rec, **over):
    a = dict(q=P, q_len=3 * 512, table=P, table_len=15, lengths=P, lengths_len=3, o=P,
             o_len=3 * 512, lse=P, lse_len=24, workspace=P, workspace_bytes=1 << 30, seqs=3,
             q_heads=8, table_cols=5, max_length=80, q_stride=512, window=0, scale=0.125)
    a.update(over)
    return L.fe2o3_paged_attention_decode(rec if rec is None else C.byref(rec), *a.values(), None)


def test_record_layout_matches_the_header(tmp_path):
    from fe2o3_amd import _lib
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    rec = _lib.Fe2o3KvCacheV1
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "fe2o3_mi355x.h"',
             "int main(void) {", 'printf("%zu %zu\\n", sizeof(Fe2o3KvCacheV1), '
             '_Alignof(Fe2o3KvCacheV1));']
    expect = [f"{C.sizeof(rec)} {C.alignment(rec)}"]
    for field, _ in rec._fields_:
        lines.append(f'printf("%zu\\n", offsetof(Fe2o3KvCacheV1, {field}));')
        expect.append(str(getattr(rec, field).offset))
    heads = [(8, 8, 64), (32, 8, 128), (128, 1, 128), (6, 2, 64), (64, 4, 128), (68, 4, 64)]
    from fe2o3_amd import kernels
    for q, kv, d in heads:
        lines.append('printf("%llu\\n", (unsigned long long)'
                     f'FE2O3_PAGED_ATTENTION_WORKSPACE_BYTES({q}u, {kv}u, {d}u));')
        expect.append(str(kernels.paged_attention_workspace_bytes(q, kv, d)))
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0;", "}"]))
    exe = tmp_path / "layout"
    subprocess.run([cc, "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n")
    assert got[:-1] == expect


def test_e4m3_quotients_by_reciprocal():
    """The cache write divides by a row's scale s through q = x r, r = RN(1 / s),
    corrected once: q + (x - q s) r with fused multiply-adds.  For every scale that a
    row of bf16 can have (s = RN(amax / 448), 128 significands) and every bf16 x up to
    amax down to where its code is 0, that is the correctly rounded quotient; powers
    of two change nothing while nothing is subnormal.  In 80-bit arithmetic, whose 64
    bits hold x - q s exactly, and q + e r to more than twice fp32's."""
    f, wide = np.float32, np.longdouble
    if np.finfo(wide).nmant < 63:
        pytest.skip("no 80-bit floating point")
    sig = np.arange(128, 256).astype(f)
    checked = 0
    for amax in sig:
        s = f(amax / f(448))
        r = f(f(1) / s)
        for k in range(-1, 24):
            x = (sig * f(2.0 ** -k)).astype(f)
            x = x[x <= amax]
            q = (x * r).astype(f)
            e = (x.astype(wide) - q.astype(wide) * wide(s)).astype(f)
            got = (q.astype(wide) + e.astype(wide) * wide(r)).astype(f)
            assert np.array_equal(got, (x / s).astype(f))
            checked += x.size
    assert checked > 350000


def test_e4m3_write_codes_are_the_divisions(tmp_path):
    """The write's own quotients (kv_cache.hpp, RowScale) for every bf16 row maximum and
    x of both signs, zeros among them: the codes of the division."""
    exe = tmp_path / "row_scale_check"
    subprocess.run(["g++", "-O2", "-std=c++17", "-fopenmp", "-ffp-contract=off", "-o", str(exe),
                    os.path.join(ROOT, "tests", "row_scale_check.cpp")], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "bad 0" in r.stdout, r.stdout


def test_page_division(tmp_path):
    exe = tmp_path / "fast_div_check"
    subprocess.run(["g++", "-O2", "-std=c++17", "-o", str(exe),
                    os.path.join(ROOT, "tests", "fast_div_check.cpp")], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "bad 0" in r.stdout, r.stdout


def test_grids_stay_within_a_launch(tmp_path):
    """Every number of workgroups has a grid of fewer than 2^32 threads a dimension,
    of 1024 threads a workgroup, that holds it with less than a row to spare."""
    src = tmp_path / "grid.cpp"
    src.write_text('#include <stdio.h>\n'
                   f'#include "{ROOT}/fe2o3_amd/csrc/kv_cache.hpp"\n' + """
int main() {
  using kv_cache::Grid;
  unsigned long long bad = 0, tried = 0;
  auto one = [&](uint64_t n) {
    if (n < 1u || n >= UINT64_C(1) << 31) return;
    const Grid g = Grid::of((uint32_t)n);
    const uint64_t held = (uint64_t)g.x * g.y;
    const bool row = g.y == 1u || g.x == kv_cache::kGridWidth;
    if (UINT64_C(1024) * g.x >> 32 != 0u || g.y > 65535u || held < n || held - n >= g.x || !row)
      ++bad;
    ++tried;
  };
  for (uint64_t n = 1; n < 5000u; ++n) one(n);
  for (int b = 10; b <= 31; ++b)
    for (uint64_t e = 0; e < 9; ++e)
      for (uint64_t m = 1; m < 8; ++m) one((UINT64_C(1) << b) * m + e - 4u);
  printf("tried %llu bad %llu\\n", tried, bad);
  return bad == 0 ? 0 : 1;
}
""")
    exe = tmp_path / "grid"
    subprocess.run(["g++", "-O2", "-std=c++17", "-o", str(exe), str(src)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and "bad 0" in r.stdout, r.stdout


CACHE_REFUSALS = [
    (dict(format=2), SHAPE), (dict(pages=0), SHAPE), (dict(page_size=0), SHAPE),
    (dict(kv_heads=0), SHAPE), (dict(head_dim=0), SHAPE),
    (dict(pages=1 << 20, page_size=1 << 11), SHAPE),  # 2^31 slots
    (dict(head_dim=1 << 31), SHAPE), (dict(head_dim=(1 << 32) - 3), SHAPE),
    (dict(head_stride=63), STRIDE), (dict(token_stride=63), STRIDE),
    (dict(token_stride=127), STRIDE),  # heads of one token reach into the next
    (dict(page_stride=16 * 128 - 1), STRIDE),
    # tokens within a head, and the next head begins before they end
    (dict(token_stride=64, head_stride=16 * 64 - 1), STRIDE),
    (dict(page_stride=1 << 63), OVERFLOW), (dict(head_stride=(1 << 64) - 1), OVERFLOW),
    (dict(k_len=4 * 16 * 128 - 1), LENGTH), (dict(v_len=0), LENGTH),
    (dict(k_scale_len=1), LENGTH),  # a bf16 cache has no scales
    (dict(k=None), NULL), (dict(v=None), NULL),
    (dict(k=P + 1), ALIGNMENT),
]


@pytest.mark.parametrize("call", [_write, _read, _decode])
def test_cache_record_is_checked(L, call):
    assert call(L, None) == NULL
    for over, status in CACHE_REFUSALS:
        assert call(L, _cache(**over)) == status, over
    e4m3 = dict(fmt=E4M3)
    assert call(L, _cache(**e4m3, k_scale_len=4 * 16 * 2 - 1)) == LENGTH
    assert call(L, _cache(**e4m3, v_scale_len=4 * 16 * 2 + 1)) == LENGTH
    assert call(L, _cache(**e4m3, v_scale=None)) == NULL
    assert call(L, _cache(**e4m3, k_scale=P + 2)) == ALIGNMENT


def test_strides_of_single_dimensions_say_nothing(L):
    """One page, one token a page or one head: its stride is not looked at; the
    call goes on to the check that this one fails."""
    for over in (dict(pages=1, page_stride=0), dict(kv_heads=1, head_stride=0),
                 dict(page_size=1, token_stride=0, page_stride=128)):
        assert _write(L, _cache(**over), slots_len=2) == LENGTH, over


def test_write_refusals(L):
    rec = _cache()
    assert _write(L, rec, slots_len=2) == LENGTH
    assert _write(L, rec, tokens=1 << 30, slots_len=1 << 30) == SHAPE
    assert _write(L, rec, token_stride=127) == STRIDE
    assert _write(L, rec, head_stride=10) == STRIDE
    assert _write(L, rec, token_stride=1 << 63) == OVERFLOW
    assert _write(L, rec, k_len=3 * 128 - 1) == LENGTH
    assert _write(L, rec, v_len=3 * 128 - 1) == LENGTH
    for name in ("k", "v", "slots"):
        assert _write(L, rec, **{name: None}) == NULL
    for name, off in (("k", 1), ("v", 3), ("slots", 2)):
        assert _write(L, rec, **{name: P + off}) == ALIGNMENT
    # no tokens: nothing is launched and no array is looked at
    assert _write(L, rec, tokens=0, slots_len=0, k=None, k_len=0, v=None, v_len=0,
                  slots=None) == 0


def test_read_refusals(L):
    rec = _cache()
    assert _read(L, rec, table_len=9) == LENGTH
    assert _read(L, rec, starts_len=2) == LENGTH
    assert _read(L, rec, tokens=1 << 30) == SHAPE
    assert _read(L, rec, seqs=1 << 31, table_cols=0, table_len=0, starts_len=(1 << 31) + 1) == SHAPE
    assert _read(L, rec, token_stride=64) == STRIDE
    assert _read(L, rec, k_len=3 * 128 - 1) == LENGTH
    for name in ("k", "v", "starts", "table"):
        assert _read(L, rec, **{name: None}) == NULL
    for name, off in (("k", 1), ("v", 3), ("starts", 2), ("table", 1)):
        assert _read(L, rec, **{name: P + off}) == ALIGNMENT
    assert _read(L, rec, tokens=0, k=None, k_len=0, v=None, v_len=0) == 0
    assert _read(L, rec, seqs=0, table_len=0, starts_len=1) == 0


def test_decode_refusals(L):
    rec = _cache()
    assert _decode(L, _cache(head_dim=96, kv_heads=2)) == SHAPE
    assert _decode(L, rec, q_heads=0) == SHAPE
    assert _decode(L, rec, q_heads=7) == SHAPE
    assert _decode(L, rec, max_length=81) == SHAPE
    assert _decode(L, rec, table_cols=0, table_len=0, max_length=1) == SHAPE
    assert _decode(L, rec, max_length=1 << 31, table_cols=1 << 30) == SHAPE
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert _decode(L, rec, scale=scale) == SHAPE
    # 2^31 tiles in all
    many = dict(table_cols=1 << 26, max_length=1 << 30, seqs=1 << 5, lengths_len=1 << 5,
                table_len=1 << 31)
    assert _decode(L, rec, **many) == SHAPE
    assert _decode(L, rec, q_stride=511) == STRIDE
    assert _decode(L, rec, q_stride=1 << 63) == OVERFLOW
    assert _decode(L, rec, q_len=3 * 512 - 1) == LENGTH
    assert _decode(L, rec, table_len=14) == LENGTH
    assert _decode(L, rec, lengths_len=2) == LENGTH
    assert _decode(L, rec, o_len=3 * 512 + 1) == LENGTH
    assert _decode(L, rec, lse_len=23) == LENGTH
    for name in ("q", "table", "lengths", "o", "workspace"):
        assert _decode(L, rec, **{name: None}) == NULL
    for name in ("q", "o", "workspace"):
        assert _decode(L, rec, **{name: P + 8}) == ALIGNMENT
    for name in ("lse", "table", "lengths"):
        assert _decode(L, rec, **{name: P + 2}) == ALIGNMENT
    assert _decode(L, rec, q_stride=516, q_len=1 << 20) == ALIGNMENT
    # rows of the cache off 16 bytes
    assert _decode(L, _cache(k=P + 2)) == ALIGNMENT
    assert _decode(L, _cache(token_stride=132, page_stride=1 << 12, k_len=1 << 20,
                             v_len=1 << 20)) == ALIGNMENT
    assert _decode(L, _cache(fmt=E4M3, page_stride=2056, k_len=1 << 20, v_len=1 << 20)) == ALIGNMENT
    from fe2o3_amd import kernels
    need = kernels.paged_attention_workspace_bytes(8, 2, 64)
    assert _decode(L, rec, workspace_bytes=need - 1) == WORKSPACE
    assert _decode(L, rec, seqs=0, lengths_len=0, table_len=0) == 0


@pytest.mark.parametrize("entry,call", [("fe2o3_kv_cache_write", _write),
                                        ("fe2o3_kv_cache_read", _read),
                                        ("fe2o3_paged_attention_decode", _decode)])
def test_fault_point_fails_closed(L, monkeypatch, entry, call):
    monkeypatch.setenv("FE2O3_FAULT_POINT", entry)
    assert call(L, _cache()) == -23


class _Fake:
    """A tensor's metadata without a GPU."""

    def __init__(self, shape, strides, dtype="torch.bfloat16", device=0):
        self.shape, self._strides, self.dtype, self._device = shape, strides, dtype, device
        self.is_cuda = device >= 0

    def stride(self, i=None):
        return self._strides if i is None else self._strides[i]

    def numel(self):
        return int(np.prod(self.shape))

    def is_contiguous(self):
        want, at = [], 1
        for n in reversed(self.shape):
            want.insert(0, at)
            at *= n
        return all(n == 1 or s == w for n, s, w in zip(self.shape, self._strides, want))

    def data_ptr(self):
        return P

    def get_device(self):
        return self._device


def test_cache_of_tensors_takes_their_strides():
    from fe2o3_amd import kernels
    k = _Fake((4, 16, 2, 64), (2048, 64, 1024, 1))
    rec = kernels.KvCache(k, k).record
    assert (rec.page_stride, rec.token_stride, rec.head_stride) == (2048, 64, 1024)
    assert rec.k_len == 8192 and rec.format == BF16
    # [pages, 2, ...]: K and V beside each other
    both = _Fake((4, 16, 2, 64), (4096, 128, 64, 1))
    rec = kernels.KvCache(both, both).record
    assert rec.page_stride == 4096 and rec.k_len == 3 * 4096 + 15 * 128 + 64 + 64
    with pytest.raises(ValueError):  # head_dim strided
        kernels.KvCache(_Fake((4, 16, 2, 64), (4096, 256, 128, 2)),
                        _Fake((4, 16, 2, 64), (4096, 256, 128, 2)))
    with pytest.raises(ValueError):
        kernels.KvCache(k, both)
    with pytest.raises(ValueError):
        kernels.KvCache(_Fake((4, 16, 128), (2048, 128, 1)), _Fake((4, 16, 128), (2048, 128, 1)))
    codes = _Fake((4, 16, 2, 64), (2048, 128, 64, 1), "torch.uint8")
    with pytest.raises(TypeError):  # codes without scales
        kernels.KvCache(codes, codes)
    with pytest.raises(TypeError):  # host memory
        kernels.KvCache(_Fake((4, 16, 2, 64), (2048, 128, 64, 1), device=-1),
                        _Fake((4, 16, 2, 64), (2048, 128, 64, 1), device=-1))
    with pytest.raises(ValueError):
        kernels.KvCache(k, k, k_scale=_Fake((4, 2, 16), (32, 16, 1), "torch.float32"))
    scale = _Fake((4, 2, 16), (32, 16, 1), "torch.float32")
    rec = kernels.KvCache(codes, codes, scale, scale).record
    assert rec.format == E4M3 and rec.k_scale_len == 128
    with pytest.raises(ValueError):  # tokens before heads
        swapped = _Fake((4, 16, 2), (32, 2, 1), "torch.float32")
        kernels.KvCache(codes, codes, swapped, swapped)


def test_arrays_on_another_device_are_refused(monkeypatch):
    """The launch goes to the current device: an array elsewhere is refused
    before the library is called."""
    from fe2o3_amd import _lib, kernels

    class Lib:
        @staticmethod
        def fe2o3_rt_get_device(out):
            out._obj.value = 0
            return 0

        def __getattr__(self, name):
            raise AssertionError(name)

    cache = kernels.KvCache(*(_Fake((4, 16, 2, 64), (2048, 128, 64, 1)) for _ in "kv"))
    here, there = _Fake((3, 2, 64), (128, 64, 1)), _Fake((3, 2, 64), (128, 64, 1), device=1)
    slots = _Fake((3,), (1,), "torch.int32")
    monkeypatch.setattr(_lib, "lib", lambda: Lib())
    with pytest.raises(ValueError, match="device 1"):
        kernels.kv_cache_write(cache, here, there, slots)
    far = kernels.KvCache(*(_Fake((4, 16, 2, 64), (2048, 128, 64, 1), device=1) for _ in "kv"))
    with pytest.raises(ValueError, match="the current one is 0"):
        kernels.kv_cache_write(far, there, there, slots)


def test_shapes_that_do_not_fit_are_refused(monkeypatch):
    """A block table or an output of as many elements in another shape."""
    from fe2o3_amd import _lib, kernels

    class Lib:
        @staticmethod
        def fe2o3_rt_get_device(out):
            out._obj.value = 0
            return 0

        def __getattr__(self, name):
            raise AssertionError(name)

    monkeypatch.setattr(_lib, "lib", lambda: Lib())
    cache = kernels.KvCache(*(_Fake((4, 16, 2, 64), (2048, 128, 64, 1)) for _ in "kv"))
    q, lengths = _Fake((3, 4, 64), (256, 64, 1)), _Fake((3,), (1,), "torch.int32")
    table, turned = (_Fake(s, (s[1], 1), "torch.int32") for s in ((3, 2), (2, 3)))
    other = _Fake((4, 3, 64), (192, 64, 1))
    ws = _Fake((1 << 20,), (1,), "torch.uint8")
    with pytest.raises(ValueError, match="block table"):
        kernels.paged_attention_decode(cache, q, turned, lengths, q, None, ws, max_length=32,
                                       scale=1.0)
    with pytest.raises(ValueError, match="out of"):
        kernels.paged_attention_decode(cache, q, table, lengths, other, None, ws, max_length=32,
                                       scale=1.0)
    rows, starts = _Fake((9, 2, 64), (128, 64, 1)), _Fake((4,), (1,), "torch.int32")
    with pytest.raises(ValueError, match="block table"):
        kernels.kv_cache_read(cache, turned, starts, rows, rows)


def test_statistics_and_outputs_of_another_shape_are_refused(monkeypatch):
    """lse of [q_heads, seqs], and out of another shape where q is a DeviceBuffer."""
    from fe2o3_amd import _lib, kernels, runtime

    class Lib:
        @staticmethod
        def fe2o3_rt_get_device(out):
            out._obj.value = 0
            return 0

        @staticmethod
        def fe2o3_paged_attention_decode(*args):
            raise OverflowError  # the checks are through

        def __getattr__(self, name):
            raise AssertionError(name)

    monkeypatch.setattr(_lib, "lib", lambda: Lib())
    cache = kernels.KvCache(*(_Fake((4, 16, 2, 64), (2048, 128, 64, 1)) for _ in "kv"))
    lengths, table = _Fake((3,), (1,), "torch.int32"), _Fake((3, 2), (2, 1), "torch.int32")
    ws = _Fake((1 << 20,), (1,), "torch.uint8")
    held = runtime.DeviceBuffer.__new__(runtime._View)
    held.ctx = type("Context", (), {"device": 0})()
    held.dtype, held.count, held.ptr = np.dtype(np.uint16), 3 * 4 * 64, P
    fits = _Fake((3, 4, 64), (256, 64, 1))
    other = _Fake((4, 3, 64), (192, 64, 1))
    stats, turned = (_Fake(s, (s[1], 1), "torch.float32") for s in ((3, 4), (4, 3)))
    for q, more in ((fits, {}), (held, dict(q_heads=4))):
        def call(out, lse):
            kernels.paged_attention_decode(cache, q, table, lengths, out, lse, ws, max_length=32,
                                           scale=1.0, **more)
        with pytest.raises(ValueError, match="out of"):
            call(other, None)
        with pytest.raises(ValueError, match="lse of"):
            call(fits, turned)
        flat = _Fake((3 * 4 * 64,), (1,)), _Fake((12,), (1,), "torch.float32")
        for out, lse in ((fits, stats), (fits, None), (held, stats), flat):
            with pytest.raises(OverflowError):
                call(out, lse)


@pytest.mark.parametrize("table", [(0, 5), (0,)])
def test_empty_batch(L, monkeypatch, table):
    """A step of no sequences, with a max_length that its tables have pages for, and a
    read of none: nothing to do, and no error."""
    from fe2o3_amd import _lib, kernels

    class Lib:
        @staticmethod
        def fe2o3_rt_get_device(out):
            out._obj.value = 0
            return 0

        def __getattr__(self, name):
            return getattr(L, name)  # returns before any HIP call

    monkeypatch.setattr(_lib, "lib", lambda: Lib())
    cache = kernels.KvCache(*(_Fake((4, 16, 2, 64), (2048, 128, 64, 1)) for _ in "kv"))
    q, lse = _Fake((0, 4, 64), (256, 64, 1)), _Fake((0, 4), (4, 1), "torch.float32")
    table = _Fake(table, (5, 1)[-len(table):], "torch.int32")
    kernels.paged_attention_decode(cache, q, table, _Fake((0,), (1,), "torch.int32"), q, lse,
                                   _Fake((1 << 20,), (1,), "torch.uint8"), max_length=80,
                                   scale=0.125, sync=False)
    rows = _Fake((3, 2, 64), (128, 64, 1))
    kernels.kv_cache_read(cache, table, _Fake((1,), (1,), "torch.int32"), rows, rows, sync=False)


def test_decode_scale_within_its_range(L):
    """Scores are taken in powers of two: a scale of which log2 e makes an infinity is
    refused, the largest below it goes on to the check that this call fails."""
    most = float(np.nextafter(np.finfo(np.float32).max / np.float32(1.4426950408889634),
                              np.float32(0)))
    assert _decode(L, _cache(), scale=3e38, workspace_bytes=0) == SHAPE
    assert _decode(L, _cache(), scale=2.4e38, workspace_bytes=0) == SHAPE
    assert _decode(L, _cache(), scale=most, workspace_bytes=0) == WORKSPACE
    assert _decode(L, _cache(), scale=1e-45, workspace_bytes=0) == WORKSPACE
