"""CPU checks of the 4-bit paged cache: every refusal of its record, as in
test_kv_cache_host.py, whose helpers it uses."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from test_kv_cache_host import (ALIGNMENT, LENGTH, NULL, OVERFLOW, P, SHAPE, STRIDE, _decode, _read,
                                _write, L)  # noqa: F401

MXFP4 = 4


def _cache(pages=4, page_size=16, kv_heads=2, head_dim=64, **over):
    from fe2o3_amd import _lib
    row = kv_heads * head_dim // 2
    n, scales = pages * page_size * row, pages * page_size * kv_heads * (head_dim // 32)
    rec = _lib.Fe2o3KvCacheV1(P, n, P, n, P, scales, P, scales, page_size * row, row,
                              head_dim // 2, MXFP4, pages, page_size, kv_heads, head_dim, 0)
    for name, value in over.items():
        setattr(rec, name, value)
    return rec


BAD = [
    (dict(format=2), SHAPE), (dict(format=3), SHAPE), (dict(head_dim=48), SHAPE), (dict(head_dim=0), SHAPE),
    (dict(head_stride=31), STRIDE), (dict(token_stride=63), STRIDE), (dict(page_stride=1023), STRIDE),
    (dict(page_stride=1 << 63), OVERFLOW), (dict(k_len=4095), LENGTH), (dict(v_len=4095), LENGTH),
    (dict(k_scale_len=255), LENGTH), (dict(v_scale_len=257), LENGTH), (dict(k_scale_len=128), LENGTH),
    (dict(k=None), NULL), (dict(v=None), NULL), (dict(k_scale=None), NULL), (dict(v_scale=None), NULL),
    (dict(k_scale=P + 2), ALIGNMENT), (dict(v_scale=P + 1), ALIGNMENT),
]


@pytest.mark.parametrize("over,want", BAD)
def test_records_refused(L, over, want):  # noqa: F811
    rec = _cache(**over)
    assert _write(L, rec) == want
    assert _read(L, rec) == want
    assert _decode(L, rec) == want


def test_good_records_reach_the_calls_own_checks(L):  # noqa: F811
    # codes may start anywhere for the write and the read, not for decode attention
    rec = _cache(k=P + 1)
    assert _write(L, rec, k=None) == NULL
    assert _read(L, rec, k=None) == NULL
    assert _decode(L, rec) == ALIGNMENT
    assert _decode(L, _cache(), q=None) == NULL
    assert _decode(L, _cache(head_dim=96, token_stride=96, head_stride=48, page_stride=1536,
                             k_len=1 << 20, v_len=1 << 20, k_scale_len=384,
                             v_scale_len=384)) == SHAPE
    assert _decode(L, _cache(token_stride=72, page_stride=1152, k_len=1 << 20,
                             v_len=1 << 20)) == ALIGNMENT


class _Fake:
    """What KvCache asks of a tensor."""

    def __init__(self, shape, dtype, strides=None):
        self.shape, self.dtype = tuple(shape), dtype
        if strides is None:
            strides, n = [], 1
            for size in reversed(self.shape):
                strides.append(n)
                n *= size
            strides.reverse()
        self._strides = tuple(strides)

    def get_device(self):
        return 0

    def stride(self):
        return self._strides

    def is_contiguous(self):
        return True

    def numel(self):
        return int(np.prod(self.shape))

    def data_ptr(self):
        return P


def test_format_from_the_scales():
    from fe2o3_amd import kernels
    k = lambda: _Fake((4, 16, 2, 32), "torch.uint8")  # noqa: E731
    s = lambda *shape: _Fake(shape, "torch.uint8")  # noqa: E731
    c = kernels.KvCache(k(), k(), s(4, 2, 16, 2), s(4, 2, 16, 2))
    assert c.format == kernels.KV_MXFP4 and c.shape == (4, 16, 2, 64)
    assert c.record.head_dim == 64 and c.record.k_scale_len == 256
    f = lambda: _Fake((4, 2, 16), "torch.float32")  # noqa: E731
    c = kernels.KvCache(k(), k(), f(), f())
    assert c.format == kernels.KV_E4M3 and c.shape == (4, 16, 2, 32)
    for bad in (s(4, 2, 16), s(4, 16, 2, 2), s(4, 2, 16, 1)):
        with pytest.raises(ValueError):
            kernels.KvCache(k(), k(), bad, bad)
    b = _Fake((4, 16, 2, 32), "torch.bfloat16")
    with pytest.raises(TypeError):
        kernels.KvCache(b, b, s(4, 2, 16, 2), s(4, 2, 16, 2))
    assert C.sizeof(c.record) == 112


def test_decode_of_a_cache_past_its_span(L):  # noqa: F811
    """Slots that span 2^36 bytes are past decode attention's row numbers; the write and
    the read take them."""
    pages = (1 << 20) + 1
    row = 64 * 8
    far = dict(pages=pages, page_size=128, kv_heads=8, head_dim=64, page_stride=128 * row,
               token_stride=row, head_stride=64, k_len=1 << 40, v_len=1 << 40,
               k_scale_len=pages * 128 * 8 * 2, v_scale_len=pages * 128 * 8 * 2)
    assert _decode(L, _cache(**far)) == SHAPE
    assert _write(L, _cache(**far), k=None, token_stride=1024, head_stride=128,
                  k_len=1 << 20, v_len=1 << 20) == NULL
    assert _decode(L, _cache(**dict(far, k=P + 8))) == ALIGNMENT


def test_decode_of_a_cache_of_too_many_rows(L):  # noqa: F811
    """One page, the heads outermost: slots span little, and there are 2^32 rows."""
    slots, heads = 1 << 30, 4
    many = dict(pages=1, page_size=slots, kv_heads=heads, head_dim=64, token_stride=32,
                head_stride=32 * slots, page_stride=0, k_len=1 << 40, v_len=1 << 40,
                k_scale_len=slots * heads * 2, v_scale_len=slots * heads * 2)
    assert _decode(L, _cache(**many)) == SHAPE
    assert _decode(L, _cache(**dict(many, k=P + 8))) == ALIGNMENT
