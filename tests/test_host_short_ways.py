"""CPU check: calls with DeviceBuffers do not try the short ways through the Python checks, which
are for tensors and give a DeviceBuffer up by an exception, a twentieth to a sixth of a small
call's time.  No call reaches the device: the entry points are replaced."""
from __future__ import annotations

import types

import numpy as np
import pytest

from fe2o3_amd import kernels, runtime


def _buffer(n, dtype):
    b = runtime.DeviceBuffer.__new__(runtime._View)
    b.ctx, b.dtype, b.count = types.SimpleNamespace(device=0), np.dtype(dtype), n
    b.nbytes, b.ptr = n * b.dtype.itemsize, 0x10000
    return b


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(kernels, "_current_device", lambda: 0)
    monkeypatch.setattr(kernels, "_call", lambda entry, *args, **more: made.append((entry, args)))

    def short(*args, **more):
        raise AssertionError("the short way of tensors")
    for name in ("_fast_rows", "_fast_decode", "_fast_rotary", "_fast_packing", "_fast_product"):
        monkeypatch.setattr(kernels, name, short)
    monkeypatch.setattr(kernels.KvCache, "_fast", short)
    return made


PAGES, PLACES, HEADS, DIM, TOKENS, SEQS = 3, 16, 2, 64, 5, 2


def _cache():
    n = PAGES * PLACES * HEADS * DIM
    return kernels.KvCache(_buffer(n, np.uint16), _buffer(n, np.uint16),
                           shape=(PAGES, PLACES, HEADS, DIM))


def _rows():
    return _buffer(TOKENS * HEADS * DIM, np.uint16)


def _write():
    kernels.kv_cache_write(_cache(), _rows(), _rows(), _buffer(TOKENS, np.uint32))


def _read():
    kernels.kv_cache_read(_cache(), _buffer(SEQS * 2, np.uint32), _buffer(SEQS + 1, np.uint32),
                          _rows(), _rows(), tokens=TOKENS)


def _decode():
    q, out = (_buffer(SEQS * 4 * DIM, np.uint16) for _ in range(2))
    kernels.paged_attention_decode(
        _cache(), q, _buffer(SEQS * 2, np.uint32), _buffer(SEQS, np.uint32), out,
        _buffer(SEQS * 4, np.float32), _buffer(1 << 20, np.uint8), max_length=32, scale=0.125,
        q_heads=4)


def _rotary(k=True):
    kernels.rotary(_rows(), _rows() if k else None, _buffer(TOKENS, np.uint32),
                   _buffer(DIM // 2, np.float64), q_shape=(HEADS, DIM), k_shape=(HEADS, DIM))


def _packed(rows, cols):
    return [_buffer(int(np.prod(s)), np.uint8) for s in kernels.mxfp4_shapes(rows, cols)]


def _quantize():
    kernels.quantize_mxfp4(_buffer(20 * 300, np.float32), *_packed(20, 300), rows=20, cols=300)


def _dequantize():
    kernels.dequantize_mxfp4(*_packed(20, 300), _buffer(20 * 300, np.uint16), rows=20, cols=300)


def _product():
    kernels.gemm_mxfp4_nt(*_packed(20, 300), *_packed(40, 300), _buffer(800, np.uint16), 20, 40,
                          300)


@pytest.mark.parametrize("call,entry", [
    (_write, "fe2o3_kv_cache_write"), (_read, "fe2o3_kv_cache_read"),
    (_decode, "fe2o3_paged_attention_decode"), (_rotary, "fe2o3_rotary"),
    (lambda: _rotary(False), "fe2o3_rotary"), (_quantize, "fe2o3_quantize_mxfp4"),
    (_dequantize, "fe2o3_dequantize_mxfp4"), (_product, "fe2o3_gemm_mxfp4_nt")])
def test_buffers_go_the_long_way(calls, call, entry):
    call()
    assert [name for name, _ in calls] == [entry]
