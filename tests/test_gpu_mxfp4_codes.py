"""GPU tests of the packing's codes and scales over everything that decides them: every largest
exponent of a block, under it every bf16 value, and in f32 both sides of every border between
two codes.  The codes are compared with the definition in 64 bits, from values that the host
made of their bits."""
from __future__ import annotations

import numpy as np
import pytest

import mxfp4_ref as ref

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

EXPONENTS = 255  # biased, of the largest magnitude: subnormal (0), 1 .. 254


def _k():
    from fe2o3_amd import kernels
    return kernels


def _values64(bits):
    """Float bits as doubles, exactly, by integers alone."""
    e, fraction = (bits >> 23 & 255).astype(np.int64), (bits & 0x7FFFFF).astype(np.int64)
    v = np.ldexp(np.where(e > 0, fraction + (1 << 23), fraction).astype(np.float64),
                 np.maximum(e, 1) - 150)
    return np.where(bits >> 31, -v, v)


def _blocks(bits, exponent):
    """Blocks of 31 of the bits and the largest value of the exponent; larger ones as +0."""
    top = np.uint32(exponent << 23 | 0x7FFFFF)
    bits = np.where((bits & 0x7FFFFFFF) <= top, bits, 0).astype(np.uint32)
    bits = np.resize(bits, -(-bits.size // 31) * 31).reshape(-1, 31)
    return np.concatenate([bits, np.full((len(bits), 1), top, np.uint32)], 1)


def _check(x, bits, exponent):
    """Packs x [rows, 256], of these bits, and compares blocks of 32 on this exponent's scale."""
    k = _k()
    rows = x.shape[0]
    q, s = (torch.full(n, 0xA5, dtype=torch.uint8, device="cuda") for n in k.mxfp4_shapes(*x.shape))
    k.quantize_mxfp4(x, q, s)
    byte = max(exponent - 2, 0)
    assert bool((s[:, :rows] == byte).all()) and bool((s[:, rows:] == 0xA5).all())
    v = torch.from_numpy(_values64(bits)).cuda()
    y = v.abs() * 2.0 ** (127 - byte)
    want = torch.zeros_like(y, dtype=torch.uint8)
    for border, up in ref.BORDERS:
        want += (y >= border) if up else (y > border)
    want += 8 * (torch.from_numpy((bits >> 31).astype(np.uint8)).cuda())
    got = torch.stack((q & 15, q >> 4), -1).view(rows, -1)
    bad = (got != want).nonzero()
    assert not len(bad), (exponent, len(bad), hex(int(bits[tuple(bad[0].tolist())])),
                          int(got[tuple(bad[0])]), int(want[tuple(bad[0])]))


def _rows(blocks):
    """Blocks as rows of 256, the last repeated."""
    n = -(-len(blocks) // 8) * 8
    return np.concatenate([blocks, np.repeat(blocks[-1:], n - len(blocks), 0)]).reshape(-1, 256)


def test_every_bf16_under_every_exponent(gpu):
    """Packed as bf16, and the same values as f32."""
    every = np.arange(65536, dtype=np.uint32) << 16
    every = every[(every >> 23 & 255) < 255]
    for exponent in range(EXPONENTS):
        blocks = _blocks(every, exponent)
        blocks[:, 31] = exponent << 23 | 0x7F0000  # the largest one that is a bf16
        bits = _rows(blocks)
        held = torch.from_numpy((bits >> 16).astype(np.uint16).view(np.int16)).cuda()
        _check(held.view(torch.bfloat16), bits, exponent)
        _check(torch.from_numpy(bits.view(np.float32)).cuda(), bits, exponent)


def test_f32_beside_every_border(gpu):
    """Three values on either side of each border and of each code's value, and random ones of
    every exponent from the top down to where all codes are zero."""
    rng = np.random.default_rng(1)
    at = np.array([b for b, _ in ref.BORDERS] + list(ref.MAGNITUDES[1:]) + [7.5])
    for exponent in range(EXPONENTS):
        with np.errstate(over="ignore"):
            middle = np.ldexp(at, max(exponent - 2, 0) - 127).astype(np.float32).view(np.uint32)
        near = (middle[:, None].astype(np.int64) + np.arange(-3, 4)).astype(np.uint32).ravel()
        low = max(exponent - 6, 0) << 23
        some = rng.integers(low, (exponent << 23) + 0x800000, 3000).astype(np.uint32)
        bits = np.concatenate([near, near | 0x80000000, some, some[::2] | 0x80000000])
        bits = _rows(_blocks(bits, exponent))
        _check(torch.from_numpy(bits.view(np.float32)).cuda(), bits, exponent)
