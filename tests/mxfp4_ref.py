"""The microscaled 4-bit format in 64 bits: codes, scales and packed matrices in numpy."""
from __future__ import annotations

import numpy as np

MAGNITUDES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
# between neighbouring magnitudes, and whether a tie there goes up (to the even code)
BORDERS = [(0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True),
           (5.0, False)]


def scale_bytes(x):
    """Scale bytes of blocks [..., 32] (float32 or float64 of float32 values)."""
    with np.errstate(invalid="ignore"):
        top = np.max(np.abs(x), -1)
    bad = ~np.isfinite(x).all(-1)
    _, e = np.frexp(np.where(bad | (top == 0), 1.0, top).astype(np.float64))
    # frexp's exponent is floor(log2) + 1
    byte = np.where(top == 0, 0, np.maximum(e - 1 - 2 + 127, 0))
    return np.where(bad, 255, byte).astype(np.uint8)


def scale_values(byte):
    byte = np.asarray(byte)
    return np.where(byte == 255, np.nan, np.ldexp(1.0, byte.astype(int) - 127))


def codes(x, byte):
    """Codes of blocks [..., 32] on their scales; those of NaN blocks are 0 here."""
    with np.errstate(invalid="ignore"):
        y = np.abs(x.astype(np.float64)) / scale_values(byte)[..., None]
        c = np.zeros(x.shape, np.uint8)
        for border, up in BORDERS:
            c += ((y >= border) if up else (y > border)).astype(np.uint8)
    return c | (np.signbit(x).astype(np.uint8) << 3)


def values(code, byte):
    """Values of codes [..., 32] in 64 bits."""
    v = MAGNITUDES[code & 7] * np.where(code & 8, -1.0, 1.0)
    return v * scale_values(byte)[..., None]


def two_to_a_byte(code):
    return (code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8)


def one_a_byte(packed):
    return np.stack((packed & 15, packed >> 4), -1).reshape(*packed.shape[:-1],
                                                             2 * packed.shape[-1])


def pack(x):
    """(codes [rows, panels * 128], scales [panels, rows to 16, 8]) of a matrix."""
    rows, cols = x.shape
    panels = -(-cols // 256)
    wide = np.zeros((rows, panels * 256), x.dtype)
    wide[:, :cols] = x
    blocks = wide.reshape(rows, panels, 8, 32)
    byte = scale_bytes(blocks)
    scales = np.zeros((panels, -(-rows // 16) * 16, 8), np.uint8)
    scales[:, :rows] = byte.transpose(1, 0, 2)
    return two_to_a_byte(codes(blocks, byte)).reshape(rows, -1), scales


def unpack(packed, scales):
    """The matrix [rows, panels * 256] in 64 bits."""
    rows, panels = packed.shape[0], scales.shape[0]
    code = one_a_byte(packed).reshape(rows, panels, 8, 32)
    return values(code, scales[:, :rows].transpose(1, 0, 2)).reshape(rows, -1)
