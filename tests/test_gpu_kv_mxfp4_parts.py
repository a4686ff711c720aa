"""Decode attention over 4-bit rows holds its probabilities in two bf16 parts: against 64 bits
with the bound that two parts allow, and one part alone exceeds.

Bound of one output, A = sum_j p_j |v_j|: a probability's first part is off by 2^-8 of it at
most and the second by 2^-8 of the rest, so A 2^-16 where test_gpu_paged_attention.py has
A 2^-8 for one; the scores, the sums and the output's own rounding as there.  Outputs whose
exact value lies that near a border between two bf16 come out on either side of it, which is
all that this path's outputs differ in from probabilities in 32 bits."""
from __future__ import annotations

import numpy as np
import pytest

from gpu_util import bf16_to_f32
from test_gpu_kv_mxfp4 import Batch4
from test_gpu_paged_attention import _bf16_bits

pytestmark = pytest.mark.gpu


def _tight(b, window):
    """(o, bound of two parts, o of probabilities in one part) in 64 bits."""
    o, _, loose, _ = b.reference(window)
    tol, one = loose.copy(), np.zeros_like(o)
    group = b.q_heads // b.kv_heads
    for s, count in enumerate(b.lengths):
        keep = np.arange(max(0, count - window) if window else 0, count)
        if not keep.size:
            continue
        for h in range(b.q_heads):
            k, v = b.k[s][keep, h // group], b.v[s][keep, h // group]
            x = k @ b.q[s, h] * b.scale
            p = np.exp(x - x.max())
            part = bf16_to_f32(_bf16_bits(p)).astype(np.float64)
            one[s, h] = part @ v / p.sum()
            mean = p @ np.abs(v) / p.sum()
            tol[s, h] -= mean * (2.0 ** -8 * (1 + 2.0 ** -7) - 2.0 ** -16)
    return o, tol, one


# query heads a KV head: two subtiles side by side, one row tile, two to four that share tiles
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("q_heads,kv_heads", [(3, 1), (32, 4), (9, 1), (32, 2), (17, 1), (48, 1),
                                              (64, 1)])
@pytest.mark.parametrize("lengths,window", [([700, 70, 1, 0, 333], 0), ([3000, 2500], 0),
                                            ([1500, 40, 999], 257)])
def test_two_parts(gpu, lengths, window, q_heads, kv_heads, head_dim):
    b = Batch4(gpu, lengths, q_heads, kv_heads, head_dim, 16)
    o, tol, one = _tight(b, window)
    got = bf16_to_f32(b.run(window)[0].download()).reshape(o.shape).astype(np.float64)
    off = np.abs(got - o)
    worst = np.unravel_index(np.argmax(off - tol), off.shape)
    assert np.all(off <= tol), (worst, got[worst], o[worst], tol[worst])
    # probabilities in one part, rounded once like these, exceed the bound
    rounded = bf16_to_f32(_bf16_bits(one.astype(np.float32))).astype(np.float64)
    assert np.any(np.abs(rounded - o) > tol)
