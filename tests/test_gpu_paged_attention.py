"""fe2o3_paged_attention_decode on the GPU against attention in 64 bits, element
by element, with the bound that its roundings allow.

Bound of one output, A = sum_j p_j |v_j| the mean magnitude that it sums:
  probabilities (times the V scale) rounded to bf16 for the MFMA: A 2^-8;
  scores: products of bf16 are exact in fp32, their sum over head_dim terms and
  the scalings are off by at most (head_dim + 4) 2^-24 of B = max_j scale
  sum_d |q_d k_jd|, which moves each probability by that share, and the sum of
  them likewise: twice, and 2^-20 for exp2, the running sums' fp32 additions
  (pairs of tiles, waves and runs: below 2^8 steps of 2^-24 each, twice) and
  the last division;
  the output's own rounding to bf16: 2^-8 |o|.
The log-sum-exp has the scores' error and 2^-20, and 2^-22 of its magnitude."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from gpu_util import Guarded, assert_same, bf16_to_f32

pytestmark = pytest.mark.gpu


def _k():
    from fe2o3_amd import kernels
    return kernels


def _bf16_bits(x):
    from oracle import oracle as orc
    return np.asarray(orc.bf16_from_f32(np.ascontiguousarray(x, np.float32).ravel()),
                      np.uint16).reshape(np.shape(x))


def _decode_table():
    from oracle import oracle as orc
    return np.asarray(orc.fp8_decode_table(), np.float32)


class Batch:
    """Sequences in a guarded paged cache.  Slots that no sequence reaches hold NaN
    (values and scales), entries behind a sequence's pages an id out of range."""

    def __init__(self, gpu, fmt, lengths, q_heads, kv_heads, head_dim, page_size, order="token",
                 pad=0, q_pad=0, cols=None, seed=0, peak=1.0, slack=2):
        rng = np.random.default_rng([seed, len(lengths), q_heads, head_dim, page_size])
        self.gpu, self.fmt, self.lengths = gpu, fmt, list(lengths)
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.page_size, self.order_name, self.pad = page_size, order, pad
        need = [-(-n // page_size) for n in lengths]
        pages = sum(need) + slack
        self.cols = max(need + [1]) if cols is None else cols
        free = rng.permutation(pages)
        self.table = np.full((len(lengths), self.cols), 0xFFFFFFF0, np.uint32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = free[at:at + n]
            at += n
        if order == "token":
            head = head_dim + pad
            token = kv_heads * head
            page = page_size * token
        else:
            token = head_dim + pad
            head = page_size * token
            page = kv_heads * head
        self.shape, self.strides = (pages, page_size, kv_heads, head_dim), (page, token, head)
        n = pages * page
        self.k, self.v, arrays, scales = [], [], [], []
        for part, held in enumerate((self.k, self.v)):
            if fmt == "bf16":
                flat, itemsize = np.full(n, 0x7FFF, np.uint16), 2
            else:
                flat, itemsize = np.full(n, 0x7F, np.uint8), 1
                scale = np.full((pages, kv_heads, page_size), np.nan, np.float32)
            rows = np.lib.stride_tricks.as_strided(
                flat, self.shape, [s * itemsize for s in self.strides] + [itemsize])
            for s, count in enumerate(lengths):
                key = np.arange(count)
                page_of, place = self.table[s, key // page_size], key % page_size
                x = rng.standard_normal((count, kv_heads, head_dim)).astype(np.float32)
                if part == 0:
                    x *= peak
                if fmt == "bf16":
                    rows[page_of, place] = _bf16_bits(x)
                    held.append(bf16_to_f32(rows[page_of, place]).astype(np.float64))
                else:
                    code = rng.integers(0, 256, x.shape).astype(np.uint8)
                    code[code & 0x7F == 0x7F] = 0x38
                    sc = (np.float32(0.004) * peak * (0.5 + rng.random((count, kv_heads)))
                          ).astype(np.float32)
                    rows[page_of, place] = code
                    scale[page_of, :, place] = sc
                    held.append(_decode_table()[code].astype(np.float64)
                                * sc.astype(np.float64)[..., None])
            arrays.append(Guarded(gpu, flat))
            if fmt == "e4m3":
                scales.append(Guarded(gpu, scale))
        self.arrays, self.scales = arrays, scales
        self.cache = _k().KvCache(*(a.body for a in arrays), *(a.body for a in scales),
                                  shape=self.shape, strides=self.strides)
        self.q_stride = q_heads * head_dim + q_pad
        qn = (len(lengths) - 1) * self.q_stride + q_heads * head_dim
        q = np.full(max(qn, 0), 0x7FFF, np.uint16)
        view = np.lib.stride_tricks.as_strided(q, (len(lengths), q_heads, head_dim),
                                               (2 * self.q_stride, 2 * head_dim, 2))
        view[...] = _bf16_bits(rng.standard_normal(view.shape))
        self.q = bf16_to_f32(view).astype(np.float64)
        self.dev_q = Guarded(gpu, q)
        self.dev_table = Guarded(gpu, self.table)
        self.dev_lengths = Guarded(gpu, np.array(lengths, np.uint32))
        self.scale = head_dim ** -0.5

    def outputs(self):
        rows = len(self.lengths) * self.q_heads
        return (Guarded(self.gpu, np.full(rows * self.head_dim, 0x7FDE, np.uint16)),
                Guarded(self.gpu, np.full(rows, 7.0, np.float32)))

    def run(self, window=0, max_length=None, lse=True, workspace=None, out=None, **more):
        kern = _k()
        o, stat = self.outputs() if out is None else out
        if workspace is None:  # whatever it holds
            n = kern.paged_attention_workspace_bytes(self.q_heads, self.kv_heads, self.head_dim)
            workspace = Guarded(self.gpu, np.full(n, 0xFF, np.uint8))
        kern.paged_attention_decode(
            self.cache, self.dev_q.body, self.dev_table.body, self.dev_lengths.body, o.body,
            stat.body if lse else None, workspace.body,
            max_length=max(self.lengths + [0]) if max_length is None else max_length,
            scale=self.scale, window=window, q_heads=self.q_heads, q_stride=self.q_stride, **more)
        assert o.guards_intact() and stat.guards_intact() and workspace.guards_intact()
        return o, stat

    def reference(self, window=0, max_length=None, drop=None):
        """(o, lse, bound of o, bound of lse) in 64 bits; drop: keys left out of a sequence."""
        d, group = self.head_dim, self.q_heads // self.kv_heads
        shape = (len(self.lengths), self.q_heads)
        o, lse = np.zeros(shape + (d,)), np.full(shape, -np.inf)
        o_tol, lse_tol = np.zeros(shape + (d,)), np.zeros(shape)
        for s, count in enumerate(self.lengths):
            end = count if max_length is None else min(count, max_length)
            keep = np.arange(max(0, end - window) if window else 0, end)
            if drop is not None:
                keep = keep[~drop(s, keep)]
            if keep.size == 0:
                continue
            for h in range(self.q_heads):
                k, v = self.k[s][keep, h // group], self.v[s][keep, h // group]
                x = k @ self.q[s, h] * self.scale
                top = x.max()
                p = np.exp(x - top)
                total = p.sum()
                p /= total
                o[s, h] = p @ v
                lse[s, h] = top + np.log(total)
                b = (np.abs(k) @ np.abs(self.q[s, h])).max() * self.scale
                score = (d + 4) * 2.0 ** -24 * b
                mean = p @ np.abs(v)
                o_tol[s, h] = mean * (2.0 ** -8 * (1 + 2.0 ** -7) + 2 * score + 2.0 ** -20) \
                    + np.abs(o[s, h]) * 2.0 ** -8 * (1 + 2.0 ** -7)
                lse_tol[s, h] = score + 2.0 ** -20 + np.abs(lse[s, h]) * 2.0 ** -22
        return o, lse, o_tol, lse_tol

    def compare(self, got, want, lse=True):
        o, stat = got
        x = bf16_to_f32(o.download()).reshape(want[0].shape).astype(np.float64)
        off = np.abs(x - want[0])
        worst = np.unravel_index(np.argmax(off - want[2]), off.shape)
        assert np.all(off <= want[2]), (worst, x[worst], want[0][worst], want[2][worst])
        # a row of no keys is +0, not -0
        empty = np.isneginf(want[1])
        assert not np.any(o.download().reshape(want[0].shape)[empty])
        y = stat.download().reshape(want[1].shape).astype(np.float64)
        if not lse:
            assert np.all(y == 7.0)
            return
        assert np.array_equal(np.isneginf(y), empty)
        with np.errstate(invalid="ignore"):
            off = np.where(empty, 0.0, np.abs(y - want[1]))
        assert np.all(off <= want[3]), (off.max(), want[3][np.unravel_index(off.argmax(), off.shape)])

    def inputs_unchanged(self):
        return all(a.unchanged() for a in
                   self.arrays + self.scales + [self.dev_q, self.dev_table, self.dev_lengths])


def _check(gpu, fmt, lengths, q_heads, kv_heads, head_dim, page_size, window=0, **more):
    b = Batch(gpu, fmt, lengths, q_heads, kv_heads, head_dim, page_size, **more)
    b.compare(b.run(window), b.reference(window))
    assert b.inputs_unchanged()


FORMATS = ["bf16", "e4m3"]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("lengths", [[1], [0], [0, 1, 2], [31, 32, 33], [127, 128, 129, 0],
                                     [255, 256, 257], [500], [1000, 3, 0, 700]])
def test_lengths(gpu, fmt, head_dim, lengths):
    _check(gpu, fmt, lengths, 8, 2, head_dim, 16)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (4, 4), (3, 1), (28, 4), (16, 1), (17, 1),
                                              (32, 1), (66, 2), (48, 1), (64, 1), (65, 1),
                                              (200, 2)])
def test_groups(gpu, fmt, q_heads, kv_heads):
    _check(gpu, fmt, [70, 700], q_heads, kv_heads, 128, 16)
    _check(gpu, fmt, [70, 700], q_heads, kv_heads, 64, 16)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("page_size", [1, 3, 7, 24, 32, 40, 64, 256, 1000])
@pytest.mark.parametrize("order", ["token", "head"])
def test_pages(gpu, fmt, head_dim, page_size, order):
    _check(gpu, fmt, [333, 1, 95], 8, 4, head_dim, page_size, order=order)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("order", ["token", "head"])
def test_strides(gpu, fmt, order):
    _check(gpu, fmt, [300, 41], 6, 2, 128, 16, order=order, pad=16, q_pad=24, cols=50)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 512, 5000])
def test_windows(gpu, fmt, window):
    _check(gpu, fmt, [0, 1, 32, 33, 450, 1600], 8, 2, 64, 16, window=window)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("q_heads,kv_heads", [(4, 2), (8, 4), (20, 1)])
@pytest.mark.parametrize("window", [1500, 2047, 2048, 2049])
def test_windows_over_many_runs(gpu, fmt, q_heads, kv_heads, window):
    _check(gpu, fmt, [5000, 0, 1999, 2100, 7000], q_heads, kv_heads, 64, 16, window=window)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lengths,q_heads,kv_heads,head_dim,page_size", [
    ([40001], 2, 1, 128, 16),           # one head of one sequence in as many runs as there are
    ([5000, 1, 0, 0, 9000, 33], 8, 2, 64, 16),
    ([2500] * 40, 4, 2, 128, 32),       # runs that end anywhere in a sequence
    ([int(x) for x in np.linspace(0, 700, 150)], 2, 1, 64, 8),  # more than a wave's lanes of sequences
    ([300] * 3 + [0] * 200 + [4000], 2, 2, 64, 64),
    # a multiple of four KV heads: a wave each
    ([40001], 8, 4, 128, 16),
    ([5000, 1, 0, 0, 9000, 33], 16, 8, 64, 16),
    ([1500, 1501, 1499, 31] * 6, 64, 4, 128, 32),
    ([int(x) for x in np.linspace(0, 1400, 70)], 4, 4, 64, 8),
    # more than one tile of query rows, more than one block of 64
    ([5000, 1, 0, 4000, 33], 20, 1, 128, 16),
    ([2500] * 9, 48, 1, 64, 16),
    ([3000, 2999, 40], 64, 1, 128, 16),
    ([3000, 0, 1700], 150, 1, 64, 16),
])
def test_many_runs(gpu, fmt, lengths, q_heads, kv_heads, head_dim, page_size):
    _check(gpu, fmt, lengths, q_heads, kv_heads, head_dim, page_size)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("seqs", [65, 129, 700, 4300])  # to several chunks of a wave's lanes
@pytest.mark.parametrize("q_heads,kv_heads", [(2, 1), (4, 4)])
def test_many_sequences(gpu, fmt, seqs, q_heads, kv_heads):
    """More heads than runs, so that most lie within one, and a long sequence
    among them that takes several; the last ones are empty."""
    lengths = [37 * i % 151 for i in range(seqs - 2)] + [0, 0]
    lengths[seqs // 3] = 2000
    lengths[seqs // 2] = 1300
    _check(gpu, fmt, lengths, q_heads, kv_heads, 64, 16)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lengths,q_heads,kv_heads,head_dim", [
    ([40001], 8, 4, 128), ([5000, 1, 0, 0, 9000, 33], 16, 8, 64),
    ([1500, 1501, 1499, 31] * 6, 64, 4, 128), ([37 * i % 151 for i in range(700)], 4, 4, 64),
])
def test_four_heads_a_workgroup(gpu, fmt, lengths, q_heads, kv_heads, head_dim):
    """A table with room for much longer sequences, for which four KV heads share a
    workgroup whatever the lengths are."""
    b = Batch(gpu, fmt, lengths, q_heads, kv_heads, head_dim, 64, cols=1700)
    b.compare(b.run(max_length=1700 * 64), b.reference())
    assert b.inputs_unchanged()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("q_heads", [20, 48, 70])  # 70: two blocks of query rows
def test_many_sequences_of_many_query_heads(gpu, fmt, q_heads):
    lengths = [41 * i % 97 for i in range(300)]
    lengths[7] = 1500
    lengths[298] = 1400
    _check(gpu, fmt, lengths, q_heads, 1, 64, 16)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("q_heads,kv_heads", [(33, 1), (48, 1), (98, 2), (64, 1)])
@pytest.mark.parametrize("window", [0, 33, 700])
def test_waves_that_share_tiles(gpu, fmt, head_dim, q_heads, kv_heads, window):
    """More than 32 query heads a KV head: runs of every number of tiles that leaves some
    of the four teams without one, pages that end inside tiles, rows that end inside a
    wave's, and calls of one workgroup a head as well as many."""
    _check(gpu, fmt, [1, 31, 33, 95, 130, 0, 257], q_heads, kv_heads, head_dim, 24, window=window)
    _check(gpu, fmt, [2500, 0, 33, 1300], q_heads, kv_heads, head_dim, 40, window=window)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("peak", [30.0, 1e-3])
def test_peaked_and_flat_scores(gpu, fmt, peak):
    """Scores up to several hundred, where one key has almost all of the weight
    and the running reference rises often, and scores of nearly 0."""
    _check(gpu, fmt, [900, 64, 3000], 8, 2, 128, 16, peak=peak)
    _check(gpu, fmt, [900, 64, 3000], 8, 4, 64, 16, peak=peak)
    _check(gpu, fmt, [900, 64, 3000], 36, 1, 128, 16, peak=peak)


def _split(y, parts):
    """f32 values as the sum of one or two bf16 parts, by rounding to nearest."""
    first = bf16_to_f32(_bf16_bits(y)).astype(np.float32)
    if parts == 1:
        return first.astype(np.float64)
    return first.astype(np.float64) + bf16_to_f32(_bf16_bits(y - first)).astype(np.float64)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("q_heads,kv_heads", [(8, 2), (16, 4), (20, 1), (40, 1), (64, 1)])
def test_probabilities_keep_sixteen_bits(gpu, fmt, head_dim, q_heads, kv_heads):
    """Keys of two scores by turns whose weighted values cancel: with probabilities
    (times the V scale) in one bf16 part the result would be off by some 2^-10 of the
    mean magnitude A that it sums, which the one-part result below shows; two leave
    2^-16.  The other errors: a score is one product here, exact, so its scalings,
    exp2 and the products with scales move a probability by less than 2^-21; sums of
    fp32 that cancel pair by pair, 2^-21 of A; the sum of the probabilities moves o
    in proportion alone, by 2^-16 of it at most, and the output's rounding by 2^-8."""
    lengths = [96, 2500, 640]
    b = Batch(gpu, fmt, lengths, q_heads, kv_heads, head_dim, 16)
    q = np.zeros_like(b.q)
    q[..., 0] = 1.0
    b.q = q
    b.dev_q = Guarded(gpu, _bf16_bits(q))
    rng = np.random.default_rng(head_dim)
    sign = np.where(np.arange(head_dim) % 2, -1.0, 1.0)

    def error(y):  # of one part
        return _split(y, 1) - y
    if fmt == "bf16":
        # the score of the second kind: the probability that one part rounds most
        c = -bf16_to_f32(np.arange(0x3F80, 0x40A0, dtype=np.uint16)).astype(np.float64)
        p = np.exp(c * b.scale).astype(np.float32)
        at = np.argmax(np.abs(error(p)) / p)
        score, weight = c[at], [1.0, float(p[at])]
        v = bf16_to_f32(_bf16_bits(rng.uniform(0.5, 1.0, head_dim))).astype(np.float64) * sign
        w = -bf16_to_f32(_bf16_bits(v / weight[1])).astype(np.float64)
        k_rows = [0, int(_bf16_bits(np.float32(score)))]
        v_rows, v_scales = [_bf16_bits(v), _bf16_bits(w)], None
        values = [v, w]
    else:
        # codes 1 and -1.5, with V scales that make them cancel: t, and t / 1.5 over p
        t = np.linspace(1.0, 2.0, 4097, dtype=np.float32)[:-1]
        t = t[np.argmax(np.abs(error(t) - 1.5 * error(t / np.float32(1.5))))]
        k_scale = np.float32(3.0)
        score = -3.0
        p = np.float32(np.exp(score * b.scale))
        v_scales = [np.float32(t), np.float32(np.float64(t) / 1.5 / np.float64(p))]
        weight = [float(t), float(np.float32(p * v_scales[1]))]
        k_rows = [0, 0xB8]
        v_rows = [np.where(sign > 0, 0x38, 0xB8), np.where(sign > 0, 0xBC, 0x3C)]
        values = [sign, -1.5 * sign]
    size = 2 if fmt == "bf16" else 1
    flats = [a.download() for a in b.arrays]
    rows = [np.lib.stride_tricks.as_strided(x, b.shape, [size * s for s in b.strides] + [size])
            for x in flats]
    if fmt == "e4m3":
        scale_flats = [a.download() for a in b.scales]
        scales = [x.reshape(b.shape[0], kv_heads, 16) for x in scale_flats]
    for s, count in enumerate(lengths):
        for kind in range(2):
            key = np.arange(kind, count, 2)
            page, place = b.table[s, key // 16], key % 16
            rows[0][page, place] = 0
            rows[0][page, place, :, 0] = k_rows[kind]
            rows[1][page, place] = v_rows[kind]
            if fmt == "e4m3":
                scales[0][page, :, place] = k_scale
                scales[1][page, :, place] = v_scales[kind]
    for a, x in zip(b.arrays, flats):
        a.body.upload(x)
    if fmt == "e4m3":
        for a, x in zip(b.scales, scale_flats):
            a.body.upload(x)
    # every sequence has as many of each kind: o of one pair
    total = 1.0 + float(np.exp(np.float64(score) * b.scale))
    exact_weight = ([1.0, total - 1.0] if fmt == "bf16" else
                    [float(v_scales[0]), (total - 1.0) * float(v_scales[1])])
    want = sum(w * v for w, v in zip(exact_weight, values)) / total
    mean = sum(w * np.abs(v) for w, v in zip(exact_weight, values)) / total
    tol = mean * (2.0 ** -16 + 2.0 ** -20) + np.abs(want) * (2.0 ** -8 * (1 + 2.0 ** -6))

    def emulated(parts):
        x = sum(_split(np.float32(w), parts) * v for w, v in zip(weight, values)) / total
        return bf16_to_f32(_bf16_bits(x.astype(np.float32))).astype(np.float64)
    assert np.all(np.abs(emulated(2) - want) <= tol)
    assert np.all(np.abs(emulated(1) - want) > 4 * tol)
    o, _ = b.run()
    x = bf16_to_f32(o.download()).reshape(len(lengths), q_heads, head_dim).astype(np.float64)
    off = np.abs(x - want)
    assert np.all(off <= tol), (off / tol).max()


def test_rising_scores(gpu):
    """Keys in rising order of score raise the reference in every tile."""
    b = Batch(gpu, "bf16", [2000], 4, 1, 128, 16)
    q = np.zeros_like(b.q)
    q[..., 0] = 1.0
    b.q = q
    b.dev_q = Guarded(gpu, _bf16_bits(q))
    x = b.k[0]
    x[:, 0, 0] = bf16_to_f32(_bf16_bits(np.linspace(-3000.0, 3000.0, 2000))).astype(np.float64)
    flat = b.arrays[0].download()
    rows = np.lib.stride_tricks.as_strided(flat, b.shape, [2 * s for s in b.strides] + [2])
    key = np.arange(2000)
    rows[b.table[0, key // 16], key % 16] = _bf16_bits(x)
    b.arrays[0].body.upload(flat)
    b.arrays[0].initial[64:64 + flat.size] = flat
    b.compare(b.run(), b.reference())


@pytest.mark.parametrize("fmt", FORMATS)
def test_length_above_max_length(gpu, fmt):
    b = Batch(gpu, fmt, [500, 20, 333], 8, 2, 128, 16)
    for most in (0, 1, 300, 333):
        b.compare(b.run(max_length=most), b.reference(max_length=most))
        b.compare(b.run(max_length=most, window=40), b.reference(max_length=most, window=40))
    b.dev_lengths.body.upload(np.array([0xFFFFFFFF, 20, 333], np.uint32))
    b.compare(b.run(max_length=500), b.reference())


@pytest.mark.parametrize("fmt", FORMATS)
def test_pages_out_of_range_are_left_out(gpu, fmt):
    b = Batch(gpu, fmt, [200, 64, 700, 16], 8, 2, 128, 16)
    bad = b.table.copy()
    bad[0, 3] = b.shape[0]
    bad[1, :] = 0xFFFFFFFF  # all of a sequence's pages
    bad[2, 40] = 0x80000000
    bad[3, 0] = b.shape[0]
    b.dev_table.body.upload(bad.ravel())

    def drop(s, key):
        return bad[s, key // 16] >= b.shape[0]
    b.compare(b.run(), b.reference(drop=drop))


@pytest.mark.parametrize("kv_heads", [2, 4])
def test_without_lse_and_repeated(gpu, kv_heads):
    b = Batch(gpu, "bf16", [4000, 17, 900], 8, kv_heads, 128, 16)
    b.compare(b.run(lse=False), b.reference(), lse=False)
    first, second = b.run(), b.run()
    assert_same(first[0].download(), second[0].download())
    assert_same(first[1].download(), second[1].download())


@pytest.mark.parametrize("length", [300, 3000])
def test_nonfinite_values_of_kept_keys(gpu, length):
    """A NaN key or value shows in its own sequence and KV head only."""
    b = Batch(gpu, "bf16", [length, length], 4, 2, 64, 16)
    want = b.reference()
    flat = b.arrays[0].download()
    rows = np.lib.stride_tricks.as_strided(flat, b.shape, [2 * s for s in b.strides] + [2])
    rows[b.table[1, 5], 3, 1, 7] = 0x7FC0
    b.arrays[0].body.upload(flat)
    o, stat = b.run()
    x = bf16_to_f32(o.download()).reshape(2, 4, 64)
    assert np.all(np.isnan(x[1, 2:])) and np.all(np.isnan(stat.download().reshape(2, 4)[1, 2:]))
    x[1, 2:] = 0.0
    clean = np.where(np.isnan(x), np.inf, x)
    want[0][1, 2:] = 0.0
    assert np.all(np.abs(clean - want[0]) <= want[2])


@pytest.mark.parametrize("length", [1, 300, 3000])
@pytest.mark.parametrize("q_heads,kv_heads", [(4, 2), (16, 4), (40, 2), (49, 1)])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_infinite_values_of_kept_keys(gpu, length, q_heads, kv_heads, head_dim):
    """An infinite element of a kept V row is that element's result, whatever
    rounding its key's probability has, the largest (1, exactly) among them; the
    other elements are as they would be."""
    b = Batch(gpu, "bf16", [length, length], q_heads, kv_heads, head_dim, 16)
    want = b.reference()
    flat = b.arrays[1].download()
    rows = np.lib.stride_tricks.as_strided(flat, b.shape, [2 * s for s in b.strides] + [2])
    first = (kv_heads - 1) * (q_heads // kv_heads)
    p = b.k[1][:, -1] @ b.q[1, first] * b.scale
    keys = [int(np.argmax(p)), length // 2, length - 1]
    elements = [7, 20, 33]
    for key, element in zip(keys, elements):
        rows[b.table[1, key // 16], key % 16, -1, element] = 0xFF80 if element == 20 else 0x7F80
    b.arrays[1].body.upload(flat)
    o, stat = b.run()
    x = bf16_to_f32(o.download()).reshape(2, q_heads, head_dim)
    for element in elements:
        assert np.all(x[1, first:, element] == (-np.inf if element == 20 else np.inf))
    x[1, first:, elements] = want[0][1, first:, elements]
    assert not np.any(np.isnan(x)) and np.all(np.abs(x - want[0]) <= want[2])
    off = np.abs(stat.download().reshape(want[1].shape) - want[1])
    assert np.all(off <= want[3])


def test_shared_pages(gpu):
    """Two sequences with a common prefix on the same pages."""
    b = Batch(gpu, "e4m3", [640, 640], 8, 2, 128, 16)
    b.table[1, :30] = b.table[0, :30]
    b.dev_table.body.upload(b.table.ravel())
    for x in (b.k, b.v):
        x[1][:480] = x[0][:480]
    b.compare(b.run(), b.reference())


def test_offsets_past_32_bits(gpu):
    """Pages more than 2^32 bytes apart."""
    kern = _k()
    stride, page_size, d = (1 << 31) + 64, 32, 128
    pages = 3
    extent = (pages - 1) * stride + page_size * d
    k, v = gpu.alloc(extent, np.uint16), gpu.alloc(extent, np.uint16)
    cache = kern.KvCache(k, v, shape=(pages, page_size, 1, d), strides=(stride, d, d))
    b = Batch(gpu, "bf16", [90], 4, 1, d, page_size, slack=0)
    for buf, held in ((k, b.k), (v, b.v)):
        for col, page in enumerate(b.table[0]):
            rows = np.zeros((page_size, d))
            part = held[0][col * page_size:(col + 1) * page_size, 0]
            rows[:len(part)] = part
            buf.view(int(page) * stride, page_size * d).upload(_bf16_bits(rows).ravel())
    b.cache = cache
    b.compare(b.run(), b.reference())
    k.free()
    v.free()


def test_more_heads_than_a_grid_row(gpu):
    """2^21 sequences and some of up to four keys, a workgroup each, with the bound of
    the other tests (scores of at most 64 in magnitude)."""
    torch = pytest.importorskip("torch")
    kern = _k()
    seqs, d, page_size, pages = (1 << 21) + 5, 64, 4, 50
    g = torch.Generator(device="cuda").manual_seed(2)
    k, v = (torch.randn(pages, page_size, 1, d, device="cuda", generator=g).bfloat16()
            for _ in "kv")
    q = torch.randn(seqs, 1, d, device="cuda", generator=g).bfloat16()
    lengths = torch.randint(0, 5, (seqs,), device="cuda", generator=g)
    lengths[-5:] = torch.tensor([4, 0, 1, 3, 4], device="cuda")
    table = torch.randint(0, pages, (seqs, 1), dtype=torch.int32, device="cuda", generator=g)
    out = torch.full_like(q, 3.0)
    lse = torch.full((seqs, 1), 7.0, device="cuda")
    ws = torch.empty(kern.paged_attention_workspace_bytes(1, 1, d), dtype=torch.uint8,
                     device="cuda")
    kern.paged_attention_decode(kern.KvCache(k, v), q, table, lengths.to(torch.int32), out, lse,
                                ws, max_length=4, scale=0.125)
    step = 1 << 19
    for at in range(0, seqs, step):
        part = slice(at, min(at + step, seqs))
        keys, values = (x[table[part, 0].long(), :, 0].double() for x in (k, v))
        x = (keys * q[part].double()).sum(-1) * 0.125
        x = x.masked_fill(torch.arange(4, device="cuda") >= lengths[part, None], -np.inf)
        assert x.max() <= 64.0
        empty = lengths[part] == 0
        p = torch.softmax(torch.where(empty[:, None], 0.0, x), -1) * ~empty[:, None]
        want = (p[..., None] * values).sum(1)
        mean = (p[..., None] * values.abs()).sum(1)
        tol = mean * (2.0 ** -8 * (1 + 2.0 ** -7) + 2 * 68 * 2.0 ** -18 + 2.0 ** -20) \
            + want.abs() * 2.0 ** -8 * (1 + 2.0 ** -7)
        assert torch.all((out[part, 0].double() - want).abs() <= tol), at
        assert not torch.any(out[part, 0][empty].view(torch.int16))
        full = torch.logsumexp(x, -1)
        off = torch.where(empty, 0.0, (lse[part, 0].double() - full).abs())
        assert torch.all(off <= 68 * 2.0 ** -18 + 2.0 ** -20 + 64 * 2.0 ** -22)
        assert torch.equal(torch.isneginf(lse[part, 0]), empty)


# ---- together, as a program uses them -----------------------------------------------------

@pytest.mark.parametrize("fmt", FORMATS)
def test_prompt_then_steps(gpu, fmt):
    """A prompt through fe2o3_flash_attention_fwd, its K and V into the cache, then
    tokens one by one: each step's attention is that of the prompt kernel's last
    row over everything so far (bf16; both within their bound of 64 bits), and of
    the values that the cache holds (e4m3)."""
    kern = _k()
    heads, d, page_size, prompt, steps = 4, 128, 16, 100, 5
    total = prompt + steps
    rng = np.random.default_rng(11)
    q, k, v = (_bf16_bits(rng.standard_normal((heads, total, d))) for _ in range(3))
    pages = 16
    dtype = np.uint16 if fmt == "bf16" else np.uint8
    arrays = [gpu.to_device(np.full(pages * page_size * heads * d, 0x7F, dtype)) for _ in "kv"]
    scales = [gpu.to_device(np.full(pages * heads * page_size, np.nan, np.float32))
              for _ in "kv"] if fmt == "e4m3" else [None, None]
    cache = kern.KvCache(*arrays, *scales, shape=(pages, page_size, heads, d))
    table = rng.permutation(pages)[:-(-total // page_size)].astype(np.uint32)
    slot = lambda t: (table[t // page_size] * page_size + t % page_size).astype(np.uint32)  # noqa: E731

    def flash(n):
        o, lse = gpu.alloc(heads * n * d, np.uint16), gpu.alloc(heads * n, np.float32)
        kern.flash_attention_fwd_gpu.Kernel.load(gpu).prepare(
            *(gpu.to_device(np.ascontiguousarray(x[:, :n]).ravel()) for x in (q, k, v)), o, lse,
            1, heads, n, d, 1, d ** -0.5).launch()
        return (bf16_to_f32(o.download()).reshape(heads, n, d)[:, -1].astype(np.float64),
                lse.download().reshape(heads, n)[:, -1])

    # [heads, seq, head_dim] rows of the prompt, as the prompt kernel takes them
    kern.kv_cache_write(cache, *(gpu.to_device(np.ascontiguousarray(x[:, :prompt]).ravel())
                                 for x in (k, v)),
                        gpu.to_device(slot(np.arange(prompt))), strides=(d, prompt * d))
    workspace = gpu.alloc(kern.paged_attention_workspace_bytes(heads, heads, d), np.uint8)
    dtable = gpu.to_device(table)
    out, lse = gpu.alloc(heads * d, np.uint16), gpu.alloc(heads, np.float32)
    for step in range(steps):
        t = prompt + step
        kern.kv_cache_write(cache, *(gpu.to_device(np.ascontiguousarray(x[:, t]).ravel())
                                     for x in (k, v)), gpu.to_device(slot(np.arange(t, t + 1))),
                            sync=False)
        kern.paged_attention_decode(
            cache, gpu.to_device(np.ascontiguousarray(q[:, t]).ravel()), dtable,
            gpu.to_device(np.array([t + 1], np.uint32)), out, lse, workspace, max_length=total,
            scale=d ** -0.5, q_heads=heads)
        got = bf16_to_f32(out.download()).reshape(heads, d).astype(np.float64)
        b = Batch.__new__(Batch)
        b.lengths, b.q_heads, b.kv_heads, b.head_dim, b.scale = [t + 1], heads, heads, d, d ** -0.5
        b.q = bf16_to_f32(q[:, t]).astype(np.float64)[None]
        read = [gpu.alloc((t + 1) * heads * d, np.uint16) for _ in "kv"]
        kern.kv_cache_read(cache, dtable, gpu.to_device(np.array([0, t + 1], np.uint32)), *read)
        if fmt == "bf16":
            for x, y in zip((k, v), read):
                assert_same(y.download().reshape(t + 1, heads, d),
                            np.ascontiguousarray(x[:, :t + 1].transpose(1, 0, 2)))
            b.k, b.v = ([bf16_to_f32(x[:, :t + 1]).transpose(1, 0, 2).astype(np.float64)]
                        for x in (k, v))
        else:
            held = []
            for x, s in zip(arrays, scales):
                key = np.arange(t + 1)
                page, place = table[key // page_size], key % page_size
                codes = x.download().reshape(pages, page_size, heads, d)[page, place]
                sc = s.download().reshape(pages, heads, page_size)[page, :, place]
                held.append([_decode_table()[codes].astype(np.float64)
                             * sc.astype(np.float64)[..., None]])
            b.k, b.v = held
        o, want_lse, o_tol, lse_tol = b.reference()
        assert np.all(np.abs(got - o[0]) <= o_tol[0])
        assert np.all(np.abs(lse.download() - want_lse[0]) <= lse_tol[0])
        if fmt == "bf16":
            last, last_lse = flash(t + 1)
            assert np.all(np.abs(got - last) <= 2 * o_tol[0])
            assert np.all(np.abs(lse.download() - last_lse) <= 2 * lse_tol[0])


class _Graph:
    """Two calls captured on one stream into a HIP graph."""

    def __init__(self, stream):
        self.hip = C.CDLL("libamdhip64.so")
        self.stream = C.c_void_p(stream.handle)
        self.ready = C.c_void_p()

    def __enter__(self):
        assert self.hip.hipStreamBeginCapture(self.stream, 2) == 0  # relaxed
        return self

    def __exit__(self, *failure):
        graph = C.c_void_p()
        rc = self.hip.hipStreamEndCapture(self.stream, C.byref(graph))
        if failure[0] is None:
            assert rc == 0
            assert self.hip.hipGraphInstantiate(C.byref(self.ready), graph, None, None,
                                                C.c_size_t(0)) == 0
        if graph:
            self.hip.hipGraphDestroy(graph)

    def replay(self):
        assert self.hip.hipGraphLaunch(self.ready, self.stream) == 0


@pytest.mark.parametrize("fmt", FORMATS)
def test_captured_and_replayed(gpu, fmt):
    """A step (write, then attention) in a graph, replayed while lengths, slots,
    rows and the table change between the replays and other work runs: every
    replay gives the eager call's bits.  Two graphs share one workspace, one
    behind the other."""
    kern = _k()
    b = Batch(gpu, fmt, [900, 64, 33, 2000], 8, 2, 128, 16, slack=40)
    rng = np.random.default_rng(3)
    stream = gpu.stream()
    n = kern.paged_attention_workspace_bytes(8, 2, 128)
    workspace = Guarded(gpu, np.full(n, 0xFF, np.uint8))
    new = [gpu.alloc(4 * 2 * 128, np.uint16) for _ in "kv"]
    slots = gpu.alloc(4, np.uint32)
    outs = [b.outputs(), b.outputs()]

    def step(out, window, on, sync):
        kern.kv_cache_write(b.cache, *new, slots, stream=on, sync=False)
        b_run = dict(max_length=2048, scale=b.scale, window=window, q_heads=8)
        kern.paged_attention_decode(b.cache, b.dev_q.body, b.dev_table.body, b.dev_lengths.body,
                                    out[0].body, out[1].body, workspace.body, stream=on,
                                    sync=sync, **b_run)

    cols = 2048 // 16
    table = np.zeros((4, cols), np.uint32)
    table[:, :b.cols] = np.minimum(b.table, b.shape[0] - 1)
    b.dev_table = Guarded(gpu, table)
    for x in new:
        x.upload(_bf16_bits(rng.standard_normal(x.count)))
    slots.upload(np.full(4, 0xFFFFFFFF, np.uint32))
    gpu.synchronize()
    graphs = []
    for out, window in zip(outs, (0, 100)):
        with _Graph(stream) as graph:
            step(out, window, stream, False)
        graphs.append(graph)
    lengths = np.array(b.lengths)
    for turn in range(4):
        page = table[np.arange(4), lengths // 16].copy()
        fresh = lengths % 16 == 0
        page[fresh] = b.shape[0] - 1 - 4 * turn - np.arange(4)[fresh]
        table[np.arange(4), lengths // 16] = page
        b.dev_table.body.upload(table.ravel())
        slots.upload((page * 16 + lengths % 16).astype(np.uint32))
        for x in new:
            x.upload(_bf16_bits(rng.standard_normal(x.count)))
        lengths = lengths + 1 if turn != 2 else np.array([5, 0, 1999, 700])
        b.dev_lengths.body.upload(lengths.astype(np.uint32))
        for graph in graphs:
            graph.replay()
        stream.synchronize()
        for out, window in zip(outs, (0, 100)):
            eager = b.outputs()
            step(eager, window, None, True)
            assert_same(out[0].download(), eager[0].download(), f"turn {turn}")
            assert_same(out[1].download(), eager[1].download(), f"turn {turn} lse")
            assert out[0].guards_intact() and out[1].guards_intact()
    assert workspace.guards_intact()


@pytest.mark.parametrize("fmt", FORMATS)
def test_two_calls_at_once(gpu, fmt):
    """Steps on two streams, each with its own cache and workspace, side by side: the
    bits of the same calls alone."""
    batches = [Batch(gpu, fmt, [9000, 0, 33, 2000], 8, 2, 128, 16, seed=1),
               Batch(gpu, fmt, [700 + 5 * i for i in range(90)], 48, 1, 64, 24, seed=2)]
    alone = [b.run() for b in batches]
    for b, got in zip(batches, alone):
        b.compare(got, b.reference())
    streams = [gpu.stream() for _ in batches]
    kern = _k()
    spaces = [Guarded(gpu, np.full(kern.paged_attention_workspace_bytes(
        b.q_heads, b.kv_heads, b.head_dim), 0xFF, np.uint8)) for b in batches]
    outs = [[b.outputs() for _ in range(4)] for b in batches]
    gpu.synchronize()
    for turn in range(4):
        for b, stream, space, out in zip(batches, streams, spaces, outs):
            kern.paged_attention_decode(
                b.cache, b.dev_q.body, b.dev_table.body, b.dev_lengths.body, out[turn][0].body,
                out[turn][1].body, space.body, max_length=max(b.lengths), scale=b.scale,
                q_heads=b.q_heads, stream=stream, sync=False)
    gpu.synchronize()
    for b, want, out in zip(batches, alone, outs):
        for o, stat in out:
            assert_same(o.download(), want[0].download())
            assert_same(stat.download(), want[1].download())
            assert o.guards_intact() and stat.guards_intact()
    assert all(space.guards_intact() for space in spaces)


def test_tensors_and_streams(gpu):
    """The same calls on torch tensors, on a stream of torch's own, with K and V in
    one allocation and the rows columns of a fused projection."""
    torch = pytest.importorskip("torch")
    kern = _k()
    g = torch.Generator(device="cuda").manual_seed(1)
    pages, page_size, heads, d, q_heads = 20, 16, 2, 64, 6
    both = torch.zeros(pages, 2, heads, page_size, d, device="cuda", dtype=torch.bfloat16)
    cache = kern.KvCache(both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2))
    rows = torch.randn(150, q_heads + 2 * heads, d, generator=g, device="cuda").bfloat16()
    k, v = rows[:, q_heads:q_heads + heads], rows[:, q_heads + heads:]
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)[None, :10].contiguous()
    at = torch.arange(150, device="cuda")
    slots = (table[0, at // page_size].long() * page_size + at % page_size).to(torch.int32)
    lengths = torch.tensor([150], device="cuda", dtype=torch.int32)
    out = torch.empty(1, q_heads, d, device="cuda", dtype=torch.bfloat16)
    lse = torch.empty(1, q_heads, device="cuda")
    ws = torch.empty(kern.paged_attention_workspace_bytes(q_heads, heads, d), dtype=torch.uint8,
                     device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    kern.kv_cache_write(cache, k, v, slots, stream=stream, sync=False)
    kern.paged_attention_decode(cache, rows[149:, :q_heads], table, lengths, out, lse, ws,
                                max_length=160, scale=0.125, stream=stream)
    x = torch.einsum("ghd,thd->hgt", rows[149, :q_heads].double().view(heads, 3, d).transpose(0, 1),
                     k.double()) * 0.125
    want = torch.matmul(torch.softmax(x, -1), v.double().transpose(0, 1).contiguous())
    assert torch.allclose(out[0].double().view(heads, 3, d), want, atol=2.0 ** -7, rtol=2.0 ** -7)
    assert torch.allclose(lse[0].double().view(heads, 3), torch.logsumexp(x, -1), atol=1e-5)
    back = [torch.full((152, heads, d), 3.0, device="cuda", dtype=torch.bfloat16) for _ in "kv"]
    starts = torch.tensor([1, 151], device="cuda", dtype=torch.int32)
    kern.kv_cache_read(cache, table, starts, *back)
    for a, b in zip((k, v), back):
        assert torch.equal(b[1:151], a) and torch.all(b[0] == 3.0) and torch.all(b[151] == 3.0)
