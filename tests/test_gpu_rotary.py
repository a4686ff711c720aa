"""fe2o3_rotary on the GPU against the rotation in 64 bits.

Bound of one output, m the scale, (a, b) its pair: the sine and cosine are f32 values of
an angle that is off by 2^-25 of a turn's half at most (pi 2^-24) and rounded with a few
units of 2^-24, then times m: 2^-21 |m| (|a| + |b|) with the two products and the sum;
and the output's own rounding, 2^-8 of it for bf16, 2^-24 for f32."""
from __future__ import annotations

import numpy as np
import pytest

from gpu_util import Guarded, assert_same, bf16_to_f32
from test_gpu_mxfp4 import _bf16_bits

pytestmark = pytest.mark.gpu

NO_SLOT = 0xFFFFFFFF


def _k():
    from fe2o3_amd import kernels
    return kernels


def _turned(x, positions, freq, interleaved, inverse, scale):
    """(result, sum of magnitudes of each output's pair) of x [tokens, heads, d] in 64 bits."""
    r = 2 * len(freq)
    x = x.astype(np.float64)
    # the angle in extended precision: 64 bits of position * freq
    t = (positions.astype(np.longdouble)[:, None] * freq.astype(np.longdouble))[:, None]
    c, s = np.cos(t).astype(np.float64), np.sin(t).astype(np.float64)
    if inverse:
        s = -s
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    p, q = scale * (a * c - b * s), scale * (b * c + a * s)
    size = abs(scale) * (np.abs(a) + np.abs(b))
    y, m = x.copy(), np.zeros_like(x)
    if interleaved:
        y[..., 0:r:2], y[..., 1:r:2] = p, q
        m[..., 0:r:2] = m[..., 1:r:2] = size
    else:
        y[..., :r // 2], y[..., r // 2:r] = p, q
        m[..., :r // 2] = m[..., r // 2:r] = size
    return y, m


class Rows:
    """Rows [tokens, heads, d] in a guarded array with strides, NaN between them."""

    def __init__(self, gpu, rng, fmt, tokens, heads, d, pad=0, heads_first=False, offset=0):
        self.fmt, self.shape = fmt, (tokens, heads, d)
        row = d + pad
        self.strides = (row, tokens * row) if heads_first else (heads * row + pad, row)
        n = (tokens - 1) * self.strides[0] + (heads - 1) * self.strides[1] + d
        flat = np.full(offset + n, np.nan, np.float32) if fmt == "f32" else \
            np.full(offset + n, 0x7F81, np.uint16)  # a signalling NaN
        self.offset = offset
        view = self.view(flat)
        x = rng.standard_normal(self.shape) * np.exp2(rng.integers(-8, 8, self.shape))
        view[...] = x if fmt == "f32" else _bf16_bits(x)
        self.values = view.copy() if fmt == "f32" else bf16_to_f32(view)
        self.dev = Guarded(gpu, flat)
        self.body = self.dev.full.view(64 + offset, n)

    def view(self, flat):
        size = flat.dtype.itemsize
        return np.lib.stride_tricks.as_strided(flat[self.offset:], self.shape,
                                               (self.strides[0] * size, self.strides[1] * size, size))

    def check(self, x, positions, freq, interleaved, inverse, scale, before):
        """The result of rows x; `before`: this array's bytes before the call."""
        assert self.dev.guards_intact()
        got = self.dev.download()
        kept = positions == NO_SLOT
        view, old = self.view(got), self.view(before)
        want, size = _turned(x, np.where(kept, 0, positions), freq, interleaved, inverse, scale)
        y = (view if self.fmt == "f32" else bf16_to_f32(view)).astype(np.float64)
        step = 2.0 ** -24 if self.fmt == "f32" else 2.0 ** -8
        bound = np.abs(want) * step * 1.01 + size * 2.0 ** -21 + 1e-44
        off = np.abs(y - want)[~kept]
        assert np.all(off <= bound[~kept]), (off - bound[~kept]).max()
        assert_same(view[kept], old[kept], "skipped tokens")
        # between the rows, and elements that no row has
        rest = got.copy()
        self.view(rest)[...] = old
        assert_same(rest, before, "between the rows")


def _check(gpu, fmt, tokens, q_heads, k_heads, d, r, interleaved=False, inverse=False, scale=1.0,
           in_place=False, first=0, spread=5000, pad=0, heads_first=False, offset=0, skip=False):
    rng = np.random.default_rng([tokens, q_heads, d, r])
    freq = _k().rotary_frequencies(r, factor=4.0, schedule="by_turns")[0]
    positions = (first + rng.integers(0, spread, tokens)).astype(np.uint32)
    if skip:
        positions[::3] = NO_SLOT
    arrays = [Rows(gpu, rng, fmt, tokens, h, d, pad, heads_first, offset)
              for h in (q_heads, k_heads) if h]
    if in_place:
        outs, names = arrays, {}
    else:  # dense
        outs = [Rows(gpu, rng, fmt, tokens, h, d) for h in (q_heads, k_heads) if h]
        names = dict(q_out=outs[0].body)
        if k_heads:
            names["k_out"] = outs[1].body
    dp, df = Guarded(gpu, positions), gpu.to_device(freq)
    before = [o.dev.download() for o in outs]
    _k().rotary(arrays[0].body, arrays[1].body if k_heads else None, dp.body, df,
                interleaved=interleaved, inverse=inverse, scale=scale, q_shape=(q_heads, d),
                k_shape=(k_heads, d), q_strides=arrays[0].strides,
                k_strides=arrays[1].strides if k_heads else None, **names)
    for a, o, b in zip(arrays, outs, before):
        o.check(a.values, positions, freq, interleaved, inverse, scale, b)
        assert in_place or a.dev.unchanged()
    assert dp.unchanged()


@pytest.mark.parametrize("fmt", ["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,r", [(2, 2), (64, 64), (128, 128), (128, 64), (128, 36), (64, 20),
                                 (80, 80), (96, 32), (100, 6), (33, 32), (256, 256), (130, 128),
                                 (5000, 4096)])
def test_dimensions(gpu, fmt, interleaved, d, r):
    _check(gpu, fmt, 19, 3, 2, d, r, interleaved)


@pytest.mark.parametrize("fmt", ["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("scale", [1.0, 1.2, -0.5])
def test_directions(gpu, fmt, interleaved, inverse, in_place, scale):
    _check(gpu, fmt, 50, 8, 2, 128, 96, interleaved, inverse, scale, in_place, skip=True)


@pytest.mark.parametrize("tokens,q_heads,k_heads", [(1, 1, 0), (1, 32, 8), (2, 64, 1), (511, 4, 4),
                                                    (1023, 1, 0), (1024, 2, 1), (2049, 3, 1),
                                                    (5000, 2, 2)])
def test_sizes(gpu, tokens, q_heads, k_heads):
    _check(gpu, "bf16", tokens, q_heads, k_heads, 64, 64, skip=True)
    _check(gpu, "f32", tokens, q_heads, k_heads, 64, 48, True)


@pytest.mark.parametrize("fmt", ["bf16", "f32"])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("pad,heads_first,offset", [(1, False, 1), (8, False, 0), (3, True, 5)])
def test_strides(gpu, fmt, in_place, pad, heads_first, offset):
    _check(gpu, fmt, 45, 5, 3, 72, 64, False, False, 1.0, in_place, pad=pad,
           heads_first=heads_first, offset=offset, skip=True)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("first,spread", [(1 << 20, 1000), (1 << 24, 1 << 20), ((1 << 32) - 3000, 2000)])
def test_far_positions(gpu, interleaved, first, spread):
    """Angles of 10^6 radians and more, where 32 bits would be off by whole parts of a turn."""
    _check(gpu, "f32", 64, 2, 1, 128, 128, interleaved, first=first, spread=spread)


def test_there_and_back(gpu):
    """The inverse undoes the turn: two roundings of f32."""
    rng = np.random.default_rng(4)
    x = rng.standard_normal((300, 4, 64)).astype(np.float32)
    k = _k()
    dx = gpu.to_device(x.ravel())
    pos = gpu.to_device(rng.integers(0, 100000, 300).astype(np.uint32))
    freq = gpu.to_device(k.rotary_frequencies(64)[0])
    k.rotary(dx, None, pos, freq, q_shape=(4, 64))
    assert not np.array_equal(dx.download(), x.ravel())
    k.rotary(dx, None, pos, freq, q_shape=(4, 64), inverse=True)
    y = dx.download().reshape(x.shape)
    pair = np.abs(x[..., :32]) + np.abs(x[..., 32:])
    assert np.all(np.abs(y - x) <= np.concatenate([pair, pair], -1) * 2.0 ** -19)


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_is_the_transposed_map(gpu, interleaved):
    """<g, R x> = <R' g, x> for the map with a scale, and the gradient of a loss against
    differences of it: (L(x + h e) - L(x - h e)) / 2 h, exact for a linear map up to the
    roundings of f32, a few 2^-21 of the pair's size over h."""
    rng = np.random.default_rng(8)
    k = _k()
    x, g = (rng.standard_normal((20, 3, 48)).astype(np.float32) for _ in range(2))
    pos = gpu.to_device(rng.integers(0, 3000, 20).astype(np.uint32))
    freq = gpu.to_device(k.rotary_frequencies(32)[0])

    def turn(v, inverse):
        d = gpu.to_device(v.ravel())
        k.rotary(d, None, pos, freq, q_shape=(3, 48), interleaved=interleaved, inverse=inverse,
                 scale=1.3)
        return d.download().reshape(v.shape).astype(np.float64)

    grad = turn(g, True)
    assert abs((g * turn(x, False)).sum() - (grad * x).sum()) <= 2.0 ** -21 * 4 * 1.3 * (
        np.abs(g).sum() * np.abs(x).max())
    h = 0.5
    for t, head, e in [(0, 0, 0), (3, 1, 17), (19, 2, 31), (7, 0, 40)]:
        step = np.zeros_like(x)
        step[t, head, e] = h
        difference = ((turn(x + step, False) - turn(x - step, False)) * g).sum() / (2 * h)
        # the identity outside the turned part has no scale either way
        assert abs(difference - grad[t, head, e]) <= 2.0 ** -18 * 4 * np.abs(x).max() * np.abs(
            g).max() / h


def test_tensors_streams_and_a_graph(gpu):
    """Q and K as columns of one projection's rows, on a stream, captured and replayed."""
    torch = pytest.importorskip("torch")
    k = _k()
    gen = torch.Generator(device="cuda").manual_seed(2)
    rows = torch.randn(40, 12, 64, generator=gen, device="cuda").to(torch.bfloat16)
    q, kk = rows[:, :6], rows[:, 6:9]
    qo, ko = torch.empty(40, 6, 64, dtype=rows.dtype, device="cuda"), torch.empty(
        40, 3, 64, dtype=rows.dtype, device="cuda")
    pos = torch.arange(40, device="cuda", dtype=torch.int32)
    table = k.rotary_frequencies(64, schedule="base", factor=8.0)[0]
    freq = torch.from_numpy(table).cuda()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()

    def check():
        torch.cuda.synchronize()
        for x, y in ((q, qo), (kk, ko)):
            want, size = _turned(x.float().cpu().numpy(), pos.cpu().numpy(), table, False, False, 1.0)
            off = np.abs(y.double().cpu().numpy() - want)
            assert np.all(off <= np.abs(want) * 2.0 ** -8 * 1.01 + size * 2.0 ** -21)

    k.rotary(q, kk, pos, freq, q_out=qo, k_out=ko, stream=side, sync=False)
    side.synchronize()
    check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        k.rotary(q, kk, pos, freq, q_out=qo, k_out=ko, stream=side, sync=False)
    for turn in range(3):
        rows.copy_(torch.randn(rows.shape, generator=gen, device="cuda"))
        pos += 100 * turn
        qo.zero_()
        graph.replay()
        check()
    before = rows.clone()
    k.rotary(q, kk, pos, freq)  # in place, V beside them left alone
    assert torch.equal(rows[:, :6], qo) and torch.equal(rows[:, 6:9], ko)
    assert torch.equal(rows[:, 9:], before[:, 9:])


def test_more_tokens_than_a_grid_row(gpu):
    """2^21 workgroups make a row of the grid."""
    torch = pytest.importorskip("torch")
    k = _k()
    n = (1 << 21) * 256 + 77  # of two elements: a pair each, 256 tokens a workgroup
    x = torch.ones(n, 1, 2, dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(n, dtype=torch.int32, device="cuda")
    pos[-77:] = 1
    freq = torch.tensor([np.pi / 2], dtype=torch.float64, device="cuda")
    k.rotary(x, None, pos, freq)
    assert bool((x[:-77] == 1).all())
    assert torch.equal(x[-77:, 0].float().cpu(), torch.tensor([[-1.0, 1.0]]).repeat(77, 1))


def test_grid_of_two_dimensions(gpu):
    """More workgroups than a grid's row has, against the same tokens in parts."""
    torch = pytest.importorskip("torch")
    k = _k()
    tokens, d = (1 << 21) + 37, 512
    x = torch.randn(tokens, 1, d, device="cuda").to(torch.bfloat16)
    positions = torch.randint(0, 1 << 20, (tokens,), dtype=torch.int32, device="cuda")
    freq = torch.from_numpy(k.rotary_frequencies(d)[0]).cuda()
    whole, part = torch.empty_like(x), torch.empty_like(x)
    k.rotary(x, None, positions, freq, q_out=whole)
    for at in range(0, tokens, 1 << 20):
        to = min(tokens, at + (1 << 20))
        k.rotary(x[at:to], None, positions[at:to], freq, q_out=part[at:to])
    assert torch.equal(whole, part)
