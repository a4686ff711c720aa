"""The paged key-value cache on the GPU (fe2o3_kv_cache_write,
fe2o3_kv_cache_read): every byte of the cache and of the outputs against plain
numpy and the oracle's e4m3 encoder, guard bands around every array."""
from __future__ import annotations

import numpy as np
import pytest

from gpu_util import Guarded, assert_same, bf16_to_f32

pytestmark = pytest.mark.gpu

NO_SLOT = 0xFFFFFFFF
TINY = np.float32(1.17549435e-38)


def _k():
    from fe2o3_amd import kernels
    return kernels


def _bf16_bits(x):
    from oracle import oracle as orc
    return np.asarray(orc.bf16_from_f32(np.ascontiguousarray(x, np.float32).ravel()),
                      np.uint16).reshape(np.shape(x))


def _codes(x, scale):
    """e4m3 codes of f32 values divided by their row's scale."""
    from oracle import oracle as orc
    y = (x / scale[..., None]).astype(np.float32)
    return np.asarray(orc.quantize_e4m3(np.ascontiguousarray(y).ravel(), np.float32(1.0)),
                      np.uint8).reshape(x.shape)


def _scales(x):
    return (np.maximum(np.abs(x).max(-1), TINY) / np.float32(448.0)).astype(np.float32)


class Paged:
    """A guarded cache of given order, every slot holding a pattern."""

    def __init__(self, gpu, rng, fmt, pages, page_size, kv_heads, head_dim, order="token", pad=0):
        self.fmt, self.shape = fmt, (pages, page_size, kv_heads, head_dim)
        if order == "token":
            head = head_dim + pad
            token = kv_heads * head
            page = page_size * token + pad
        else:
            token = head_dim + pad
            head = page_size * token
            page = kv_heads * head + pad
        self.strides = (page, token, head)
        n = (pages - 1) * page + (page_size - 1) * token + (kv_heads - 1) * head + head_dim
        dtype = np.uint16 if fmt == "bf16" else np.uint8
        # as they come, NaN among them
        self.init = [rng.integers(0, np.iinfo(dtype).max + 1, n).astype(dtype) for _ in "kv"]
        self.dev = [Guarded(gpu, x) for x in self.init]
        self.scale_init, self.scale_dev = [], [None, None]
        if fmt == "e4m3":
            m = pages * kv_heads * page_size
            self.scale_init = [rng.random(m, np.float32) + 0.5 for _ in "kv"]
            self.scale_dev = [Guarded(gpu, x) for x in self.scale_init]
        self.cache = _k().KvCache(*(g.body for g in self.dev),
                                  *(g.body if g else None for g in self.scale_dev),
                                  shape=self.shape, strides=self.strides)

    def rows(self, flat):
        """View [pages, page_size, kv_heads, head_dim] of a flat host array."""
        size = flat.dtype.itemsize
        return np.lib.stride_tricks.as_strided(flat, self.shape,
                                               [s * size for s in self.strides] + [size])

    def scales(self, flat):
        pages, page_size, kv_heads, _ = self.shape
        return flat.reshape(pages, kv_heads, page_size).transpose(0, 2, 1)

    def check(self, want, want_scales, what):
        for name, g, w in zip("kv", self.dev, want):
            assert g.guards_intact(), (what, name)
            assert_same(g.download(), w, f"{what} {name}")
        for name, g, w in zip("kv", self.scale_dev, want_scales):
            assert g.guards_intact(), (what, name)
            assert_same(g.download(), w, f"{what} {name} scales")


def _write_case(gpu, fmt, tokens, kv_heads, head_dim, page_size, order="token", pad=0,
                row_pad=0, heads_first=False, values=None, seed=0):
    rng = np.random.default_rng([seed, tokens, kv_heads, head_dim, page_size])
    pages = -(-tokens // page_size) + 2
    p = Paged(gpu, rng, fmt, pages, page_size, kv_heads, head_dim, order, pad)
    if heads_first:
        token_stride = head_dim + row_pad
        head_stride = tokens * token_stride
    else:
        head_stride = head_dim + row_pad
        token_stride = kv_heads * head_stride + row_pad
    n = (tokens - 1) * token_stride + (kv_heads - 1) * head_stride + head_dim
    rows, host = [], []
    for part in range(2):
        flat = _bf16_bits(rng.standard_normal(n).astype(np.float32) * 3.0)
        view = np.lib.stride_tricks.as_strided(flat, (tokens, kv_heads, head_dim),
                                               (2 * token_stride, 2 * head_stride, 2))
        if values is not None:
            view[...] = values(rng, view.shape, part)
        rows.append(Guarded(gpu, flat))
        host.append(view)
    slots = rng.permutation(pages * page_size)[:tokens].astype(np.uint32)
    if tokens > 2:
        slots[1::5] = NO_SLOT
        slots[2] = pages * page_size  # the first past the cache
    dslots = Guarded(gpu, slots)
    _k().kv_cache_write(p.cache, rows[0].body, rows[1].body, dslots.body,
                        strides=(token_stride, head_stride))
    want = [x.copy() for x in p.init]
    want_scales = [x.copy() for x in p.scale_init]
    ok = slots < pages * page_size
    page, place = slots[ok] // page_size, slots[ok] % page_size
    for part in range(2):
        x = host[part][ok]
        if fmt == "e4m3":
            f = bf16_to_f32(x)
            scale = _scales(f)
            p.scales(want_scales[part])[page, place] = scale
            x = _codes(f, scale)
        p.rows(want[part])[page, place] = x
    p.check(want, want_scales, "write")
    assert all(g.unchanged() for g in rows) and dslots.unchanged()


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("head_dim", [1, 7, 8, 20, 64, 100, 128, 256, 513, 1000])
def test_write_head_dims(gpu, fmt, head_dim):
    _write_case(gpu, fmt, 37, 3, head_dim, 16)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("tokens,kv_heads,page_size", [(1, 1, 1), (1, 8, 16), (5, 1, 1),
                                                       (64, 32, 16), (1000, 8, 24),
                                                       (333, 2, 7), (4099, 1, 256)])
def test_write_sizes(gpu, fmt, tokens, kv_heads, page_size):
    _write_case(gpu, fmt, tokens, kv_heads, 64, page_size)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("order,pad,row_pad,heads_first", [
    ("head", 0, 0, False), ("head", 3, 0, True), ("token", 1, 1, False), ("token", 5, 7, True),
    ("token", 128, 8, False)])
def test_write_orders_and_strides(gpu, fmt, order, pad, row_pad, heads_first):
    _write_case(gpu, fmt, 53, 4, 128, 16, order, pad, row_pad, heads_first)


def test_write_every_finite_value(gpu):
    """Rows that hold every finite bf16 value once, of like magnitude and mixed:
    subnormals, zeros of both signs, and the largest among them."""
    def values(rng, shape, part):
        finite = np.array([b for b in range(1 << 16) if b & 0x7F80 != 0x7F80], np.uint16)
        n = int(np.prod(shape))
        x = np.resize(finite, n)
        if part:
            x = rng.permutation(x)
        return x.reshape(shape)
    _write_case(gpu, "e4m3", 1024, 1, 64, 32, values=values)


def test_write_zero_rows_and_ties(gpu):
    """All-zero rows (scale of the smallest normal), and rows whose quotients
    fall on the midpoints of e4m3 values."""
    def values(rng, shape, part):
        x = np.zeros(shape, np.float32)
        x[1::2, ..., 0] = 448.0
        x[1::2, ..., 1:] = rng.integers(-448 * 2, 448 * 2, shape)[1::2, ..., 1:] / 2.0
        return _bf16_bits(x)
    _write_case(gpu, "e4m3", 40, 2, 128, 16, values=values)


def test_write_zeros_of_both_signs(gpu):
    """Every row, of ordinary magnitude, holds zeros of both signs: the codes keep
    the sign, as the encoder does."""
    def values(rng, shape, part):
        x = _bf16_bits(rng.standard_normal(shape).astype(np.float32))
        x[..., 3::7] = 0x8000
        x[..., 5::7] = 0
        return x
    for head_dim in (64, 100):
        _write_case(gpu, "e4m3", 41, 2, head_dim, 16, values=values)


def test_write_small_rows(gpu):
    """Rows whose largest value lies anywhere from the smallest normal to far above
    the scales that divide as they are, x of any significand and sign down to 2^-20
    of it: the division's codes."""
    def values(rng, shape, part):
        top = 1 + np.arange(shape[0])[:, None, None] % 70
        exponent = np.maximum(top - rng.integers(0, 20, shape), 0)
        exponent[..., 0] = top[..., 0]
        return (exponent << 7 | rng.integers(0, 128, shape)
                | rng.integers(0, 2, shape) << 15).astype(np.uint16)
    _write_case(gpu, "e4m3", 700, 2, 256, 16, values=values)


def test_write_nonfinite_rows(gpu):
    """A NaN stays a NaN and leaves the rest of its row as it would be; a row with
    an infinity has an infinite scale."""
    kern = _k()
    p = Paged(gpu, np.random.default_rng(1), "e4m3", 2, 4, 1, 64)
    x = np.random.default_rng(2).standard_normal((3, 1, 64)).astype(np.float32)
    bits = _bf16_bits(x)
    bits[0, 0, 5] = 0x7FC0
    bits[1, 0, 6] = 0x7F80
    d = gpu.to_device(bits.ravel())
    kern.kv_cache_write(p.cache, d, d, gpu.to_device(np.arange(3, dtype=np.uint32)))
    codes = p.rows(p.dev[0].download())[0]
    scales = p.scales(p.scale_dev[0].download())[0]
    plain = bf16_to_f32(bits)
    rest = np.delete(plain[0, 0], 5)
    assert scales[0, 0] == _scales(rest)
    assert codes[0, 0, 5] & 0x7F == 0x7F
    assert_same(np.delete(codes[0, 0], 5), _codes(rest, _scales(rest)))
    assert np.isinf(scales[1, 0]) and codes[1, 0, 6] & 0x7F == 0x7F
    assert_same(codes[2], _codes(plain[2], _scales(plain[2])))


# ---- reading back ---------------------------------------------------------------------------

def _read_case(gpu, fmt, lengths, kv_heads, head_dim, page_size, order="token", pad=0,
               row_pad=0, heads_first=False, first=0, tail=3, bad_page=False, cols=None, seed=0):
    rng = np.random.default_rng([seed, len(lengths), kv_heads, head_dim, page_size])
    need = [-(-n // page_size) for n in lengths]
    pages = sum(need) + 2
    p = Paged(gpu, rng, fmt, pages, page_size, kv_heads, head_dim, order, pad)
    cols = max(need + [1]) if cols is None else cols
    order_of_pages = rng.permutation(pages)
    # entries behind a sequence's pages are never looked at
    table = np.full((len(lengths), cols), 0xDEADBEEF, np.uint32)
    at = 0
    for s, n in enumerate(need):
        table[s, :min(n, cols)] = order_of_pages[at:at + min(n, cols)]
        at += n
    if bad_page:
        table[-1, 0] = pages
    starts = (first + np.concatenate([[0], np.cumsum(lengths)])).astype(np.uint32)
    tokens = int(starts[-1]) + tail
    if heads_first:
        token_stride = head_dim + row_pad
        head_stride = tokens * token_stride
    else:
        head_stride = head_dim + row_pad
        token_stride = kv_heads * head_stride + row_pad
    n = (tokens - 1) * token_stride + (kv_heads - 1) * head_stride + head_dim
    outs = [Guarded(gpu, rng.integers(0, 1 << 16, n).astype(np.uint16)) for _ in "kv"]
    want = [g.initial[64:64 + n].copy() for g in outs]
    dt, ds = Guarded(gpu, table), Guarded(gpu, starts)
    _k().kv_cache_read(p.cache, dt.body, ds.body, outs[0].body, outs[1].body, tokens=tokens,
                       strides=(token_stride, head_stride))
    from oracle import oracle as orc
    decode = np.asarray(orc.fp8_decode_table(), np.float32)
    for part in range(2):
        rows = p.rows(p.init[part])
        if fmt == "e4m3":
            with np.errstate(invalid="ignore"):
                f = decode[rows] * p.scales(p.scale_init[part])[..., None]
            rows = np.where(np.isnan(f), np.uint16(0x7FC0), _bf16_bits(np.nan_to_num(f)))
        out = np.lib.stride_tricks.as_strided(want[part], (tokens, kv_heads, head_dim),
                                              (2 * token_stride, 2 * head_stride, 2))
        for s, count in enumerate(lengths):
            for i in range(count):
                col = i // page_size
                page = table[s, col] if col < cols else pages
                out[starts[s] + i] = rows[page, i % page_size] if page < pages else 0
        got = outs[part].download()
        if fmt == "e4m3":  # any NaN for a NaN
            nan = ((got & 0x7F80) == 0x7F80) & ((got & 0x7F) != 0)
            written = np.zeros(n, bool)
            np.lib.stride_tricks.as_strided(written, (tokens, kv_heads, head_dim),
                                            (token_stride, head_stride, 1))[
                int(starts[0]):int(starts[-1])] = True
            got = np.where(nan & written, np.uint16(0x7FC0), got)
        assert_same(got, want[part], f"read {'kv'[part]}")
        assert outs[part].guards_intact()
    assert dt.unchanged() and ds.unchanged()
    p.check(p.init, p.scale_init, "cache after read")


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("head_dim", [1, 7, 8, 20, 64, 128, 513])
def test_read_head_dims(gpu, fmt, head_dim):
    _read_case(gpu, fmt, [5, 0, 33, 1], 3, head_dim, 16)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("lengths,kv_heads,page_size", [
    ([1], 1, 1), ([0], 2, 16), ([0, 0, 0], 2, 16), ([17], 8, 16), ([7, 8, 9, 1, 64], 2, 8),
    ([100, 3, 250], 32, 24), ([1] * 70, 1, 16), ([3, 0] * 600, 1, 2)])
def test_read_lengths(gpu, fmt, lengths, kv_heads, page_size):
    _read_case(gpu, fmt, lengths, kv_heads, 64, page_size)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("order,pad,row_pad,heads_first", [
    ("head", 0, 0, True), ("head", 3, 1, False), ("token", 5, 7, True)])
def test_read_orders_and_strides(gpu, fmt, order, pad, row_pad, heads_first):
    _read_case(gpu, fmt, [40, 19], 4, 128, 16, order, pad, row_pad, heads_first, first=2, tail=5)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_read_out_of_range(gpu, fmt):
    """Rows past the table's pages and on a page past the cache's are +0."""
    _read_case(gpu, fmt, [40, 19], 2, 64, 8, bad_page=True)
    _read_case(gpu, fmt, [40, 19], 2, 64, 8, cols=3)


def test_write_then_read_is_the_rounding(gpu):
    """A row through an e4m3 cache is off by at most half a step of the format:
    2^-4 of the value, or 2^-10 of the scale below its smallest normal (2^-6), and
    the product's and bf16's own roundings, 2^-24 and 2^-8 of the result."""
    kern = _k()
    rng = np.random.default_rng(4)
    tokens, heads, d = 100, 2, 128
    p = Paged(gpu, rng, "e4m3", 10, 16, heads, d)
    x = [_bf16_bits(rng.standard_normal((tokens, heads, d)).astype(np.float32)) for _ in "kv"]
    slots = np.arange(tokens, dtype=np.uint32)
    kern.kv_cache_write(p.cache, *(gpu.to_device(v.ravel()) for v in x), gpu.to_device(slots))
    out = [gpu.alloc(tokens * heads * d, np.uint16) for _ in "kv"]
    kern.kv_cache_read(p.cache, gpu.to_device(np.arange(10, dtype=np.uint32)),
                       gpu.to_device(np.array([0, tokens], np.uint32)), *out)
    for a, b in zip(x, out):
        a = bf16_to_f32(a).astype(np.float64)
        b = bf16_to_f32(b.download()).reshape(a.shape).astype(np.float64)
        scale = np.abs(a).max(-1, keepdims=True) / 448.0
        half = np.maximum(np.abs(a) * 2.0 ** -4, scale * 2.0 ** -10)
        # the scale's own rounding (2^-24) moves code and result alike
        assert np.all(np.abs(a - b) <= half * (1 + 2.0 ** -7) + np.abs(b) * (2.0 ** -8 + 2.0 ** -22))


def test_offsets_past_32_bits(gpu):
    """Pages 2^32 bytes apart and more: only the touched rows of 13 GiB."""
    kern = _k()
    stride = (1 << 31) + 64  # elements
    pages, page_size, heads, d = 3, 4, 2, 64
    extent = (pages - 1) * stride + page_size * heads * d
    k, v = gpu.alloc(extent, np.uint16), gpu.alloc(extent, np.uint16)
    cache = kern.KvCache(k, v, shape=(pages, page_size, heads, d), strides=(stride, heads * d, d))
    rng = np.random.default_rng(5)
    x = [rng.integers(0, 0x7F00, (5, heads, d)).astype(np.uint16) for _ in "kv"]
    slots = np.array([11, 8, 5, 0, 9], np.uint32)
    kern.kv_cache_write(cache, *(gpu.to_device(a.ravel()) for a in x), gpu.to_device(slots))
    for a, buf in zip(x, (k, v)):
        for row, slot in enumerate(slots):
            at = int(slot) // page_size * stride + int(slot) % page_size * heads * d
            assert_same(buf.view(at, heads * d).download().reshape(heads, d), a[row])
    out = [gpu.alloc(page_size * heads * d, np.uint16) for _ in "kv"]
    kern.kv_cache_read(cache, gpu.to_device(np.array([2], np.uint32)),
                       gpu.to_device(np.array([0, page_size], np.uint32)), *out)
    for a, buf in zip(x, out):
        got = buf.download().reshape(page_size, heads, d)
        for row, slot in enumerate(slots):
            if slot >= 8:
                assert_same(got[slot - 8], a[row])


def test_more_workgroups_than_a_grid_row(gpu):
    """A write of more rows than one turn of the largest grid, and a read of more
    tokens than a grid's first row, back from the written cache."""
    torch = pytest.importorskip("torch")
    kern = _k()
    tokens, heads, page_size = (1 << 22) + 9, 64, 1024
    pages = tokens // page_size + 2
    g = torch.Generator(device="cuda").manual_seed(3)

    def bits(*shape):
        return torch.randint(-32768, 32768, shape, dtype=torch.int16, device="cuda", generator=g)

    held = [bits(pages, page_size, heads, 1) for _ in "kv"]
    rows = [bits(tokens, heads, 1) for _ in "kv"]
    slots = torch.randperm(pages * page_size, device="cuda", generator=g)[:tokens]
    slots[5::7] = -1
    want = [x.clone().view(-1, heads, 1) for x in held]
    kept = slots >= 0
    for w, x in zip(want, rows):
        w[slots[kept]] = x[kept]
    bf16 = torch.bfloat16
    cache = kern.KvCache(*(x.view(bf16) for x in held))
    kern.kv_cache_write(cache, *(x.view(bf16) for x in rows), slots.to(torch.int32))
    for x, w in zip(held, want):
        assert torch.equal(x.view(-1, heads, 1), w)

    # one head of the cache: tokens past the first row of workgroups
    narrow = [x[:, :, :1] for x in held]
    starts = torch.tensor([3, 11, 11, tokens - 2], dtype=torch.int32, device="cuda")
    cols = -(-tokens // page_size)
    table = torch.randint(0, pages, (3, cols), dtype=torch.int32, device="cuda", generator=g)
    out = [bits(tokens, 1, 1) for _ in "kv"]
    expect = [x.clone() for x in out]
    kern.kv_cache_read(kern.KvCache(*(x.view(bf16) for x in narrow)), table, starts,
                       *(x.view(bf16) for x in out))
    for s, (start, end) in enumerate([(3, 11), (11, 11), (11, tokens - 2)]):
        at = torch.arange(end - start, device="cuda")
        page = table[s, at // page_size].long()
        for w, x in zip(expect, narrow):
            w[start:end] = x[page, at % page_size]
    for x, w in zip(out, expect):
        assert torch.equal(x, w)
