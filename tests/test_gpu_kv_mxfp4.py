"""The 4-bit paged cache on the GPU: rows written and read back bit for bit against the
format's definition, and decode attention over it against attention in 64 bits within
the bound that test_gpu_paged_attention.py derives (a 4-bit value is exact in bf16, so
nothing is added to it)."""
from __future__ import annotations

import numpy as np
import pytest

import mxfp4_ref as ref
from gpu_util import Guarded, assert_same, bf16_to_f32
from test_gpu_paged_attention import Batch, _bf16_bits

pytestmark = pytest.mark.gpu

NO_SLOT = 0xFFFFFFFF


def _k():
    from fe2o3_amd import kernels
    return kernels


def _strides(order, page_size, kv_heads, row, pad):
    """(page, token, head) strides in bytes."""
    if order == "token":
        head = row + pad
        token = kv_heads * head
        return page_size * token, token, head
    token = row + pad
    head = page_size * token
    return kv_heads * head, token, head


class Cache4:
    """A guarded 4-bit cache; every slot holds bytes as they come, NaN scales among them."""

    def __init__(self, gpu, rng, pages, page_size, kv_heads, head_dim, order="token", pad=0):
        self.shape = (pages, page_size, kv_heads, head_dim)
        self.strides = _strides(order, page_size, kv_heads, head_dim // 2, pad)
        n = pages * self.strides[0]
        self.init = [rng.integers(0, 256, n).astype(np.uint8) for _ in "kv"]
        self.blocks = [rng.integers(0, 256, (pages, kv_heads, page_size, head_dim // 32))
                       .astype(np.uint8) for _ in "kv"]
        self.dev = [Guarded(gpu, x) for x in self.init]
        self.dev_blocks = [Guarded(gpu, x) for x in self.blocks]
        self.cache = _k().KvCache(*(g.body for g in self.dev), *(g.body for g in self.dev_blocks),
                                  shape=self.shape, strides=self.strides)

    def rows(self, flat):
        """View [pages, page_size, kv_heads, head_dim / 2]."""
        pages, page_size, kv_heads, head_dim = self.shape
        return np.lib.stride_tricks.as_strided(
            flat, (pages, page_size, kv_heads, head_dim // 2), (*self.strides, 1))

    def check(self, want, want_blocks):
        for g, w in zip(self.dev + self.dev_blocks, want + want_blocks):
            assert g.guards_intact()
            assert_same(g.download(), np.ravel(w), "cache")


def _encode(x):
    """Row bytes and scale bytes of rows [..., head_dim]."""
    blocks = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    byte = ref.scale_bytes(blocks)
    code = ref.two_to_a_byte(ref.codes(blocks, byte))
    return code.reshape(*x.shape[:-1], x.shape[-1] // 2), byte


def _write(gpu, tokens, kv_heads, head_dim, page_size, order="token", pad=0, row_pad=0,
           values=None, seed=0):
    rng = np.random.default_rng([seed, tokens, kv_heads, head_dim, page_size])
    pages = -(-tokens // page_size) + 2
    c = Cache4(gpu, rng, pages, page_size, kv_heads, head_dim, order, pad)
    head_stride = head_dim + row_pad
    token_stride = kv_heads * head_stride + row_pad
    n = (tokens - 1) * token_stride + (kv_heads - 1) * head_stride + head_dim
    rows, host = [], []
    for _ in range(2):
        flat = _bf16_bits(rng.standard_normal(n) * np.exp2(rng.integers(-20, 20, n) / 4))
        view = np.lib.stride_tricks.as_strided(flat, (tokens, kv_heads, head_dim),
                                               (2 * token_stride, 2 * head_stride, 2))
        if values is not None:
            view[...] = _bf16_bits(values(rng, view.shape))
        rows.append(Guarded(gpu, flat))
        host.append(bf16_to_f32(view))
    slots = rng.permutation(pages * page_size)[:tokens].astype(np.uint32)
    if tokens > 2:
        slots[1::5] = NO_SLOT
        slots[2] = pages * page_size  # the first past the cache
    dslots = Guarded(gpu, slots)
    _k().kv_cache_write(c.cache, rows[0].body, rows[1].body, dslots.body,
                        strides=(token_stride, head_stride))
    want, blocks = [x.copy() for x in c.init], [x.copy() for x in c.blocks]
    ok = slots < pages * page_size
    page, place = slots[ok] // page_size, slots[ok] % page_size
    nan = []
    for part in range(2):
        code, byte = _encode(host[part][ok])
        c.rows(want[part])[page, place] = code
        blocks[part].transpose(0, 2, 1, 3)[page, place] = byte
        nan.append(np.repeat(byte == 255, 16, -1))
    got = [g.download() for g in c.dev]
    for part in range(2):  # codes on a NaN scale may be any
        seen = c.rows(got[part])[page, place]
        c.rows(want[part])[page, place] = np.where(nan[part], seen,
                                                   c.rows(want[part])[page, place])
    c.check(want, blocks)
    assert all(g.unchanged() for g in rows) and dslots.unchanged()


@pytest.mark.parametrize("head_dim", [32, 64, 96, 128, 160, 256, 512, 1024])
def test_write_head_dims(gpu, head_dim):
    _write(gpu, 37, 3, head_dim, 16)


@pytest.mark.parametrize("tokens,kv_heads,page_size", [(1, 1, 1), (1, 8, 16), (5, 1, 1),
                                                       (64, 32, 16), (1000, 8, 24), (333, 2, 7),
                                                       (4099, 1, 256)])
def test_write_sizes(gpu, tokens, kv_heads, page_size):
    _write(gpu, tokens, kv_heads, 128, page_size)


@pytest.mark.parametrize("order", ["token", "head"])
@pytest.mark.parametrize("pad,row_pad", [(0, 0), (1, 1), (3, 5), (16, 8)])
def test_write_orders_and_strides(gpu, order, pad, row_pad):
    _write(gpu, 77, 3, 64, 16, order, pad, row_pad)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_write_rows_that_are_not_finite(gpu, bad):
    def values(rng, shape):
        x = rng.standard_normal(shape)
        x[rng.random(shape) < 0.01] = bad
        return x.astype(np.float32)
    _write(gpu, 50, 2, 128, 16, values=values)


def test_write_zeros_and_the_smallest(gpu):
    def values(rng, shape):
        x = rng.standard_normal(shape) * 2.0 ** -128
        x[::3] = 0.0
        x[1::3] = -0.0
        return x.astype(np.float32)
    _write(gpu, 50, 2, 128, 16, values=values)


def _read(gpu, lengths, kv_heads, head_dim, page_size, order="token", pad=0, row_pad=0, lead=2,
          behind=3, short_table=0):
    rng = np.random.default_rng([len(lengths), kv_heads, head_dim, page_size])
    need = [-(-n // page_size) for n in lengths]
    pages, cols = sum(need) + 2, max(need + [1]) - short_table
    c = Cache4(gpu, rng, pages, page_size, kv_heads, head_dim, order, pad)
    for blocks, g in zip(c.blocks, c.dev_blocks):  # whose values are finite in bf16
        np.minimum(blocks, 251, out=blocks)
        g.body.upload(blocks.ravel())
        g.initial[64:-64] = blocks.ravel()
    table = np.full((len(lengths), cols), 0xFFFFFFF0, np.uint32)
    free, at = rng.permutation(pages), 0
    for s, n in enumerate(need):
        table[s, :n] = free[at:at + min(n, cols)]
        at += n
    if len(lengths) > 1 and lengths[1] > page_size:
        table[1, 0] = pages  # out of range: +0
    starts = (lead + np.concatenate([[0], np.cumsum(lengths)])).astype(np.uint32)
    tokens = int(starts[-1]) + behind
    head_stride = head_dim + row_pad
    token_stride = kv_heads * head_stride
    n = (tokens - 1) * token_stride + (kv_heads - 1) * head_stride + head_dim
    outs = [Guarded(gpu, rng.integers(0, 65536, n).astype(np.uint16)) for _ in "kv"]
    dt, ds = Guarded(gpu, table), Guarded(gpu, starts)
    _k().kv_cache_read(c.cache, dt.body, ds.body, outs[0].body, outs[1].body, tokens=tokens,
                       strides=(token_stride, head_stride))
    for part, out in enumerate(outs):
        want = out.initial[64:-64].copy()
        view = np.lib.stride_tricks.as_strided(want, (tokens, kv_heads, head_dim),
                                               (2 * token_stride, 2 * head_stride, 2))
        rows = c.rows(c.init[part])
        for s, count in enumerate(lengths):
            key = np.arange(count)
            inside = key // page_size < cols
            page = table[s, np.minimum(key // page_size, cols - 1)]
            ok = inside & (page < pages)
            page, place = np.where(ok, page, 0), key % page_size
            code = ref.one_a_byte(rows[page, place]).reshape(count, kv_heads, head_dim // 32, 32)
            x = ref.values(code, c.blocks[part].transpose(0, 2, 1, 3)[page, place])
            bits = _bf16_bits(x.reshape(count, kv_heads, head_dim).astype(np.float32))
            view[starts[s]:starts[s] + count] = np.where(ok[:, None, None], bits, 0)
        assert out.guards_intact()
        assert_same(out.download(), want, "read")
    c.check(c.init, c.blocks)


@pytest.mark.parametrize("head_dim", [32, 64, 96, 128, 256, 1024])
def test_read_head_dims(gpu, head_dim):
    _read(gpu, [37, 0, 5], 3, head_dim, 16)


@pytest.mark.parametrize("order", ["token", "head"])
@pytest.mark.parametrize("pad,row_pad", [(0, 0), (1, 3), (16, 8)])
@pytest.mark.parametrize("lengths,kv_heads,page_size", [([1], 1, 1), ([0, 100, 33], 8, 24),
                                                        ([700, 650], 2, 64)])
def test_read_orders_and_strides(gpu, order, pad, row_pad, lengths, kv_heads, page_size):
    _read(gpu, lengths, kv_heads, 64, page_size, order, pad, row_pad)


def test_read_past_the_table(gpu):
    _read(gpu, [70, 65], 2, 128, 16, short_table=2)


# ---- decode attention ----------------------------------------------------------------------


class Batch4(Batch):
    """A Batch over a 4-bit cache.  Slots that no sequence reaches hold NaN scales."""

    def __init__(self, gpu, lengths, q_heads, kv_heads, head_dim, page_size, order="token", pad=0,
                 q_pad=0, cols=None, seed=0, peak=1.0, slack=2):
        rng = np.random.default_rng([seed, len(lengths), q_heads, head_dim, page_size])
        self.gpu, self.fmt, self.lengths = gpu, "mxfp4", list(lengths)
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.page_size, self.order_name, self.pad = page_size, order, pad
        need = [-(-n // page_size) for n in lengths]
        pages = sum(need) + slack
        self.cols = max(need + [1]) if cols is None else cols
        free, at = rng.permutation(pages), 0
        self.table = np.full((len(lengths), self.cols), 0xFFFFFFF0, np.uint32)
        for s, n in enumerate(need):
            self.table[s, :n] = free[at:at + n]
            at += n
        self.shape = (pages, page_size, kv_heads, head_dim)
        self.strides = _strides(order, page_size, kv_heads, head_dim // 2, pad)
        self.k, self.v, self.arrays, self.scales = [], [], [], []
        for part, held in enumerate((self.k, self.v)):
            flat = rng.integers(0, 256, pages * self.strides[0]).astype(np.uint8)
            blocks = np.full((pages, kv_heads, page_size, head_dim // 32), 255, np.uint8)
            rows = np.lib.stride_tricks.as_strided(
                flat, (pages, page_size, kv_heads, head_dim // 2), (*self.strides, 1))
            for s, count in enumerate(lengths):
                key = np.arange(count)
                page, place = self.table[s, key // page_size], key % page_size
                x = rng.standard_normal((count, kv_heads, head_dim)).astype(np.float32)
                x *= np.exp2(rng.integers(-2, 2, (count, kv_heads, head_dim // 32)).repeat(32, -1))
                if part == 0:
                    x *= peak
                code, byte = _encode(x)
                rows[page, place] = code
                blocks.transpose(0, 2, 1, 3)[page, place] = byte
                held.append(ref.values(ref.one_a_byte(code).reshape(*byte.shape, 32), byte)
                            .reshape(x.shape))
            self.arrays.append(Guarded(gpu, flat))
            self.scales.append(Guarded(gpu, blocks))
        self.cache = _k().KvCache(*(a.body for a in self.arrays), *(a.body for a in self.scales),
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

    def reference(self, *args, **kwargs):
        """With scores hundreds apart a 4-bit V has zeros under the largest probability, and
        an output may come from probabilities near 2^-126 of it alone.  Both the exponential
        and the MFMA's two parts of one flush below 2^-126: 2^-125 |v| a key, over a sum
        that the largest one makes at least 1."""
        o, lse, o_tol, lse_tol = super().reference(*args, **kwargs)
        for s, v in enumerate(self.v):
            o_tol[s] += 2.0 ** -125 * np.abs(v).sum(0).max(initial=0.0)
        return o, lse, o_tol, lse_tol


def _check(gpu, lengths, q_heads, kv_heads, head_dim, page_size, window=0, **more):
    b = Batch4(gpu, lengths, q_heads, kv_heads, head_dim, page_size, **more)
    b.compare(b.run(window), b.reference(window))
    assert b.inputs_unchanged()


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("lengths", [[1], [0], [0, 1, 2], [31, 32, 33], [63, 64, 65],
                                     [127, 128, 129, 0], [255, 256, 257], [500], [511, 513],
                                     [1000, 3, 0, 700]])
def test_lengths(gpu, head_dim, lengths):
    _check(gpu, lengths, 8, 2, head_dim, 16)


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (4, 4), (3, 1), (8, 2), (10, 2), (28, 4),
                                              (9, 1), (12, 1), (16, 1), (17, 1), (32, 1), (66, 2),
                                              (48, 1), (64, 1), (65, 1), (200, 2)])
def test_groups(gpu, head_dim, q_heads, kv_heads):
    _check(gpu, [70, 700], q_heads, kv_heads, head_dim, 16)


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("page_size", [1, 3, 7, 24, 32, 40, 64, 256, 1000])
@pytest.mark.parametrize("order", ["token", "head"])
def test_pages(gpu, head_dim, page_size, order):
    _check(gpu, [333, 1, 95], 8, 4, head_dim, page_size, order=order)


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("order", ["token", "head"])
def test_strides(gpu, head_dim, order):
    _check(gpu, [300, 41], 6, 2, head_dim, 16, order=order, pad=16, q_pad=24, cols=50)


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 512, 5000])
def test_windows(gpu, head_dim, window):
    _check(gpu, [0, 1, 32, 33, 450, 1600], 8, 2, head_dim, 16, window=window)


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("q_heads,kv_heads", [(4, 2), (8, 4), (20, 1)])
@pytest.mark.parametrize("window", [1500, 2047, 2048, 2049])
def test_windows_over_many_runs(gpu, head_dim, q_heads, kv_heads, window):
    _check(gpu, [5000, 0, 1999, 2100, 7000], q_heads, kv_heads, head_dim, 16, window=window)


@pytest.mark.parametrize("lengths,q_heads,kv_heads,head_dim,page_size", [
    ([40001], 2, 1, 128, 16),
    ([40001], 2, 1, 64, 16),
    ([5000, 1, 0, 0, 9000, 33], 8, 2, 64, 16),
    ([2500] * 40, 4, 2, 128, 32),
    ([int(x) for x in np.linspace(0, 700, 150)], 2, 1, 64, 8),
    ([300] * 3 + [0] * 200 + [4000], 2, 2, 64, 64),
    ([40001], 8, 4, 128, 16),
    ([5000, 1, 0, 0, 9000, 33], 16, 8, 128, 16),
    ([1500, 1501, 1499, 31] * 6, 64, 4, 128, 32),
    ([int(x) for x in np.linspace(0, 1400, 70)], 4, 4, 64, 8),
    ([5000, 1, 0, 4000, 33], 20, 1, 128, 16),
    ([2500] * 9, 48, 1, 64, 16),
    ([3000, 2999, 40], 64, 1, 128, 16),
    ([3000, 0, 1700], 150, 1, 64, 16),
])
def test_many_runs(gpu, lengths, q_heads, kv_heads, head_dim, page_size):
    _check(gpu, lengths, q_heads, kv_heads, head_dim, page_size)


@pytest.mark.parametrize("seqs", [65, 700, 4300])
@pytest.mark.parametrize("q_heads,kv_heads", [(2, 1), (4, 4)])
def test_many_sequences(gpu, seqs, q_heads, kv_heads):
    lengths = [37 * i % 151 for i in range(seqs - 2)] + [0, 0]
    lengths[seqs // 3] = 2000
    lengths[seqs // 2] = 1300
    _check(gpu, lengths, q_heads, kv_heads, 64, 16)


@pytest.mark.parametrize("lengths,q_heads,kv_heads,head_dim", [
    ([40001], 8, 4, 128), ([5000, 1, 0, 0, 9000, 33], 16, 8, 64),
    ([1500, 1501, 1499, 31] * 6, 64, 4, 128), ([37 * i % 151 for i in range(700)], 4, 4, 64),
])
def test_four_heads_a_workgroup(gpu, lengths, q_heads, kv_heads, head_dim):
    b = Batch4(gpu, lengths, q_heads, kv_heads, head_dim, 64, cols=1700)
    b.compare(b.run(max_length=1700 * 64), b.reference())
    assert b.inputs_unchanged()


@pytest.mark.parametrize("peak", [0.0, 1e-3, 8.0, 100.0])
def test_peaked_and_flat_scores(gpu, peak):
    _check(gpu, [700, 41, 2100], 8, 2, 128, 16, peak=peak)
    _check(gpu, [700, 41], 40, 1, 64, 16, peak=peak)


@pytest.mark.parametrize("head_dim", [64, 128])
def test_length_above_max_length_and_bad_pages(gpu, head_dim):
    b = Batch4(gpu, [300, 777, 40], 8, 2, head_dim, 16)
    b.compare(b.run(max_length=500), b.reference(max_length=500))
    table = b.table.copy()
    table[0, 3] = 0xFFFFFFFF
    table[1, ::2] = b.shape[0]
    b.dev_table = Guarded(gpu, table)
    b.compare(b.run(), b.reference(drop=lambda s, key: table[s, key // 16] >= b.shape[0]))


@pytest.mark.parametrize("lengths", [[77], [3000]])
@pytest.mark.parametrize("part", [0, 1])
def test_nan_blocks_of_kept_keys(gpu, lengths, part):
    """A NaN block of V makes NaN of its 32 outputs, one of K of the whole head."""
    b = Batch4(gpu, lengths, 8, 2, 128, 16)
    blocks = b.scales[part].download().reshape(b.shape[0], 2, 16, 4)
    key = lengths[0] // 2
    blocks[b.table[0, key // 16], 1, key % 16, 2] = 255
    b.scales[part].body.upload(blocks.ravel())
    o, lse = b.run()
    nan = np.isnan(bf16_to_f32(o.download())).reshape(2, 4, 128)
    want = np.zeros_like(nan)
    want[1, :, slice(None) if part == 0 else slice(64, 96)] = True
    assert np.array_equal(nan, want)
    assert np.array_equal(np.isnan(lse.download()).reshape(2, 4),
                          [[False] * 4, [part == 0] * 4])


def test_without_lse_and_repeated(gpu):
    b = Batch4(gpu, [5000, 33, 1200], 16, 4, 128, 16)
    first = b.run()
    b.compare(b.run(lse=False), b.reference(), lse=False)
    again = b.run()
    for x, y in zip(first, again):
        assert_same(x.download(), y.download(), "repeated")


def test_offsets_past_32_bits(gpu):
    """The pages in use lie behind 2^32 bytes of the cache."""
    pages, page_size = (1 << 32) // (64 * 8 * 64) + 40, 64
    # a cache of torch's allocator, so that only the pages in use are written
    torch = pytest.importorskip("torch")
    k = _k()
    gen = torch.Generator(device="cuda").manual_seed(1)
    cache = [torch.empty(pages, page_size, 8, 64, dtype=torch.uint8, device="cuda") for _ in "kv"]
    blocks = [torch.empty(pages, 8, page_size, 4, dtype=torch.uint8, device="cuda") for _ in "kv"]
    held = k.KvCache(*cache, *blocks)
    n = 300
    rows = torch.randn(2, n, 8, 128, generator=gen, device="cuda").to(torch.bfloat16)
    table = torch.arange(pages - 5, pages, device="cuda", dtype=torch.int32)[None]
    at = torch.arange(n, device="cuda")
    slots = (table[0, at // page_size].long() * page_size + at % page_size).to(torch.int32)
    k.kv_cache_write(held, rows[0], rows[1], slots)
    back = torch.zeros_like(rows)
    k.kv_cache_read(held, table, torch.tensor([0, n], device="cuda", dtype=torch.int32), back[0],
                    back[1])
    code, byte = _encode(rows.float().cpu().numpy())
    want = ref.values(ref.one_a_byte(code).reshape(*byte.shape, 32), byte).reshape(code.shape[:3]
                                                                                  + (128,))
    assert np.array_equal(back.float().cpu().numpy(), want)
    q = torch.randn(1, 32, 128, generator=gen, device="cuda").to(torch.bfloat16)
    out, lse = torch.empty_like(q), torch.empty(1, 32, device="cuda")
    work = torch.empty(k.paged_attention_workspace_bytes(32, 8, 128), dtype=torch.uint8,
                       device="cuda")
    k.paged_attention_decode(held, q, table, torch.tensor([n], device="cuda", dtype=torch.int32),
                             out, lse, work, max_length=n, scale=128 ** -0.5)
    qh = q[0].double().cpu().numpy().reshape(8, 4, 128)
    s = np.einsum("hgd,nhd->hgn", qh, want[0]) * 128 ** -0.5
    p = np.exp(s - s.max(-1, keepdims=True))
    o = np.einsum("hgn,nhd->hgd", p / p.sum(-1, keepdims=True), want[1]).reshape(32, 128)
    mean = np.einsum("hgn,nhd->hgd", p / p.sum(-1, keepdims=True), np.abs(want[1])).reshape(32, 128)
    assert np.all(np.abs(out[0].double().cpu().numpy() - o) <= mean * 2.0 ** -7)


def test_layer_steps_in_a_graph(gpu):
    """Steps of a layer as a program makes them, captured once and replayed: a new
    token's K and V written into their slots, then its attention, the length growing
    on the device; against the same steps made eagerly, bit for bit, and 64 bits."""
    torch = pytest.importorskip("torch")
    k = _k()
    seqs, heads, kv_heads, d, page_size, cols = 3, 8, 2, 64, 16, 6
    gen = torch.Generator(device="cuda").manual_seed(9)
    pages = seqs * cols + 1
    table = torch.randperm(pages, generator=gen, device="cuda")[:seqs * cols].reshape(
        seqs, cols).to(torch.int32)
    work = torch.empty(k.paged_attention_workspace_bytes(heads, kv_heads, d), dtype=torch.uint8,
                       device="cuda")

    def program():
        cache = [torch.zeros(pages, page_size, kv_heads, d // 2, dtype=torch.uint8, device="cuda")
                 for _ in "kv"]
        blocks = [torch.full((pages, kv_heads, page_size, d // 32), 255, dtype=torch.uint8,
                             device="cuda") for _ in "kv"]
        held = k.KvCache(*cache, *blocks)
        state = dict(q=torch.zeros(seqs, heads, d, dtype=torch.bfloat16, device="cuda"),
                     kv=torch.zeros(seqs, 2, kv_heads, d, dtype=torch.bfloat16, device="cuda"),
                     lengths=torch.tensor([0, 17, 40], dtype=torch.int32, device="cuda"),
                     out=torch.empty(seqs, heads, d, dtype=torch.bfloat16, device="cuda"),
                     lse=torch.empty(seqs, heads, device="cuda"))

        def step(stream):
            at = state["lengths"].long()
            slot = (table.gather(1, (at // page_size)[:, None])[:, 0].long() * page_size
                    + at % page_size).to(torch.int32)
            k.kv_cache_write(held, state["kv"][:, 0], state["kv"][:, 1], slot, stream=stream,
                             sync=False)
            state["lengths"] += 1
            k.paged_attention_decode(held, state["q"], table, state["lengths"], state["out"],
                                     state["lse"], work, max_length=cols * page_size,
                                     scale=d ** -0.5, stream=stream, sync=False)
        return state, step, held

    rows = torch.randn(40, 2, kv_heads, d, generator=gen, device="cuda").to(torch.bfloat16)
    side = torch.cuda.Stream()
    eager, graphed = program(), program()
    history = [[], [], []]
    for state, _, held in (eager, graphed):  # the prefixes of sequences 1 and 2
        for s, n in ((1, 17), (2, 40)):
            at = torch.arange(n, device="cuda")
            slot = (table[s, at // page_size].long() * page_size + at % page_size).to(torch.int32)
            k.kv_cache_write(held, rows[:n, 0], rows[:n, 1], slot)
    history[1], history[2] = list(rows[:17].float().cpu()), list(rows[:40].float().cpu())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    state, step, _ = graphed
    before = state["lengths"].clone()
    with torch.cuda.graph(graph, stream=side):
        step(side)
    state["lengths"].copy_(before)
    for turn in range(4):
        q = torch.randn(seqs, heads, d, generator=gen, device="cuda").to(torch.bfloat16)
        kv = torch.randn(seqs, 2, kv_heads, d, generator=gen, device="cuda").to(torch.bfloat16)
        for state, _, _ in (eager, graphed):
            state["q"].copy_(q)
            state["kv"].copy_(kv)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager[1](None)
        torch.cuda.synchronize()
        assert torch.equal(eager[0]["out"], graphed[0]["out"])
        assert torch.equal(eager[0]["lse"], graphed[0]["lse"])
        for s in range(seqs):
            history[s].append(kv[s].float().cpu())
            x = np.stack([h.numpy() for h in history[s]])
            code, byte = _encode(x)
            x = ref.values(ref.one_a_byte(code).reshape(*byte.shape, 32), byte).reshape(x.shape)
            qh = q[s].double().cpu().numpy().reshape(kv_heads, heads // kv_heads, d)
            sc = np.einsum("hgd,nhd->hgn", qh, x[:, 0]) * d ** -0.5
            p = np.exp(sc - sc.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            o = np.einsum("hgn,nhd->hgd", p, x[:, 1]).reshape(heads, d)
            mean = np.einsum("hgn,nhd->hgd", p, np.abs(x[:, 1])).reshape(heads, d)
            got = eager[0]["out"][s].double().cpu().numpy()
            assert np.all(np.abs(got - o) <= mean * 2.0 ** -7), turn


def test_grid_of_two_dimensions(gpu):
    """More workgroups than a grid's row has, one a head, against the same sequences in parts."""
    torch = pytest.importorskip("torch")
    k = _k()
    seqs, heads, d, pages, page, cols = (1 << 18) + 3, 8, 64, 64, 16, 16
    gen = torch.Generator(device="cuda").manual_seed(2)

    def byte(*shape, low=0, high=256):
        return torch.randint(low, high, shape, dtype=torch.uint8, device="cuda", generator=gen)

    cache = k.KvCache(byte(pages, page, heads, d // 2), byte(pages, page, heads, d // 2),
                      byte(pages, heads, page, d // 32, low=120, high=128),
                      byte(pages, heads, page, d // 32, low=120, high=128))
    q = torch.randn(seqs, heads, d, device="cuda", generator=gen).to(torch.bfloat16)
    table = torch.randint(0, pages, (seqs, cols), dtype=torch.int32, device="cuda", generator=gen)
    lengths = torch.randint(0, 41, (seqs,), dtype=torch.int32, device="cuda", generator=gen)
    work = torch.empty(k.paged_attention_workspace_bytes(heads, heads, d), dtype=torch.uint8,
                       device="cuda")
    results = []
    for step in (seqs, 1 << 17):
        out = torch.full_like(q, 3.0)
        lse = torch.full((seqs, heads), 3.0, device="cuda")
        for at in range(0, seqs, step):
            to = min(seqs, at + step)
            # the last part by itself would be a call of one workgroup of eight waves a head
            at = max(0, min(at, to - 1024))
            k.paged_attention_decode(cache, q[at:to], table[at:to], lengths[at:to], out[at:to],
                                     lse[at:to], work, max_length=page * cols, scale=0.125)
        results.append((out, lse))
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    empty = lengths == 0
    assert not bool(results[0][0][empty].any())
    assert bool(torch.isneginf(results[0][1][empty]).all())
