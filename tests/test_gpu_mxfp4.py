"""GPU tests of the microscaled 4-bit matrices: packing and unpacking, bit for bit against
the format's definition, and the product against 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import mxfp4_ref as ref
from gpu_util import Guarded, assert_same, bf16_to_f32

pytestmark = pytest.mark.gpu


def _k():
    from fe2o3_amd import kernels
    return kernels


def _bf16_bits(x):
    x = np.ascontiguousarray(x, np.float32)
    u = x.view(np.uint32)
    r = (u + 0x7FFF + ((u >> 16) & 1)) >> 16
    return np.where(np.isnan(x), 0x7FC0, r).astype(np.uint16)


def _strided(x, stride, fill):
    """Rows of x, `stride` elements apart, as one flat array."""
    rows, cols = x.shape
    flat = np.full(max((rows - 1) * stride + cols, 0), fill, x.dtype)
    np.lib.stride_tricks.as_strided(flat, x.shape, (stride * x.itemsize, x.itemsize))[...] = x
    return flat


def _matrix(rng, rows, cols):
    """Blocks of every size of value, ties and zeros among them."""
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-30, 30, (rows, cols)) / 8)
    x *= np.exp2(rng.integers(-60, 60, (rows, 1)))
    tie = rng.random(x.shape) < 0.1
    x[tie] = np.exp2(np.floor(np.log2(np.abs(x[tie]) + 1e-30))) * 1.25
    x[rng.random(x.shape) < 0.05] = 0.0
    x[rng.random(x.shape) < 0.05] = -0.0
    return x.astype(np.float32)


def _quantize(gpu, x, fmt, stride=None, offset=0):
    """(codes, scales) of the kernel and x as it saw it; offset: elements before x."""
    rows, cols = x.shape
    held = x if fmt == "f32" else _bf16_bits(x)
    stride = cols if stride is None else stride
    flat = _strided(held, stride, np.nan if fmt == "f32" else 0x7FC0)
    dev = Guarded(gpu, np.concatenate([np.zeros(offset, held.dtype), flat]))
    panels = -(-cols // 256)
    q = Guarded(gpu, np.full(rows * panels * 128, 0xA5, np.uint8))
    s = Guarded(gpu, np.full(-(-rows // 16) * 16 * panels * 8, 0xA5, np.uint8))
    _k().quantize_mxfp4(dev.full.view(64 + offset, flat.size), q.body, s.body, rows=rows,
                        cols=cols, stride=stride)
    assert q.guards_intact() and s.guards_intact() and dev.unchanged()
    return (q.download().reshape(rows, -1), s.download().reshape(panels, -1, 8),
            x if fmt == "f32" else bf16_to_f32(held).reshape(x.shape))


def _check_packed(got, x):
    q, s, seen = got
    rows = seen.shape[0]
    want_q, want_s = ref.pack(seen)
    assert_same(s[:, :rows], want_s[:, :rows], "scales")
    # rows past the last keep their bytes
    assert np.all(s[:, rows:] == 0xA5)
    blocks = np.repeat(want_s[:, :rows].transpose(1, 0, 2).reshape(rows, -1) == 255, 16, 1)
    assert_same(np.where(blocks, 0, q), np.where(blocks, 0, want_q), "codes")


SHAPES = [(1, 1), (1, 32), (1, 33), (3, 255), (16, 256), (17, 257), (33, 4096), (5, 700),
          (100, 31), (1000, 40), (700, 2049), (40, 20000)]


@pytest.mark.parametrize("fmt", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize(gpu, fmt, rows, cols):
    x = _matrix(np.random.default_rng(rows * 7 + cols), rows, cols)
    _check_packed(_quantize(gpu, x, fmt), x)


@pytest.mark.parametrize("fmt", ["bf16", "f32"])
@pytest.mark.parametrize("stride,offset", [(300, 0), (301, 1), (307, 3), (1000, 5)])
def test_quantize_strides(gpu, fmt, stride, offset):
    x = _matrix(np.random.default_rng(stride), 45, 299)
    _check_packed(_quantize(gpu, x, fmt, stride, offset), x)


def test_quantize_every_bf16(gpu):
    """Every finite bf16 beside every largest magnitude's exponent: all scales there are."""
    bits = np.arange(65536, dtype=np.uint32)
    v = (bits << 16).view(np.float32)
    v = v[np.isfinite(v)]
    v = v[np.abs(v) <= 1.0]
    rows = []
    for e in range(-126, 128, 11):  # 31 values under a largest one of this exponent
        top = np.float32(2.0) ** e
        with np.errstate(under="ignore"):
            y = (v.astype(np.float64) * float(top)).astype(np.float32)
        y = bf16_to_f32(_bf16_bits(y))
        y = np.resize(y, -(-y.size // 31) * 31).reshape(-1, 31)
        rows.append(np.concatenate([y, np.full((len(y), 1), top, np.float32)], 1).ravel())
    x = np.stack(rows)
    _check_packed(_quantize(gpu, x, "bf16"), x)
    _check_packed(_quantize(gpu, x, "f32"), x)


@pytest.mark.parametrize("fmt", ["bf16", "f32"])
def test_quantize_smallest_and_largest(gpu, fmt):
    tiny = np.float32(2.0 ** -133)  # a subnormal of both types
    x = np.zeros((6, 256), np.float32)
    x[0, :32] = tiny * np.arange(32)
    x[1, :32] = 2.0 ** -126 * np.linspace(-1, 1, 32)
    x[2, :32] = 2.0 ** -124 * np.linspace(-2, 2, 32)
    x[3, :32] = 2.0 ** 127 * np.linspace(-1.9, 1.9, 32)
    x[4] = -0.0
    x[5, 3] = tiny
    _check_packed(_quantize(gpu, x, fmt), x)


@pytest.mark.parametrize("fmt", ["bf16", "f32"])
@pytest.mark.parametrize("bad", [np.nan, -np.nan, np.inf, -np.inf])
def test_blocks_that_are_not_finite(gpu, fmt, bad):
    """The block alone reads back as NaN."""
    x = _matrix(np.random.default_rng(5), 20, 600)
    x[3, 70] = x[17, 599] = bad
    got = _quantize(gpu, x, fmt)
    _check_packed(got, x)
    back = _dequantize(gpu, got[0], got[1], 600, "f32")
    nan = np.isnan(back)
    want = np.zeros_like(nan)
    want[3, 64:96] = want[17, 576:] = True
    assert np.array_equal(nan, want)


def _dequantize(gpu, q, s, cols, fmt, stride=None):
    rows = q.shape[0]
    stride = cols if stride is None else stride
    n = (rows - 1) * stride + cols
    out = Guarded(gpu, np.full(n, 7.0, np.float32) if fmt == "f32"
                  else np.full(n, 0x40E0, np.uint16))
    dq, ds = Guarded(gpu, q), Guarded(gpu, s)
    _k().dequantize_mxfp4(dq.body, ds.body, out.body, rows=rows, cols=cols, stride=stride)
    assert out.guards_intact() and dq.unchanged() and ds.unchanged()
    y = out.download()
    y = y if fmt == "f32" else bf16_to_f32(y)
    view = np.lib.stride_tricks.as_strided(y, (rows, cols), (4 * stride, 4))
    if stride > cols:  # between the rows: as before
        gaps = np.lib.stride_tricks.as_strided(y[cols:], (rows - 1, stride - cols), (4 * stride, 4))
        assert np.all(gaps == 7.0)
    return view.copy()


@pytest.mark.parametrize("fmt", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_dequantize(gpu, fmt, rows, cols):
    rng = np.random.default_rng(rows + cols)
    panels = -(-cols // 256)
    q = rng.integers(0, 256, (rows, panels * 128)).astype(np.uint8)
    s = rng.integers(0, 252, (panels, -(-rows // 16) * 16, 8)).astype(np.uint8)
    got = _dequantize(gpu, q, s, cols, fmt)
    want = ref.unpack(q, s)[:, :cols].astype(np.float32)
    assert_same(got, want, "values")
    if rows > 1:
        assert_same(_dequantize(gpu, q, s, cols, fmt, cols + 3), want, "strided values")


@pytest.mark.parametrize("fmt", ["bf16", "f32"])
def test_dequantize_every_scale(gpu, fmt):
    q = np.tile((np.arange(16) * 17).astype(np.uint8), (256, 8))
    s = np.zeros((1, 256, 8), np.uint8)
    s[0] = np.arange(256)[:, None]
    got = _dequantize(gpu, q, s, 256, fmt)
    with np.errstate(over="ignore"):
        want = ref.unpack(q, s).astype(np.float32)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan) and nan.sum() == 256
    assert_same(np.where(nan, 0, got), np.where(nan, 0, want), "values")


# ---- the product -------------------------------------------------------------------------

def _operand(rng, rows, k, low=118, high=132):
    """A random packed operand: codes of every value, its padding zeros."""
    panels = -(-k // 256)
    q = rng.integers(0, 256, (rows, panels * 128)).astype(np.uint8)
    code = ref.one_a_byte(q)
    code[:, k:] = 0
    s = rng.integers(low, high, (panels, -(-rows // 16) * 16, 8)).astype(np.uint8)
    s[:, rows:] = 255  # rows past the last have no effect
    return ref.two_to_a_byte(code), s


def _product(gpu, a, b, m, n, k, c_offset=0):
    bufs = [Guarded(gpu, x) for x in (a[0], a[1], b[0], b[1])]
    c = Guarded(gpu, np.full(m * n + c_offset, 0x7FDE, np.uint16))
    out = c.full.view(64 + c_offset, m * n)
    _k().gemm_mxfp4_nt(*(x.body for x in bufs), out, m, n, k)
    assert c.guards_intact() and all(x.unchanged() for x in bufs)
    got = c.download()
    assert np.all(got[:c_offset] == 0x7FDE)
    return got[c_offset:].reshape(m, n)


def _check_product(gpu, m, n, k, c_offset=0, **scales):
    """Against 64 bits: half a bf16 step of the result, and f32 sums of K products, each
    partial sum at most the sum of magnitudes (2^-24 of it for each of K additions at the
    most; the matrix core adds 128 at a time)."""
    rng = np.random.default_rng(m * 31 + n * 7 + k)
    a, b = _operand(rng, m, k, **scales), _operand(rng, n, k, **scales)
    got = bf16_to_f32(_product(gpu, a, b, m, n, k, c_offset)).astype(np.float64)
    x, y = ref.unpack(*a), ref.unpack(*b)
    want = x @ y.T
    bound = np.abs(want) * 2.0 ** -8 * (1 + 2.0 ** -7) + (np.abs(x) @ np.abs(y).T) * k * 2.0 ** -24
    off = np.abs(got - want)
    worst = np.unravel_index(np.argmax(off - bound), off.shape)
    assert np.all(off <= bound), (worst, got[worst], want[worst], bound[worst])
    # and no more than the rounding over all outputs: half a step at most, a third on average
    assert np.linalg.norm(off) <= 2.0 ** -8 * np.linalg.norm(want)


# a row, few rows or columns (the weights' stream), tiles of 128, of 256, last rounds as
# quarters, and edges of each
@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 1, 32), (1, 17, 700), (3, 5, 256), (16, 16, 257), (16, 4096, 4096),
    (17, 1000, 1030), (1, 14336, 512), (4096, 16, 1024), (64, 512, 5000), (33, 65, 8192),
    (128, 128, 256), (129, 127, 300), (256, 256, 512), (1000, 1500, 700), (700, 3000, 1281),
    (2048, 2048, 768), (2047, 2049, 513), (2560, 2500, 256), (4352, 4096, 256),
    (4300, 4100, 512), (4352, 4099, 700)])
def test_product(gpu, m, n, k):
    _check_product(gpu, m, n, k)


@pytest.mark.parametrize("m,n,k", [(16, 48, 512), (300, 301, 512), (2304, 2048, 256)])
@pytest.mark.parametrize("offset", [1, 4])
def test_product_c_at_any_element(gpu, m, n, k, offset):
    _check_product(gpu, m, n, k, offset)


@pytest.mark.parametrize("panels", [1, 2, 3, 4, 5, 6, 7, 8, 9, 13])
@pytest.mark.parametrize("m,n", [(20, 40), (384, 256), (1300, 1200), (2816, 1536)])
def test_product_of_every_number_of_panels(gpu, m, n, panels):
    _check_product(gpu, m, n, 256 * panels)


@pytest.mark.parametrize("m,n,k", [(20, 40000, 2048), (1, 66000, 2300), (36000, 17, 2048)])
def test_product_streams_more_than_a_round(gpu, m, n, k):
    _check_product(gpu, m, n, k)


@pytest.mark.parametrize("m,n,k", [(5120, 5120, 512), (8192, 4096, 1024), (5120, 4864, 768)])
def test_product_in_rounds(gpu, m, n, k):
    """More whole tiles than a device has CUs, the last round part full or not; stages of k
    that a round hands to the next, and (768) that it does not."""
    _check_product(gpu, m, n, k)


@pytest.mark.parametrize("m,n,k", [(20, 40, 600), (200, 300, 600), (2500, 2000, 512)])
def test_product_scales_of_every_size(gpu, m, n, k):
    """Scales down to 2^-127 beside others, whose products are subnormal or vanish."""
    rng = np.random.default_rng(m)
    a, b = _operand(rng, m, k, 60, 190), _operand(rng, n, k, 60, 190)
    a[1][:, : m // 2] = rng.integers(0, 3, a[1][:, : m // 2].shape)
    b[1][:, : n // 2] = rng.integers(120, 253, b[1][:, : n // 2].shape)
    got = bf16_to_f32(_product(gpu, a, b, m, n, k)).astype(np.float64)
    x, y = ref.unpack(*a), ref.unpack(*b)
    want = x @ y.T
    total = np.abs(x) @ np.abs(y).T
    fine = total < 2.0 ** 127  # others may overflow on the way
    bound = np.abs(want) * 2.0 ** -8 * (1 + 2.0 ** -7) + total * k * 2.0 ** -24 + 2.0 ** -126
    assert fine.mean() > 0.5
    assert np.all(np.abs(got - want)[fine] <= bound[fine])


@pytest.mark.parametrize("m,n", [(20, 40), (200, 300), (2500, 2000)])
def test_product_nan_scales(gpu, m, n):
    """A NaN block makes NaN of its row or column, and of nothing else."""
    rng = np.random.default_rng(m)
    a, b = _operand(rng, m, 700), _operand(rng, n, 700)
    a[1][2, m - 1, 3] = 255
    a[1][0, 3, 0] = 255
    b[1][1, n - 2, 7] = 255
    got = np.isnan(bf16_to_f32(_product(gpu, a, b, m, n, 700)))
    want = np.zeros((m, n), bool)
    want[[3, m - 1]] = True
    want[:, n - 2] = True
    assert np.array_equal(got, want)


def test_product_of_nothing(gpu):
    c = Guarded(gpu, np.full(20 * 30, 0x7FDE, np.uint16))
    none = Guarded(gpu, np.zeros(0, np.uint8)).body
    _k().gemm_mxfp4_nt(none, none, none, none, c.body, 20, 30, 0)
    assert c.guards_intact() and not np.any(c.download())


def test_tiles_and_split_agree_with_one_another(gpu):
    """The same rows in products of other sizes: the tiles' bits do not depend on them."""
    rng = np.random.default_rng(3)
    a, b = _operand(rng, 2560, 1000), _operand(rng, 2304, 1000)
    whole = _product(gpu, a, b, 2560, 2304, 1000)
    part = (a[0][:300], a[1][:, :304])  # scale rows 300 to 303 are of no effect
    assert_same(_product(gpu, part, b, 300, 2304, 1000), whole[:300], "first rows")


# ---- with torch: streams, graphs, tensors ---------------------------------------------------

def test_linear_on_tensors_streams_and_graphs(gpu):
    """Packing of activations and the product with packed weights, eager on a stream of
    its own and replayed from a graph over new activations."""
    torch = pytest.importorskip("torch")
    k = _k()
    gen = torch.Generator(device="cuda").manual_seed(5)
    m, n, cols = 37, 1100, 1000
    w = torch.randn(n, cols, generator=gen, device="cuda")
    packed = [torch.zeros(s, dtype=torch.uint8, device="cuda") for s in k.mxfp4_shapes(n, cols)]
    k.quantize_mxfp4(w, *packed)
    x = torch.randn(m, 2 * cols, generator=gen, device="cuda").to(torch.bfloat16)[:, cols:]
    acts = [torch.zeros(s, dtype=torch.uint8, device="cuda") for s in k.mxfp4_shapes(m, cols)]
    c = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    back = torch.empty(m, cols, device="cuda")

    def step(stream):
        k.quantize_mxfp4(x, *acts, stream=stream, sync=False)
        k.gemm_mxfp4_nt(*acts, *packed, c, stream=stream, sync=False)
        k.dequantize_mxfp4(*acts, back, stream=stream, sync=False)

    def check():
        torch.cuda.synchronize()
        host = x.float().cpu().numpy()
        want_q, want_s = ref.pack(host)
        assert np.array_equal(acts[0].cpu().numpy(), want_q)
        a = ref.unpack(want_q, want_s)
        assert np.array_equal(back.cpu().numpy(), a[:, :cols].astype(np.float32))
        b = ref.unpack(*ref.pack(w.cpu().numpy()))
        want = a @ b.T
        off = np.abs(c.float().cpu().numpy() - want)
        assert np.all(off <= np.abs(want) * 2.0 ** -8 * (1 + 2.0 ** -7)
                      + (np.abs(a) @ np.abs(b).T) * 2.0 ** -24 * cols)

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    step(side)
    side.synchronize()
    check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(side)
    for _ in range(3):
        x.copy_(torch.randn(m, cols, generator=gen, device="cuda"))
        c.zero_()
        graph.replay()
        check()


def test_packing_in_a_grid_of_two_dimensions(gpu):
    """More workgroups than a grid's row has, against the same rows in parts."""
    torch = pytest.importorskip("torch")
    k = _k()
    rows = 16 * (1 << 21) + 37
    x = torch.randn(rows, 1, device="cuda").to(torch.bfloat16)
    whole = [torch.full(s, 7, dtype=torch.uint8, device="cuda") for s in k.mxfp4_shapes(rows, 1)]
    back = torch.empty_like(x)
    k.quantize_mxfp4(x, *whole)
    k.dequantize_mxfp4(*whole, back)
    at = 0
    while at < rows:
        n = min(rows - at, 1 << 23)
        part = [torch.empty(s, dtype=torch.uint8, device="cuda") for s in k.mxfp4_shapes(n, 1)]
        values = torch.empty(n, 1, dtype=torch.bfloat16, device="cuda")
        k.quantize_mxfp4(x[at:at + n], *part)
        k.dequantize_mxfp4(*part, values)
        assert torch.equal(part[0], whole[0][at:at + n])
        assert torch.equal(part[1][:, :n], whole[1][:, at:at + n])
        assert torch.equal(values, back[at:at + n])
        at += n
    assert bool((whole[1][:, rows:] == 7).all())
