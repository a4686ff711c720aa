"""GPU tests of the 4-bit product's large tiles: every way that a launch takes, over its whole
loop, with all outputs compared.

The codes are any and the scales 1 and 2, so that a product is a multiple of 2^-2 below 2^8
and a sum of up to 2^14 of them a multiple of 2^-2 below 2^22: 24 bits hold every partial sum,
in any order, and C is the exact sum rounded once, bit for bit."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

GUARD, CANARY = 64, -7.0
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _k():
    from fe2o3_amd import kernels
    return kernels


def _operand(rows, k, seed, low=127, high=129):
    """A packed operand of any codes, scale bytes low .. high - 1; the columns past k are
    zeros, the scales of rows past the last NaN (they have no effect)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    codes, scales = _k().mxfp4_shapes(rows, k)
    q = torch.randint(0, 256, codes, generator=gen, device="cuda", dtype=torch.uint8)
    if k % 2:
        q[:, k // 2] &= 15
    q[:, (k + 1) // 2:] = 0
    s = torch.randint(low, high, scales, generator=gen, device="cuda", dtype=torch.uint8)
    s[:, rows:] = 255
    return q, s


def _unpack(q, s):
    """The matrix [rows, panels * 256] in 64 bits."""
    rows, panels = q.shape[0], s.shape[0]
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), device="cuda", dtype=torch.float64)
    code = torch.stack((q & 15, q >> 4), -1).view(rows, panels, 8, 32)
    byte = s[:, :rows].transpose(0, 1)
    scale = torch.exp2(byte.double() - 127).masked_fill(byte == 255, float("nan"))
    return (table[code.int()] * scale[..., None]).view(rows, panels * 256)


def _product(a, b, offset=0):
    """C at `offset` elements past 128 bytes, its surroundings unchanged."""
    m, n = a[0].shape[0], b[0].shape[0]
    held = torch.full((m * n + offset + 2 * GUARD,), CANARY, dtype=torch.bfloat16, device="cuda")
    c = held[GUARD + offset:GUARD + offset + m * n].view(m, n)
    _k().gemm_mxfp4_nt(*a, *b, c)
    assert bool((held[:GUARD + offset] == CANARY).all()) and bool((held[-GUARD:] == CANARY).all())
    return c


def _check_exact(m, n, k, offset=0):
    a, b = _operand(m, k, 2 * k + m), _operand(n, k, 2 * k + n + 1)
    got = _product(a, b, offset)
    want = torch.matmul(_unpack(*a), _unpack(*b).T.contiguous())
    assert float(want.abs().max()) < 2.0 ** 22
    bad = got != want.float().to(torch.bfloat16)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[0].tolist())


@pytest.mark.parametrize("panels", [2, 4, 6, 8, 10, 14])
def test_rounds(gpu, panels):
    """Tiles one after another in a workgroup: 400 on 256 CUs, from two stages of k a tile on;
    from six on the loop between a tile's first and last steps runs."""
    _check_exact(5120, 5120, 256 * panels)


@pytest.mark.parametrize("m,n,k", [(8192, 4096, 8192), (6144, 6144, 1536), (8192, 5120, 2048),
                                   (5120, 6656, 2550)])
def test_whole_rounds_and_a_tail(gpu, m, n, k):
    """Two whole rounds, and two with a last part round as quarters (three stages or two);
    k that ends within a panel."""
    _check_exact(m, n, k)


@pytest.mark.parametrize("m,n,k", [(512, 24576, 16384), (1024, 24576, 16384), (24576, 768, 16128)])
def test_staged_stores(gpu, m, n, k):
    """Operands of 192 MiB and more, whose tiles store C through LDS: less than a round, and a
    round with a tail of two stages, and of three under a tall C and an odd number of panels."""
    assert (m + n) * (-(-k // 256) * 128) >= 192 << 20
    _check_exact(m, n, k)


# more than 128 tiles of 256 x 256, where they run as such: whole tiles, and edges on both sides
ONE_ROUND = [(3328, 2816), (3300, 2801)]


@pytest.mark.parametrize("k", [256, 512, 700, 1280, 1536, 2304, 3328])
@pytest.mark.parametrize("m,n", ONE_ROUND)
def test_one_round(gpu, m, n, k):
    _check_exact(m, n, k)


@pytest.mark.parametrize("m,n", [*ONE_ROUND, (5120, 5120), (8192, 4096)])
@pytest.mark.parametrize("offset", [1, 4, 8])
def test_c_at_any_element_of_large_tiles(gpu, m, n, offset):
    """Whole tiles whose C is not at 16 bytes (8 elements are) end as edge tiles do."""
    _check_exact(m, n, 1024, offset)


# and in rounds with quarters behind or not, on small tiles, and split over a workgroup's waves
# (the last three: few tiles, a few rows of a wide C, a few columns of a tall one)
EVERY_WAY = [*ONE_ROUND, (5120, 5120), (6144, 6144), (1300, 1200), (300, 1100), (20, 4096),
             (4096, 17)]


@pytest.mark.parametrize("m,n", EVERY_WAY)
def test_nan_scales_of_large_tiles(gpu, m, n):
    """A NaN block makes NaN of its row or column and of nothing else: in the first, a middle
    and the last panel, in every block of a panel."""
    panels = 4
    a, b = _operand(m, 256 * panels, 1), _operand(n, 256 * panels, 2)
    gen = torch.Generator(device="cpu").manual_seed(m)
    rows = torch.randperm(m, generator=gen)[:min(m // 2, 24)].tolist() + [0, m - 1]
    cols = torch.randperm(n, generator=gen)[:min(n // 2, 24)].tolist() + [n - 1]
    for i, row in enumerate(rows):
        a[1][i % panels, row, i // 3 % 8] = 255
    for i, col in enumerate(cols):
        b[1][(i + 1) % panels, col, i // 3 % 8] = 255
    got = torch.isnan(_product(a, b))
    want = torch.zeros_like(got)
    want[rows] = True
    want[:, cols] = True
    assert torch.equal(got, want)


@pytest.mark.parametrize("m,n", EVERY_WAY)
def test_scales_of_every_size_of_large_tiles(gpu, m, n):
    """Scales down to 2^-127 beside others up to 2^125, whose products are subnormal or vanish.
    The bound: half a bf16 step of the result, for each of k additions 2^-24 of the sum of
    magnitudes, and what vanishes below the normal range."""
    k = 1024
    a, b = _operand(m, k, 3, 60, 190), _operand(n, k, 4, 60, 190)
    gen = torch.Generator(device="cuda").manual_seed(n)
    low, high = a[1][:, :m // 2], b[1][:, :n // 2]
    low.copy_(torch.randint(0, 3, low.shape, generator=gen, device="cuda"))
    high.copy_(torch.randint(120, 253, high.shape, generator=gen, device="cuda"))
    x, y = _unpack(*a), _unpack(*b)
    got = _product(a, b).double()
    want = torch.matmul(x, y.T.contiguous())
    total = torch.matmul(x.abs(), y.abs().T.contiguous())
    bound = want.abs() * 2.0 ** -8 * (1 + 2.0 ** -7) + total * k * 2.0 ** -24 + 2.0 ** -126
    fine = total < 2.0 ** 127  # others may overflow on the way
    assert float(fine.double().mean()) > 0.5
    assert bool((~fine | ((got - want).abs() <= bound)).all())


def test_every_tile_has_the_same_bits(gpu):
    """Rows of one product in tiles one after another with a last round of quarters, and the
    same rows of smaller products: in rounds alone, in one round of whole tiles and of edge
    tiles, in quarters' tiles of two stages and of three.  Scales of 14 octaves, so that sums
    round on the way and another order would show."""
    k = 2048
    a, b = _operand(8192, k, 5, 118, 132), _operand(5120, k, 6, 118, 132)
    whole = _product(a, b)

    def rows(x, first, count):
        up = (count + 15) // 16 * 16
        return x[0][first:first + count].contiguous(), x[1][:, first:first + up].contiguous()

    x, y = _unpack(*rows(a, 0, 256)), _unpack(*b)
    want = torch.matmul(x, y.T.contiguous())
    total = torch.matmul(x.abs(), y.abs().T.contiguous())
    bound = want.abs() * 2.0 ** -8 * (1 + 2.0 ** -7) + total * k * 2.0 ** -24
    assert bool(((whole[:256].double() - want).abs() <= bound).all())
    for first, count, cols in [(0, 5120, 5120), (4096, 4096, 5120), (1024, 1792, 5120),
                               (16, 1790, 5001), (6896, 1296, 5120), (7888, 300, 5120),
                               (32, 301, 4999)]:
        got = _product(rows(a, first, count), rows(b, 0, cols))
        same = got.view(torch.int16) == whole[first:first + count, :cols].view(torch.int16)
        assert bool(same.all()), (first, count, cols, int((~same).sum()))


@pytest.mark.parametrize("m,n,k", [(4300, 4900, 700), (4300, 4100, 1300), (4480, 4864, 1280),
                                   (4224, 4224, 512)])
def test_edges_and_a_tail(gpu, m, n, k):
    """A round of edge tiles and a last round of quarters, of two stages or three; the last two
    have whole quarters all the same."""
    _check_exact(m, n, k)
