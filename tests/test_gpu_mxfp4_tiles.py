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
