"""Products of 4-bit operands whose blocks' exponents are any distance apart, against 64 bits.

Bound: S = the sum of the magnitudes of a result's products.  A product that is far below the largest of its
instruction, or below the sum that it is added to, is cut off where fp32 ends: what an instruction loses is taken as
2^-20 of its largest product at most, 2^-20 S in all, whatever the distance, and each of the K / 64 additions of
instructions' results, and of three more partial sums, as 2^-24 of a partial sum <= S."""
import pytest
import torch

from home_seek_amd import ops

pytestmark = pytest.mark.gpu

F64 = torch.float64
VALUES = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=F64)
VALUES = torch.cat((VALUES, -VALUES))


def operand(dev, g, rows, k, lo, hi):
    """(codes, scales), any of each, and what they stand for in 64 bits."""
    b = torch.randint(0, 256, (rows, k // 2), generator=g)
    e = torch.randint(lo, hi + 1, (rows, k // 32), generator=g)
    v = VALUES[torch.stack((b & 15, b >> 4), dim=-1).flatten(-2)] * torch.exp2(e.double()).repeat_interleave(32, dim=-1)
    return b.to(torch.uint8).view(torch.int8).to(dev), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu).to(dev), v


# few rows (by 16, 32, 48, 64), tiles of 64 whole and in halves, of 128, of 256
@pytest.mark.parametrize("m,n,k", ((1, 64, 1024), (5, 40, 96), (20, 64, 1024), (40, 64, 544), (64, 72, 2048), (80, 64, 256), (100, 136, 4096),
                                   (700, 4096, 256), (2100, 2056, 256), (4000, 4096, 96)))
@pytest.mark.parametrize("x,w", (((-4, 4), (-4, 4)), ((-24, 24), (-24, 24)), ((-50, 50), (-50, 50)), ((0, 0), (-100, 100)), ((-127, -100), (100, 127))))
def test_any_distance(dev, m, n, k, x, w):
    g = torch.Generator().manual_seed(m + k + x[1])
    xp, xs, xv = operand(dev, g, m, k, *x)
    wp, ws, wv = operand(dev, g, n, k, *w)
    out = ops.fp4_linear(xp, wp, ws, x_scale=xs, out_dtype=torch.float32)
    rows = torch.arange(m) if m <= 700 else torch.cat((torch.arange(0, 64), torch.randint(0, m, (100,), generator=g), torch.arange(m - 40, m)))
    xv = xv[rows]
    want, size = xv @ wv.T, xv.abs() @ wv.abs().T
    assert size.max() < 2.0 ** 126  # every partial sum is finite
    tol = size * (2.0 ** -20 + (k / 64 + 4) * 2.0 ** -24) + want.abs() * 2.0 ** -24 + 2.0 ** -149
    err = (out.cpu()[rows].double() - want).abs()
    assert (err <= tol).all(), float((err / size.clamp(min=2.0 ** -149)).max())
