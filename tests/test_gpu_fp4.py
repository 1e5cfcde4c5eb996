"""Quantisation to the experts' 4-bit format, and products of two quantised
operands, against restatements in 64 bits: codes and exponents exactly, products
within a bound of their sums.

The bound: S = the sum of the magnitudes of a result's products.  Results of the
matrix instruction are summed in fp32, at most K / 64 of them and three more
partial sums: each addition is off by 2^-24 of a partial sum <= S at most, so
(K / 64 + 4) 2^-24 S.  Inside an instruction products of blocks whose exponents
are up to 20 apart lose 2^-20 of its largest product at most: 2^-20 S in all.
Then half a step of the output's type."""
import pytest
import torch

from home_seek_amd import ops

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E8M0 = torch.float8_e8m0fnu
GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=F64)


def normal(dev, seed, shape, dtype=BF16, std=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=dev) * std).to(dtype)


def plain_quant(x):
    """Codes [M, K] and exponent bytes [M, K/32] of finite rows, on the host in 64 bits."""
    v = x.cpu().double().reshape(x.shape[0], -1, 32)
    top = v.abs().amax(dim=2)
    e = torch.full_like(top, -127.0)
    for k in range(-126, 127):
        e = torch.where(6 * 2.0 ** (k - 1) < top, float(k), e)
    a = (v / torch.exp2(e)[:, :, None]).abs()
    lo = (torch.searchsorted(GRID, a, right=True) - 1).clamp(max=6)  # GRID[lo] <= a, and the next one above it
    down, above = a - GRID[lo], GRID[lo + 1] - a
    code = torch.where((above < down) | ((above == down) & (lo % 2 == 1)), lo + 1, lo)
    code = torch.where(torch.signbit(v), code + 8, code)
    return code.reshape(x.shape).to(torch.uint8), (e + 127).to(torch.uint8)


def pack(codes):
    return codes[..., 0::2] | codes[..., 1::2] << 4


def values(packed, scale):
    b = packed.view(torch.uint8).cpu()
    code = torch.stack((b & 15, b >> 4), dim=-1).flatten(-2).long()
    v = torch.cat((GRID, -GRID))[code]
    byte = scale.view(torch.uint8).cpu().double()
    s = torch.where(byte == 255, float("nan"), torch.exp2(byte - 127))
    return v * s.repeat_interleave(32, dim=-1)


@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("m,k", ((1, 32), (3, 64), (5, 96), (2, 1120), (7, 4096), (130, 544), (1025, 512), (1, 65536), (8200, 96), (4099, 1024), (4101, 544),
                                 (2731, 1536), (2050, 2048), (1367, 2592)))
def test_codes_and_scales(dev, m, k, dtype):
    x = normal(dev, m + k, (m, k), dtype)
    x[0, :32] = 0
    x[-1, -32:] *= 1e-30
    x[:, 3] *= 1e6
    packed, scale = ops.fp4_quant(x)
    code, byte = plain_quant(x)
    assert packed.dtype == torch.int8 and scale.dtype == E8M0
    assert torch.equal(scale.view(torch.uint8).cpu(), byte)
    assert torch.equal(packed.view(torch.uint8).cpu(), pack(code))
    back = ops.fp4_dequant_bf16(packed, scale)
    assert torch.equal(back.cpu().double(), values(packed, scale))


@pytest.mark.parametrize("dtype", (BF16, F32))
def test_ties_and_the_ends_of_the_range(dev, dtype):
    """Every border between two codes, and one step to both sides, under every exponent that the type holds them in."""
    edges = torch.tensor([0.0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6], dtype=F64)
    step = 1 + torch.finfo(dtype).eps
    row = torch.cat((edges, edges * step, -edges / step, -edges, torch.tensor([6.0, -6.0, -0.0, 0.0], dtype=F64)))
    row = torch.cat((row, torch.zeros(-row.numel() % 32, dtype=F64)))
    blocks = row.reshape(-1, 32)
    blocks = torch.cat((blocks, blocks.flip(1), blocks.clamp(-4.5, 4.5), blocks.clamp(-1, 1)))  # other largest values
    rows = [blocks.reshape(1, -1) * 2.0 ** e for e in (*range(-128, -120), -60, 0, 1, 77, *range(120, 126))]
    x = torch.cat(rows).to(dtype).to(dev)
    assert torch.isfinite(x).all()
    packed, scale = ops.fp4_quant(x)
    code, byte = plain_quant(x)
    assert torch.equal(scale.view(torch.uint8).cpu(), byte)
    assert torch.equal(packed.view(torch.uint8).cpu(), pack(code))


@pytest.mark.parametrize("dtype", (BF16, F32))
def test_largest_and_smallest_values(dev, dtype):
    fi = torch.finfo(dtype)
    x = torch.zeros(4, 64, dtype=dtype)
    x[0, 5], x[0, 40] = fi.max, -fi.max
    x[1, 0], x[1, 33] = fi.smallest_normal, -fi.smallest_normal
    x[2, 1], x[2, 60] = fi.smallest_normal * 2.0 ** -5, 2.0 ** -127
    packed, scale = ops.fp4_quant(x.to(dev))
    code, byte = plain_quant(x)
    assert torch.equal(scale.view(torch.uint8).cpu(), byte)
    assert torch.equal(packed.view(torch.uint8).cpu(), pack(code))


@pytest.mark.parametrize("bad", (float("inf"), -float("inf"), float("nan")))
def test_infinity_and_nan_take_their_block_only(dev, bad):
    x = normal(dev, 1, (5, 128))
    x[2, 70] = bad
    packed, scale = ops.fp4_quant(x)
    got = ops.fp4_dequant_bf16(packed, scale)
    keep = torch.ones_like(x, dtype=torch.bool)
    keep[2, 64:96] = False
    assert got[~keep].isnan().all()
    x[2, 70] = 0
    assert torch.equal(got[keep], ops.fp4_dequant_bf16(*ops.fp4_quant(x))[keep])
    for m in (5, 200):  # in a product: its row, whole
        xx = normal(dev, 2, (m, 128))
        xx[m - 2, 70] = bad
        w = ops.fp4_quant(normal(dev, 3, (24, 128)))
        out = ops.fp4_linear(xx, *w)
        rows = out.isnan().all(dim=1)
        assert rows[m - 2] and int(rows.sum()) == 1 and int(out.isnan().any(dim=1).sum()) == 1
    cols = normal(dev, 4, (200, 128))  # and as a column of the other operand, whole
    cols[198, 70] = bad
    for m in (5, 200):
        out = ops.fp4_linear(normal(dev, 5, (m, 128)), *ops.fp4_quant(cols))
        assert out[:, 198].isnan().all() and int(out.isnan().sum()) == m


def test_quant_of_views(dev):
    base = normal(dev, 4, (6, 5, 256))
    want = ops.fp4_quant(base.contiguous())
    for x in (base[:, :, 64:192], base[::2], base.transpose(0, 1), base[:, 1:3, 32:64], base.reshape(-1)[8:7 * 32 + 8].view(7, 32)):
        packed, scale = ops.fp4_quant(x)
        p, s = ops.fp4_quant(x.contiguous().clone())
        assert packed.shape == x.shape[:-1] + (x.shape[-1] // 2,) and scale.shape == x.shape[:-1] + (x.shape[-1] // 32,)
        assert torch.equal(packed, p) and torch.equal(scale.view(torch.uint8), s.view(torch.uint8))
    assert torch.equal(want[0][3, 2], ops.fp4_quant(base[3, 2])[0])
    empty = ops.fp4_quant(base[:0])
    assert empty[0].shape == (0, 5, 128) and empty[1].shape == (0, 5, 8)


def check(out, x, w, k, dtype):
    """x, w: (packed, scale)."""
    xv, wv = values(*x), values(*w)
    want, size = xv @ wv.T, xv.abs() @ wv.abs().T
    tol = size * (2.0 ** -20 + (k / 64 + 4) * 2.0 ** -24) + want.abs() * (torch.finfo(dtype).eps / 2)
    err = (out.cpu().double() - want).abs()
    assert out.dtype == dtype and (err <= tol).all(), float((err - tol).max())


# rows that take each kernel: a workgroup's own quantisation, few rows (16, 32, 48, 64), tiles of 64; ragged reductions
SIZES = [
    (1, 64, 4096), (1, 8, 32), (2, 24, 96), (3, 136, 512), (4, 64, 4096), (5, 48, 4096), (16, 40, 1024), (17, 64, 2048),
    (33, 72, 544), (48, 64, 480), (49, 128, 1056), (64, 520, 4096), (64, 8, 64), (65, 64, 64), (65, 8, 32), (66, 200, 96),
    (100, 136, 4096), (127, 72, 2016), (300, 264, 768), (513, 1000, 288), (16, 4096, 64), (1, 64, 32768), (130, 64, 16384),
    (100, 1032, 1056), (250, 4096, 1024), (200, 520, 2336), (70, 72, 2048), (66, 264, 2592), (2, 32776, 2080), (16, 24008, 512), (33, 16392, 1024), (64, 8200, 2080), (1, 40000, 512), (2, 12000, 544),
]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_products(dev, m, n, k):
    x, w = normal(dev, m, (m, k)), ops.fp4_quant(normal(dev, n, (n, k)))
    x[:, 1] *= 40
    xq = ops.fp4_quant(x)
    for dtype in (BF16, F32):
        out = ops.fp4_linear(x, *w, out_dtype=dtype)
        check(out, xq, w, k, dtype)
        if k % 512 == 0 or m > 16:
            assert torch.equal(out, ops.fp4_linear(xq[0], *w, x_scale=xq[1], out_dtype=dtype))
    x32 = x.float() * 1.001  # fp32 rows with more bits than bf16's
    check(ops.fp4_linear(x32, *w), ops.fp4_quant(x32), w, k, BF16)
    xq32 = ops.fp4_quant(x32)
    check(ops.fp4_linear(xq32[0], *w, x_scale=xq32[1]), xq32, w, k, BF16)


@pytest.mark.parametrize("m,n,k", ((2050, 2056, 96), (2049, 2040, 544), (4097, 4104, 320), (4090, 4000, 1024), (3900, 4008, 96), (4095, 4088, 544),
                                   (7700, 4096, 32)))
def test_products_of_large_tiles(dev, m, n, k):
    x, w = normal(dev, m, (m, k)), ops.fp4_quant(normal(dev, n, (n, k)))
    check(ops.fp4_linear(x, *w), ops.fp4_quant(x), w, k, BF16)
    check(ops.fp4_linear(x, *w, out_dtype=F32), ops.fp4_quant(x), w, k, F32)


@pytest.mark.parametrize("m", (1, 20, 80, 2100, 4000))
def test_far_exponents(dev, m):
    """Scales over the whole range: sums whose blocks are far apart, results that no output type holds."""
    n, k = {2100: 2056, 4000: 4096}.get(m, 64), 256
    g = torch.Generator(device=dev).manual_seed(m)
    x = normal(dev, m, (m, k), F32) * torch.exp2(torch.randint(-10, 10, (m, k // 32, 1), generator=g, device=dev).expand(-1, -1, 32).reshape(m, k).float())
    wq = ops.fp4_quant(normal(dev, 9, (n, k)))
    check(ops.fp4_linear(x, *wq, out_dtype=F32), ops.fp4_quant(x), wq, k, F32)
    big = ops.fp4_linear(torch.full((m, k), 2.0 ** 120, device=dev), *ops.fp4_quant(torch.full((n, k), 2.0 ** 20, device=dev)))
    assert (big == float("inf")).all()
    small = ops.fp4_linear(torch.full((m, k), 2.0 ** -120, device=dev), *ops.fp4_quant(torch.full((n, k), 2.0 ** -60, device=dev)))
    assert (small == 0).all()
    ends = ops.fp4_linear(torch.full((m, k), 2.0 ** -120, device=dev), *ops.fp4_quant(torch.full((n, k), 2.0 ** 122, device=dev)))
    assert (ends == k * 4).all()


def test_shapes_views_and_no_rows(dev):
    k, n = 256, 40
    w, s = ops.fp4_quant(normal(dev, 1, (n, k)))
    base = normal(dev, 2, (4, 5, k + 64))
    x = base[:, :, 32:32 + k]
    out = ops.fp4_linear(x, w, s)
    assert out.shape == (4, 5, n) and torch.equal(out.reshape(20, n), ops.fp4_linear(x.reshape(20, k).contiguous(), w, s))
    assert ops.fp4_linear(x[0, 0], w, s).shape == (n,)
    assert ops.fp4_linear(x[:0], w, s).shape == (0, 5, n)
    p, e = ops.fp4_quant(x)
    assert torch.equal(ops.fp4_linear(p, w, s, x_scale=e), ops.fp4_linear(x, w, s))
    assert torch.equal(ops.fp4_linear(p.transpose(0, 1), w, s, x_scale=e.transpose(0, 1)), ops.fp4_linear(x, w, s).transpose(0, 1))
    wide, wide_s = ops.fp4_quant(normal(dev, 3, (n, 2 * k)))
    half, half_s = wide[:, : k // 2], wide_s[:, : k // 32]  # rows that are not contiguous
    assert torch.equal(ops.fp4_linear(x, half, half_s), ops.fp4_linear(x, half.contiguous(), half_s.contiguous()))
    assert torch.equal(ops.fp4_linear(x, w.view(torch.uint8), s), ops.fp4_linear(x, w, s))


@pytest.mark.parametrize("m", (1, 40, 333))
def test_other_stream_and_replayed(dev, m):
    k, n = 1024, 128
    w, s = ops.fp4_quant(normal(dev, 1, (n, k)))
    x = normal(dev, 2, (m, k))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = ops.fp4_linear(x, w, s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, q = ops.fp4_linear(x, w, s), ops.fp4_quant(x)
    torch.cuda.synchronize()
    assert torch.equal(first, ops.fp4_linear(x, w, s))
    for seed in range(3):
        x.copy_(normal(dev, 10 + seed, (m, k)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.fp4_linear(x, w, s))
        p, e = ops.fp4_quant(x)
        assert torch.equal(q[0], p) and torch.equal(q[1].view(torch.uint8), e.view(torch.uint8))


def test_nothing_behind_the_operands_counts(dev):
    """Rows and columns of tiles that are not there: what lies behind the operands in memory changes nothing."""
    for m, n, k in ((3, 24, 96), (20, 24, 96), (70, 72, 352)):
        x, wx = normal(dev, m, (m, k)), normal(dev, n, (n, k))
        w, s = ops.fp4_quant(wx)
        xp, xs = ops.fp4_quant(x)
        want = ops.fp4_linear(x, w, s)

        def inside(t):
            big = torch.full((t.numel() + 65536,), 0xff if t.element_size() == 1 else float("nan"), device=dev,
                             dtype=torch.uint8 if t.element_size() == 1 else t.dtype)
            part = big[: t.numel()]
            part.copy_(t.reshape(-1).view(torch.uint8) if t.element_size() == 1 else t.reshape(-1))
            return part.view(t.dtype).view(t.shape)

        assert torch.equal(want, ops.fp4_linear(inside(x), inside(w), inside(s)))
        assert torch.equal(ops.fp4_linear(xp, w, s, x_scale=xs), ops.fp4_linear(inside(xp), inside(w), inside(s), x_scale=inside(xs)))


def test_refusals(dev):
    x = normal(dev, 1, (4, 64))
    w, s = ops.fp4_quant(normal(dev, 2, (16, 64)))
    for bad, exc in ((lambda: ops.fp4_quant(x.half()), TypeError), (lambda: ops.fp4_quant(x[:, :40]), ValueError),
                     (lambda: ops.fp4_quant(x[:, :0]), ValueError), (lambda: ops.fp4_quant(x.cpu()), RuntimeError),
                     (lambda: ops.fp4_linear(x[:, :32], w, s), ValueError), (lambda: ops.fp4_linear(x, w, s.float()), TypeError),
                     (lambda: ops.fp4_linear(x, w, s[:8]), ValueError), (lambda: ops.fp4_linear(x, w.float(), s), TypeError),
                     (lambda: ops.fp4_linear(x, w[:12], s[:12]), RuntimeError), (lambda: ops.fp4_linear(x, w, s, out_dtype=torch.float16), TypeError),
                     (lambda: ops.fp4_linear(x, w[0], s[0]), ValueError), (lambda: ops.fp4_linear(w[:4], w, s, x_scale=s[:3]), ValueError),
                     (lambda: ops.fp4_linear(x, w, s, x_scale=s[:4]), ValueError)):
        with pytest.raises(exc):
            bad()
