"""Products with bias, activation and residual, dense and per expert, and their
gradients, against 64-bit restatements.

Inputs are small integers over a power of two where that can be: every sum is
then exact in fp32, in any order, so results without an activation are the
correctly rounded 64-bit ones, bit for bit.  Behind an activation a result is
off by the fp32 evaluation (the exponential, the sum, the quotient and up to
four products: 16 x 2^-24 of the magnitudes that enter) plus half a step of its
type; a gradient also carries the bf16 rounding of dz, half a step of every term
(2^-8, half a step of bf16 being 2^-9 of the next power of two above the value,
at most 2^-8 of the value)."""
import pytest
import torch

from home_seek_amd import ops

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
LIMIT = 1.5


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def ints(dev, seed, shape, top=3, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randint(-top, top + 1, shape, generator=g, device=dev) * scale).to(BF16)


def some_order(dev, m, k, e, seed, drop=0.0, skew=False):
    g = torch.Generator(device=dev).manual_seed(seed)
    u = torch.rand((m, k), generator=g, device=dev)
    idx = ((u * u if skew else u) * e).long().clamp(max=e - 1)
    if drop:
        idx = torch.where(torch.rand((m, k), generator=g, device=dev) < drop, -1, idx)
    return ops.moe_sort(idx, e)


def spans(order, rows):
    if order is None:
        return [(None, 0, rows)]
    off = order.offsets.tolist()
    return [(e, a, b) for e, (a, b) in enumerate(zip(off[:-1], off[1:]))]


def at(t, e):
    return t if e is None else t[e]


def act64(act, z, zu):
    """(y, y' by z, y' by zu, the magnitudes that enter y)"""
    if act is None:
        return z, torch.ones_like(z), None, z.abs()
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s), None, z.abs()
    g, u = z.clamp(max=LIMIT), zu.clamp(-LIMIT, LIMIT)
    s = torch.sigmoid(g)
    return (g * s * u, (s + g * s * (1 - s)) * u * (z <= LIMIT), g * s * (zu.abs() <= LIMIT), (g * u).abs())


def forward64(x, w, w_up, bias, bias_up, residual, act, order):
    p, n = x.shape[0], w.shape[-2]
    y = torch.zeros(p, n, dtype=F64, device=x.device)
    size = torch.zeros_like(y)
    zs = [torch.zeros_like(y) for _ in range(2 if act == "swiglu" else 1)]
    for e, a, b in spans(order, p):
        for z, ww, bb in zip(zs, (w, w_up), (bias, bias_up)):
            z[a:b] = x[a:b].double() @ at(ww, e).double().T + (0 if bb is None else at(bb, e).double())
        y[a:b], _, _, size[a:b] = act64(act, zs[0][a:b], zs[-1][a:b])
        if residual is not None:
            y[a:b] += residual[a:b].double()
            size[a:b] += residual[a:b].double().abs()
    return y, size, torch.cat(zs, dim=1)


def check_forward(dev, m, n, k, act, order=None, lead=(), with_bias=True, with_res=True, out_dtype=BF16):
    scale = 1.0 if act is None else 2.0 ** -(k.bit_length() // 2 + 2)
    x, w = ints(dev, 1, (m, k)), ints(dev, 2, lead + (n, k), scale=scale)
    w_up = ints(dev, 3, lead + (n, k), scale=scale) if act == "swiglu" else None
    bias = ints(dev, 4, lead + (n,), scale=scale) if with_bias else None
    bias_up = ints(dev, 5, lead + (n,), scale=scale) if with_bias and act == "swiglu" else None
    res = ints(dev, 6, (m, n), top=9) if with_res else None
    limit = LIMIT if act == "swiglu" else None
    out, pre = ops.linear(x, w, bias, res, act=act, w_up=w_up, bias_up=bias_up, limit=limit, order=order,
                          out_dtype=out_dtype, want_pre=True)
    alone = ops.linear(x, w, bias, res, act=act, w_up=w_up, bias_up=bias_up, limit=limit, order=order, out_dtype=out_dtype)
    y, size, z = forward64(x, w, w_up, bias, bias_up, res, act, order)
    assert out.dtype == out_dtype and torch.equal(out, alone)
    assert torch.equal(pre, z.to(F32).to(BF16))  # exact sums, one rounding
    if act is None:
        assert torch.equal(out, y.to(F32).to(out_dtype))
    else:
        bound = 16 * 2.0 ** -24 * size
        assert bool(((out.double() - y).abs() <= bound + half_step(out_dtype) * (y.abs() + bound)).all())


SHAPES = [(1, 8, 8), (1, 4096, 4096), (3, 64, 72), (5, 1000, 520), (8, 2048, 1024), (16, 256, 64), (17, 136, 4096),
          (31, 520, 2048), (33, 4096, 128), (64, 72, 1000), (100, 264, 136), (127, 128, 64), (129, 1288, 200),
          (500, 2048, 512), (1000, 504, 1032), (2049, 4096, 256), (4093, 2056, 64),
          (4100, 4104, 72),  # more than 256 tiles of 256 x 256
          # every tile, whole and with its reduction split, for one matrix and for swiglu's two
          (1500, 4096, 136), (1900, 2048, 136), (200, 4104, 136), (500, 4104, 136), (2000, 4104, 136), (2500, 2056, 520),
          (3001, 136, 4104)]


@pytest.mark.parametrize("act", [None, "silu", "swiglu"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_dense(dev, m, n, k, act):
    check_forward(dev, m, n, k, act)


@pytest.mark.parametrize("with_bias,with_res,out_dtype", [(False, False, BF16), (True, False, F32), (False, True, F32)])
@pytest.mark.parametrize("act", [None, "swiglu"])
@pytest.mark.parametrize("m", [1, 7, 40, 300])
def test_dense_without_the_options(dev, m, act, with_bias, with_res, out_dtype):
    check_forward(dev, m, 392, 264, act, None, (), with_bias, with_res, out_dtype)


GROUPS = [(1, 6, 256, 64, 128, 0.0), (8, 6, 256, 512, 512, 0.0), (8, 2, 3, 72, 200, 0.5), (40, 4, 16, 264, 72, 0.3),
          (37, 16, 5, 520, 136, 0.1), (300, 6, 64, 136, 64, 0.2), (512, 6, 8, 512, 256, 0.0), (700, 3, 1, 256, 128, 0.4),
          (50, 2, 1024, 8, 8, 0.0), (90, 3, 7, 64, 64, 1.0), (1500, 4, 20, 1032, 328, 0.1), (1200, 4, 12, 2056, 136, 0.0), (1200, 4, 12, 136, 2056, 0.0),
          (750, 2, 16, 1032, 136, 0.1), (750, 2, 8, 4104, 136, 0.1), (1250, 2, 3, 2056, 520, 0.1), (750, 2, 8, 136, 4104, 0.1),
          (1250, 2, 3, 520, 2056, 0.1), (750, 2, 8, 2056, 136, 0.1), (1000, 2, 3, 136, 2056, 0.1), (100, 2, 16, 4104, 1032, 0.1)]


@pytest.mark.parametrize("act", [None, "silu", "swiglu"])
@pytest.mark.parametrize("m,top_k,e,n,k,drop", GROUPS)
def test_per_expert(dev, m, top_k, e, n, k, drop, act):
    order = some_order(dev, m, top_k, e, m, drop, skew=True)
    check_forward(dev, m * top_k, n, k, act, order, (e,))


def test_random_values_within_the_sums_error(dev):
    """Sums that round: n additions are off by at most n 2^-23 of the magnitudes (2^-23: whichever way the matrix
    cores round)."""
    m, n, k = 333, 520, 2048
    x, w = torch.randn(m, k, device=dev).to(BF16), torch.randn(n, k, device=dev).to(BF16)
    out = ops.linear(x, w, out_dtype=F32)
    want = x.double() @ w.double().T
    assert bool(((out.double() - want).abs() <= k * 2.0 ** -23 * (x.double().abs() @ w.double().abs().T)).all())


def test_leading_dimensions_and_strides(dev):
    base, wide = ints(dev, 1, (6, 10, 3, 264)), ints(dev, 2, (2, 520, 320))
    x, w = base[:, :, 1, :200], wide[0, :, 8:208]
    res = ints(dev, 3, (6, 10, 1040))[:, :, 520:]
    want = (x.double() @ w.double().T + res.double()).to(F32).to(BF16)
    assert torch.equal(ops.linear(x, w, residual=res), want)
    assert torch.equal(ops.linear(base[:, :, 1, 3:203], wide[0, :, 5:205]),  # rows that are not 16-byte aligned
                       (base[:, :, 1, 3:203].double() @ wide[0, :, 5:205].double().T).to(F32).to(BF16))
    assert torch.equal(ops.linear(x, w.T.contiguous().T, residual=res), want)
    assert torch.equal(ops.linear(x[0, 0], w), (x[0, 0].double() @ w.double().T).to(F32).to(BF16))
    assert torch.equal(ops.linear(x[:1, :1].expand(6, 10, 200), w, residual=res),
                       (x[:1, :1].double() @ w.double().T + res.double()).to(F32).to(BF16))


def test_views_of_stacked_expert_weights(dev):
    """w and w_up as halves of one [E, 2 N, K] tensor, as a checkpoint may stack them."""
    e, n, k = 6, 136, 72
    w13 = ints(dev, 1, (e, 2 * n, k), scale=0.125)
    order = some_order(dev, 30, 2, e, 1)
    x = ints(dev, 2, (60, k))
    a = ops.linear(x, w13[:, :n], act="swiglu", w_up=w13[:, n:], limit=LIMIT, order=order)
    b = ops.linear(x, w13[:, :n].contiguous(), act="swiglu", w_up=w13[:, n:].contiguous(), limit=LIMIT, order=order)
    assert torch.equal(a, b)


def test_no_rows(dev):
    w = ints(dev, 1, (64, 72))
    assert ops.linear(torch.empty(0, 72, dtype=BF16, device=dev), w).shape == (0, 64)
    order = ops.moe_sort(torch.empty(0, 2, dtype=torch.int64, device=dev), 3)
    w3 = ints(dev, 2, (3, 64, 72))
    x = torch.empty(0, 72, dtype=BF16, device=dev)
    assert ops.linear(x, w3, order=order).shape == (0, 64)
    g = ops.linear_grad(torch.empty(0, 64, dtype=BF16, device=dev), x, w3, order=order, need_bias=True)
    assert g.x.shape == (0, 72) and not bool(g.w.any()) and not bool(g.bias.any()) and g.w.shape == w3.shape


def test_infinities_and_nan_stay_in_their_rows(dev):
    """A row's values reach that row's results only, and padding reaches none."""
    m, n, k = 70, 136, 72
    x, w = ints(dev, 1, (m, k)), ints(dev, 2, (n, k))
    want = ops.linear(x, w)
    x[3, 5], x[40, 0], x[69, 71] = float("inf"), float("nan"), float("-inf")
    got = ops.linear(x, w)
    rest = [r for r in range(m) if r not in (3, 40, 69)]
    assert torch.equal(got[rest], want[rest]) and bool(got[40].isnan().all())
    assert not bool(got[3].isfinite().any()) and not bool(got[69].isfinite().any())
    order = some_order(dev, 20, 2, 3, 1, 0.5)
    rows = ints(dev, 3, (40, k))
    rows[int(order.offsets[-1]):] = float("nan")
    out = ops.linear(rows, ints(dev, 4, (3, n, k)), order=order, residual=torch.full((40, n), float("nan"), device=dev).to(BF16))
    assert not bool(out[int(order.offsets[-1]):].any())


def test_swiglu_at_its_limit(dev):
    """Beyond the limit, infinite, at it, and NaN: as torch's clamp."""
    vals = torch.tensor([float("-inf"), -100.0, -LIMIT, -1.0, 0.0, 1.0, LIMIT, 2.0, 1e30, float("inf"), float("nan")])
    z, zu = torch.meshgrid(vals, vals, indexing="ij")
    x = torch.zeros(1, 8, device=dev, dtype=BF16)
    n = 128
    bias, bias_up = torch.zeros(n, device=dev, dtype=BF16), torch.zeros(n, device=dev, dtype=BF16)
    bias[:121], bias_up[:121] = z.reshape(-1), zu.reshape(-1)
    w = torch.zeros(n, 8, device=dev, dtype=BF16)
    for limit in (LIMIT, None):
        out, pre = ops.linear(x, w, bias, act="swiglu", w_up=w, bias_up=bias_up, limit=limit, out_dtype=F32, want_pre=True)
        g = bias.double() if limit is None else bias.double().clamp(max=limit)
        u = bias_up.double() if limit is None else bias_up.double().clamp(-limit, limit)
        want = (g * torch.sigmoid(g) * u)[None]
        finite = want.isfinite() & (want.abs() < 3e38)
        assert torch.equal(out.isnan(), want.isnan())
        assert bool(((out.double() - want).abs() <= 2.0 ** -20 * (g * u).abs() + 1e-30)[finite].all())
        assert torch.equal(out[~finite & ~want.isnan()].double().sign(), want[~finite & ~want.isnan()].sign())


def grads64(d_out, x, w, w_up, pre, act, order):
    """(dx, dw's, db's) and bounds of what the bf16 rounding of dz and the fp32 evaluation can change in each."""
    p, n = d_out.shape
    d = d_out.double()
    if act is None:
        dz, err = [d], [torch.zeros_like(d)]
    else:
        z = pre.double()
        _, a, b, _ = act64(act, z[:, :n], z[:, -n:])
        if act == "silu":
            dz, size = [d * a], [d.abs() * (1 + z.abs())]
        else:
            lim = torch.clamp(z[:, n:].abs(), max=LIMIT)
            dz = [d * a, d * b]
            gate = z[:, :n].clamp(max=LIMIT).abs()
            size = [d.abs() * lim * (1 + gate), d.abs() * gate]
        err = [half_step(BF16) * v.abs() + 16 * 2.0 ** -24 * s for v, s in zip(dz, size)]
    ws = (w, w_up)[: len(dz)]
    dx, ex = torch.zeros(x.shape, dtype=F64, device=x.device), torch.zeros(x.shape, dtype=F64, device=x.device)
    dw = [torch.zeros(t.shape, dtype=F64, device=x.device) for t in ws]
    ew = [torch.zeros_like(t) for t in dw]
    db = [torch.zeros(t.shape[:-1], dtype=F64, device=x.device) for t in ws]
    eb = [torch.zeros_like(t) for t in db]
    for e, a, b in spans(order, p):
        for j, t in enumerate(ws):
            dx[a:b] += dz[j][a:b] @ at(t, e).double()
            ex[a:b] += err[j][a:b] @ at(t, e).double().abs()
            ix = slice(None) if e is None else e
            dw[j][ix] = dz[j][a:b].T @ x[a:b].double()
            ew[j][ix] = err[j][a:b].T @ x[a:b].double().abs()
            db[j][ix] = dz[j][a:b].sum(dim=0)
            # summed before the rounding of dz, in fp32
            eb[j][ix] = (b - a + 16) * 2.0 ** -24 * (dz[j][a:b].abs().sum(dim=0) + (0 if act is None else size[j][a:b].sum(dim=0)))
    return (dx, ex), list(zip(dw, ew)), list(zip(db, eb))


def within(got, want, err, terms=0):
    slack = err + terms * 2.0 ** -23 * err + half_step(got.dtype) * (want.abs() + err)
    return bool(((got.double() - want).abs() <= slack + 1e-300).all())


def check_grad(dev, m, n, k, act, order=None, lead=()):
    d_out, x, w = ints(dev, 1, (m, n)), ints(dev, 2, (m, k)), ints(dev, 3, lead + (n, k))
    w_up = ints(dev, 4, lead + (n, k)) if act == "swiglu" else None
    mats = 2 if act == "swiglu" else 1
    pre = ints(dev, 5, (m, mats * n), top=20, scale=0.125) if act else None
    limit = LIMIT if act == "swiglu" else None
    if order is not None:  # rows of no expert are not read
        last = int(order.offsets[-1])
        for t in (d_out, x, pre):
            if t is not None:
                t[last:] = float("nan")
    kw = dict(act=act, pre=pre, w_up=w_up, limit=limit, order=order)
    got = ops.linear_grad(d_out, x, w, need_bias=True, **kw)
    got32 = ops.linear_grad(d_out, x, w, need_x=False, w_dtype=F32, **kw)
    clean = [None if t is None else t.nan_to_num(nan=0.0) for t in (d_out, x, pre)]
    dx, dw, db = grads64(clean[0], clean[1], w, w_up, clean[2], act, order)
    if act is None:  # exact sums
        assert torch.equal(got.x, dx[0].to(F32).to(BF16))
        assert torch.equal(got.w, dw[0][0].to(F32).to(BF16)) and torch.equal(got32.w, dw[0][0].to(F32))
        assert torch.equal(got.bias, db[0][0].to(F32))
        assert got.w_up is None and got.bias_up is None and got32.x is None and got32.bias is None
        return
    assert within(got.x, *dx, terms=2 * n)
    for j, (t, t32, b) in enumerate(zip((got.w, got.w_up)[:mats], (got32.w, got32.w_up)[:mats], (got.bias, got.bias_up)[:mats])):
        # the bf16 one is the fp32 one rounded
        assert torch.equal(t, t32.to(BF16))
        assert bool(((t32.double() - dw[j][0]).abs() <=
                     dw[j][1] + m * 2.0 ** -23 * (dw[j][0].abs() + dw[j][1] * 2.0 ** 9) + 1e-300).all())
        assert bool(((b.double() - db[j][0]).abs() <= db[j][1] + 1e-300).all())


@pytest.mark.parametrize("act", [None, "silu", "swiglu"])
@pytest.mark.parametrize("m,n,k", [(1, 8, 8), (1, 1024, 512), (3, 64, 72), (17, 136, 264), (64, 256, 128), (65, 72, 1000),
                                   (130, 520, 136), (500, 512, 512), (1001, 264, 520), (300, 2048, 4096), (4100, 72, 4104), (72, 4104, 4104),
                                   (1500, 136, 4096), (2000, 1024, 1024), (500, 136, 4104), (2000, 136, 4104),
                                   (2500, 520, 2056), (3001, 136, 2056), (500, 4104, 4104)])
def test_dense_gradient(dev, m, n, k, act):
    check_grad(dev, m, n, k, act)


@pytest.mark.parametrize("act", [None, "silu", "swiglu"])
@pytest.mark.parametrize("m,top_k,e,n,k,drop", GROUPS)
def test_per_expert_gradient(dev, m, top_k, e, n, k, drop, act):
    order = some_order(dev, m, top_k, e, m + 1, drop, skew=True)
    check_grad(dev, m * top_k, n, k, act, order, (e,))


def test_gradient_parts(dev):
    d_out, x, w = ints(dev, 1, (70, 64)), ints(dev, 2, (70, 72)), ints(dev, 3, (64, 72))
    pre = ints(dev, 4, (70, 64), scale=0.5)
    whole = ops.linear_grad(d_out, x, w, act="silu", pre=pre, need_bias=True)
    parts = [ops.linear_grad(d_out, x, w, act="silu", pre=pre, need_x=a, need_w=b, need_bias=c)
             for a, b, c in ((True, False, False), (False, True, False), (False, False, True), (False, False, False))]
    assert torch.equal(parts[0].x, whole.x) and parts[0].w is None and parts[0].bias is None
    assert torch.equal(parts[1].w, whole.w) and parts[1].x is None
    assert torch.equal(parts[2].bias, whole.bias) and all(t is None for t in parts[3])


def test_gradient_against_differences(dev):
    """y is smooth between the limits: a central difference of the fp32 result along a direction gives the
    gradient's product with it, up to the step's third-order term and the rounding over the step."""
    m, n, k = 24, 64, 72
    g = torch.Generator(device=dev).manual_seed(3)
    x = ints(dev, 1, (m, k), scale=0.25)
    w, w_up = ints(dev, 2, (n, k), scale=0.0625), ints(dev, 3, (n, k), scale=0.0625)
    d_out = ints(dev, 4, (m, n))
    step = ints(dev, 5, (m, k), top=1, scale=0.03125)  # x +- step are bf16 values
    _, pre = ops.linear(x, w, act="swiglu", w_up=w_up, want_pre=True)
    grad = ops.linear_grad(d_out, x, w, act="swiglu", pre=pre, w_up=w_up)
    f = [(ops.linear(x + s, w, act="swiglu", w_up=w_up, out_dtype=F32).double() * d_out.double()).sum()
         for s in (step, -step)]
    assert torch.equal((x + step).double(), x.double() + step.double())
    want = float((f[0] - f[1]) / 2)
    got = float((grad.x.double() * step.double()).sum())
    # third derivatives of silu(g) u along the step: |g'''| <= 1 with |u| <= 8 and |dz| <= |step| |w|_1 <= 0.5 per sum,
    # plus bf16 roundings of pre (2^-8 of |z| <= 8, on a slope that changes by at most 8 per unit), dz and dx
    dz_step = (step.double().abs() @ w.double().abs().T + step.double().abs() @ w_up.double().abs().T)
    bound = float((d_out.double().abs() * (dz_step ** 3 * 2 + dz_step * 2.0 ** -7 * 16)).sum())
    assert abs(got - want) <= bound and abs(want) > 0


def test_deterministic_and_replayed(dev):
    """A captured expert layer (sort, gather, products, combine, and back) replays what eager calls give."""
    m, k, e, d, i = 60, 4, 12, 256, 136
    g = torch.Generator(device=dev).manual_seed(1)
    x = ints(dev, 1, (m, d), scale=0.25)
    idx = torch.randint(0, e, (m, k), generator=g, device=dev)
    w = torch.rand((m, k), generator=g, device=dev)
    w1, w3, w2 = ints(dev, 2, (e, i, d), scale=0.03125), ints(dev, 3, (e, i, d), scale=0.03125), ints(dev, 4, (e, d, i), scale=0.03125)

    def step():
        order = ops.moe_sort(idx, e)
        rows = ops.moe_gather(x, order)
        a, pre = ops.linear(rows, w1, act="swiglu", w_up=w3, limit=10.0, order=order, want_pre=True)
        y = ops.linear(a, w2, order=order)
        out = ops.moe_combine(y, order, w, residual=x)
        d_y, d_w = ops.moe_combine_grad(out, y, order, w)
        down = ops.linear_grad(d_y, a, w2, order=order)
        up = ops.linear_grad(down.x, rows, w1, act="swiglu", pre=pre, w_up=w3, limit=10.0, order=order, need_bias=True)
        return (out, d_w, down.w, up.w, up.w_up, up.bias, up.bias_up, ops.moe_combine(up.x, order, residual=out))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step()
    torch.cuda.current_stream().wait_stream(side)
    for seed in range(3):
        idx.copy_(torch.randint(0, e, (m, k), generator=g, device=dev))
        x.copy_(ints(dev, 50 + seed, (m, d), scale=0.25))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step()):
            assert torch.equal(a, b)


def test_matrices_that_are_read_once(dev):
    """64 experts of 2048 x 4096 with a few rows each: the kernels for which w's stream is what counts."""
    e, n, k = 64, 2048, 4096
    w = ints(dev, 1, (e, n, k))
    for m, top_k in ((40, 2), (700, 2), (3000, 2)):
        order = some_order(dev, m, top_k, e, m)
        x, d = ints(dev, 2, (m * top_k, k), top=1), ints(dev, 3, (m * top_k, n), top=1)
        out, dx = ops.linear(x, w, order=order), ops.linear_grad(d, x, w, order=order, need_w=False).x
        for i, a, b in spans(order, m * top_k):
            if b > a:
                assert torch.equal(out[a:b], (x[a:b].double() @ w[i].double().T).to(F32).to(BF16))
                assert torch.equal(dx[a:b], (d[a:b].double() @ w[i].double()).to(F32).to(BF16))


def test_two_graphs_at_once(dev):
    """Products whose reduction is split hand their sums through a workspace: each call's own, so that graphs of
    several streams may run together."""
    m, n, k = 64, 4096, 4096
    w = ints(dev, 1, (n, k))
    runs = []
    for seed in (2, 3):
        x, d = ints(dev, seed, (m, k)), ints(dev, seed + 5, (m, n))
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            ops.linear(x, w)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs = [(ops.linear(x, w), ops.linear_grad(d, x, w, need_bias=True)) for _ in range(4)]
        # x and d stay alive with the graph that reads them
        runs.append((stream, graph, outs, ops.linear(x, w), ops.linear_grad(d, x, w, need_bias=True), x, d))
    torch.cuda.synchronize()
    for _ in range(5):
        for stream, graph, *_ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, outs, y, g, *_ in runs:
            for out, grad in outs:
                assert torch.equal(out, y)
                assert all(torch.equal(a, b) for a, b in zip(grad[:3], g[:3]))


def test_offsets_beyond_the_rows_are_cut(dev):
    """An order that does not come from moe_sort: what its offsets say beyond the rows that there are counts for nothing."""
    x, w, d = ints(dev, 1, (4, 64)), ints(dev, 2, (2, 8, 64)), ints(dev, 3, (4, 8))
    good = ops.ExpertOrder(*(torch.tensor(t, dtype=torch.int32, device=dev) for t in ([0, 2, 4], [0, 1, 2, 3], [[0, 1], [2, 3]])))
    far = good._replace(offsets=torch.tensor([-7, 2, 1 << 30], dtype=torch.int32, device=dev))
    assert torch.equal(ops.linear(x, w, order=far), ops.linear(x, w, order=good))
    for a, b in zip(ops.linear_grad(d, x, w, order=far, need_bias=True), ops.linear_grad(d, x, w, order=good, need_bias=True)):
        assert a is None and b is None or torch.equal(a, b)


@pytest.mark.parametrize("m", [4, 40, 1000])
def test_groups_that_overlap_stay_inside(dev, m):
    """Offsets that rise and fall, which no sort gives: rows are undefined then, what is summed per group is not."""
    x, w = ints(dev, 1, (m, 64)), ints(dev, 2, (3, 8, 64))
    off = torch.tensor([0, m, 0, m], dtype=torch.int32, device=dev)  # groups 0 and 2 have all rows, group 1 none
    order = ops.ExpertOrder(off, torch.arange(m, dtype=torch.int32, device=dev), torch.arange(m, dtype=torch.int32, device=dev)[:, None].contiguous())
    assert ops.linear(x, w, order=order).shape == (m, 8)
    grad = ops.linear_grad(ints(dev, 3, (m, 8)), x, w, order=order)
    assert not bool(grad.w[1].any())
    for g in (0, 2):
        assert torch.equal(grad.w[g], ops.linear_grad(ints(dev, 3, (m, 8)), x, w[g], need_x=False).w)


def test_weights_beyond_32_bits(dev):
    """Expert matrices that lie beyond 2^32 bytes."""
    e, n, k = 40, 8192, 8192  # 5.4 GB
    w = torch.empty(e, n, k, dtype=BF16, device=dev)
    w[0], w[-1] = ints(dev, 1, (n, k)), ints(dev, 2, (n, k))
    order = ops.moe_sort(torch.tensor([[0, e - 1]] * 20, device=dev), e)
    x = ints(dev, 3, (40, k))
    want = [(x[a:b].double() @ w[i].double().T).to(F32).to(BF16) for i, a, b in ((0, 0, 20), (-1, 20, 40))]
    assert torch.equal(ops.linear(x, w, order=order), torch.cat(want))
    d = ints(dev, 4, (40, n))
    dx = ops.linear_grad(d, x, w, order=order, need_w=False).x
    assert torch.equal(dx[20:], (d[20:].double() @ w[-1].double()).to(F32).to(BF16))


def test_refusals(dev):
    x, w = ints(dev, 1, (4, 64)), ints(dev, 2, (8, 64))
    err = ops._lib.HsmoeError
    with pytest.raises(ValueError, match="activation"):
        ops.linear(x, w, act="relu")
    with pytest.raises(ValueError, match="up weight"):
        ops.linear(x, w, act="swiglu")
    with pytest.raises(ValueError, match="up weight"):
        ops.linear(x, w, w_up=w)
    with pytest.raises(ValueError, match="limit"):
        ops.linear(x, w, act="silu", limit=1.0)
    for bad in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="positive"):
            ops.linear(x, w, act="swiglu", w_up=w, limit=bad)
    with pytest.raises(TypeError, match="bf16"):
        ops.linear(x.float(), w)
    with pytest.raises(TypeError, match="bf16"):
        ops.linear(x, w.half())
    with pytest.raises(TypeError, match="output"):
        ops.linear(x, w, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="rows of"):
        ops.linear(x[:, :56], w)
    with pytest.raises(ValueError, match="weights"):
        ops.linear(x, w, act="swiglu", w_up=w[:4])
    with pytest.raises(ValueError, match="bias"):
        ops.linear(x, w, bias=x[0])
    with pytest.raises(ValueError, match="up bias"):
        ops.linear(x, w, bias_up=w[:, 0])
    with pytest.raises(ValueError, match="residual"):
        ops.linear(x, w, residual=x)
    with pytest.raises(err, match="multiples of 8"):
        ops.linear(x, w[:7])
    with pytest.raises(err, match="multiples of 8"):
        ops.linear(x[:, :60], w[:, :60])
    order = ops.moe_sort(torch.zeros(2, 2, dtype=torch.int64, device=dev), 3)
    w3 = ints(dev, 2, (3, 8, 64))
    with pytest.raises(ValueError, match="order"):
        ops.linear(x, w3[:2], order=order)
    with pytest.raises(ValueError, match="weights"):
        ops.linear(x, w, order=order)
    with pytest.raises(ValueError, match="rows"):
        ops.linear(x[:3], w3, order=order)
    d = ints(dev, 3, (4, 8))
    with pytest.raises(ValueError, match="pre"):
        ops.linear_grad(d, x, w, act="silu")
    with pytest.raises(ValueError, match="pre"):
        ops.linear_grad(d, x, w, act="silu", pre=x)
    with pytest.raises(ValueError, match="d_out"):
        ops.linear_grad(x, x, w)
    with pytest.raises(TypeError, match="gradient"):
        ops.linear_grad(d, x, w, w_dtype=torch.float16)
    with pytest.raises(err, match="cpu"):
        ops.linear(x, w.cpu())
