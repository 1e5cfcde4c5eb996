"""linear's gradients against central differences of linear itself, along the direction in which each gradient counts
most: every element moves by the same step, with the sign of its own gradient, so that what is compared is the step
times the sum of the gradient's magnitudes, and nothing of it cancels.

The bound is made of the formulas in 64 bits and of the roundings that the calls make:
  * what a central difference of this step misses: that of the formulas, less their derivative (exact);
  * the fp32 results on both sides: 16 x 2^-24 of the magnitudes that enter one;
  * pre kept in bf16: the derivative at pre, less that at the unrounded sums (exact);
  * dz rounded to bf16, each factor off by 2^-8 of its value (half a step), its evaluation in fp32 (16 x 2^-24 of the
    magnitudes that enter), the gradient itself, 2^-8 again where it is bf16, and the fp32 sums, n 2^-23 of the
    magnitudes of their n terms.
It has to stay below a tenth of what is compared: a gradient that is zero, turned, or lacks one matrix's part is
rejected, which the first test shows on the CPU."""
import pytest
import torch

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
M, N, K = 24, 24, 72
STEP = {"x": 2.0 ** -6, "w": 2.0 ** -7, "w_up": 2.0 ** -7, "bias": 2.0 ** -5, "bias_up": 2.0 ** -5}
CASES = [(None, None, 0), ("silu", None, 0), ("swiglu", None, 0), ("swiglu", 2.0, 0), ("silu", None, 3), ("swiglu", None, 3)]


def inputs(act, experts):
    """bf16 inputs to which a step can be added exactly; with experts, rows in groups of unequal size and some of none."""
    g = torch.Generator().manual_seed(7)
    lead = (experts,) if experts else ()

    def ints(shape, scale):
        return (torch.randint(-3, 4, shape, generator=g) * scale).to(BF16)

    t = {"x": ints((M, K), 0.25), "w": ints(lead + (N, K), 0.0625), "bias": ints(lead + (N,), 0.25)}
    if act == "swiglu":
        t["w_up"], t["bias_up"] = ints(lead + (N, K), 0.0625), ints(lead + (N,), 0.25)
    spans = [(0, 0, 11), (1, 11, 11), (2, 11, 20)] if experts else [(None, 0, M)]
    return t, ints((M, N), 1.0), spans


def of(t, e):
    return t if e is None else t[e]


def sums64(t, spans):
    zs = []
    for w, b in (("w", "bias"), ("w_up", "bias_up")):
        if w in t:
            z = torch.zeros(M, N, dtype=F64)
            for e, a, end in spans:
                z[a:end] = t["x"][a:end].double() @ of(t[w], e).double().T + of(t[b], e).double()
            zs.append(z)
    return zs


def value64(act, limit, zs):
    """(y, the magnitudes that enter it)"""
    if act is None:
        return zs[0], zs[0].abs()
    g = zs[0] if limit is None else zs[0].clamp(max=limit)
    y = g / (1 + torch.exp(-g))
    if act == "silu":
        return y, g.abs()
    u = zs[1] if limit is None else zs[1].clamp(-limit, limit)
    return y * u, (g * u).abs()


def slopes64(act, limit, zs):
    """y' by each sum"""
    if act is None:
        return [torch.ones_like(zs[0])]
    g = zs[0] if limit is None else zs[0].clamp(max=limit)
    s = 1 / (1 + torch.exp(-g))
    slope = s + g * s * (1 - s)
    if act == "silu":
        return [slope]
    u = zs[1] if limit is None else zs[1].clamp(-limit, limit)
    inside = [torch.ones_like(g)] * 2 if limit is None else [zs[0] <= limit, zs[1].abs() <= limit]
    return [slope * u * inside[0], g * s * inside[1]]


def slope_sizes64(act, limit, zs):
    """the magnitudes that enter each y'"""
    if act is None:
        return [torch.zeros_like(zs[0])]
    g = (zs[0] if limit is None else zs[0].clamp(max=limit)).abs()
    if act == "silu":
        return [1 + g]
    u = (zs[1] if limit is None else zs[1].clamp(-limit, limit)).abs()
    return [(1 + g) * u, g]


def live(spans):
    rows = torch.zeros(M, 1, dtype=F64)
    for _, a, end in spans:
        rows[a:end] = 1
    return rows


def gradient64(t, spans, dz):
    """name -> gradient, and name -> the sum of its terms' magnitudes"""
    grad, size = {}, {}
    dz = [d * live(spans) for d in dz]
    x = t["x"].double()
    grad["x"], size["x"] = torch.zeros_like(x), torch.zeros_like(x)
    for d, w, b in zip(dz, ("w", "w_up"), ("bias", "bias_up")):
        grad[w], size[w] = torch.zeros(t[w].shape, dtype=F64), torch.zeros(t[w].shape, dtype=F64)
        grad[b], size[b] = torch.zeros(t[b].shape, dtype=F64), torch.zeros(t[b].shape, dtype=F64)
        for e, a, end in spans:
            at = slice(None) if e is None else e
            for out, f in ((grad, lambda v: v), (size, torch.abs)):
                out["x"][a:end] += f(d[a:end]) @ f(of(t[w], e).double())
                out[w][at] = f(d[a:end]).T @ f(x[a:end])
                out[b][at] = f(d[a:end]).sum(dim=0)
    return grad, size


def moved(t, name, step):
    return {**t, name: (t[name].double() + step).to(BF16)}


def derive(act, limit, experts, name):
    """inputs, d_out, spans, step, what the difference has to be near, the bound, and the formulas' gradient"""
    t, d_out, spans = inputs(act, experts)
    d = d_out.double() * live(spans)
    zs = sums64(t, spans)
    grad, _ = gradient64(t, spans, [d * s for s in slopes64(act, limit, zs)])
    step = STEP[name] * grad[name].sign()
    assert all(torch.equal(moved(t, name, s)[name].double(), t[name].double() + s) for s in (step, -step))
    sides = [value64(act, limit, sums64(moved(t, name, s), spans)) for s in (step, -step)]
    exact = float((grad[name] * step).sum())
    difference = float((d * (sides[0][0] - sides[1][0])).sum() / 2)
    bound = abs(difference - exact)
    bound += sum(float((d.abs() * y_size).sum()) for _, y_size in sides) / 2 * 16 * 2.0 ** -24
    rounded = [z.to(BF16).double() for z in zs]
    dz = [d * s for s in slopes64(act, limit, rounded)]
    at_pre, size_pre = gradient64(t, spans, dz)
    bound += abs(float(((at_pre[name] - grad[name]) * step).sum()))
    half = 2.0 ** -8 if act is not None and not name.startswith("bias") else 0.0
    errors = [half * v.abs() + 16 * 2.0 ** -24 * d.abs() * s for v, s in zip(dz, slope_sizes64(act, limit, rounded))]
    off = gradient64(t, spans, errors)[1][name] + (M + 2 * N) * 2.0 ** -23 * size_pre[name]
    if not name.startswith("bias"):
        off = off + 2.0 ** -8 * (at_pre[name].abs() + off)
    bound += float((off * step.abs()).sum())
    return t, d_out, spans, step, exact, bound, grad[name]


def parts_missing(act, limit, experts, name, step):
    """The step's product with gradients that are wrong: zero, turned, without one matrix's part."""
    t, d_out, spans = inputs(act, experts)
    d = d_out.double() * live(spans)
    dz = [d * s for s in slopes64(act, limit, sums64(t, spans))]
    full = float((gradient64(t, spans, dz)[0][name] * step).sum())
    wrong = [0.0, -full]
    if act == "swiglu" and name == "x":
        for keep in (0, 1):
            part = [v * (i == keep) for i, v in enumerate(dz)]
            wrong.append(float((gradient64(t, spans, part)[0][name] * step).sum()))
    return wrong


def names_of(act):
    return ["x", "w", "bias"] + (["w_up", "bias_up"] if act == "swiglu" else [])


ALL = [(act, limit, experts, name) for act, limit, experts in CASES for name in names_of(act)]


@pytest.mark.parametrize("act,limit,experts,name", ALL)
def test_the_bound_rejects_wrong_gradients(act, limit, experts, name):
    *_, step, exact, bound, _ = derive(act, limit, experts, name)
    assert exact > 0 and bound < exact / 10
    for wrong in parts_missing(act, limit, experts, name, step):
        assert abs(wrong - exact) > bound


@pytest.mark.gpu
@pytest.mark.parametrize("act,limit,experts,name", ALL)
def test_gradient_against_differences(dev, act, limit, experts, name):
    from home_seek_amd import ops
    t, d_out, spans, step, exact, bound, _ = derive(act, limit, experts, name)
    order = None
    if experts:  # one slot per token: the rows behind the last are dropped pairs
        ids = torch.full((M, 1), -1)
        for e, a, end in spans:
            ids[a:end] = e
        order = ops.moe_sort(ids.to(dev), experts)
        assert order.offsets.tolist() == [0, 11, 11, 20]

    def forward(t, **kw):
        t = {k: v.to(dev) for k, v in t.items()}
        return ops.linear(t["x"], t["w"], t["bias"], None, act, t.get("w_up"), t.get("bias_up"), limit, order, **kw)

    sides = [forward(moved(t, name, s), out_dtype=F32).double().cpu() for s in (step, -step)]
    difference = float((d_out.double() * (sides[0] - sides[1])).sum() / 2)
    pre = forward(t, want_pre=True)[1]
    on = {k: v.to(dev) for k, v in t.items()}
    grad = ops.linear_grad(d_out.to(dev), on["x"], on["w"], act, None if act is None else pre, on.get("w_up"), limit, order,
                           need_bias=True)
    got = float((getattr(grad, name).double().cpu() * step).sum())
    assert abs(got - difference) <= bound, (got, difference, exact, bound)
