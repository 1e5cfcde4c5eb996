"""The norms around a block with its gate, residual scale and stream, and their
gradient, against the formulas in 64 bits.

Bounds, with e = 2^-24 and s = half a step of a type.  A sum of D terms is off by at
most D e of the sum of their magnitudes; half of that goes into 1 / rms.  So a norm
y = w v r is off by (D / 2 + 8) e |y|, a product of k factors by k e.  The gradients
are sums of terms of which each is a product with such factors; their errors are
bounded by (2 D + 32) e times the sum of the terms' magnitudes, and sums over M rows
by (M + 2 D + 32) e times that of their terms."""
import pytest
import torch

from home_seek_amd import _lib, ops

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def normal(dev, seed, shape, dtype=BF16, std=1.0, mean=0.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=dev) * std + mean).to(dtype)


def make(dev, m, d, t, s, w, gate, post, pre, seed=0):
    a = {"f": normal(dev, seed + 1, (m, d), t, 3.0), "h": normal(dev, seed + 2, (m, d), s, 2.0)}
    a["post_w"] = normal(dev, seed + 3, (d,), w, 0.2, 1.0) if post else None
    a["pre_w"] = normal(dev, seed + 4, (d,), w, 0.2, 1.0) if pre else None
    shape = {"none": None, "channel": (d,), "token": (m, 1), "full": (m, d)}[gate]
    a["gate"] = None if shape is None else normal(dev, seed + 5, shape, t, 0.5, 0.3)
    return a


def rms_inv(v, eps):
    return 1 / torch.sqrt((v * v).mean(dim=-1, keepdim=True) + eps)


def check_forward(a, out, n, scale, eps):
    d = a["f"].shape[-1]
    f, h = a["f"].double(), a["h"].double()
    u = f if a["post_w"] is None else f * rms_inv(f, eps) * a["post_w"].double()
    t = scale * (1 if a["gate"] is None else a["gate"].double()) * u
    want = h + t
    tol = half(out.dtype) * want.abs() + (d / 2 + 16) * E * t.abs() + 2 * E * want.abs() + torch.finfo(out.dtype).smallest_normal
    assert out.dtype == a["h"].dtype and ((out.double() - want).abs() <= tol).all()
    if a["pre_w"] is None:
        assert n is None
        return
    held = out.double()  # the norm is that of the stream as it is held
    want = held * rms_inv(held, eps) * a["pre_w"].double()
    tol = (half(n.dtype) + (d / 2 + 16) * E) * want.abs() + torch.finfo(n.dtype).smallest_normal
    assert n.dtype == a["f"].dtype and ((n.double() - want).abs() <= tol).all()


def check_grad(a, d_h, d_n, scale, eps, g):
    """a["h"]: the stream after the block."""
    m, d = a["f"].shape
    f, h = a["f"].double(), a["h"].double()
    k = (2 * d + 32) * E
    total = torch.zeros_like(h) if d_h is None else d_h.double()
    size = total.abs()
    if d_n is not None:
        r = rms_inv(h, eps)
        dn = d_n.double()
        q = dn * a["pre_w"].double()
        total = total + r * q - h * r ** 3 * (q * h).mean(dim=1, keepdim=True)
        size = size + (r * q).abs() + h.abs() * r ** 3 * (q * h).abs().mean(dim=1, keepdim=True)
        if g.pre_w is not None:
            t = dn * h * r
            assert ((g.pre_w.double() - t.sum(dim=0)).abs() <= (m + 2 * d + 32) * E * t.abs().sum(dim=0)).all()
    elif g.pre_w is not None:
        assert (g.pre_w == 0).all()
    if g.h is not None:
        assert g.h.dtype == a["h"].dtype and ((g.h.double() - total).abs() <= k * size + half(g.h.dtype) * total.abs() + 1e-38).all()
    dt, dt_size = scale * total, abs(scale) * size
    y = f * rms_inv(f, eps)
    u = f if a["post_w"] is None else y * a["post_w"].double()
    if a["gate"] is not None and g.gate is not None:
        t, s = dt * u, dt_size * u.abs()
        if a["gate"].shape == (m, d):
            assert g.gate.dtype == a["gate"].dtype
            assert ((g.gate.double() - t).abs() <= 2 * k * s + half(g.gate.dtype) * t.abs() + 1e-38).all()
        else:
            dim = 0 if a["gate"].dim() == 1 else 1
            assert g.gate.dtype == F32 and g.gate.shape == a["gate"].shape
            err = (g.gate.double() - t.sum(dim=dim).reshape(g.gate.shape)).abs()
            assert (err <= (m + 4 * d + 64) * E * s.sum(dim=dim).reshape(g.gate.shape)).all()
    gate = 1.0 if a["gate"] is None else a["gate"].double()
    du, du_size = dt * gate, dt_size * (gate if isinstance(gate, float) else gate.abs())
    if a["post_w"] is None:
        want, s = du, du_size
    else:
        if g.post_w is not None:
            t, s = du * y, du_size * y.abs()
            assert ((g.post_w.double() - t.sum(dim=0)).abs() <= (m + 4 * d + 64) * E * s.sum(dim=0)).all()
        r, w = rms_inv(f, eps), a["post_w"].double()
        want = r * du * w - f * r ** 3 * (du * w * f).mean(dim=1, keepdim=True)
        s = r * du_size * w.abs() + f.abs() * r ** 3 * (du_size * w.abs() * f.abs()).mean(dim=1, keepdim=True)
    if g.f is not None:
        assert g.f.dtype == a["f"].dtype and ((g.f.double() - want).abs() <= 2 * k * s + half(g.f.dtype) * want.abs() + 1e-38).all()


SIZES = [(1, 8), (3, 64), (33, 72), (5, 128), (17, 136), (9, 256), (7, 264), (6, 512), (5, 520), (4, 1024), (3, 4096),
         (2, 4104), (2, 8192), (1, 8200), (2, 16384), (1030, 64), (2100, 512), (1500, 1536), (700, 4096), (300, 8192), (300, 6152), (3, 12296), (300, 16384),
         (900, 776), (2300, 1024)]
KINDS = [(BF16, BF16, BF16), (BF16, F32, F32), (F32, F32, F32), (F32, BF16, BF16)]


@pytest.mark.parametrize("m,d", SIZES)
@pytest.mark.parametrize("t,s,w", KINDS)
def test_forward_and_gradient(dev, m, d, t, s, w):
    for i, (gate, post, pre) in enumerate((("channel", True, True), ("full", True, True), ("token", True, True),
                                           ("none", True, False), ("none", False, True), ("token", False, False), ("channel", False, True))):
        if m * d > 400000 and i not in (0, 2):
            continue
        a = make(dev, m, d, t, s, w, gate, post, pre, seed=10 * i)
        scale, eps = (0.5, 1e-6) if i % 2 else (-1.25, 1e-3)
        out, n = ops.block_norm(a["f"], a["h"], a["post_w"], a["gate"], scale, a["pre_w"], eps)
        check_forward(a, out, n, scale, eps)
        d_h = normal(dev, 97 + i, (m, d), s)
        d_n = normal(dev, 98 + i, (m, d), t) if pre else None
        g = ops.block_norm_grad(d_h, d_n, a["f"], a["h"], a["post_w"], a["gate"], scale, a["pre_w"], eps)
        assert [x is None for x in g] == [False, False, not post, gate == "none", not pre]
        check_grad(a, d_h, d_n, scale, eps, g)


def test_one_of_the_two_results(dev):
    a = make(dev, 50, 264, BF16, F32, BF16, "channel", True, True)
    for d_h, d_n in ((normal(dev, 1, (50, 264), F32), None), (None, normal(dev, 2, (50, 264)))):
        g = ops.block_norm_grad(d_h, d_n, a["f"], a["h"], a["post_w"], a["gate"], 0.7, a["pre_w"])
        check_grad(a, d_h, d_n, 0.7, 1e-6, g)
        for i in range(5):
            need = [j == i for j in range(5)]
            part = ops.block_norm_grad(d_h, d_n, a["f"], a["h"], a["post_w"], a["gate"], 0.7, a["pre_w"], need=need)
            for j in range(5):
                assert (part[j] is None) != need[j]
            assert torch.equal(part[i], g[i])


def test_weights_of_two_types_and_gate_of_another(dev):
    a = make(dev, 20, 512, BF16, BF16, F32, "channel", True, True)
    a["pre_w"], a["gate"] = a["pre_w"].to(BF16), a["gate"].float()
    out, n = ops.block_norm(a["f"], a["h"], a["post_w"], a["gate"], 1.0, a["pre_w"])
    check_forward(a, out, n, 1.0, 1e-6)
    d_h, d_n = normal(dev, 1, (20, 512)), normal(dev, 2, (20, 512))
    check_grad(a, d_h, d_n, 1.0, 1e-6, ops.block_norm_grad(d_h, d_n, a["f"], a["h"], a["post_w"], a["gate"], 1.0, a["pre_w"]))
    a["gate"] = normal(dev, 3, (20, 512), F32)
    check_grad(a, d_h, d_n, 1.0, 1e-6, ops.block_norm_grad(d_h, d_n, a["f"], a["h"], a["post_w"], a["gate"], 1.0, a["pre_w"]))


def test_agrees_with_the_norms_that_were_there(dev):
    """Without a gate and a norm after the block it is add_rms_norm's function: the stream bit for bit."""
    f, h, w = normal(dev, 1, (37, 4096)), normal(dev, 2, (37, 4096)), normal(dev, 3, (4096,), BF16, 0.1, 1.0)
    out, n = ops.block_norm(f, h, pre_w=w)
    h2, n2 = ops.add_rms_norm(h, w, add=f, want_sum=True)
    assert torch.equal(out, h2)
    err = (n.double() - n2.double()).abs()
    assert (err <= 2 * half(BF16) * n2.double().abs() * (1 + 1e-3)).all()


def test_rows_of_zeros_infinities_and_nan_stay_rows(dev):
    a = make(dev, 70, 520, BF16, BF16, BF16, "channel", True, True)
    clean = ops.block_norm(a["f"], a["h"], a["post_w"], a["gate"], 1.0, a["pre_w"])
    a["f"][3] = 0
    a["h"][4], a["f"][4] = 0, 0
    a["f"][5, 7], a["f"][6, 8] = float("inf"), float("nan")
    out, n = ops.block_norm(a["f"], a["h"], a["post_w"], a["gate"], 1.0, a["pre_w"])
    rest = [i for i in range(70) if not 3 <= i <= 6]
    assert torch.equal(out[rest], clean[0][rest]) and torch.equal(n[rest], clean[1][rest])
    assert torch.equal(out[3], a["h"][3]) and (out[4] == 0).all() and (n[4] == 0).all()
    assert out[5].isnan().any() and out[6].isnan().all() and n[5].isnan().all() and n[6].isnan().all()
    d = normal(dev, 9, (70, 520))
    g = ops.block_norm_grad(d, d, a["f"], out, a["post_w"], a["gate"], 1.0, a["pre_w"])
    assert torch.isfinite(g.f[rest]).all() and torch.isfinite(g.f[3:5]).all() and g.f[6].isnan().all()


@pytest.mark.parametrize("m,d", ((33, 72), (5, 128), (9, 256), (3, 512), (3, 1024), (1, 64)))
def test_without_eps(dev, m, d):
    """Rows beyond the last of a group of rows are zeros to the kernels, and have no rms: they may not reach the sums."""
    a = make(dev, m, d, BF16, BF16, BF16, "channel", True, True)
    out, n = ops.block_norm(a["f"], a["h"], a["post_w"], a["gate"], 0.5, a["pre_w"], 0.0)
    check_forward(a, out, n, 0.5, 0.0)
    d_h, d_n = normal(dev, 1, (m, d)), normal(dev, 2, (m, d))
    g = ops.block_norm_grad(d_h, d_n, a["f"], a["h"], a["post_w"], a["gate"], 0.5, a["pre_w"], 0.0)
    assert all(torch.isfinite(x).all() for x in g)
    check_grad(a, d_h, d_n, 0.5, 0.0, g)


def test_shapes_strides_and_no_rows(dev):
    f, h = normal(dev, 1, (3, 4, 96))[:, :, 16:80], normal(dev, 2, (4, 3, 64), F32).transpose(0, 1)
    w = normal(dev, 3, (128,), BF16, 0.1, 1.0)[::2]
    gate = normal(dev, 4, (3, 4, 1))
    out, n = ops.block_norm(f, h, w, gate, 0.5, w)
    flat = ops.block_norm(f.reshape(12, 64), h.reshape(12, 64), w.contiguous(), gate.reshape(12, 1), 0.5, w.contiguous())
    assert out.shape == n.shape == (3, 4, 64) and torch.equal(out.reshape(12, 64), flat[0]) and torch.equal(n.reshape(12, 64), flat[1])
    one = ops.block_norm(f[0, 0], h[0, 0], w, None, 0.5, w)
    assert one[0].shape == (64,)
    none = ops.block_norm(f[:0], h[:0], w, gate[:0], 0.5, w)
    assert none[0].shape == (0, 4, 64)
    g = ops.block_norm_grad(none[0], none[1], f[:0], none[0], w, w, 0.5, w)
    assert (g.post_w == 0).all() and (g.pre_w == 0).all() and (g.gate == 0).all() and g.f.shape == (0, 4, 64)
    d_h, d_n = normal(dev, 5, (4, 3, 64), F32).transpose(0, 1), normal(dev, 6, (3, 4, 128))[:, :, ::2]
    a = ops.block_norm_grad(d_h, d_n, f, out, w, gate, 0.5, w)
    b = ops.block_norm_grad(d_h.reshape(12, 64), d_n.reshape(12, 64), f.reshape(12, 64), out.reshape(12, 64), w, gate.reshape(12, 1), 0.5, w)
    assert all(torch.equal(x.reshape(y.shape), y) for x, y in zip(a, b))


def test_deterministic_and_replayed(dev):
    a = make(dev, 3000, 1024, BF16, F32, BF16, "channel", True, True)
    d_h, d_n = normal(dev, 1, (3000, 1024), F32), normal(dev, 2, (3000, 1024))

    def step():
        out, n = ops.block_norm(a["f"], a["h"], a["post_w"], a["gate"], 0.5, a["pre_w"])
        return [out, n, *ops.block_norm_grad(d_h, d_n, a["f"], out, a["post_w"], a["gate"], 0.5, a["pre_w"])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step()
    torch.cuda.synchronize()
    for seed in range(3):
        a["f"].copy_(normal(dev, 50 + seed, (3000, 1024)))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(outs, step()):
            assert torch.equal(x, y)


def test_refusals(dev):
    f, h, w = normal(dev, 1, (4, 64)), normal(dev, 2, (4, 64)), normal(dev, 3, (64,))
    for bad, exc in ((lambda: ops.block_norm(f, h[:3]), ValueError), (lambda: ops.block_norm(f[:, :60], h[:, :60]), ValueError),
                     (lambda: ops.block_norm(f.half(), h), TypeError), (lambda: ops.block_norm(f, h.double()), TypeError),
                     (lambda: ops.block_norm(f, h, w[:32]), ValueError), (lambda: ops.block_norm(f, h, w, w[:1]), ValueError),
                     (lambda: ops.block_norm(f, h, w, f[:2]), ValueError), (lambda: ops.block_norm(f, h, w.half()), TypeError),
                     (lambda: ops.block_norm(f, h, w, eps=-1.0), RuntimeError), (lambda: ops.block_norm(f, h.cpu()), RuntimeError),
                     (lambda: ops.block_norm_grad(None, None, f, h), ValueError), (lambda: ops.block_norm_grad(h, f, f, h), ValueError),
                     (lambda: ops.block_norm_grad(h.float(), None, f, h), ValueError),
                     (lambda: ops.block_norm(normal(dev, 1, (1, 16392)), normal(dev, 1, (1, 16392))), RuntimeError)):
        with pytest.raises(exc):
            bad()


@pytest.mark.parametrize("m,d", ((37, 64), (9, 512), (600, 2056), (300, 8192), (270, 12296)))
@pytest.mark.parametrize("gate", ("channel", "token", "full"))
def test_written_over_what_was_read(dev, m, d, gate):
    """The entry points may write the stream over the stream, n over f, and gradients over d_h and f or d_n."""
    L = _lib.lib()
    a = make(dev, m, d, BF16, F32, BF16, gate, True, True)
    out, n = ops.block_norm(a["f"], a["h"], a["post_w"], a["gate"], 0.5, a["pre_w"])
    d_h, d_n = normal(dev, 1, (m, d), F32), normal(dev, 2, (m, d))
    want = ops.block_norm_grad(d_h, d_n, a["f"], out, a["post_w"], a["gate"], 0.5, a["pre_w"])
    spec, _, keep = ops._block_norm_spec(a["f"], F32, a["post_w"], a["gate"], a["pre_w"])
    f, h = a["f"].clone(), a["h"].clone()
    stream = torch.cuda.current_stream().cuda_stream
    assert L.hsmoe_block_norm(f.data_ptr(), h.data_ptr(), m, d, spec, 0.5, 1e-6, h.data_ptr(), f.data_ptr(), stream) == 0
    assert torch.equal(h, out) and torch.equal(f, n)
    nbytes = L.hsmoe_block_norm_grad_workspace_size(m, d)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    for over_f in (True, False):
        f, dx, dn = a["f"].clone(), d_h.clone(), d_n.clone()
        post, pre = torch.empty(d, device=dev), torch.empty(d, device=dev)
        d_gate = torch.empty_like(want.gate)
        df = f if over_f else dn
        assert L.hsmoe_block_norm_grad(dx.data_ptr(), dn.data_ptr(), f.data_ptr(), out.data_ptr(), m, d, spec, 0.5, 1e-6, df.data_ptr(),
                                       dx.data_ptr(), post.data_ptr(), d_gate.data_ptr(), pre.data_ptr(), ws.data_ptr(), nbytes, stream) == 0
        for got, ref in ((df, want.f), (dx, want.h), (post, want.post_w), (d_gate, want.gate), (pre, want.pre_w)):
            assert torch.equal(got, ref)
