"""The expert layer as torch.autograd functions: the gradients that loss.backward()
leaves are those of the ops (each checked against 64 bits elsewhere), bit for bit."""
import pytest
import torch

from home_seek_amd import autograd, ops

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def rnd(dev, seed, shape, std=1.0, dtype=BF16):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=dev) * std).to(dtype)


def leaf(t):
    return t.detach().clone().requires_grad_()


@pytest.mark.parametrize("act", [None, "silu", "swiglu"])
@pytest.mark.parametrize("lead", [(5,), (2, 3, 7), (300,)])
def test_linear_backward(dev, act, lead):
    n, k = 72, 136
    x, w, b, r = (leaf(rnd(dev, i, s)) for i, s in enumerate((lead + (k,), (n, k), (n,), lead + (n,))))
    up, bu = (leaf(rnd(dev, 7, (n, k))), leaf(rnd(dev, 8, (n,)))) if act == "swiglu" else (None, None)
    limit = 2.0 if act == "swiglu" else None
    d = rnd(dev, 9, lead + (n,))
    out = autograd.linear(x, w, b, r, act, up, bu, limit)
    out.backward(d)
    want, pre = ops.linear(x, w, b, r, act, up, bu, limit, want_pre=True)
    g = ops.linear_grad(d, x, w, act, pre, up, limit, need_bias=True)
    assert torch.equal(out, want)
    assert torch.equal(x.grad, g.x) and torch.equal(w.grad, g.w) and torch.equal(r.grad, d)
    assert torch.equal(b.grad, g.bias.to(BF16)) and b.grad.dtype == BF16
    if act == "swiglu":
        assert torch.equal(up.grad, g.w_up) and torch.equal(bu.grad, g.bias_up.to(BF16))


def test_only_what_is_needed(dev):
    x, w = rnd(dev, 1, (4, 64)), leaf(rnd(dev, 2, (8, 64)))
    autograd.linear(x, w, act="silu", out_dtype=F32).sum().backward()  # an expanded gradient, in fp32
    ones = torch.ones(4, 8, dtype=BF16, device=dev)
    assert torch.equal(w.grad, ops.linear_grad(ones, x, w, "silu", ops.linear(x, w, act="silu", want_pre=True)[1]).w)
    assert not autograd.linear(x, w.detach()).requires_grad


def test_without_gradients_no_sums_are_kept(dev, monkeypatch):
    x, w = rnd(dev, 1, (4, 64)), leaf(rnd(dev, 2, (8, 64)))
    kept, plain = [], ops.linear
    monkeypatch.setattr(ops, "linear", lambda *a, **kw: (kept.append(kw.get("want_pre", False)), plain(*a, **kw))[1])
    a = autograd.linear(x, w, act="silu")
    with torch.no_grad():
        b = autograd.linear(x, w, act="silu")
    assert a.requires_grad and not b.requires_grad and torch.equal(a, b) and kept == [True, False]


def test_one_matrix_for_both_weights_and_for_all_experts(dev):
    order = ops.moe_sort(torch.tensor([[0, 2], [2, 1], [0, 0]], device=dev), 3)
    x, w = rnd(dev, 1, (6, 64)), leaf(rnd(dev, 2, (72, 64)))
    each = w.expand(3, 72, 64)
    out = autograd.linear(x, each, act="swiglu", w_up=each, limit=3.0, order=order)
    d = rnd(dev, 3, out.shape)
    out.backward(d)
    wide = w.detach().expand(3, 72, 64).contiguous()
    want, pre = ops.linear(x, wide, act="swiglu", w_up=wide, limit=3.0, order=order, want_pre=True)
    g = ops.linear_grad(d, x, wide, "swiglu", pre, wide, 3.0, order)
    assert torch.equal(out, want)
    # torch adds the six bf16 gradients: five sums, each off by half a step of at most the sum of the sizes
    size = (g.w.double().abs() + g.w_up.double().abs()).sum(0)
    assert bool(((w.grad.double() - (g.w.double() + g.w_up.double()).sum(0)).abs() <= 5 * 1.02 * 2.0 ** -8 * size).all())


def test_no_tokens_and_bf16_weights(dev):
    e, d, i = 3, 64, 72
    w1, w3, w2 = leaf(rnd(dev, 4, (e, i, d))), leaf(rnd(dev, 5, (e, i, d))), leaf(rnd(dev, 6, (e, d, i)))
    for m in (0, 5):
        x, tw = leaf(rnd(dev, 1, (m, d))), leaf(rnd(dev, 2, (m, 2)))
        idx = torch.arange(2 * m, device=dev).reshape(m, 2) % e
        out = autograd.moe_ffn(x, idx, tw, w1, w3, w2)
        grads = torch.autograd.grad(out.float().sum(), (x, tw, w1, w3, w2))
        assert out.shape == (m, d) and out.dtype == BF16
        for g, t in zip(grads, (x, tw, w1, w3, w2)):
            assert g.shape == t.shape and g.dtype == BF16
            assert bool(g.any()) == (m > 0 and g.numel() > 0)


@pytest.mark.parametrize("drop", [0.0, 0.4])
def test_moe_ffn_backward(dev, drop):
    m, k, e, d, i = 40, 3, 9, 128, 72
    idx = torch.randint(0, e, (m, k), device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    if drop:
        idx = torch.where(torch.rand((m, k), device=dev, generator=torch.Generator(device=dev).manual_seed(2)) < drop, -1, idx)
    x, res, tw = leaf(rnd(dev, 1, (m, d))), leaf(rnd(dev, 2, (m, d))), leaf(rnd(dev, 3, (m, k), dtype=F32))
    w1, w3, w2 = leaf(rnd(dev, 4, (e, i, d), 0.1)), leaf(rnd(dev, 5, (e, i, d), 0.1)), leaf(rnd(dev, 6, (e, d, i), 0.1))
    g = rnd(dev, 7, (m, d))
    out = autograd.moe_ffn(x, idx, tw, w1, w3, w2, 2.0, res)
    out.backward(g)
    order = ops.moe_sort(idx, e)
    rows = ops.moe_gather(x, order)
    a, pre = ops.linear(rows, w1, act="swiglu", w_up=w3, limit=2.0, order=order, want_pre=True)
    y = ops.linear(a, w2, order=order)
    assert torch.equal(out, ops.moe_combine(y, order, tw, res))
    d_y, d_w = ops.moe_combine_grad(g, y, order, tw)
    down = ops.linear_grad(d_y, a, w2, order=order)
    up = ops.linear_grad(down.x, rows, w1, "swiglu", pre, w3, 2.0, order)
    for got, want in ((tw.grad, d_w), (w2.grad, down.w), (w1.grad, up.w), (w3.grad, up.w_up), (res.grad, g),
                      (x.grad, ops.moe_combine(up.x, order))):
        assert torch.equal(got, want)


def test_moe_ffn_against_float64(dev):
    """The layer as a whole: the norm of the error of a result behind r bf16 roundings, each off by at most 2^-8 of
    its value, stays below what the roundings carry through the layer's (absolute) linear maps."""
    m, k, e, d, i = 30, 2, 4, 64, 64
    idx = torch.randint(0, e, (m, k), device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    x, tw = rnd(dev, 1, (m, d)), rnd(dev, 3, (m, k), dtype=F32).abs()
    w1, w3, w2 = rnd(dev, 4, (e, i, d), 0.1), rnd(dev, 5, (e, i, d), 0.1), rnd(dev, 6, (e, d, i), 0.1)
    out = autograd.moe_ffn(x, idx, tw, w1, w3, w2, None).double()
    want, size = torch.zeros(m, d, dtype=torch.float64, device=dev), torch.zeros(m, d, dtype=torch.float64, device=dev)
    for t in range(m):
        for j in range(k):
            ex = int(idx[t, j])
            z, u = w1[ex].double() @ x[t].double(), w3[ex].double() @ x[t].double()
            a = z * torch.sigmoid(z) * u
            want[t] += tw[t, j].double() * (w2[ex].double() @ a)
            size[t] += tw[t, j].double() * (w2[ex].double().abs() @ a.abs())
    # the activation's rounding, the product's and the result's
    assert bool(((out - want).abs() <= 3.1 * 2.0 ** -8 * size + 1e-6).all())


def test_residual_of_dropped_rows_has_no_gradient(dev):
    idx = torch.tensor([[0, -1], [1, -1]], device=dev)
    order = ops.moe_sort(idx, 2)
    x, w, r = rnd(dev, 1, (4, 64)), rnd(dev, 2, (2, 8, 64)), leaf(rnd(dev, 3, (4, 8)))
    autograd.linear(x, w, residual=r, order=order).sum().backward()
    assert r.grad[:2].tolist() == [[1.0] * 8] * 2 and not bool(r.grad[2:].any())


def test_captured_training_step(dev):
    """Forward and backward captured together, replayed on new inputs, against eager steps on other leaves."""
    m, k, e, d, i = 64, 2, 6, 128, 64
    gen = torch.Generator(device=dev).manual_seed(5)
    base = [rnd(dev, s, sh, 0.1) for s, sh in ((4, (e, i, d)), (5, (e, i, d)), (6, (e, d, i)))]
    x, idx, tw = rnd(dev, 1, (m, d)), torch.randint(0, e, (m, k), device=dev, generator=gen), torch.rand((m, k), device=dev, generator=gen)

    def step(ws):
        return torch.autograd.grad(autograd.moe_ffn(x, idx, tw, *ws).float().square().sum(), ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ws = [leaf(t) for t in base]
        step(ws)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            grads = step(ws)
    torch.cuda.current_stream().wait_stream(side)
    for seed in range(3):
        x.copy_(rnd(dev, 20 + seed, (m, d)))
        idx.copy_(torch.randint(0, e, (m, k), device=dev, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(grads, step([leaf(t) for t in base])):
            assert torch.equal(a, b)
