"""Embedding, block norms, experts, clipping and the way back into the store, as a
training step uses them: autograd's gradients are the ops' own (each checked against
64 bits elsewhere), bit for bit; the trained experts are served from the store."""
import pytest
import torch

from home_seek_amd import autograd, expert_store, ops

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
D, I, E, K, V, M = 1024, 512, 8, 2, 301, 24


def rnd(dev, seed, shape, std=1.0, dtype=BF16, mean=0.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=dev) * std + mean).to(dtype)


def leaf(t):
    return t.detach().clone().requires_grad_()


@pytest.mark.parametrize("gate", ("channel", "token", "full", None))
@pytest.mark.parametrize("stream", (BF16, F32))
def test_block_norm_backward(dev, gate, stream):
    f, h = leaf(rnd(dev, 1, (3, 5, 64))), leaf(rnd(dev, 2, (3, 5, 64), dtype=stream))
    a, b = leaf(rnd(dev, 3, (64,), 0.1, F32, 1.0)), leaf(rnd(dev, 4, (64,), 0.1, F32, 1.0))
    g = None if gate is None else leaf(rnd(dev, 5, {"channel": (64,), "token": (3, 5, 1), "full": (3, 5, 64)}[gate]))
    d_h, d_n = rnd(dev, 6, (3, 5, 64), dtype=stream), rnd(dev, 7, (3, 5, 64))
    out, n = autograd.block_norm(f, h, a, g, 0.5, b, 1e-5)
    torch.autograd.backward([out, n], [d_h, d_n])
    want = ops.block_norm_grad(d_h, d_n, f, out, a, g, 0.5, b, 1e-5)
    for t, w in zip((f, h, a, g, b), want):
        if t is not None:
            assert t.grad.dtype == t.dtype and torch.equal(t.grad, w.to(t.dtype))
    # one result alone, and without the norm before the next block
    for which in (0, 1):
        for t in (f, h, a, b):
            t.grad = None
        autograd.block_norm(f, h, a, g, 0.5, b, 1e-5)[which].backward((d_h, d_n)[which])
        want = ops.block_norm_grad(None if which else d_h, d_n if which else None, f, out, a, g, 0.5, b, 1e-5)
        assert torch.equal(f.grad, want.f) and torch.equal(h.grad, want.h) and torch.equal(a.grad, want.post_w)
    f.grad = None
    out, n = autograd.block_norm(f, h.detach(), None, None if g is None else g.detach(), 0.5)
    assert n is None
    out.sum().backward()  # an expanded gradient
    assert torch.equal(f.grad, ops.block_norm_grad(torch.ones_like(out), None, f, out, None, g, 0.5).f)


@pytest.mark.parametrize("dtype", (BF16, F32))
def test_embed_backward(dev, dtype):
    table, ids = leaf(rnd(dev, 1, (V, 72), dtype=dtype)), torch.randint(-2, V + 2, (4, 9), device=dev)
    out = autograd.embed(ids, table, 8.0, F32)
    d = rnd(dev, 2, (4, 9, 72), dtype=F32)
    out.backward(d)
    assert table.grad.dtype == dtype and torch.equal(table.grad, ops.embed_grad(d, ids, V, 8.0, dtype))
    ids2 = ids.clone()
    out = autograd.embed(ids2, table)
    ids2.fill_(0)
    with pytest.raises(RuntimeError, match="modified"):
        out.sum().backward()


def test_gradients_against_differences(dev):
    """fp32 stream and rows: the directional derivative along the gradients' signs."""
    m, d = 6, 64
    t = {k: rnd(dev, i, s, 1.0, F32, 1.0 if len(s) == 1 else 0.0) for i, (k, s) in enumerate(
        dict(f=(m, d), h=(m, d), post_w=(d,), gate=(d,), pre_w=(d,)).items())}
    c_h, c_n = rnd(dev, 20, (m, d), 1.0, F32), rnd(dev, 21, (m, d), 1.0, F32)

    def loss(t):
        out, n = ops.block_norm(t["f"], t["h"], t["post_w"], t["gate"], 0.7, t["pre_w"])
        return (out.double() * c_h.double()).sum() + (n.double() * c_n.double()).sum()

    out, _ = ops.block_norm(t["f"], t["h"], t["post_w"], t["gate"], 0.7, t["pre_w"])
    g = ops.block_norm_grad(c_h, c_n, t["f"], out, t["post_w"], t["gate"], 0.7, t["pre_w"])._asdict()
    step = 2.0 ** -9
    for k in t:
        sign = torch.sign(g[k])
        far = [loss({**t, k: t[k] + s * step * sign}) for s in (2, 1, -1, -2)]
        slope = (8 * (far[1] - far[2]) - (far[0] - far[3])) / (12 * step)  # off by step^4 / 30 of the fifth derivative
        want = g[k].double().abs().sum()
        # fp32 results: 2 m d values of size ~3 off by 2^-22 each, eight differences over 12 steps
        assert abs(float(slope - want)) <= 2 * m * d * 3 * 2.0 ** -22 * 18 / (12 * step) * 0.1 + 1e-3 * float(want), k


def model(dev):
    return {"table": leaf(rnd(dev, 1, (V, D), 0.05)), "gate": leaf(rnd(dev, 2, (D,), 0.1, BF16, 0.5)),
            **{f"{n}{j}": leaf(rnd(dev, 10 * j + i, (D,), 0.1, F32, 1.0)) for j in (0, 1) for i, n in enumerate(("post", "pre"))},
            **{f"w{n}{j}": leaf(rnd(dev, 100 * j + n, (E, D, I) if n == 2 else (E, I, D), 0.03)) for j in (0, 1) for n in (1, 3, 2)}}


def forward(p, ids, idx, w):
    h = autograd.embed(ids, p["table"], 4.0)
    zero = torch.zeros_like(h)
    h, n = autograd.block_norm(zero, h, pre_w=p["pre0"])  # the first norm: no block before it
    for j in (0, 1):
        f = autograd.moe_ffn(n, idx, w, p[f"w1{j}"], p[f"w3{j}"], p[f"w2{j}"])
        h, n = autograd.block_norm(f, h, p[f"post{j}"], p["gate"], 0.5, p["pre1"])
    return h, n


def step(p, ids, idx, w, d):
    _, n = forward(p, ids, idx, w)
    return torch.autograd.grad(n, list(p.values()), d)


def inputs(dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    ids = torch.randint(-1, V, (M,), generator=g, device=dev)
    idx = torch.rand(M, E, generator=g, device=dev).topk(K).indices
    return ids, idx, torch.rand(M, K, generator=g, device=dev) + 0.1, rnd(dev, seed + 1, (M, D))


def plain_step(p, ids, idx, w, d):
    """The same model in 64 bits on the host, by torch's differentiation."""
    q = {k: v.detach().cpu().double().requires_grad_() for k, v in p.items()}
    ids, idx, w, d = ids.cpu(), idx.cpu(), w.cpu().double(), d.cpu().double()
    norm = lambda v, g: v * torch.rsqrt((v * v).mean(dim=-1, keepdim=True) + 1e-6) * g
    h = torch.where((ids >= 0)[:, None], q["table"][ids.clamp(min=0)], 0.0) * 4.0
    n = norm(h, q["pre0"])
    for j in (0, 1):
        f = torch.zeros_like(n)
        for s in range(K):
            for e in range(E):
                at = torch.nonzero(idx[:, s] == e)[:, 0]
                g = (n[at] @ q[f"w1{j}"][e].T).clamp(max=10.0)
                u = (n[at] @ q[f"w3{j}"][e].T).clamp(-10.0, 10.0)
                f = f.index_add(0, at, w[at, s, None] * ((g * torch.sigmoid(g) * u) @ q[f"w2{j}"][e].T))
        h = h + 0.5 * q["gate"] * norm(f, q[f"post{j}"])
        n = norm(h, q["pre1"])
    return torch.autograd.grad(n, list(q.values()), d)


def test_step_clip_and_serve(dev):
    p = model(dev)
    ids, idx, w, d = inputs(dev, 5)
    grads = step(p, ids, idx, w, d)
    # Between the ops everything is bf16: about 12 roundings on the longest way forward and as many back, each off by
    # 2^-9 of the values' size at random (2^-8 at most), so 24 2^-8 of the gradient's norm is more than they add up to
    for k, g, want in zip(p, grads, plain_step(p, ids, idx, w, d)):
        assert float((g.cpu().double() - want).norm()) <= 24 * 2.0 ** -8 * float(want.norm()), k
    before = [g.clone() for g in grads]
    norm = ops.clip_grads(grads, 0.5)
    want = sum(float((g.double() ** 2).sum()) for g in before) ** 0.5
    assert want > 0.5 and abs(float(norm) - want) <= 2.0 ** -23 * want
    c = torch.tensor(0.5 / (want + 1e-6), dtype=F32).to(dev)
    for g, b in zip(grads, before):
        assert ((g.double() - b.double() * c.double()).abs() <= (torch.finfo(g.dtype).eps / 2 + 2.0 ** -22) * (b.double() * c.double()).abs() + 1e-38).all()
    with torch.no_grad():
        for t, g in zip(p.values(), grads):
            t -= g.to(t.dtype)
    # back into the store, and served: the kernels of the 4-bit experts on what the codes stand for
    store = expert_store.HbmExpertStore(1, E, D, I, dev, with_shared=False)
    store.mark_absent(0, 3)
    table = store.table(0)
    assert (table[3] == 0).all() and (table[2] != 0).all()
    for e in range(E):
        store.put_expert(0, e, p["w10"][e], p["w30"][e], p["w20"][e])
    assert store.has_expert(0, 3) and store.table(0) is table and (table != 0).all()
    fresh = expert_store.HbmExpertStore(1, E, D, I, dev, with_shared=False).table(0)
    assert torch.equal(table - table[0, 0], fresh - fresh[0, 0])
    x = rnd(dev, 77, (M, D))
    got = ops.moe_prefill(x, idx, w, store.table(0), ops.SCALE_E8M0, None, 10.0, i=I)[0].double()
    held = [[ops.fp4_dequant_bf16(c, s) for c, s in zip(store.expert_views(0, e)[0::2], store.expert_views(0, e)[1::2])] for e in range(E)]
    assert torch.equal(held[2][0], ops.fp4_dequant_bf16(*ops.fp4_quant(p["w10"][2].detach())))
    want = torch.zeros(M, D, dtype=torch.float64, device=dev)
    for s in range(K):
        for e in range(E):
            at = torch.nonzero(idx[:, s] == e)[:, 0]
            w1, w3, w2 = (t.double() for t in held[e])
            g, u = (x[at].double() @ w1.T).clamp(max=10.0), (x[at].double() @ w3.T).clamp(-10.0, 10.0)
            want[at] += w[at, s, None].double() * ((g * torch.sigmoid(g) * u) @ w2.T)
    assert float((got - want).norm()) <= 2.0 ** -8 * float(want.norm())


def test_step_replayed(dev):
    """Forward, backward and clipping in one captured graph."""
    p = model(dev)
    ids, idx, w, d = inputs(dev, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(p, ids, idx, w, d)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            grads = step(p, ids, idx, w, d)
            norm = ops.clip_grads(grads, 0.5)
    torch.cuda.synchronize()
    for seed in (7, 9, 11):
        for a, b in zip((ids, idx, w, d), inputs(dev, seed)):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want = step(p, ids, idx, w, d)
        assert torch.equal(ops.clip_grads(want, 0.5), norm)
        assert all(torch.equal(a, b) for a, b in zip(grads, want))


def test_what_autograd_is_told(dev):
    x = leaf(rnd(dev, 1, (4, 64)))
    y = x * 2
    z = (y * y).sum()  # saves y
    with torch.no_grad():
        ops.clip_grads([y], 0.1)
    with pytest.raises(RuntimeError, match="modified"):
        z.backward()
    for bad in (lambda: ops.clip_grads([x], 1.0), lambda: ops.clip_grads([x.detach()], 1.0, out=[x * 1]),
                lambda: ops.embed_grad(rnd(dev, 1, (2, 64)), torch.zeros(2, dtype=torch.int64, device=dev), 4, out=x)):
        with pytest.raises(ValueError, match="no_grad"):
            bad()
    assert float(ops.grad_norm([x])) > 0


def test_put_expert_refuses_other_shapes(dev):
    store = expert_store.HbmExpertStore(1, 2, D, I, dev, with_shared=False)
    a, b = rnd(dev, 1, (I, D)), rnd(dev, 2, (D, I))
    for bad, exc in (((0, 0, a, a, a), ValueError), ((0, 0, b, a, b), ValueError), ((0, 2, a, a, b), IndexError), ((0, 0, a, a, b.half()), TypeError),
                     ((0, 0, a, a.cpu(), b), ValueError)):
        store.expert_record(0, 0).fill_(7)
        with pytest.raises(exc):
            store.put_expert(*bad)
        assert (store.expert_record(0, 0) == 7).all()  # nothing is written before everything is looked at
