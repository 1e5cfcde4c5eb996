"""The norm of many tensors and clipping to it, against 64-bit restatements.

Bounds: squares and sums are in 64 bits, so the norm is off by half a step of fp32
(and 2^-50 of it from the sums).  A clipped value is off by the factor's rounding and
its own product's, 2^-24 each, and half a step of its type."""
import math

import pytest
import torch

from home_seek_amd import ops

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
E = 2.0 ** -24


def normal(dev, seed, shape, dtype=BF16, std=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=dev) * std).to(dtype)


def plain_norm(grads, kind):
    live = [g.double() for g in grads if g.numel()]
    if kind == 2.0:
        return math.sqrt(sum(float((g * g).sum()) for g in live))
    return max((float(g.abs().max()) for g in live), default=0.0)


def check(grads, max_norm, kind, norm, outs):
    want = plain_norm(grads, kind)
    assert norm.dtype == F32 and norm.dim() == 0
    assert abs(float(norm) - want) <= (E + 2.0 ** -45) * want + 1e-45
    c = min(1.0, max_norm / (want + 1e-6))
    for g, o in zip(grads, outs):
        w = g.double() * c
        assert ((o.double() - w).abs() <= (2.2 * E + torch.finfo(o.dtype).eps / 2) * w.abs() + torch.finfo(o.dtype).smallest_normal * 2.0 ** -7).all()


LISTS = {
    "one value": [(1,)],
    "an empty one and a scalar": [(0,), (), (3, 0, 2)],
    "a layer": [(64, 33), (64,), (7,), (128, 16), (1,)],
    "one workgroup's most": [(32768,)],
    "a value more": [(32768,), (1,)],
    "odd sizes": [(16384,), (16385,), (16383,), (8,), (9,), (100003,), (2, 3, 5)],
    "a launch's most": [(37,)] * 112,
    "more than a launch": [(411 + i % 7,) for i in range(113)],
    "many": [(1 + 37 * i % 2999,) for i in range(700)],
    "large": [(3000, 4099), (1, 70001), (4096,), (2048, 4096)],
    "large and more than a launch": [(411 + i % 7,) for i in range(113)] + [(4099, 4097), (16385,)],
}


@pytest.mark.parametrize("name", LISTS)
@pytest.mark.parametrize("kind", (2.0, math.inf))
def test_lists(dev, name, kind):
    shapes = LISTS[name]
    types = [BF16 if i % 3 else F32 for i in range(len(shapes))]
    grads = [normal(dev, i, s, t, 0.1 * (1 + i % 5)) for i, (s, t) in enumerate(zip(shapes, types))]
    norm = ops.grad_norm(grads, kind)
    for max_norm in (0.25, 0.0, 1e9, math.inf):
        kept = [g.clone() for g in grads]
        got = ops.clip_grads(kept, max_norm, kind)
        assert torch.equal(got, norm)
        check(grads, max_norm, kind, got, kept)
        if max_norm > 1e6:
            assert all(torch.equal(a, b) for a, b in zip(kept, grads))
        outs = [torch.full_like(g, 7.0, dtype=BF16 if i % 2 else F32) for i, g in enumerate(grads)]
        before = [g.clone() for g in grads]
        assert torch.equal(ops.clip_grads(grads, max_norm, kind, out=outs), norm)
        check(grads, max_norm, kind, norm, outs)
        assert all(torch.equal(a, b) for a, b in zip(before, grads))
        for a, b in zip(outs, kept):
            if a.dtype == b.dtype:
                assert torch.equal(a, b)


@pytest.mark.parametrize("max_norm", (1.0, 1e9))
def test_some_in_place(dev, max_norm):
    base = normal(dev, 1, (9000001,))
    grads = [base[1:], normal(dev, 2, (9000000,), F32), normal(dev, 3, (40000,)), normal(dev, 4, (70003,), F32)]
    before = [g.clone() for g in grads]
    outs = [torch.empty(9000000, dtype=F32, device=dev), torch.empty(9000000, device=dev), grads[2], grads[3]]
    norm = ops.clip_grads(grads, max_norm, out=outs)
    check(before, max_norm, 2.0, norm, outs)
    assert torch.equal(grads[0], before[0]) and torch.equal(grads[1], before[1])


@pytest.mark.parametrize("n", (5, 40000))
def test_far_values(dev, n):
    for v in (1e-30, 3e-38, 1e-42, 1e30, 3.3e38):
        g = torch.full((n,), v, device=dev)
        want = float(g[0].double()) * math.sqrt(n)
        got = float(ops.grad_norm([g]))
        assert got == math.inf if want > torch.finfo(F32).max else abs(got - want) <= 2 * E * want + 1e-45
        assert float(ops.grad_norm([g], math.inf)) == float(g[0])
        ops.clip_grads([g], 1.0)
        c = min(1.0, 1.0 / (want + 1e-6))
        assert abs(float(g[0]) - v * c) <= 4 * E * v * c + 1e-44
    mixed = [torch.full((n,), 1e-20, device=dev), torch.full((1,), 1e20, device=dev)]
    assert abs(float(ops.grad_norm(mixed)) - 1e20) <= 1e20 * 2 * E


@pytest.mark.parametrize("n", (5, 40000))
@pytest.mark.parametrize("kind", (2.0, math.inf))
def test_infinities_and_nan(dev, n, kind):
    for bad in (math.inf, -math.inf, math.nan):
        grads = [normal(dev, 1, (n,)), normal(dev, 2, (n,), F32)]
        grads[1][n // 2] = bad
        norm = ops.clip_grads(grads, 1.0, kind)
        if math.isnan(bad):
            assert norm.isnan() and all(g.isnan().all() for g in grads)
        else:
            assert norm == math.inf and (grads[0] == 0).all() and grads[1][n // 2].isnan()
            assert int(grads[1].isnan().sum()) == 1


def test_views_and_orders_of_memory(dev):
    base, other = normal(dev, 1, (200, 70)), normal(dev, 2, (70001,), F32)
    grads = [base.t(), base.clone().as_strided((70, 200), (1, 70)), other[1:], other.clone()[3:60000], normal(dev, 3, (5, 6, 7)).permute(2, 0, 1),
             normal(dev, 5, (40001,))[1:]]
    kept = [g.clone() for g in grads]
    norm = ops.clip_grads(grads, 0.5)
    check(kept, 0.5, 2.0, norm, grads)
    assert float(other[0]) == float(normal(dev, 2, (70001,), F32)[0])
    outs = [torch.empty_like(g, dtype=F32) for g in kept]  # the same order of memory
    check(kept, 0.5, 2.0, ops.clip_grads(kept, 0.5, out=outs), outs)
    shifted = torch.empty(40002, dtype=F32, device=dev)
    check(kept[-1:], 0.5, 2.0, ops.clip_grads(kept[-1:], 0.5, out=[shifted[1:40001]]), [shifted[1:40001]])


def test_tensor_beyond_32_bits(dev):
    n = 2 ** 32 + 40005
    g = torch.zeros(n, dtype=BF16, device=dev)
    g[5], g[2 ** 31 + 3], g[n - 1] = 3.0, 4.0, 12.0
    norm = ops.clip_grads([g], 1.3)
    assert float(norm) == 13.0
    c = torch.tensor(1.3, dtype=F32).double() / (13.0 + 1e-6)
    for at, v in ((5, 3.0), (2 ** 31 + 3, 4.0), (n - 1, 12.0)):
        assert float(g[at]) == float(torch.tensor(v * float(c)).to(BF16))


@pytest.mark.parametrize("n", (500, 100000))
def test_deterministic_and_replayed(dev, n):
    grads = [normal(dev, i, (n + i,), BF16 if i % 2 else F32) for i in range(5)]
    outs = [torch.empty_like(g) for g in grads]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.clip_grads(grads, 1.0, out=outs)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            norm = ops.clip_grads(grads, 1.0, out=outs)
            alone = ops.grad_norm(grads)
    torch.cuda.synchronize()
    for seed in range(3):
        for i, g in enumerate(grads):
            g.copy_(normal(dev, 100 * seed + i, g.shape, g.dtype))
        graph.replay()
        torch.cuda.synchronize()
        want = [torch.empty_like(g) for g in grads]
        assert torch.equal(ops.clip_grads(grads, 1.0, out=want), norm) and torch.equal(norm, alone)
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_refusals(dev):
    a, b = normal(dev, 1, (64, 8)), normal(dev, 2, (64, 8), F32)
    for bad, exc in ((lambda: ops.clip_grads([a, a], 1.0), RuntimeError), (lambda: ops.clip_grads([a, a[3:5]], 1.0), RuntimeError),
                     (lambda: ops.clip_grads([a, b], 1.0, out=[a, a]), RuntimeError), (lambda: ops.clip_grads([a, b], 1.0, out=[b, a]), RuntimeError),
                     (lambda: ops.clip_grads([b], 1.0, out=[b.view(-1).view(BF16)[:512].view(64, 8)]), RuntimeError),
                     (lambda: ops.clip_grads([a], 1.0, out=[a, b]), ValueError), (lambda: ops.clip_grads([a], 1.0, out=[a[:3]]), ValueError),
                     (lambda: ops.clip_grads([a], 1.0, out=[torch.empty(8, 64, device=dev).t()]), ValueError),
                     (lambda: ops.clip_grads([a[:, ::2]], 1.0), ValueError), (lambda: ops.grad_norm([a[:, :4]]), ValueError),
                     (lambda: ops.grad_norm([a[:1].expand(64, 8)]), ValueError),
                     (lambda: ops.grad_norm([a.half()]), TypeError), (lambda: ops.grad_norm([]), ValueError),
                     (lambda: ops.grad_norm([a], 1.0), RuntimeError), (lambda: ops.clip_grads([a], -1.0), RuntimeError),
                     (lambda: ops.clip_grads([a], math.nan), RuntimeError), (lambda: ops.grad_norm([a, b.cpu()]), RuntimeError)):
        with pytest.raises(exc):
            bad()
    assert float(ops.grad_norm([a, a])) > 0  # read twice is no harm


def test_large_replayed(dev):
    """Much data into other tensors, captured: the norm, the factor and the copy follow the values of each replay."""
    grads = [normal(dev, 1, (4099, 4097)), normal(dev, 2, (70001,), F32)]
    outs = [torch.empty_like(g) for g in grads]
    ops.clip_grads(grads, 1.0, out=outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ops.clip_grads(grads, 1.0, out=outs)
    for i in range(4):
        for j, g in enumerate(grads):
            g.copy_(normal(dev, 10 * i + j, g.shape, g.dtype, (0.5, 2.0, 1e-6, 1.0)[i]))
        graph.replay()
        torch.cuda.synchronize()
        check(grads, 1.0, 2.0, norm, outs)
        got = [o.clone() for o in outs]
        assert torch.equal(ops.clip_grads(grads, 1.0, out=outs), norm)
        assert all(torch.equal(a, b) for a, b in zip(got, outs))
