"""Clipping to an infinite limit: nothing is cut down, whatever the norm, so every value stays as it is, bit for bit."""
import math

import pytest
import torch

from home_seek_amd import ops

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def make(dev, counts):
    g = torch.Generator(device=dev).manual_seed(len(counts))
    return [torch.randn(n, generator=g, device=dev).to(F32 if i % 2 else BF16) for i, n in enumerate(counts)]


# one workgroup; several; several launches; much data, which the second pass takes by pieces
LISTS = {"few": [5, 6], "more": [40000, 3001], "launches": [411 + i % 7 for i in range(120)], "much": [(1 << 24) + 7, 1000]}


@pytest.mark.parametrize("name", LISTS)
@pytest.mark.parametrize("kind", (2.0, math.inf))
@pytest.mark.parametrize("bad", (None, math.inf, -math.inf))
def test_nothing_is_cut_down(dev, name, kind, bad):
    grads = make(dev, LISTS[name])
    if bad is not None:
        grads[1][3] = bad
    kept = [g.clone() for g in grads]
    outs = [torch.zeros_like(g, dtype=F32) for g in grads]
    norm = ops.clip_grads(grads, math.inf, kind, out=outs)
    assert torch.equal(norm, ops.grad_norm(grads, kind)) and (bad is None) == math.isfinite(float(norm))
    assert all(torch.equal(o, k.float()) and torch.equal(g, k) for o, g, k in zip(outs, grads, kept))
    assert torch.equal(ops.clip_grads(grads, math.inf, kind), norm)
    assert all(torch.equal(g, k) for g, k in zip(grads, kept))


@pytest.mark.parametrize("name", LISTS)
@pytest.mark.parametrize("kind", (2.0, math.inf))
def test_nan_is_nan_all_the_same(dev, name, kind):
    grads = make(dev, LISTS[name])
    grads[1][3], grads[0][1] = math.nan, math.inf
    outs = [torch.zeros_like(g) for g in grads]
    assert ops.clip_grads(grads, math.inf, kind, out=outs).isnan() and all(o.isnan().all() for o in outs)
    ops.clip_grads(grads, math.inf, kind)
    assert all(g.isnan().all() for g in grads)


def test_a_norm_beyond_fp32(dev):
    """Finite values whose norm fp32 does not hold: the limit is compared in 64 bits, the norm comes out infinite."""
    for n in (100, 50000):
        g = torch.full((n,), 3e38, device=dev)
        assert ops.clip_grads([g], math.inf) == math.inf and (g == torch.full_like(g, 3e38)).all()
