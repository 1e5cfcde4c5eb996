"""Sums within a bf16 step of SwiGLU's limit: the forward call cuts the fp32 sum, the gradient goes by pre, the sum as
it is kept in bf16."""
import math

import pytest
import torch

from home_seek_amd import ops

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
LIMIT, STEP = 10.0, 0.0625  # a bf16 step between 8 and 16


def products(dev, values):
    """x [1, 8] and w [len(values), 8] whose product is the values, exactly, though they are no bf16 values."""
    head = torch.tensor(values, dtype=F32).to(BF16)
    rest = torch.tensor(values, dtype=F32) - head.float()
    w = torch.zeros(len(values), 8, dtype=BF16)
    w[:, 0], w[:, 1] = head, rest.to(BF16)
    assert torch.equal(w[:, 0].double() + w[:, 1].double(), torch.tensor(values, dtype=torch.float64))
    return torch.ones(1, 8, dtype=BF16, device=dev), w.to(dev)


VALUES = [LIMIT - STEP / 4, LIMIT, LIMIT + STEP / 64, LIMIT + STEP / 4, LIMIT + STEP / 2, LIMIT + STEP * 3 / 4, LIMIT + STEP]
KEPT = [LIMIT] * 5 + [LIMIT + STEP] * 2  # half a step rounds to the even value, the limit


@pytest.mark.parametrize("m", [1, 40])
def test_gates_at_the_limit(dev, m):
    values = VALUES + [0.0]
    x, w = products(dev, values)
    _, w_up = products(dev, [2.0] * len(values))
    x = x.expand(m, 8).contiguous()
    out, pre = ops.linear(x, w, act="swiglu", w_up=w_up, limit=LIMIT, out_dtype=F32, want_pre=True)
    assert pre[:, :7].tolist() == [KEPT] * m
    cut = min(VALUES), LIMIT
    want = [2 * g / (1 + math.exp(-g)) for g in [cut[0]] + [cut[1]] * 6]
    assert bool(((out[:, :7].double().cpu() - torch.tensor(want, dtype=torch.float64)).abs() <= 16 * 2.0 ** -24 * 20).all())
    db = ops.linear_grad(torch.ones(m, 8, dtype=BF16, device=dev), x, w, "swiglu", pre, w_up, LIMIT, need_bias=True).bias
    s = 1 / (1 + math.exp(-LIMIT))
    slope = 2 * (s + LIMIT * s * (1 - s))
    assert bool(((db[:5].double() - m * slope).abs() <= (m + 16) * 2.0 ** -24 * m * 22).all())
    assert db[5:7].tolist() == [0.0, 0.0]


@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_up_values_at_the_limit(dev, sign):
    values = VALUES + [0.0]
    x, w_up = products(dev, [sign * v for v in values])
    _, w = products(dev, [1.0] * len(values))
    out, pre = ops.linear(x, w, act="swiglu", w_up=w_up, limit=LIMIT, out_dtype=F32, want_pre=True)
    assert pre[0, 8:15].tolist() == [sign * v for v in KEPT]
    gate = 1 / (1 + math.exp(-1.0))
    want = torch.tensor([sign * gate * min(v, LIMIT) for v in VALUES], dtype=torch.float64)
    assert bool(((out[0, :7].double().cpu() - want).abs() <= 16 * 2.0 ** -24 * LIMIT).all())
    db = ops.linear_grad(torch.ones(1, 8, dtype=BF16, device=dev), x, w, "swiglu", pre, w_up, LIMIT, need_bias=True).bias_up
    assert bool(((db[:5].double() - gate).abs() <= 17 * 2.0 ** -24).all()) and db[5:7].tolist() == [0.0, 0.0]
