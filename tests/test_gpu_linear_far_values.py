"""SiLU and SwiGLU of gates far below zero: the sigmoid is a number there that fp32
does not hold, and the product with the gate has to be next to nothing all the
same, in every kernel that has an epilogue and in the gradient.

With s <= 2^-124 from z = -86 on and the gate counted as -86 below, |z s| <= 86.5 x
2^-124 and |s + z s (1 - s)| <= 87 x 2^-124, both below 2^-117; the true values are
smaller still (86 e^-86 < 2^-117)."""
import pytest
import torch

from home_seek_amd import ops

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
FAR = [-87.0, -90.0, -126.0, -200.0, -1e4, -2.0 ** 30, -23336016.0, -1e30, -1e36, -1e38, -3e38]
NEXT_TO_NOTHING = 2.0 ** -117


def far_gates(dev, n):
    return torch.tensor(FAR, device=dev).to(BF16).repeat(n // len(FAR) + 1)[:n].contiguous()


# one row (no tiles), tiles, tiles whose reduction is split (the join's epilogue)
SHAPES = [(1, 128, 64), (40, 128, 64), (300, 264, 72), (64, 4096, 4096)]


@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_far_gates_give_next_to_nothing(dev, m, n, k, out_dtype):
    x, w, gate = torch.zeros(m, k, dtype=BF16, device=dev), torch.zeros(n, k, dtype=BF16, device=dev), far_gates(dev, n)
    y = ops.linear(x, w, gate, act="silu", out_dtype=out_dtype)
    assert bool((y <= 0).all()) and bool((y.double().abs() <= NEXT_TO_NOTHING).all())
    for up in (3.0, -3.0):
        y = ops.linear(x, w, gate, act="swiglu", w_up=w, bias_up=torch.full_like(gate, up), limit=10.0, out_dtype=out_dtype)
        assert bool((y * up <= 0).all()) and bool((y.double().abs() <= 3 * NEXT_TO_NOTHING).all())


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_far_gates_times_an_infinite_up_value(dev, m, n, k):
    """Next to nothing, but not nothing: no NaN."""
    x, w, gate = torch.zeros(m, k, dtype=BF16, device=dev), torch.zeros(n, k, dtype=BF16, device=dev), far_gates(dev, n)
    for up in (float("inf"), float("-inf")):
        y = ops.linear(x, w, gate, act="swiglu", w_up=w, bias_up=torch.full_like(gate, up))
        assert bool((y == -up).all())


@pytest.mark.parametrize("with_bias", [True, False])
@pytest.mark.parametrize("act", ["silu", "swiglu"])
def test_far_gates_have_next_to_no_gradient(dev, act, with_bias):
    m, n = 70, 128
    gate = far_gates(dev, n).expand(m, n)
    eye = torch.eye(n, dtype=BF16, device=dev)
    kw = dict(act=act, need_bias=with_bias)
    if act == "silu":
        g = ops.linear_grad(torch.ones(m, n, dtype=BF16, device=dev), torch.ones(m, n, dtype=BF16, device=dev), eye,
                            pre=gate, **kw)
        got = [g.x, g.w, g.bias]
    else:
        pre = torch.cat((gate, torch.full_like(gate, 3.0)), dim=1)
        g = ops.linear_grad(torch.ones(m, n, dtype=BF16, device=dev), torch.ones(m, n, dtype=BF16, device=dev), eye,
                            pre=pre, w_up=eye, limit=10.0, **kw)
        got = [g.x, g.w, g.bias, g.w_up, g.bias_up]
    for t in got:
        if t is not None:  # sums of at most 2 m such values, times 3
            assert bool((t.double().abs() <= 6 * m * NEXT_TO_NOTHING).all())


def test_gates_that_matter_keep_their_bits(dev):
    """Down to -80 a result is off by the fp32 evaluation and half a step of its type: the exponential (3 ulp), the
    sum, the quotient (1 ulp) and the product, below 8 x 2^-23 of the value."""
    n = 4096
    z = torch.linspace(-80.0, 20.0, n, device=dev).to(BF16)
    x, w = torch.zeros(1, 8, dtype=BF16, device=dev), torch.zeros(n, 8, dtype=BF16, device=dev)
    want = z.double() / (1 + torch.exp(-z.double()))
    y = ops.linear(x, w, z, act="silu", out_dtype=F32)[0].double()
    assert bool(((y - want).abs() <= 8 * 2.0 ** -23 * want.abs()).all())
