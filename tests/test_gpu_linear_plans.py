"""The ways of doing a product (tile, whole or with its reduction in parts, dense or per expert, one matrix or
swiglu's two) that the shapes of test_gpu_linear.py do not reach, by the same 64-bit comparisons.
test_linear_plans_host.py holds that both lists together reach every way there is."""
import pytest
import torch

from test_gpu_linear import BF16, F32, check_forward, check_grad, ints, some_order, spans

from home_seek_amd import ops

pytestmark = pytest.mark.gpu

# m, n, k
FORWARD = [(8, 8144, 5728), (8259, 8, 4312), (8305, 8, 3544), (388, 6256, 7400), (5140, 728, 8312)]
# tokens, slots, experts, n, k
FORWARD_GROUPS = [(10, 2, 4, 3608, 4096), (3373, 2, 50, 8, 4584), (4138, 2, 2, 8, 5016), (2188, 2, 2, 8, 7048),
                  (7428, 2, 10, 232, 8104)]
GRAD = [(3, 5528, 7920), (2, 2560, 8112), (8228, 3472, 8), (15692, 144, 8296), (5619, 144, 8256), (7594, 912, 6952)]
GRAD_GROUPS = [(1021, 2, 2, 1808, 8), (3432, 2, 108, 8608, 8), (4256, 2, 4, 3968, 8), (4069, 2, 7, 1880, 8),
               (5328, 2, 2, 160, 8408), (5087, 2, 2, 152, 5568)]
ACTS = [None, "swiglu"]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", FORWARD)
def test_dense(dev, m, n, k, act):
    check_forward(dev, m, n, k, act)


@pytest.mark.parametrize("drop", [0.0, 0.2])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,top_k,e,n,k", FORWARD_GROUPS)
def test_per_expert(dev, m, top_k, e, n, k, act, drop):
    check_forward(dev, m * top_k, n, k, act, some_order(dev, m, top_k, e, m, drop, skew=True), (e,))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", GRAD)
def test_dense_gradient(dev, m, n, k, act):
    check_grad(dev, m, n, k, act)


@pytest.mark.parametrize("drop", [0.0, 0.2])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,top_k,e,n,k", GRAD_GROUPS)
def test_per_expert_gradient(dev, m, top_k, e, n, k, act, drop):
    check_grad(dev, m * top_k, n, k, act, some_order(dev, m, top_k, e, m, drop, skew=True), (e,))


def test_a_token_of_eight_over_many_experts(dev):
    """Decode: one or no row per expert, tiles for matrices that are read once in two parts, each XCD's begun
    elsewhere in its part."""
    e, n, k = 64, 4096, 4096
    w = ints(dev, 1, (e, n, k))
    for drop in (0.0, 0.4):
        order = some_order(dev, 4, 2, e, 5, drop)
        x, d = ints(dev, 2, (8, k)), ints(dev, 3, (8, n))
        out, dx = ops.linear(x, w, order=order), ops.linear_grad(d, x, w, order=order, need_w=False).x
        last = int(order.offsets[-1])
        assert not bool(out[last:].any()) and not bool(dx[last:].any())
        for i, a, b in spans(order, 8):
            if b > a:
                assert torch.equal(out[a:b], (x[a:b].double() @ w[i].double().T).to(F32).to(BF16))
                assert torch.equal(dx[a:b], (d[a:b].double() @ w[i].double()).to(F32).to(BF16))
