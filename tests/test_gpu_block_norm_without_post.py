"""The gradient of a block's result f that has no norm of its own, h' = h + scale gate f: f is no factor of it, so what
stands in f, an infinity or NaN in a padded row for one, changes nothing."""
import pytest
import torch

from home_seek_amd import ops

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def normal(dev, seed, shape, dtype=BF16):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn(shape, generator=g, device=dev).to(dtype)


# rows by 8, 16, 32 and 64 threads, by a wave twice, by workgroups, by the widest ones twice
@pytest.mark.parametrize("m,d", ((40, 64), (33, 128), (19, 256), (9, 512), (7, 768), (300, 2056), (5, 8192), (270, 12296)))
@pytest.mark.parametrize("gate", (None, "channel", "token", "full"))
@pytest.mark.parametrize("t,s", ((BF16, BF16), (BF16, F32), (F32, BF16), (F32, F32)))
def test_far_values_of_f_change_nothing(dev, m, d, gate, t, s):
    f, h, d_h, d_n, w = normal(dev, 1, (m, d), t), normal(dev, 2, (m, d), s), normal(dev, 3, (m, d), s), normal(dev, 4, (m, d), t), normal(dev, 5, (d,), t)
    g = None if gate is None else normal(dev, 6, {"channel": (d,), "token": (m, 1), "full": (m, d)}[gate], t)
    far = f.clone()
    far[0], far[1, 3], far[2, d - 1], far[m - 1, d // 2] = float("nan"), float("inf"), -float("inf"), float("nan")
    for grads in ((d_h, None, None), (d_h, d_n, w), (None, d_n, w)):
        dh, dn, pre = grads
        want = ops.block_norm_grad(dh, dn, f, h, None, g, 0.75, pre)
        got = ops.block_norm_grad(dh, dn, far, h, None, g, 0.75, pre)
        assert torch.isfinite(got.f).all() and torch.equal(got.f, want.f) and torch.equal(got.h, want.h)
        assert pre is None or torch.equal(got.pre_w, want.pre_w)
        part = ops.block_norm_grad(dh, dn, far, h, None, g, 0.75, pre, need=(True, False, False, False, False))
        assert torch.equal(part.f, want.f)
    plain = 0.75 * d_h.float()
    plain = (plain if g is None else plain * g.float()).to(t)  # the products in their order, each rounded to fp32
    assert torch.equal(ops.block_norm_grad(d_h, None, far, h, None, g, 0.75).f, plain)
