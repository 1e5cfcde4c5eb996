"""A stream that is written after the block norm, where no norm of it follows: the gradients are those of the call."""
import pytest
import torch

from home_seek_amd import autograd, ops

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("stream", (BF16, F32))
@pytest.mark.parametrize("d", (64, 2056, 12296))
def test_written_afterwards(dev, stream, d):
    g = torch.Generator(device=dev).manual_seed(d)
    rnd = lambda *s, t=BF16: torch.randn(s, generator=g, device=dev).to(t)
    f, h, w, gate = (t.requires_grad_() for t in (rnd(5, d), rnd(5, d, t=stream), rnd(d), rnd(5, 1)))
    out, _ = autograd.block_norm(f, h, w, gate, 0.5)
    kept, d_h = out.detach().clone(), rnd(5, d, t=stream)
    want = ops.block_norm_grad(d_h, None, f, kept, w, gate, 0.5)
    with torch.no_grad():
        out.fill_(float("nan"))
    out.backward(d_h)
    for t, x in ((f, want.f), (h, want.h), (w, want.post_w), (gate, want.gate)):
        assert torch.equal(t.grad, x.to(t.dtype))
    out, _ = autograd.block_norm(f, h, w, gate, 0.5)
    f.grad = None
    out.sum().backward()  # an expanded gradient
    assert torch.equal(f.grad, ops.block_norm_grad(torch.ones_like(out), None, f, out, w, gate, 0.5).f)
