"""What torch.autograd is told about the block norm: which tensors its backward pass reads (no GPU needed: plain sums
that torch's differentiation does not see, in place of the kernels)."""
import pytest
import torch

from home_seek_amd import autograd, ops

F32 = torch.float32


@pytest.fixture()
def plain(monkeypatch):
    given = []

    def block_norm(f, h, post_w=None, gate=None, scale=1.0, pre_w=None, eps=1e-6):
        out = h.detach() + scale * f.detach().to(h.dtype)
        return out, None if pre_w is None else out.to(f.dtype) * pre_w.detach()

    def block_norm_grad(d_h, d_n, f, h_out, post_w=None, gate=None, scale=1.0, pre_w=None, eps=1e-6, need=(True,) * 5):
        given.append(h_out)
        assert h_out.shape == f.shape and (d_h is None or h_out.dtype == d_h.dtype)
        d = torch.zeros_like(h_out)
        return ops.BlockNormGrad(d.to(f.dtype), d, post_w, gate, pre_w)

    monkeypatch.setattr(ops, "block_norm", block_norm)
    monkeypatch.setattr(ops, "block_norm_grad", block_norm_grad)
    return given


@pytest.mark.parametrize("stream", (torch.bfloat16, F32))
def test_a_stream_without_a_norm_before_the_next_block_may_be_written(plain, stream):
    """No gradient needs it then, as no gradient of a plain sum needs its result."""
    f, h, w = torch.randn(3, 64).bfloat16().requires_grad_(), torch.randn(3, 64).to(stream).requires_grad_(), torch.ones(64).requires_grad_()
    out, n = autograd.block_norm(f, h, w, None, 0.5)
    assert n is None
    out += 1.0
    out.sum().backward()
    assert f.grad.dtype == torch.bfloat16 and h.grad.dtype == stream and plain[0].dtype == stream


def test_a_stream_that_the_norm_is_of_may_not(plain):
    f, h, w = torch.randn(3, 64).requires_grad_(), torch.randn(3, 64).requires_grad_(), torch.ones(64).requires_grad_()
    out, n = autograd.block_norm(f, h, w, None, 0.5, w)
    (out.sum() + n.sum()).backward()
    assert len(plain) == 1 and torch.equal(plain[0], out)
    out, n = autograd.block_norm(f, h, w, None, 0.5, w)
    out.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        n.sum().backward()


def test_what_else_it_reads_may_not_change(plain):
    for i in range(4):
        t = [torch.randn(3, 64) for _ in range(2)] + [torch.ones(64), torch.ones(64)]  # f, h, post_w, gate
        f, h, w, g = (v.requires_grad_() * 1 for v in t)
        out, _ = autograd.block_norm(f, h, w, g, 0.5)
        (f, h, w, g)[i].add_(1.0)
        if i == 1:  # the stream before the block is no part of any gradient
            out.sum().backward()
            continue
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()
