"""What torch.autograd is told about the expert layer's functions, with plain products in place of the kernels (no GPU
needed)."""
import pytest
import torch
from torch.autograd import forward_ad

from home_seek_amd import autograd, ops

BF16 = torch.bfloat16


@pytest.fixture()
def plain_linear(monkeypatch):
    """ops.linear as a product that torch's differentiation does not see, as the kernels are."""
    kept = []

    def linear(x, w, bias=None, residual=None, act=None, w_up=None, bias_up=None, limit=None, order=None,
               out_dtype=BF16, want_pre=False):
        kept.append(want_pre)
        pre = (x.detach().float() @ w.detach().float().T).to(BF16)
        out = torch.nn.functional.silu(pre) if act == "silu" else pre
        return (out, pre) if want_pre else out

    monkeypatch.setattr(ops, "linear", linear)
    return kept


@pytest.mark.parametrize("mode", ["grad", "no_grad"])
def test_a_forward_mode_tangent_is_never_dropped(plain_linear, mode):
    """Forward-mode differentiation stays on under no_grad: what has no rule for it says so, as with gradients on."""
    x, w = torch.randn(4, 8).to(BF16), torch.randn(16, 8).to(BF16)
    with torch.set_grad_enabled(mode == "grad"), forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="jvp|forward mode"):
            autograd.linear(dual, w, act="silu")
        with pytest.raises(RuntimeError, match="jvp|forward mode"):
            autograd.linear(x, forward_ad.make_dual(w, torch.ones_like(w)))
        autograd.linear(x, w)  # a call without tangents goes through


def test_no_sums_are_kept_where_no_gradient_can_be_asked_for(plain_linear):
    x, w = torch.randn(4, 8).to(BF16), torch.randn(16, 8).to(BF16).requires_grad_()
    y = autograd.linear(x, w, act="silu")
    with torch.no_grad():
        a = autograd.linear(x, w, act="silu")
    with torch.inference_mode():
        b = autograd.linear(x, w, act="silu")
    c = autograd.linear(x, w.detach(), act="silu")
    assert plain_linear == [True, False, False, False]
    assert y.requires_grad and not any(t.requires_grad for t in (a, b, c))
    assert all(torch.equal(y, t) for t in (a, b, c))
