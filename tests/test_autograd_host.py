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


def order_of(rows):
    """An order of `rows` single-slot tokens in one expert."""
    at = torch.arange(rows, dtype=torch.int32)
    return ops.ExpertOrder(torch.tensor([0, rows], dtype=torch.int32), at.clone(), at.clone()[:, None].contiguous())


@pytest.fixture()
def plain_rows(plain_linear, monkeypatch):
    monkeypatch.setattr(ops, "moe_gather", lambda x, order: x.detach().clone())
    monkeypatch.setattr(ops, "moe_combine", lambda rows, order, w=None, residual=None, out_dtype=None: rows.detach().clone())
    monkeypatch.setattr(ops, "moe_combine_grad", lambda d, rows, order, w=None, need_rows=True, need_w=True:
                        (d if need_rows else None, w if need_w else None))
    monkeypatch.setattr(ops, "linear_grad", lambda d, x, w, *a, **kw:
                        ops.LinearGrad(torch.zeros_like(x), torch.zeros_like(w), None, None, None))


CALLS = {
    "linear": lambda x, w, order: autograd.linear(x, w, order=order),
    "moe_gather": lambda x, w, order: autograd.moe_gather(x, order),
    "moe_combine": lambda x, w, order: autograd.moe_combine(x, order),
}


@pytest.mark.parametrize("what", CALLS)
def test_an_order_that_changes_before_the_backward_pass_is_refused(plain_rows, what):
    """As any tensor that a backward pass reads: its gradients would be those of another order."""
    for i in range(3):
        x, w, order = torch.randn(4, 8).to(BF16).requires_grad_(), torch.randn(16, 8).to(BF16), order_of(4)
        y = CALLS[what](x, w, order)
        y.sum().backward()
        assert x.grad.shape == x.shape
        y = CALLS[what](x, w, order)
        order[i].add_(0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_a_function_keeps_its_own_order(plain_rows, monkeypatch):
    """The order that the backward pass hands on is the forward call's."""
    seen = []
    monkeypatch.setattr(ops, "moe_combine", lambda rows, order, *a: (seen.append(order), rows.detach().clone())[1])
    x, order = torch.randn(4, 8).requires_grad_(), order_of(4)
    autograd.moe_gather(x, order).sum().backward()
    assert isinstance(seen[0], ops.ExpertOrder) and all(torch.equal(a, b) for a, b in zip(seen[0], order))
