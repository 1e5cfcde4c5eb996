"""The bf16 expert layer for training: ops.linear, moe_gather and moe_combine as
torch.autograd functions, and moe_ffn, the routed SwiGLU experts made of them.

The gradients are the ops' own (linear_grad, moe_combine_grad): weights' and
rows' in bf16, routing weights' in fp32, biases' rounded to the bias's dtype.
Between the ops everything is bf16, as between torch's: the activations, the
experts' results, the sums kept for the backward pass and their gradients.
Under graph capture, capture the forward and the backward pass together, and let
go of every eager graph that reaches the same leaves first: torch ties a leaf's
gradient accumulation to the stream of the first graph that used it, and a
captured backward pass that meets an eager one's ends the process.
Second derivatives and forward-mode ones are refused by torch.
"""
from __future__ import annotations

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import ops
from .ops import ExpertOrder

__all__ = ["linear", "moe_gather", "moe_combine", "moe_ffn"]


# The order's tensors are saved as the others are, so that torch notices a change
# of one before the backward pass has read it.
def _saved_order(tensors: list) -> ExpertOrder | None:
    return ExpertOrder(*tensors) if tensors else None


class _Linear(Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, w_up, bias_up, act, limit, order, out_dtype, grad_enabled):
        need = grad_enabled and any(ctx.needs_input_grad)  # (needs_input_grad says yes under no_grad too)
        out = ops.linear(x, w, bias, residual, act, w_up, bias_up, limit, order, out_dtype, want_pre=need and act is not None)
        out, pre = out if isinstance(out, tuple) else (out, None)
        ctx.save_for_backward(x, w, w_up, pre, *(order or ()))
        ctx.act, ctx.limit = act, limit
        ctx.bias_dtypes = [None if b is None else b.dtype for b in (bias, bias_up)]
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        x, w, w_up, pre, *order = ctx.saved_tensors
        order = _saved_order(order)
        need = ctx.needs_input_grad
        d_out = d_out.to(torch.bfloat16)
        g = ops.linear_grad(d_out, x, w, ctx.act, pre, w_up, ctx.limit, order, need_x=need[0], need_w=need[1] or need[4],
                            need_bias=need[2] or need[5])
        db = [b.to(t) if b is not None and t is not None else None for b, t in zip((g.bias, g.bias_up), ctx.bias_dtypes)]
        d_res = None
        if need[3]:  # rows of no expert have no residual either
            d_res = d_out if order is None else _cleared_behind(d_out, order)
        return (g.x, g.w if need[1] else None, db[0], d_res, g.w_up if need[4] else None, db[1], None, None, None, None, None)


def _cleared_behind(rows: torch.Tensor, order: ExpertOrder) -> torch.Tensor:
    return torch.where((order.pairs >= 0)[:, None], rows, 0)


class _Gather(Function):
    @staticmethod
    def forward(ctx, x, order):
        ctx.save_for_backward(*order)
        return ops.moe_gather(x, order)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_rows):
        return ops.moe_combine(d_rows, _saved_order(ctx.saved_tensors)), None


class _Combine(Function):
    @staticmethod
    def forward(ctx, rows, order, topk_w, residual, out_dtype):
        out = ops.moe_combine(rows, order, topk_w, residual, out_dtype)
        ctx.save_for_backward(rows, topk_w, *order)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        rows, topk_w, *order = ctx.saved_tensors
        need = ctx.needs_input_grad
        d_rows = d_w = None
        if need[0] or need[2]:
            d_rows, d_w = ops.moe_combine_grad(d_out, rows, _saved_order(order), topk_w, need_rows=need[0], need_w=need[2])
        return d_rows, None, None if d_w is None else d_w.to(topk_w.dtype), d_out if need[3] else None, None


def linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, residual: torch.Tensor | None = None,
           act: str | None = None, w_up: torch.Tensor | None = None, bias_up: torch.Tensor | None = None,
           limit: float | None = None, order: ExpertOrder | None = None,
           out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """ops.linear with its gradient (for x, w, bias, residual, w_up, bias_up).  The gradient of an fp32 result is
    rounded to bf16 on its way in: the matrix cores take bf16."""
    # (a Function under no_grad too: it refuses forward-mode tangents, which stay on there)
    return _Linear.apply(x, w, bias, residual, w_up, bias_up, act, limit, order, out_dtype, torch.is_grad_enabled())


def moe_gather(x: torch.Tensor, order: ExpertOrder) -> torch.Tensor:
    """ops.moe_gather with its gradient."""
    return _Gather.apply(x, order)


def moe_combine(rows: torch.Tensor, order: ExpertOrder, topk_w: torch.Tensor | None = None,
                residual: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """ops.moe_combine with its gradient (for rows, topk_w, residual)."""
    return _Combine.apply(rows, order, topk_w, residual, out_dtype)


def moe_ffn(x: torch.Tensor, topk_idx: torch.Tensor, topk_w: torch.Tensor, w1: torch.Tensor, w3: torch.Tensor,
            w2: torch.Tensor, limit: float | None = 10.0, residual: torch.Tensor | None = None) -> torch.Tensor:
    """Routed SwiGLU experts of bf16 weights for any number of tokens, differentiable: x [M, D],
    topk_idx / topk_w [M, k], w1 and w3 [E, I, D], w2 [E, D, I] (the reference's 3-tuples, stacked) ->
    sum_j topk_w[t, j] FFN_{topk_idx[t, j]}(x[t]) (+ residual [M, D]) in bf16.  Ids that are no expert are dropped."""
    order = ops.moe_sort(topk_idx, w1.shape[0])
    a = linear(moe_gather(x, order), w1, act="swiglu", w_up=w3, limit=limit, order=order)
    return moe_combine(linear(a, w2, order=order), order, topk_w, residual)
