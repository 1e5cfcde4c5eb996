"""The bf16 expert layer for training: ops.linear, moe_gather and moe_combine as
torch.autograd functions, moe_ffn, the routed SwiGLU experts made of them, and what
stands around it: the embedding lookup and the norms between two blocks.

The gradients are the ops' own (linear_grad, moe_combine_grad, embed_grad,
block_norm_grad): weights' and rows' in bf16, routing weights' in fp32, biases',
norms' weights' and broadcast gates' rounded to their tensor's dtype.
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

__all__ = ["linear", "moe_gather", "moe_combine", "moe_ffn", "embed", "block_norm"]


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


class _Embed(Function):
    @staticmethod
    def forward(ctx, ids, table, scale, out_dtype):
        ctx.save_for_backward(ids)
        ctx.scale, ctx.vocab, ctx.dtype = scale, table.shape[0], table.dtype
        return ops.embed(ids, table, scale, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        ids, = ctx.saved_tensors
        return None, ops.embed_grad(d_out, ids, ctx.vocab, ctx.scale, ctx.dtype), None, None


class _BlockNorm(Function):
    @staticmethod
    def forward(ctx, f, h, post_w, gate, pre_w, scale, eps):
        ctx.set_materialize_grads(False)  # a result that is not used has no gradient to be read
        out, n = ops.block_norm(f, h, post_w, gate, scale, pre_w, eps)
        # (only the norm before the next block reads the stream again: without it, it may be written)
        ctx.save_for_backward(f, None if pre_w is None else out, post_w, gate, pre_w)
        ctx.scale, ctx.eps = scale, eps
        return out, n

    @staticmethod
    @once_differentiable
    def backward(ctx, d_h, d_n):
        f, out, post_w, gate, pre_w = ctx.saved_tensors
        if d_h is None and d_n is None:
            return (None,) * 7
        if out is None:
            out = d_h = d_h.contiguous()  # (the stream's type; not read as it)
        g = ops.block_norm_grad(d_h, d_n, f, out, post_w, gate, ctx.scale, pre_w, ctx.eps, need=ctx.needs_input_grad[:5])
        like = lambda d, t: None if d is None else d.to(t.dtype)
        return g.f, g.h, like(g.post_w, post_w), like(g.gate, gate), like(g.pre_w, pre_w), None, None


def embed(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """ops.embed with its gradient (for the table, in its dtype, every row written; a training loop
    that keeps a gradient buffer of its own adds to it with ops.embed_grad(..., out=))."""
    return _Embed.apply(ids, table, scale, out_dtype)


def block_norm(f: torch.Tensor, h: torch.Tensor, post_w: torch.Tensor | None = None, gate: torch.Tensor | None = None,
               scale: float = 1.0, pre_w: torch.Tensor | None = None, eps: float = 1e-6):
    """ops.block_norm with its gradient (for f, h, the norms' weights and the gate) -> (h', n)."""
    return _BlockNorm.apply(f, h, post_w, gate, pre_w, scale, eps)
