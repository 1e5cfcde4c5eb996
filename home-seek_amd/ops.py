"""Torch-facing wrappers of the libhsmoe entry points.

Each function takes device tensors, checks shapes on the host, and enqueues
the HIP kernels on the current torch stream.  Workspaces are zero-filled once
per (device, stream, purpose) and reused; kernels leave their counters at
zero, so stream-ordered calls can share them.
"""
from __future__ import annotations

import array
import contextlib
import ctypes
from typing import NamedTuple

import torch

from . import _lib
from ._lib import SCALE_E8M0, SCALE_F32, check, lib, ptr, require_cuda, stream_ptr

__all__ = [
    "SCALE_E8M0", "SCALE_F32", "scale_kind_of", "fp4_dequant_bf16", "fp8_dequant_bf16", "router_topk",
    "moe_decode", "moe_layer_decode", "moe_layer_decode_routed", "NormTail", "moe_layer_status", "moe_layer_status_words",
    "clear_moe_layer_status", "check_moe_layer_status", "lm_head_accept", "expert_table", "shared_entry",
    "dequant_blocked", "xor_checksum", "MAX_DECODE_TOKENS", "MAX_LAYER_EXPERTS", "embed_add_rms_norm", "mtp_input",
    "decode_step_record", "ExpertOrder", "moe_sort", "moe_gather", "moe_combine", "moe_combine_grad",
    "linear", "linear_grad", "LinearGrad",
]

MAX_DECODE_TOKENS = 8
MAX_LAYER_EXPERTS = 256  # expert count the one-launch layer kernel handles

_workspaces: dict[tuple, torch.Tensor] = {}
# Workspaces replaced by larger ones.  A HIP graph captured before the growth
# still holds the old address, so the old tensor stays allocated for the life
# of the process (a graph replay must never touch freed memory).
_retired_workspaces: list[tuple[tuple, torch.Tensor]] = []


def _workspace(device: torch.device, purpose: str, nbytes: int) -> torch.Tensor:
    """Zero-filled device workspace of at least nbytes, one per (device,
    stream, purpose), grown when a call needs more.  A grown layer workspace
    keeps the sticky status word of the one it replaces; the replaced one is
    kept alive (graphs captured against it may still replay)."""
    key = (device.index, stream_ptr(device), purpose)
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        new = torch.zeros(max(nbytes, 256), dtype=torch.uint8, device=device)
        if ws is not None:
            if purpose == "layer":
                off = lib().hsmoe_moe_layer_status_offset()
                new[off:off + 4].copy_(ws[off:off + 4])
            _retired_workspaces.append((key, ws))
        ws = new
        _workspaces[key] = ws
    return ws


def scale_kind_of(scale: torch.Tensor) -> tuple[int, torch.Tensor]:
    """E8M0 bytes stay bytes; every other dtype is taken by value as fp32 (as
    `sf.float()` does in fused_moe.py:25)."""
    if scale.dtype == torch.float8_e8m0fnu:
        return SCALE_E8M0, scale.view(torch.uint8)
    if scale.dtype != torch.float32:
        scale = scale.to(torch.float32)
    return SCALE_F32, scale


def fp4_dequant_bf16(packed: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """bf16 [N, K] from packed e2m1 [N, K/2] and per-32-column scales [N, K/32]."""
    dev = require_cuda(packed, scale)
    if packed.dtype not in (torch.int8, torch.uint8):
        raise TypeError(f"packed FP4 must be int8/uint8, got {packed.dtype}")
    if packed.dim() != 2:
        raise ValueError("packed FP4 must be 2-D [N, K/2]")
    n, kh = packed.shape
    k = kh * 2
    kind, sc = scale_kind_of(scale)
    if sc.numel() == 1:
        sc = sc.reshape(1, 1).expand(n, k // 32)
    if tuple(sc.shape) != (n, k // 32):
        raise ValueError(f"scale shape {tuple(scale.shape)} does not match [{n}, {k // 32}]")
    packed = packed.contiguous()
    sc = sc.contiguous()
    out = torch.empty(n, k, dtype=torch.bfloat16, device=dev)
    rc = lib().hsmoe_fp4_dequant_bf16(ptr(packed), ptr(sc), kind, n, k, kh, k // 32, ptr(out), k, stream_ptr(dev))
    check(rc, "hsmoe_fp4_dequant_bf16")
    return out


def fp8_dequant_bf16(data: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """bf16 [N, K] from e4m3 [N, K] and fp32 (or E8M0) 128x128 block scales."""
    dev = require_cuda(data, scale)
    if data.dtype not in (torch.float8_e4m3fn, torch.uint8, torch.int8):
        raise TypeError(f"FP8 weight must be float8_e4m3fn, got {data.dtype}")
    n, k = data.shape
    if scale.dtype == torch.float8_e8m0fnu or scale.element_size() == 1:
        # _ue8m0_to_f32 (weight_loader.py:14-19): bits = e << 23
        scale = (scale.view(torch.uint8).to(torch.int32) << 23).view(torch.float32)
    scale = scale.to(torch.float32).contiguous()
    if tuple(scale.shape) != ((n + 127) // 128, (k + 127) // 128):
        raise ValueError(f"block scale shape {tuple(scale.shape)} does not match {n}x{k} / 128")
    data = data.contiguous().view(torch.uint8)
    out = torch.empty(n, k, dtype=torch.bfloat16, device=dev)
    check(lib().hsmoe_fp8_dequant_bf16(ptr(data), ptr(scale), n, k, ptr(out), stream_ptr(dev)),
          "hsmoe_fp8_dequant_bf16")
    return out


def dequant_blocked(data: torch.Tensor, scale: torch.Tensor, block: tuple[int, int],
                    out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """[N, K] fp32 or bf16 from FP4 (int8/uint8 packed [N, K/2]) or e4m3 ([N, K])
    data with fp32 scales, one per (block[0] x block[1]) block (hsmoe_dequant_blocked)."""
    dev = require_cuda(data, scale)
    if data.dim() != 2:
        raise ValueError("dequant_blocked takes 2-D data")
    if data.dtype in (torch.int8, torch.uint8):
        kind, k = _lib.DATA_FP4, data.shape[1] * 2
    elif data.dtype == torch.float8_e4m3fn:
        kind, k = _lib.DATA_E4M3, data.shape[1]
    else:
        raise TypeError(f"dequant_blocked takes packed FP4 (int8) or float8_e4m3fn data, got {data.dtype}")
    if out_dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("dequant_blocked writes fp32 or bf16")
    br, bc = int(block[0]), int(block[1])
    n = data.shape[0]
    scale = scale.to(torch.float32)
    if scale.dim() != 2 or br < 1 or bc < 1 or scale.shape[0] * br < n or scale.shape[1] * bc < k:
        raise ValueError(f"scale {tuple(scale.shape)} with block {tuple(block)} does not cover [{n}, {k}]")
    scale = scale.contiguous()
    data = data.contiguous().view(torch.uint8)
    out = torch.empty(n, k, dtype=out_dtype, device=dev)
    check(lib().hsmoe_dequant_blocked(ptr(data), kind, ptr(scale), n, k, br, bc, scale.shape[1], ptr(out),
                                      _lib.OUT_F32 if out_dtype == torch.float32 else _lib.OUT_BF16,
                                      stream_ptr(dev)), "hsmoe_dequant_blocked")
    return out


def router_topk(x: torch.Tensor, gate_w: torch.Tensor, bias: torch.Tensor | None, top_k: int = 6,
                scaling: float = 1.5, want_logits: bool = False, out: tuple | None = None):
    """(idx int64 [M, k], w fp32 [M, k][, logits bf16 [M, E]]) -- see hsmoe_router_topk.
    `out` = (idx, w) preallocated outputs to fill."""
    dev = require_cuda(x, gate_w, bias)
    x = x.to(torch.bfloat16).contiguous()
    gate_w = gate_w.to(torch.bfloat16).contiguous()
    m, d = x.shape
    e = gate_w.shape[0]
    if gate_w.shape[1] != d:
        raise ValueError(f"gate weight {tuple(gate_w.shape)} does not match hidden size {d}")
    if bias is not None:
        bias = bias.to(torch.float32).contiguous()
    if out is not None:
        idx, w = out
        if idx.shape != (m, top_k) or w.shape != (m, top_k) or idx.dtype != torch.int64 or w.dtype != torch.float32:
            raise ValueError("router_topk out tensors must be int64 / fp32 [M, top_k]")
    else:
        idx = torch.empty(m, top_k, dtype=torch.int64, device=dev)
        w = torch.empty(m, top_k, dtype=torch.float32, device=dev)
    logits = torch.empty(m, e, dtype=torch.bfloat16, device=dev) if want_logits else None
    nbytes = lib().hsmoe_router_workspace_size(m, e)
    ws = _workspace(dev, "router", nbytes)
    rc = lib().hsmoe_router_topk(ptr(x), ptr(gate_w), ptr(bias), m, d, e, top_k, scaling, ptr(idx), ptr(w),
                                 ptr(logits), ptr(ws), ws.numel(), stream_ptr(dev))
    check(rc, "hsmoe_router_topk")
    return (idx, w, logits) if want_logits else (idx, w)


def _capturing(device: torch.device) -> bool:
    """Whether the stream that copies to `device`, current or not, is being captured."""
    if device.index is None or device.index == torch.cuda.current_device():
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def expert_table(entries: list, device: torch.device, wait: bool = True) -> torch.Tensor:
    """uint64 [n][6] device table from per-expert tuples.

    An entry is None (absent expert), a 6-tuple (w1, s1, w3, s3, w2, s2) of FP4
    tensors, or a 3-tuple (w1, w3, w2) of bf16 tensors.
    The table is on the device when this returns, for kernels on any stream;
    with wait=False it is there for what the current stream runs next only."""
    flat = array.array("q")
    for ent in entries:
        if ent is None:
            flat.extend((0, 0, 0, 0, 0, 0))
        elif len(ent) == 6:
            flat.extend([t.data_ptr() for t in ent])
        elif len(ent) == 3:
            w1, w3, w2 = ent
            flat.extend((w1.data_ptr(), 0, w3.data_ptr(), 0, w2.data_ptr(), 0))
        else:
            raise ValueError(f"expert entry of length {len(ent)}")
    if not flat:
        return torch.empty(0, dtype=torch.int64, device=device)
    rows = torch.frombuffer(flat, dtype=torch.int64).reshape(-1, 6)
    # The copy of a pageable tensor waits for the whole stream.  Without that
    # wait: through pinned memory (torch's cached host allocator keeps it until
    # the copy is done).  A graph would read the host memory again when others
    # own it: refused under capture.
    device = torch.device(device)
    if device.type == "cuda":
        if _capturing(device):
            raise RuntimeError("an expert table is made from host memory: not under graph capture")
        if not wait:
            return rows.pin_memory().to(device, non_blocking=True)
    return rows.to(device)


def shared_entry(w1, s1, w3, s3, w2, s2, device: torch.device) -> torch.Tensor:
    """uint64 [6] device entry of the shared expert (e4m3 + fp32 block scales,
    or bf16 weights with s1 = s3 = s2 = None)."""
    vals = [t.data_ptr() if t is not None else 0 for t in (w1, s1, w3, s3, w2, s2)]
    return torch.tensor(vals, dtype=torch.int64).to(device)


def moe_decode(x: torch.Tensor, topk_idx: torch.Tensor, topk_w: torch.Tensor, table: torch.Tensor,
               scale_kind: int, shared: torch.Tensor | None = None, swiglu_limit: float = 10.0,
               out_bf16: torch.Tensor | None = None, out_f32: torch.Tensor | None = None,
               d: int | None = None, i: int | None = None):
    """Routed (+ shared) SwiGLU FFN for M <= 8 tokens; returns (out_bf16, out_f32)."""
    dev = require_cuda(x, topk_idx, topk_w, table, shared)
    if x.dtype != torch.bfloat16:
        raise TypeError(f"hidden states must be bf16, got {x.dtype}")
    x = x.contiguous()
    m, dd = x.shape
    d = dd if d is None else d
    if i is None:
        raise ValueError("intermediate size i is required")
    if m > MAX_DECODE_TOKENS:
        raise ValueError(f"moe_decode handles at most {MAX_DECODE_TOKENS} tokens, got {m}")
    topk_idx = topk_idx.to(torch.int64).contiguous()
    topk_w = topk_w.to(torch.float32).contiguous()
    k = topk_idx.shape[1]
    if out_bf16 is None:
        out_bf16 = torch.empty(m, d, dtype=torch.bfloat16, device=dev)
    nbytes = lib().hsmoe_moe_decode_workspace_size(m, d, i, k)
    ws = _workspace(dev, "decode", nbytes)
    rc = lib().hsmoe_moe_decode(ptr(x), m, d, i, ptr(topk_idx), ptr(topk_w), k, ptr(table), table.shape[0],
                                scale_kind, ptr(shared), swiglu_limit, ptr(out_f32), ptr(out_bf16), ptr(ws),
                                ws.numel(), stream_ptr(dev))
    check(rc, "hsmoe_moe_decode")
    return out_bf16, out_f32


MAX_PREFILL_PAIRS = 12288  # m * top_k per hsmoe_moe_prefill call


def moe_prefill(x: torch.Tensor, topk_idx: torch.Tensor, topk_w: torch.Tensor, table: torch.Tensor,
                scale_kind: int, shared: torch.Tensor | None = None, swiglu_limit: float = 10.0,
                out_bf16: torch.Tensor | None = None, out_f32: torch.Tensor | None = None, i: int | None = None):
    """Routed (+ shared) SwiGLU FFN for any number of tokens as a grouped GEMM
    (hsmoe_moe_prefill); returns (out_bf16, out_f32).  Token blocks of at most
    MAX_PREFILL_PAIRS // top_k rows go to one call each."""
    dev = require_cuda(x, topk_idx, topk_w, table, shared)
    if x.dtype != torch.bfloat16:
        raise TypeError(f"hidden states must be bf16, got {x.dtype}")
    if i is None:
        raise ValueError("intermediate size i is required")
    x = x.contiguous()
    m, d = x.shape
    topk_idx = topk_idx.to(torch.int64).reshape(m, -1).contiguous()
    topk_w = topk_w.to(torch.float32).reshape(m, -1).contiguous()
    k = topk_idx.shape[1]
    if out_bf16 is None:
        out_bf16 = torch.empty(m, d, dtype=torch.bfloat16, device=dev)
    step = max(1, MAX_PREFILL_PAIRS // k)
    for a in range(0, m, step):
        b = min(m, a + step)
        nbytes = lib().hsmoe_moe_prefill_workspace_size(b - a, d, i, table.shape[0], k)
        ws = _workspace(dev, "prefill", nbytes)
        rc = lib().hsmoe_moe_prefill(ptr(x[a:b]), b - a, d, i, ptr(topk_idx[a:b]), ptr(topk_w[a:b]), k, ptr(table),
                                     table.shape[0], scale_kind, ptr(shared), swiglu_limit,
                                     None if out_f32 is None else ptr(out_f32[a:b]), ptr(out_bf16[a:b]), ptr(ws),
                                     ws.numel(), stream_ptr(dev))
        check(rc, "hsmoe_moe_prefill")
    return out_bf16, out_f32


_ROW_KINDS = {torch.bfloat16: _lib.OUT_BF16, torch.float32: _lib.OUT_F32}
_NO_GUARD = contextlib.nullcontext()


def _on(dev: torch.device):
    """Makes dev the current device around a launch (its stream belongs to it)."""
    return _NO_GUARD if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)


def _row_kind(dtype: torch.dtype, what: str) -> int:
    kind = _ROW_KINDS.get(dtype)
    if kind is None:
        raise TypeError(f"{what} must be bf16 or fp32, got {dtype}")
    return kind


class ExpertOrder(NamedTuple):
    """(token, slot) pairs in the order of their experts (moe_sort), int32 device tensors.
    Pair q = t * top_k + j is token t's slot j."""
    offsets: torch.Tensor  # [E + 1]: expert e has rows offsets[e] .. offsets[e + 1] - 1
    pairs: torch.Tensor    # [M * top_k]: the pair of each row, -1 from row offsets[E] on
    rows: torch.Tensor     # [M, top_k]: the row of each pair, -1 for a dropped one

    @property
    def n_experts(self) -> int:
        return self.offsets.numel() - 1

    def check(self) -> tuple[int, int]:
        """(tokens, top_k) of a well-formed order."""
        off, pairs, rows = self
        for t in self:
            if t.dtype != torch.int32 or not t.is_contiguous():
                raise TypeError("an expert order holds contiguous int32 tensors")
        if rows.dim() != 2 or pairs.numel() != rows.numel() or off.dim() != 1 or off.numel() < 2:
            raise ValueError("an expert order is offsets [E + 1], pairs [M * top_k], rows [M, top_k]")
        return rows.shape


def moe_sort(topk_idx: torch.Tensor, n_experts: int) -> ExpertOrder:
    """The (token, slot) pairs of topk_idx [M, k] sorted by expert, stably; ids < 0
    or >= n_experts are dropped (hsmoe_moe_sort)."""
    dev = require_cuda(topk_idx)
    if topk_idx.dim() != 2:
        raise ValueError("topk_idx must be [M, top_k]")
    if topk_idx.is_floating_point() or topk_idx.dtype == torch.bool:
        raise TypeError(f"topk_idx must hold integers, got {topk_idx.dtype}")
    topk_idx = topk_idx.to(torch.int64).contiguous()
    m, k = topk_idx.shape
    offsets = torch.empty(max(n_experts, 0) + 1, dtype=torch.int32, device=dev)
    pairs = torch.empty(m * k, dtype=torch.int32, device=dev)
    rows = torch.empty(m, k, dtype=torch.int32, device=dev)
    # a workspace of the call's own: calls of two captured graphs may run at once
    nbytes = lib().hsmoe_moe_sort_workspace_size(m, k, n_experts)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    with _on(dev):
        check(lib().hsmoe_moe_sort(ptr(topk_idx), m, k, n_experts, ptr(offsets), ptr(pairs), ptr(rows), ptr(ws), nbytes,
                                   stream_ptr(dev)), "hsmoe_moe_sort")
    return ExpertOrder(offsets, pairs, rows)


def moe_gather(x: torch.Tensor, order: ExpertOrder) -> torch.Tensor:
    """[M * k, D] rows of x [M, D] (bf16 or fp32) in the order's sequence; the rows
    behind the last sorted one are zeros (hsmoe_moe_gather).  Its gradient is
    moe_combine(d_rows, order)."""
    dev = require_cuda(x, *order)
    m, k = order.check()
    kind = _row_kind(x.dtype, "rows")
    if x.dim() != 2 or x.shape[0] != m:
        raise ValueError(f"x {tuple(x.shape)} does not have the order's {m} tokens")
    d = x.shape[1]
    if x.stride(1) != 1 or x.stride(0) < d:
        x = x.contiguous()
    out = torch.empty(m * k, d, dtype=x.dtype, device=dev)
    with _on(dev):
        check(lib().hsmoe_moe_gather(ptr(x), max(x.stride(0), d), m, d, kind, ptr(order.offsets), order.n_experts,
                                     ptr(order.rows), k, ptr(out), stream_ptr(dev)), "hsmoe_moe_gather")
    return out


def moe_combine(rows: torch.Tensor, order: ExpertOrder, topk_w: torch.Tensor | None = None,
                residual: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """[M, D]: every token's rows summed with its weights topk_w [M, k] (1 when
    None) in fp32, in slot order, plus residual [M, D] (hsmoe_moe_combine); bf16 or
    fp32 as out_dtype, the residual or the rows say."""
    dev = require_cuda(rows, topk_w, residual, *order)
    m, k = order.check()
    kind = _row_kind(rows.dtype, "rows")
    if out_dtype is None:
        out_dtype = rows.dtype if residual is None else residual.dtype
    out_kind = _row_kind(out_dtype, "the output")
    if rows.dim() != 2 or rows.shape[0] != m * k:
        raise ValueError(f"rows {tuple(rows.shape)} do not match the order's {m} x {k} pairs")
    d = rows.shape[1]
    rows = rows.contiguous()
    if topk_w is not None:
        if topk_w.shape != order.rows.shape:
            raise ValueError(f"weights {tuple(topk_w.shape)} do not match the order's [{m}, {k}]")
        topk_w = topk_w.to(torch.float32).contiguous()
    if residual is not None:
        if residual.shape != (m, d) or residual.dtype != out_dtype:
            raise ValueError(f"the residual must be [{m}, {d}] of the output's dtype")
        residual = residual.contiguous()
    out = torch.empty(m, d, dtype=out_dtype, device=dev)
    with _on(dev):
        check(lib().hsmoe_moe_combine(ptr(rows), kind, m * k, m, d, ptr(order.rows), ptr(topk_w), k, ptr(residual),
                                      out_kind, ptr(out), stream_ptr(dev)), "hsmoe_moe_combine")
    return out


def moe_combine_grad(d_out: torch.Tensor, rows: torch.Tensor, order: ExpertOrder, topk_w: torch.Tensor | None = None,
                     need_rows: bool = True, need_w: bool = True):
    """The gradient of moe_combine for d_out [M, D]: (d_rows like rows, those behind
    the last sorted one zeros; d_w fp32 [M, k], 0 where a pair is dropped), None
    where not needed (hsmoe_moe_combine_grad).  The residual's is d_out."""
    dev = require_cuda(d_out, rows, topk_w, *order)
    m, k = order.check()
    kind, out_kind = _row_kind(rows.dtype, "rows"), _row_kind(d_out.dtype, "d_out")
    if rows.dim() != 2 or rows.shape[0] != m * k or d_out.shape != (m, rows.shape[1]):
        raise ValueError(f"rows {tuple(rows.shape)} and d_out {tuple(d_out.shape)} do not match the order's {m} x {k} pairs")
    d_out, rows = d_out.contiguous(), rows.contiguous()
    if topk_w is not None:
        if topk_w.shape != order.rows.shape:
            raise ValueError(f"weights {tuple(topk_w.shape)} do not match the order's [{m}, {k}]")
        topk_w = topk_w.to(torch.float32).contiguous()
    d_rows = torch.empty_like(rows) if need_rows else None
    d_w = torch.empty(m, k, dtype=torch.float32, device=dev) if need_w else None
    with _on(dev):
        check(lib().hsmoe_moe_combine_grad(ptr(d_out), out_kind, ptr(rows), kind, m, rows.shape[1], ptr(order.offsets),
                                           order.n_experts, ptr(order.rows), ptr(topk_w), k, ptr(d_rows), ptr(d_w),
                                           stream_ptr(dev)), "hsmoe_moe_combine_grad")
    return d_rows, d_w


_ACTS = {None: _lib.ACT_NONE, "silu": _lib.ACT_SILU, "swiglu": _lib.ACT_SWIGLU}


def _act(act: str | None, limit: float | None, w_up: torch.Tensor | None) -> tuple[int, float]:
    if act not in _ACTS:
        raise ValueError(f"activation must be None, 'silu' or 'swiglu', got {act!r}")
    if (act == "swiglu") != (w_up is not None):
        raise ValueError("an up weight (w_up) goes with act='swiglu', and only with it")
    if limit is not None and act != "swiglu":
        raise ValueError("a limit goes with act='swiglu'")
    limit = float("inf") if limit is None else float(limit)
    if not limit > 0:
        raise ValueError("the limit must be positive")
    return _ACTS[act], limit


def _bf16_matrix(t: torch.Tensor, what: str) -> torch.Tensor:
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{what} must be bf16, got {t.dtype}")
    return t


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """t, or a contiguous copy where its rows are not 16-byte aligned ones of consecutive elements."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t  # (a row that is no multiple of 8 values is refused below)
    if t.stride(-1) != 1 or t.data_ptr() % 16 or any(s % 8 or s < 0 for s in t.stride()[:-1]):
        return t.contiguous() if not t.is_contiguous() else t.clone()
    if t.dim() > 1 and t.shape[-2] > 1 and t.stride(-2) < t.shape[-1]:
        return t.contiguous()
    return t


def _row_stride(t: torch.Tensor) -> int:
    return max(t.stride(-2), t.shape[-1]) if t.shape[-2] > 1 else t.shape[-1]


def _weights(w: torch.Tensor, w_up: torch.Tensor | None, order: ExpertOrder | None):
    """(w, w_up, row stride, group stride) of weights [N, K] or, with an order, [E, N, K]."""
    dims = 2 if order is None else 3
    for t in (w, w_up):
        if t is not None and (t.dim() != dims or t.shape != w.shape):
            raise ValueError(f"weights must be {'[N, K]' if order is None else '[E, N, K]'} tensors of one shape, got "
                             f"{tuple(t.shape)}")
    if order is not None and w.shape[0] != order.n_experts:
        raise ValueError(f"{w.shape[0]} weight matrices for an order of {order.n_experts} experts")
    w = _rows16(_bf16_matrix(w, "weights"))
    if w_up is not None:
        w_up = _rows16(_bf16_matrix(w_up, "weights"))
        if w_up.stride() != w.stride():
            w, w_up = w.contiguous(), w_up.contiguous()
    return w, w_up, _row_stride(w), (w.stride(0) if order is not None else 0)


def _bias(b: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    if b.shape != w.shape[:-1]:
        raise ValueError(f"bias {tuple(b.shape)} does not match weights {tuple(w.shape)}")
    b = _bf16_matrix(b, "bias").contiguous()
    return b if b.data_ptr() % 16 == 0 else b.clone()


def _linear_rows(x: torch.Tensor, what: str, cols: int, order: ExpertOrder | None) -> torch.Tensor:
    """x as rows [M, cols] that the kernels can read."""
    _bf16_matrix(x, what)
    if x.dim() < 1 or x.shape[-1] != cols:
        raise ValueError(f"{what} {tuple(x.shape)} does not have rows of {cols}")
    if order is not None and (x.dim() != 2 or x.shape[0] != order.pairs.numel()):
        raise ValueError(f"{what} {tuple(x.shape)} does not have the order's {order.pairs.numel()} rows")
    return _rows16(x if x.dim() == 2 else x.reshape(-1, cols))


def linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, residual: torch.Tensor | None = None,
           act: str | None = None, w_up: torch.Tensor | None = None, bias_up: torch.Tensor | None = None,
           limit: float | None = None, order: ExpertOrder | None = None, out_dtype: torch.dtype = torch.bfloat16,
           want_pre: bool = False):
    """act(x w^T + bias) + residual for bf16 tensors (hsmoe_linear): x [..., K],
    w [N, K], bias [N], residual [..., N] -> [..., N] bf16 or fp32.

    act: None, "silu", or "swiglu" = silu(min(g, limit)) * clamp(u, -limit, limit)
    with g from w, bias and u from w_up, bias_up.  With `order` (moe_sort) x and
    the result are its sorted rows [M * k, .], w is [E, N, K] and bias [E, N], and
    a row goes through its expert's; the rows behind the last sorted one are zeros.
    want_pre: -> (result, pre), pre the bf16 sums (with bias) before the
    activation, [..., N] or [..., 2 N] (gate, up), for linear_grad.
    N and K must be multiples of 8."""
    dev = require_cuda(x, w, w_up, bias, bias_up, residual, *(order or ()))
    code, limit = _act(act, limit, w_up)
    if order is not None:
        order.check()
    w, w_up, ldw, group = _weights(w, w_up, order)
    n, k = w.shape[-2:]
    lead = x.shape[:-1]
    x = _linear_rows(x, "x", k, order)
    m = x.shape[0]
    if bias_up is not None and act != "swiglu":
        raise ValueError("an up bias goes with act='swiglu'")
    if bias is not None:
        bias = _bias(bias, w)
    if bias_up is not None:
        bias_up = _bias(bias_up, w)
    ld_res = n
    if residual is not None:
        if residual.shape != lead + (n,):
            raise ValueError(f"residual {tuple(residual.shape)} does not match the result's {tuple(lead) + (n,)}")
        residual = _linear_rows(residual, "residual", n, None)
        ld_res = _row_stride(residual)
    kind = _row_kind(out_dtype, "the output")
    out = torch.empty((m, n) if len(lead) == 1 else lead + (n,), dtype=out_dtype, device=dev)
    pre = torch.empty(lead + (2 * n if act == "swiglu" else n,), dtype=torch.bfloat16, device=dev) if want_pre else None
    with _on(dev):
        nbytes = lib().hsmoe_linear_workspace_size(m, n, k, 1 if order is None else order.n_experts, code)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None  # the call's own, as in moe_sort
        check(lib().hsmoe_linear(ptr(x), _row_stride(x), m, k, ptr(w), ptr(w_up), ldw, group, n,
                                 None if order is None else ptr(order.offsets),
                                 1 if order is None else order.n_experts, ptr(bias), ptr(bias_up), ptr(residual),
                                 ld_res, code, limit, kind, ptr(out), ptr(pre), ptr(ws), nbytes, stream_ptr(dev)),
              "hsmoe_linear")
    return (out, pre) if want_pre else out


class LinearGrad(NamedTuple):
    """The gradient of linear; None where not needed."""
    x: torch.Tensor | None
    w: torch.Tensor | None
    bias: torch.Tensor | None
    w_up: torch.Tensor | None
    bias_up: torch.Tensor | None


def linear_grad(d_out: torch.Tensor, x: torch.Tensor, w: torch.Tensor, act: str | None = None,
                pre: torch.Tensor | None = None, w_up: torch.Tensor | None = None, limit: float | None = None,
                order: ExpertOrder | None = None, need_x: bool = True, need_w: bool = True, need_bias: bool = False,
                w_dtype: torch.dtype = torch.bfloat16) -> LinearGrad:
    """The gradient of linear(x, w, ...) for d_out [..., N] (bf16): x in bf16, the
    weights in w_dtype (bf16 or fp32), the biases in fp32; the residual's is d_out.
    pre: what linear(want_pre=True) returned (not needed without an activation).
    Behind an activation d_out y'(pre) goes to the products rounded to bf16, half a
    step (2^-8) of each term; the biases' gradients are summed before that.  What the
    limit cuts off is decided on pre: a sum beyond the limit that rounds onto it (up
    to 10.03 at limit 10) has a gradient though linear cut it.
    With `order`, an expert without rows has gradient zero, and so have the rows
    behind the last sorted one (hsmoe_linear_act_grad, _grad_input, _grad_weight)."""
    dev = require_cuda(d_out, x, w, w_up, pre, *(order or ()))
    code, limit = _act(act, limit, w_up)
    if order is not None:
        order.check()
    w, w_up, ldw, group = _weights(w, w_up, order)
    n, k = w.shape[-2:]
    lead = x.shape[:-1]
    if d_out.shape != lead + (n,):
        raise ValueError(f"d_out {tuple(d_out.shape)} does not match the result's {tuple(lead) + (n,)}")
    x = _linear_rows(x, "x", k, order)
    d_out = _linear_rows(d_out, "d_out", n, order)
    m = x.shape[0]
    mats = 2 if act == "swiglu" else 1
    kind = _row_kind(w_dtype, "the weights' gradient")
    off = None if order is None else ptr(order.offsets)
    groups = 1 if order is None else order.n_experts
    if act is not None:
        if pre is None:
            raise ValueError("the gradient of an activation needs pre (linear(..., want_pre=True))")
        if pre.shape != lead + (mats * n,):
            raise ValueError(f"pre {tuple(pre.shape)} must be {tuple(lead) + (mats * n,)}")
        pre = _linear_rows(pre, "pre", mats * n, None).contiguous()
    need_dz = act is not None and (need_x or need_w)
    dz = torch.empty(m, mats * n, dtype=torch.bfloat16, device=dev) if need_dz else d_out
    db = [None, None]
    dx = None
    dw = [None, None]
    with _on(dev):
        if need_bias or need_dz:
            nbytes = lib().hsmoe_linear_act_grad_workspace_size(m, n, groups, code) if need_bias else 0
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None  # the call's own, as in moe_sort
            if need_bias:
                db[:mats] = [torch.empty(w.shape[:-1], dtype=torch.float32, device=dev) for _ in range(mats)]
            check(lib().hsmoe_linear_act_grad(ptr(d_out), _row_stride(d_out), ptr(pre) if act else None, m, n, code, limit,
                                              off, groups, ptr(dz) if need_dz else None, ptr(db[0]), ptr(db[1]), ptr(ws),
                                              nbytes, stream_ptr(dev)), "hsmoe_linear_act_grad")
        nbytes = lib().hsmoe_linear_grad_workspace_size(m, n, k, groups, code) if need_x or need_w else 0
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None  # one product after the other
        if need_x:
            dx = torch.empty(lead + (k,), dtype=torch.bfloat16, device=dev)
            check(lib().hsmoe_linear_grad_input(ptr(dz), _row_stride(dz), m, n, ptr(w), ptr(w_up), ldw, group, k, off,
                                                groups, ptr(dx), ptr(ws), nbytes, stream_ptr(dev)),
                  "hsmoe_linear_grad_input")
        if need_w:
            dw[:mats] = [torch.empty(w.shape, dtype=w_dtype, device=dev) for _ in range(mats)]
            check(lib().hsmoe_linear_grad_weight(ptr(dz), _row_stride(dz), ptr(x), _row_stride(x), m, n, k, off, groups,
                                                 kind, ptr(dw[0]), ptr(dw[1]), ptr(ws), nbytes, stream_ptr(dev)),
                  "hsmoe_linear_grad_weight")
    return LinearGrad(dx, dw[0], db[0], dw[1], db[1])


def moe_decode_stage(stage: int, x: torch.Tensor, topk_idx: torch.Tensor, topk_w: torch.Tensor,
                     table: torch.Tensor, scale_kind: int, shared: torch.Tensor | None, swiglu_limit: float,
                     d: int, i: int, out_bf16: torch.Tensor | None = None, out_f32: torch.Tensor | None = None):
    """Launches stage 1 (gate/up) or stage 2 (down) of moe_decode alone; inputs
    must already be contiguous bf16 / int64 / fp32 device tensors."""
    dev = x.device
    m = x.shape[0]
    k = topk_idx.shape[1]
    ws = _workspace(dev, "decode", lib().hsmoe_moe_decode_workspace_size(m, d, i, k))
    if stage == 1:
        rc = lib().hsmoe_moe_gate_up(ptr(x), m, d, i, ptr(topk_idx), ptr(topk_w), k, ptr(table), table.shape[0],
                                     scale_kind, ptr(shared), swiglu_limit, ptr(ws), ws.numel(), stream_ptr(dev))
    else:
        rc = lib().hsmoe_moe_down(ptr(x), m, d, i, ptr(topk_idx), ptr(topk_w), k, ptr(table), table.shape[0],
                                  scale_kind, ptr(shared), ptr(out_f32), ptr(out_bf16), ptr(ws), ws.numel(),
                                  stream_ptr(dev))
    check(rc, f"moe_decode stage {stage}")


class NormTail:
    """The next layer's residual adds and RMSNorm, done at the end of a layer
    launch (the _norm entry points): with out = the layer's output in bf16,
    h_out = bf16(bf16(h + out) + residual) and norm_out = RMSNorm(h_out) *
    weight, bit-identical to add_rms_norm(h, weight, add=out, residual=...).
    h [M, D] bf16; residual [D] or None; weight [D]; the outputs are
    allocated when not given (h_out may be h)."""

    def __init__(self, h: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None,
                 eps: float = 1e-6, h_out: torch.Tensor | None = None, norm_out: torch.Tensor | None = None):
        require_cuda(h, weight, residual, h_out, norm_out)
        if h.dtype != torch.bfloat16 or h.dim() != 2 or not h.is_contiguous():
            raise ValueError("norm tail h must be a contiguous bf16 [M, D] tensor")
        d = h.shape[1]
        self.h = h
        self.weight = weight.to(torch.bfloat16).reshape(-1).contiguous()
        self.residual = None if residual is None else residual.to(torch.bfloat16).reshape(-1).contiguous()
        if self.weight.numel() != d or (self.residual is not None and self.residual.numel() != d):
            raise ValueError("norm tail weight and residual must be one row of the hidden size")
        self.eps = float(eps)
        self.h_out = torch.empty_like(h) if h_out is None else h_out
        self.norm_out = torch.empty_like(h) if norm_out is None else norm_out
        for t in (self.h_out, self.norm_out):
            if t.shape != h.shape or t.dtype != torch.bfloat16 or not t.is_contiguous():
                raise ValueError("norm tail outputs must be contiguous bf16 tensors shaped like h")

    def struct(self, x: torch.Tensor) -> "_lib.NormTail":
        if tuple(self.h.shape) != tuple(x.shape):
            raise ValueError(f"norm tail rows {tuple(self.h.shape)} do not match the layer's {tuple(x.shape)}")
        return _lib.NormTail(ptr(self.h), ptr(self.residual), ptr(self.weight), self.eps, ptr(self.h_out),
                             ptr(self.norm_out))


def moe_layer_decode(x: torch.Tensor, gate_w: torch.Tensor, gate_bias: torch.Tensor | None, table: torch.Tensor,
                     scale_kind: int, shared: torch.Tensor | None, i: int, top_k: int = 6, scaling: float = 1.5,
                     swiglu_limit: float = 10.0, out_bf16: torch.Tensor | None = None,
                     out_f32: torch.Tensor | None = None, idx_out: torch.Tensor | None = None,
                     w_out: torch.Tensor | None = None, want_logits: bool = False, norm: NormTail | None = None):
    """Router + routed experts + shared expert of one layer for M <= 8 tokens in
    one launch; returns (out_bf16, out_f32, idx, w[, logits]).  With `norm`
    the launch ends with its norm tail (norm.h_out, norm.norm_out receive
    it) and no output is allocated unless asked for.

    Same results as router_topk followed by moe_decode.  Inputs must already be
    contiguous device tensors of the right dtypes when called inside a graph
    capture (no conversions are enqueued then)."""
    dev = require_cuda(x, gate_w, gate_bias, table, shared)
    if x.dtype != torch.bfloat16 or gate_w.dtype != torch.bfloat16:
        raise TypeError("hidden states and gate weight must be bf16")
    x = x.contiguous()
    gate_w = gate_w.contiguous()
    m, d = x.shape
    n_exp = gate_w.shape[0]
    if gate_w.shape[1] != d:
        raise ValueError(f"gate weight {tuple(gate_w.shape)} does not match hidden size {d}")
    if m > MAX_DECODE_TOKENS:
        raise ValueError(f"moe_layer_decode handles at most {MAX_DECODE_TOKENS} tokens, got {m}")
    if gate_bias is not None:
        gate_bias = gate_bias.to(torch.float32).contiguous()
    if idx_out is None:
        idx_out = torch.empty(m, top_k, dtype=torch.int64, device=dev)
    if w_out is None:
        w_out = torch.empty(m, top_k, dtype=torch.float32, device=dev)
    if tuple(idx_out.shape) != (m, top_k) or tuple(w_out.shape) != (m, top_k):
        raise ValueError("idx_out / w_out must be [M, top_k]")
    if out_bf16 is None and out_f32 is None and norm is None:
        out_bf16 = torch.empty(m, d, dtype=torch.bfloat16, device=dev)
    logits = torch.empty(m, n_exp, dtype=torch.bfloat16, device=dev) if want_logits else None
    nbytes = lib().hsmoe_moe_layer_workspace_size(m, d, i, n_exp, top_k)
    ws = _workspace(dev, "layer", nbytes)
    args = (ptr(x), m, d, i, ptr(gate_w), ptr(gate_bias), n_exp, top_k, scaling, ptr(table), scale_kind, ptr(shared),
            swiglu_limit, ptr(idx_out), ptr(w_out), ptr(logits), ptr(out_f32), ptr(out_bf16))
    if norm is None:
        rc = lib().hsmoe_moe_layer_decode(*args, ptr(ws), ws.numel(), stream_ptr(dev))
        check(rc, "hsmoe_moe_layer_decode")
    else:
        tail = norm.struct(x)
        rc = lib().hsmoe_moe_layer_decode_norm(*args, ctypes.addressof(tail), ptr(ws), ws.numel(), stream_ptr(dev))
        check(rc, "hsmoe_moe_layer_decode_norm")
    res = (out_bf16, out_f32, idx_out, w_out)
    return res + (logits,) if want_logits else res


def moe_layer_decode_routed(x: torch.Tensor, topk_idx: torch.Tensor, table: torch.Tensor, scale_kind: int,
                            shared: torch.Tensor | None, i: int, topk_w: torch.Tensor | None = None,
                            weight_all: float = 1.0, token_ids: torch.Tensor | None = None, top_k: int | None = None,
                            swiglu_limit: float = 10.0, out_bf16: torch.Tensor | None = None,
                            out_f32: torch.Tensor | None = None, norm: NormTail | None = None):
    """Routed + shared experts of M <= 8 tokens in one launch with the routing
    given (hsmoe_moe_layer_decode_routed); returns (out_bf16, out_f32).  With
    `norm` the launch ends with its norm tail, as in moe_layer_decode.

    token_ids None: topk_idx [M, k] are the ids.  Otherwise topk_idx is a
    token table [V, k] (a hash layer's tid2eid) and token t's ids are row
    token_ids[t].  topk_w [M, k] or None (every weight weight_all).  Same
    results as moe_decode on the same ids and weights.  Inside a graph capture
    the inputs must already be contiguous device tensors of the right dtypes."""
    dev = require_cuda(x, topk_idx, table, shared, topk_w, token_ids)
    if x.dtype != torch.bfloat16:
        raise TypeError("hidden states must be bf16")
    x = x.contiguous()
    m, d = x.shape
    if m > MAX_DECODE_TOKENS:
        raise ValueError(f"moe_layer_decode_routed handles at most {MAX_DECODE_TOKENS} tokens, got {m}")
    topk_idx = topk_idx.to(torch.int64).contiguous()
    k = topk_idx.shape[-1] if top_k is None else top_k
    rows = 0
    if token_ids is not None:
        token_ids = token_ids.reshape(-1).to(torch.int64).contiguous()
        if token_ids.numel() != m:
            raise ValueError("token_ids must hold one id per token")
        rows = topk_idx.shape[0]
        if topk_idx.dim() != 2 or topk_idx.shape[1] != k:
            raise ValueError("a token table must be [V, top_k]")
    elif topk_idx.numel() != m * k:
        raise ValueError("topk_idx must be [M, top_k]")
    if topk_w is not None:
        topk_w = topk_w.to(torch.float32).contiguous()
        if topk_w.numel() != m * k:
            raise ValueError("topk_w must be [M, top_k]")
    if out_bf16 is None and out_f32 is None and norm is None:
        out_bf16 = torch.empty(m, d, dtype=torch.bfloat16, device=dev)
    n_exp = table.shape[0]
    ws = _workspace(dev, "layer", lib().hsmoe_moe_layer_workspace_size(m, d, i, n_exp, k))
    args = (ptr(x), m, d, i, ptr(topk_idx), ptr(token_ids), rows, ptr(topk_w), float(weight_all), k, ptr(table),
            n_exp, scale_kind, ptr(shared), swiglu_limit, ptr(out_f32), ptr(out_bf16))
    if norm is None:
        rc = lib().hsmoe_moe_layer_decode_routed(*args, ptr(ws), ws.numel(), stream_ptr(dev))
        check(rc, "hsmoe_moe_layer_decode_routed")
    else:
        tail = norm.struct(x)
        rc = lib().hsmoe_moe_layer_decode_routed_norm(*args, ctypes.addressof(tail), ptr(ws), ws.numel(),
                                                      stream_ptr(dev))
        check(rc, "hsmoe_moe_layer_decode_routed_norm")
    return out_bf16, out_f32


def _layer_workspaces(device: torch.device, stream: int | None = None) -> list[torch.Tensor]:
    """The layer workspaces of `stream` (or of every stream) on the device,
    the retired ones included (a graph captured against one still writes it)."""
    return [ws for (d, st, purpose), ws in list(_workspaces.items()) + _retired_workspaces
            if purpose == "layer" and d == device.index and (stream is None or st == stream)]


def moe_layer_status_words(device: torch.device | None = None, stream: int | None = None) -> list[torch.Tensor]:
    """int32 [1] device views of the layer kernel's sticky status word in the
    layer workspaces of `stream` (a raw stream handle), or of every stream of
    the device (a decode graph's capture stream included) when None."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    off = lib().hsmoe_moe_layer_status_offset()
    return [ws[off:off + 4].view(torch.int32) for ws in _layer_workspaces(device, stream)]


def moe_layer_status(device: torch.device | None = None, stream: int | None = None) -> int:
    """The layer kernel's sticky status word: 0 when every cross-workgroup wait
    of every launch completed, else 1 + the code of a wait that gave up (the
    outputs of that launch are not valid).  Reads the workspaces of `stream`,
    or of every stream of the device when None.  Synchronises the device."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    status = 0
    for w in moe_layer_status_words(device, stream):
        status = status or int(w.item())
    return status


def clear_moe_layer_status(device: torch.device | None = None, stream: int | None = None) -> None:
    """Zeroes the sticky status words (of `stream`'s layer workspaces, or of
    every stream of the device), stream-ordered on the current stream, so that
    a reported give-up does not fail every later launch's check."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    for w in moe_layer_status_words(device, stream):
        w.zero_()


def check_moe_layer_status(device: torch.device | None = None, stream: int | None = None) -> None:
    """Raises HsmoeError when moe_layer_status is not 0; the status words are
    cleared first, so the error is reported once."""
    st = moe_layer_status(device, stream)
    if st:
        clear_moe_layer_status(device, stream)
        raise _lib.HsmoeError(f"moe_layer_kernel: a cross-workgroup wait gave up (status {st}); "
                              "the outputs of that launch are not valid")


def lm_head_accept(h: torch.Tensor, lm_head: torch.Tensor, ids: torch.Tensor | None = None,
                   want_logits: bool = True, pred: torch.Tensor | None = None):
    """(logits bf16 [T, V] | None, pred int64 [T], result int64 [2] = (n_accept, bonus_row)).
    pred, if given, is where the argmax goes (contiguous int64 [T], e.g. a
    slice of the next call's id buffer)."""
    dev = require_cuda(h, lm_head, ids, pred)
    h = h.to(torch.bfloat16).contiguous()
    n, d = h.shape
    vocab = lm_head.shape[0]
    if lm_head.dtype != torch.bfloat16 or not lm_head.is_contiguous():
        raise TypeError("lm_head must be a contiguous bf16 [V, D] tensor")
    if ids is not None:
        ids = ids.reshape(-1).to(torch.int64).contiguous()
        if ids.numel() != n:
            raise ValueError("ids must have one entry per hidden row")
    logits = torch.empty(n, vocab, dtype=torch.bfloat16, device=dev) if want_logits else None
    if pred is None:
        pred = torch.empty(n, dtype=torch.int64, device=dev)
    elif pred.dtype != torch.int64 or not pred.is_contiguous() or pred.numel() != n:
        raise ValueError("pred must be a contiguous int64 tensor of one entry per hidden row")
    result = torch.empty(2, dtype=torch.int64, device=dev)
    nbytes = lib().hsmoe_lm_head_workspace_size(n, vocab)
    ws = _workspace(dev, "lm_head", nbytes)
    rc = lib().hsmoe_lm_head_accept(ptr(h), ptr(lm_head), n, d, vocab, ptr(ids), ptr(logits), ptr(pred),
                                    ptr(result), ptr(ws), ws.numel(), stream_ptr(dev))
    check(rc, "hsmoe_lm_head_accept")
    return logits, pred, result


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """bf16 RMSNorm over the last dimension (utils.py:6-9)."""
    return add_rms_norm(x, weight, eps=eps)[1]


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, add: torch.Tensor | None = None,
                 residual: torch.Tensor | None = None, eps: float = 1e-6, want_sum: bool = False):
    """h = x (+ add) (+ residual), as torch bf16 adds; -> (h if want_sum else None, RMSNorm(h)).
    x, add: [..., D] bf16 of one shape; residual: [D] bf16, added to every row."""
    dev = require_cuda(x, weight, add, residual)
    if x.dtype != torch.bfloat16 or (add is not None and add.dtype != torch.bfloat16):
        raise TypeError("add_rms_norm takes bf16 rows")
    shape = x.shape
    d = shape[-1]
    x2 = x.reshape(-1, d).contiguous()
    if add is not None:
        if add.shape != shape:
            raise ValueError(f"add {tuple(add.shape)} does not match x {tuple(shape)}")
        add = add.reshape(-1, d).contiguous()
    if residual is not None:
        residual = residual.to(torch.bfloat16).reshape(-1).contiguous()
        if residual.numel() != d:
            raise ValueError("residual must be one row of the hidden size")
    w = weight.to(torch.bfloat16).reshape(-1).contiguous()
    if w.numel() != d:
        raise ValueError("norm weight must be one row of the hidden size")
    out = torch.empty_like(x2)
    h = torch.empty_like(x2) if want_sum else None
    check(lib().hsmoe_add_rms_norm(ptr(x2), ptr(add), ptr(residual), ptr(w), x2.shape[0], d, eps, ptr(h), ptr(out),
                                   stream_ptr(dev)), "hsmoe_add_rms_norm")
    return (None if h is None else h.reshape(shape)), out.reshape(shape)


def _bf16_row(t: torch.Tensor, d: int, what: str) -> torch.Tensor:
    t = t.to(torch.bfloat16).reshape(-1).contiguous()
    if t.numel() != d:
        raise ValueError(f"{what} must be one row of the hidden size")
    return t


def embed_add_rms_norm(ids: torch.Tensor, table: torch.Tensor, weight: torch.Tensor,
                       residual: torch.Tensor | None = None, eps: float = 1e-6):
    """The embedding lookup table[ids] followed by add_rms_norm(x, weight,
    residual=residual, want_sum=True), in one launch -> (h, RMSNorm(h)), each
    bf16 [*ids.shape, D]; an id outside [0, V) reads a row of zeros."""
    dev = require_cuda(ids, table, weight, residual)
    if table.dtype != torch.bfloat16 or table.dim() != 2 or not table.is_contiguous():
        raise TypeError("the embedding table must be a contiguous bf16 [V, D] tensor")
    vocab, d = table.shape
    ids_flat = ids.reshape(-1).to(torch.int64).contiguous()
    w = _bf16_row(weight, d, "norm weight")
    res = None if residual is None else _bf16_row(residual, d, "residual")
    rows = ids_flat.numel()
    h = torch.empty(rows, d, dtype=torch.bfloat16, device=dev)
    out = torch.empty_like(h)
    check(lib().hsmoe_embed_add_rms_norm(ptr(ids_flat), rows, ptr(table), vocab, ptr(res), ptr(w), d, eps, ptr(h),
                                         ptr(out), stream_ptr(dev)), "hsmoe_embed_add_rms_norm")
    shape = tuple(ids.shape) + (d,)
    return h.reshape(shape), out.reshape(shape)


def mtp_input(tok: torch.Tensor, embed: torch.Tensor, h_prev: torch.Tensor, enorm: torch.Tensor,
              hnorm: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-6):
    """The MTP block's input for one draft token (tok: one int64 on the device):
    h = RMSNorm(h_prev) * hnorm + RMSNorm(embed[tok]) * enorm (+ residual), as
    bf16 adds -> (h [1, D], RMSNorm(h) * weight [1, D]), in one launch."""
    dev = require_cuda(tok, embed, h_prev, enorm, hnorm, weight, residual)
    if embed.dtype != torch.bfloat16 or embed.dim() != 2 or not embed.is_contiguous():
        raise TypeError("the embedding table must be a contiguous bf16 [V, D] tensor")
    vocab, d = embed.shape
    tok = tok.reshape(-1).to(torch.int64).contiguous()
    if tok.numel() != 1:
        raise ValueError("mtp_input takes one token")
    hp = _bf16_row(h_prev, d, "h_prev")
    en, hn, w = (_bf16_row(t, d, "norm weight") for t in (enorm, hnorm, weight))
    res = None if residual is None else _bf16_row(residual, d, "residual")
    h = torch.empty(1, d, dtype=torch.bfloat16, device=dev)
    out = torch.empty_like(h)
    check(lib().hsmoe_mtp_input(ptr(tok), ptr(embed), vocab, ptr(hp), ptr(en), ptr(hn), ptr(res), ptr(w), d, eps,
                                ptr(h), ptr(out), stream_ptr(dev)), "hsmoe_mtp_input")
    return h, out


def decode_step_record(tokens: torch.Tensor, pred: torch.Tensor | None = None, result: torch.Tensor | None = None,
                       record: tuple | None = None, cur: torch.Tensor | None = None):
    """A greedy step's emission from the verify's outputs, in one launch.
    tokens int64 [1 + n] = [a, drafts]; pred int64 [1 + n] and result int64 [2]
    (n_accept, bonus_row) of lm_head_accept (unused when n == 0).  -> (row
    [n + 2] (or [1]), count, next, n_accept) device int64 tensors.  record =
    (rows [cap, width], counts [cap], n_accepts [cap], k []) also writes row
    k and advances k on the device; cur (one int64) receives next."""
    dev = require_cuda(tokens, pred, result, cur)
    tokens = tokens.reshape(-1)
    n = tokens.numel() - 1
    for t in (tokens, pred, result, cur) + (tuple(record) if record else ()):
        if t is not None and (t.dtype != torch.int64 or not t.is_contiguous()):
            raise TypeError("decode_step_record takes contiguous int64 tensors")
    width = n + 2 if n > 0 else 1
    outs = torch.empty(width + 3, dtype=torch.int64, device=dev)
    rows = counts = naccs = k = None
    cap = 0
    if record is not None:
        rows, counts, naccs, k = record
        cap = rows.shape[0]
        if rows.shape[1] != width or counts.numel() < cap or naccs.numel() < cap or k.numel() != 1:
            raise ValueError("record buffers do not match the step's row width and capacity")
    check(lib().hsmoe_decode_step_record(ptr(tokens), n, ptr(pred), ptr(result), ptr(outs),
                                         outs.data_ptr() + 8 * width, outs.data_ptr() + 8 * (width + 1),
                                         outs.data_ptr() + 8 * (width + 2), ptr(rows), ptr(counts), ptr(naccs),
                                         ptr(k), cap, ptr(cur), stream_ptr(dev)), "hsmoe_decode_step_record")
    return outs[:width], outs[width], outs[width + 1], outs[width + 2]


def xor_checksum(data: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """uint8 [16] device tensor: the XOR of the 16-byte words of `data`'s bytes
    (a contiguous device tensor whose byte size is a multiple of 16)."""
    dev = require_cuda(data, out)
    if not data.is_contiguous():
        raise ValueError("xor_checksum needs a contiguous tensor")
    nbytes = data.numel() * data.element_size()
    if out is None:
        out = torch.empty(16, dtype=torch.uint8, device=dev)
    elif out.numel() * out.element_size() != 16 or not out.is_contiguous():
        raise ValueError("xor_checksum out must be 16 contiguous bytes")
    ws = _workspace(dev, "checksum", lib().hsmoe_xor_checksum_workspace_size())
    check(lib().hsmoe_xor_checksum(ptr(data) if nbytes else None, nbytes, ptr(out), ptr(ws), ws.numel(),
                                   stream_ptr(dev)), "hsmoe_xor_checksum")
    return out


# ---------------------------------------------------------------- generators

def gen_bytes(key: int, out: torch.Tensor, e4m3: bool = False) -> torch.Tensor:
    dev = require_cuda(out)
    fn = lib().hsmoe_gen_e4m3 if e4m3 else lib().hsmoe_gen_bytes
    check(fn(key, out.numel() * out.element_size(), ptr(out), stream_ptr(dev)), "hsmoe_gen_bytes")
    return out


def gen_e8m0(key: int, out: torch.Tensor, lo: int = 119, span: int = 6) -> torch.Tensor:
    dev = require_cuda(out)
    check(lib().hsmoe_gen_e8m0(key, out.numel(), lo, span, ptr(out), stream_ptr(dev)), "hsmoe_gen_e8m0")
    return out


def gen_normal(key: int, out: torch.Tensor, mean: float, std: float) -> torch.Tensor:
    dev = require_cuda(out)
    if out.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("gen_normal fills bf16 or fp32 tensors")
    check(lib().hsmoe_gen_normal(key, out.numel(), mean, std, int(out.dtype == torch.bfloat16), ptr(out),
                                 stream_ptr(dev)), "hsmoe_gen_normal")
    return out


def gen_uniform(key: int, out: torch.Tensor, lo: float, hi: float, mul: float = 1.0) -> torch.Tensor:
    dev = require_cuda(out)
    if out.dtype != torch.float32:
        raise TypeError("gen_uniform fills fp32 tensors")
    check(lib().hsmoe_gen_uniform(key, out.numel(), lo, hi, mul, ptr(out), stream_ptr(dev)), "hsmoe_gen_uniform")
    return out


def gen_index(key: int, out: torch.Tensor, n_values: int) -> torch.Tensor:
    dev = require_cuda(out)
    if out.dtype != torch.int64:
        raise TypeError("gen_index fills int64 tensors")
    check(lib().hsmoe_gen_index(key, out.numel(), n_values, ptr(out), stream_ptr(dev)), "hsmoe_gen_index")
    return out


def key(seed: int, tag: int) -> int:
    """Stream key = splitmix64 output number tag+1 for `seed` (same as the device's rand64)."""
    from .synthetic import rand64
    return rand64(seed, tag)
