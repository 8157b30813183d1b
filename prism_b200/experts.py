"""Operators of a mixture-of-experts layer: routing of rows to experts, matrix products grouped by expert and products
with 4-bit weights.

    r = route_topk(logits, k)                                # choices, their weights, and the rows' order by expert
    xs = route_gather(x, r.pos)                              # rows of x in that order
    hs = grouped_gemm_bf16(xs, w, r.offsets)                 # each group times its expert's matrix (or gemv_w4)
    y = route_combine(ys, r.pos, r.weights)                  # back into token order, weighted and added up

and their gradients: route_combine_grad, grouped_gemm_bf16_dgrad and _wgrad, route_combine without weights (of the
gather) and route_topk_grad.  They are called by name: nothing is recorded for autograd.  How many rows an expert gets
stays on the device, so all of this can run without a host synchronisation and be captured in a CUDA graph (after one
grouped or 4-bit product on the device).  Everything runs on the current stream of the tensors' device through the C ABI
in include/prism_b200.h, which states the operators in full; nothing falls back to PyTorch.

A row matrix is a 2-D tensor whose rows are contiguous (its row stride may be larger than its width).  Buffers made for
tokens * k rows hold their groups in front; what lies behind offsets[-1] does not matter and is not written.
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from . import _lib
from ._lib import load

__all__ = ["Routing", "route_workspace_size", "route_topk", "route_topk_grad", "route_gather", "route_combine", "route_combine_grad",
           "grouped_gemm_bf16", "grouped_gemm_bf16_dgrad", "grouped_gemm_bf16_wgrad", "gemv_w4"]

_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class Routing(NamedTuple):
    """What route_topk computes for T tokens and E experts."""
    ids: torch.Tensor      # (T, k) int32, -1: no expert
    weights: torch.Tensor  # (T, k) float32
    pos: torch.Tensor      # (T, k) int32: the choice's row in expert order, -1: none
    order: torch.Tensor    # (T * k,) int32: the choice (token * k + j) of each row, -1 behind the last
    offsets: torch.Tensor  # (E + 1,) int32: borders of the experts' rows


def _tensor(name: str, t: torch.Tensor, device, dtype, shape=None) -> None:
    """A contiguous tensor on `device` of the given type and shape."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor (prism_b200 has no CPU path)")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.dtype != dtype:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _rows(name: str, t: torch.Tensor, device=None, dtype=None, rows=None, width=None) -> int:
    """A 2-D tensor with contiguous rows; returns its row stride in elements."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor (prism_b200 has no CPU path)")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if t.dim() != 2:
        raise ValueError(f"{name} must have two dimensions")
    n, m = t.shape
    if (rows is not None and n != rows) or (width is not None and m != width):
        raise ValueError(f"{name} has shape {(n, m)}, expected {(n if rows is None else rows, m if width is None else width)}")
    if m > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} must have contiguous rows")
    if n <= 1:
        return m
    ld = t.stride(0)
    if ld < m:
        raise ValueError(f"{name} must not have overlapping rows")
    return ld


def _code(name: str, dtype) -> int:
    code = _CODES.get(dtype)
    if code is None:
        raise TypeError(f"{name} has dtype {dtype}, expected float32, bfloat16 or float16")
    return code


def _run(device, fn, *args) -> None:
    """fn(*args, current stream of `device`) with that device current."""
    stream = torch._C._cuda_getCurrentRawStream(device.index)   # torch.cuda.current_stream(device).cuda_stream, 2 us sooner
    if device.index == torch.cuda.current_device():
        status = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            status = fn(*args, stream)
    if status:
        _lib.check(status)


# ---------------------------------------------------------------------------
# routing
# ---------------------------------------------------------------------------
@functools.lru_cache(maxsize=256)
def route_workspace_size(tokens: int, experts: int, k: int) -> int:
    """Bytes of scratch that route_topk needs (0 up to 64 tokens)."""
    out = ctypes.c_size_t(0)
    _lib.check(load().prism_b200_route_workspace_size(int(tokens), int(experts), int(k), ctypes.byref(out)))
    return int(out.value)


def route_topk(logits: torch.Tensor, k: int, renormalize: bool = True, out=None, workspace: torch.Tensor | None = None) -> Routing:
    """The k experts of the largest logits of each token, and the order of the chosen rows by expert.

    logits (T, E) in fp32, bf16 or fp16; a logit of -inf or NaN is never chosen, and of equal logits the lowest expert
    is.  weights are the softmax over the chosen logits, or over all of them with renormalize=False.  `out` takes the
    five tensors of a Routing (or of an earlier result) to write into; `workspace` scratch of route_workspace_size bytes.
    """
    ld = _rows("logits", logits)
    code, device, k = _code("logits", logits.dtype), logits.device, int(k)
    tokens, experts = logits.shape
    if out is None:
        if not 1 <= k <= max(experts, 1):
            raise ValueError(f"k must be 1 .. experts, got {k} of {experts}")
        i32 = dict(dtype=torch.int32, device=device)
        out = Routing(torch.empty((tokens, k), **i32), torch.empty((tokens, k), dtype=torch.float32, device=device),
                      torch.empty((tokens, k), **i32), torch.empty(tokens * k, **i32), torch.empty(experts + 1, **i32))
    else:
        out = Routing(*out)
        _tensor("ids", out.ids, device, torch.int32, (tokens, k))
        _tensor("weights", out.weights, device, torch.float32, (tokens, k))
        _tensor("pos", out.pos, device, torch.int32, (tokens, k))
        _tensor("order", out.order, device, torch.int32, (tokens * k,))
        _tensor("offsets", out.offsets, device, torch.int32, (experts + 1,))
    need = route_workspace_size(tokens, experts, k)
    if workspace is None:   # kept until both launches are queued: whoever gets its memory next comes behind them
        workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    else:
        if not isinstance(workspace, torch.Tensor) or workspace.device != device or not workspace.is_contiguous():
            raise ValueError("workspace must be a contiguous tensor on the device of logits")
        if workspace.numel() * workspace.element_size() < need:
            raise ValueError("workspace too small; see route_workspace_size(tokens, experts, k)")
    _run(device, load().prism_b200_route_topk, tokens, experts, k, code, logits.data_ptr(), ld, int(bool(renormalize)),
         out.ids.data_ptr(), out.weights.data_ptr(), out.pos.data_ptr(), out.order.data_ptr(), out.offsets.data_ptr(),
         workspace.data_ptr() if need else None)
    return out


def route_topk_grad(logits: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, dweights: torch.Tensor,
                    renormalize: bool = True, out: torch.Tensor | None = None) -> torch.Tensor:
    """Gradient of route_topk's weights with respect to the logits (T, E), in their type."""
    ld = _rows("logits", logits)
    code, device = _code("logits", logits.dtype), logits.device
    tokens, experts = logits.shape
    if not isinstance(ids, torch.Tensor) or ids.dim() != 2:
        raise ValueError("ids must have two dimensions")
    k = ids.shape[1]
    _tensor("ids", ids, device, torch.int32, (tokens, k))
    _tensor("weights", weights, device, torch.float32, (tokens, k))
    _tensor("dweights", dweights, device, torch.float32, (tokens, k))
    if out is None:
        out = logits.new_empty((tokens, experts))
    else:
        _tensor("out", out, device, logits.dtype, (tokens, experts))
    _run(device, load().prism_b200_route_topk_grad, tokens, experts, k, code, logits.data_ptr(), ld, int(bool(renormalize)),
         ids.data_ptr(), weights.data_ptr(), dweights.data_ptr(), out.data_ptr())
    return out


def _pos(pos: torch.Tensor, device, tokens=None) -> tuple[int, int]:
    if not isinstance(pos, torch.Tensor) or pos.dim() != 2:
        raise ValueError("pos must have two dimensions")
    t, k = pos.shape
    _tensor("pos", pos, device, torch.int32, (t if tokens is None else tokens, k))
    return t, k


def route_gather(x: torch.Tensor, pos: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """out[pos[t, j]] = x[t] for x (T, H); out (T * k, H) by default, rows that no position names stay as they are.
    Gradient: route_combine(dout, pos)."""
    ldx = _rows("x", x)
    tokens, width = x.shape
    _, k = _pos(pos, x.device, tokens)
    if out is None:
        out, ldo = x.new_empty((tokens * k, width)), width
    else:
        ldo = _rows("out", out, x.device, x.dtype, None, width)
    _run(x.device, load().prism_b200_route_gather, _code("x", x.dtype), tokens, k, width, x.data_ptr(), ldx, pos.data_ptr(),
         out.shape[0], out.data_ptr(), ldo)
    return out


def route_combine(y: torch.Tensor, pos: torch.Tensor, weights: torch.Tensor | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """out[t] = sum over j of weights[t, j] * y[pos[t, j]] for y (rows, H): fp32 sums, rounded once.  Without weights the
    rows are added up as they are."""
    ldy = _rows("y", y)
    rows, width = y.shape
    tokens, k = _pos(pos, y.device)
    if weights is not None:
        _tensor("weights", weights, y.device, torch.float32, (tokens, k))
    if out is None:
        out, ldo = y.new_empty((tokens, width)), width
    else:
        ldo = _rows("out", out, y.device, y.dtype, tokens, width)
    _run(y.device, load().prism_b200_route_combine, _code("y", y.dtype), tokens, k, width, y.data_ptr(), ldy, rows, pos.data_ptr(),
         None if weights is None else weights.data_ptr(), out.data_ptr(), ldo)
    return out


def route_combine_grad(dout: torch.Tensor, y: torch.Tensor, pos: torch.Tensor, weights: torch.Tensor,
                       dy: torch.Tensor | None = None, dweights: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Gradients of route_combine: dy (shaped like y; rows that no position names stay as they are) and dweights."""
    ldd = _rows("dout", dout)
    tokens, width = dout.shape
    ldy = _rows("y", y, dout.device, dout.dtype, None, width)
    _, k = _pos(pos, dout.device, tokens)
    _tensor("weights", weights, dout.device, torch.float32, (tokens, k))
    rows = y.shape[0]
    if dy is None:
        dy, lddy = y.new_empty((rows, width)), width
    else:
        lddy = _rows("dy", dy, dout.device, dout.dtype, rows, width)
    if dweights is None:
        dweights = weights.new_empty((tokens, k))
    else:
        _tensor("dweights", dweights, dout.device, torch.float32, (tokens, k))
    _run(dout.device, load().prism_b200_route_combine_grad, _code("dout", dout.dtype), tokens, k, width, dout.data_ptr(), ldd,
         y.data_ptr(), ldy, rows, pos.data_ptr(), weights.data_ptr(), dy.data_ptr(), lddy, dweights.data_ptr())
    return dy, dweights


# ---------------------------------------------------------------------------
# products grouped by expert
# ---------------------------------------------------------------------------
def _weights3(w: torch.Tensor, device) -> tuple[int, int, int]:
    if not isinstance(w, torch.Tensor) or w.dim() != 3:
        raise ValueError("w must have three dimensions (experts, n, k)")
    _tensor("w", w, device, torch.bfloat16)
    return tuple(w.shape)


def grouped_gemm_bf16(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """out[r] = w[e] @ x[r] for the rows offsets[e] <= r < offsets[e + 1] of x (rows, k); w (experts, n, k); out (rows, n),
    bf16 with fp32 accumulation.  Rows outside every group are not written."""
    ldx = _rows("x", x, None, torch.bfloat16)
    experts, n, k = _weights3(w, x.device)
    rows = x.shape[0]
    if x.shape[1] != k:
        raise ValueError(f"k mismatch: x {tuple(x.shape)}, w {tuple(w.shape)}")
    _tensor("offsets", offsets, x.device, torch.int32, (experts + 1,))
    if out is None:
        out, ldo = x.new_empty((rows, n)), n
    else:
        ldo = _rows("out", out, x.device, torch.bfloat16, rows, n)
    _run(x.device, load().prism_b200_grouped_gemm_bf16, experts, rows, n, k, x.data_ptr(), ldx, w.data_ptr(), offsets.data_ptr(),
         out.data_ptr(), ldo)
    return out


def grouped_gemm_bf16_dgrad(dy: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """dx[r] = w[e].T @ dy[r]: the gradient of grouped_gemm_bf16 with respect to x."""
    lddy = _rows("dy", dy, None, torch.bfloat16)
    experts, n, k = _weights3(w, dy.device)
    rows = dy.shape[0]
    if dy.shape[1] != n:
        raise ValueError(f"n mismatch: dy {tuple(dy.shape)}, w {tuple(w.shape)}")
    _tensor("offsets", offsets, dy.device, torch.int32, (experts + 1,))
    if out is None:
        out, ldo = dy.new_empty((rows, k)), k
    else:
        ldo = _rows("out", out, dy.device, torch.bfloat16, rows, k)
    _run(dy.device, load().prism_b200_grouped_gemm_bf16_dgrad, experts, rows, n, k, dy.data_ptr(), lddy, w.data_ptr(),
         offsets.data_ptr(), out.data_ptr(), ldo)
    return out


def grouped_gemm_bf16_wgrad(dy: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor, out: torch.Tensor | None = None,
                            dtype=torch.bfloat16) -> torch.Tensor:
    """dw[e] = dy[group].T @ x[group]: the gradient with respect to w, (experts, n, k) in fp32 or bf16 (`dtype`, or that of
    `out`); zeros for an empty group."""
    lddy = _rows("dy", dy, None, torch.bfloat16)
    rows, n = dy.shape
    ldx = _rows("x", x, dy.device, torch.bfloat16, rows)
    k = x.shape[1]
    if not isinstance(offsets, torch.Tensor) or offsets.dim() != 1 or offsets.numel() < 1:
        raise ValueError("offsets must have one dimension of experts + 1")
    experts = offsets.numel() - 1
    _tensor("offsets", offsets, dy.device, torch.int32)
    if out is None:
        out = torch.empty((experts, n, k), dtype=dtype, device=dy.device)
    else:
        dtype = out.dtype
        _tensor("out", out, dy.device, dtype, (experts, n, k))
    if dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"dw has dtype {dtype}, expected float32 or bfloat16")
    _run(dy.device, load().prism_b200_grouped_gemm_bf16_wgrad, experts, rows, n, k, dy.data_ptr(), lddy, x.data_ptr(), ldx,
         offsets.data_ptr(), _CODES[dtype], out.data_ptr())
    return out


# ---------------------------------------------------------------------------
# 4-bit weights
# ---------------------------------------------------------------------------
def gemv_w4(x: torch.Tensor, q: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None,
            offsets: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Products of a few rows x (rows, k), bf16 or fp16, with matrices of 4-bit weights scales * (q - zeros).

    q (n, k / 2) uint8 holds two weights per byte, the even k in the low half; scales (n, k / group) in x's type; zeros
    (n, k / group) uint8 or None (8 everywhere); the group (32, 64 or 128) follows from the shapes.  With offsets
    (experts + 1) q, scales and zeros have a first dimension of experts, and each expert's matrix takes its rows;
    without, every row takes the one matrix.  out (rows, n) in x's type, sums in fp32.  The weights are read once for
    every eight rows.
    """
    ldx = _rows("x", x)
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"x has dtype {x.dtype}, expected bfloat16 or float16")
    device = x.device
    rows, k = x.shape
    dims = 2 if offsets is None else 3
    if not isinstance(q, torch.Tensor) or not isinstance(scales, torch.Tensor) or q.dim() != dims or scales.dim() != dims:
        raise ValueError(f"q and scales must have {dims} dimensions ({'no ' if offsets is None else ''}offsets given)")
    if q.shape[-1] * 2 != k:
        raise ValueError(f"k mismatch: x {tuple(x.shape)}, q {tuple(q.shape)}")
    n, groups = q.shape[-2], scales.shape[-1]
    if groups == 0 or k % groups:
        raise ValueError(f"scales of {groups} groups do not divide k = {k}")
    experts = q.shape[0] if dims == 3 else 1
    lead = (experts, n) if dims == 3 else (n,)
    _tensor("q", q, device, torch.uint8)
    _tensor("scales", scales, device, x.dtype, (*lead, groups))
    if zeros is not None:
        _tensor("zeros", zeros, device, torch.uint8, (*lead, groups))
    if offsets is not None:
        _tensor("offsets", offsets, device, torch.int32, (experts + 1,))
    if out is None:
        out, ldo = x.new_empty((rows, n)), n
    else:
        ldo = _rows("out", out, device, x.dtype, rows, n)
    _run(device, load().prism_b200_gemv_w4, _CODES[x.dtype], rows, experts, n, k, k // groups, x.data_ptr(), ldx, q.data_ptr(),
         scales.data_ptr(), None if zeros is None else zeros.data_ptr(), None if offsets is None else offsets.data_ptr(),
         out.data_ptr(), ldo)
    return out
