"""The residual sum and the norms around a block, in one launch.

A decoder layer adds each block's output to the residual stream and norms the sum
for the next block (``qwen3_8/decoder_layer.py:57-81``, ``qwen3_8/rms_norm.py:19-24``);
``add_rms_norm`` does both, with the forms in which models vary that step (a norm
of the block's output, a gate, a residual multiplier), and hands the result on as
bf16 / fp32 or quantised for ``block_scaled_linear`` and ``gated_mlp``.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _native
from .block_fp8 import DTYPES, new_rows, new_scales, rows16

MAX_COLS = 16384
_VALUES = (torch.bfloat16, torch.float32)


def _check(name: str, t: torch.Tensor, shape, device) -> None:
    if t.dtype not in _VALUES or t.shape != shape or t.device != device:
        raise ValueError(f"add_rms_norm: {name} must be bf16 or fp32 {tuple(shape)} on x's device")


def _vector(t: torch.Tensor) -> torch.Tensor:
    """``t`` itself if it lies dense and 16-byte aligned, else a copy."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _extent(t: torch.Tensor) -> int:
    """Bytes from the first to behind the last element."""
    return (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _clash(r: torch.Tensor, t: Optional[torch.Tensor]) -> bool:
    """Whether rows written over ``r`` may change what another row or thread reads of
    ``t``: they share memory and are not the very same elements (those are read by the
    thread that writes them) or other columns of the same rows."""
    if t is None or t.numel() == 0 or r.numel() == 0:
        return False
    off = t.data_ptr() - r.data_ptr()
    if off >= _extent(r) or -off >= _extent(t):
        return False
    if t.shape != r.shape:
        return True
    strides = zip(t.shape, t.stride(), r.stride())     # (a single row's says nothing)
    if off == 0 and t.dtype == r.dtype and all(n == 1 or a == b for n, a, b in strides):
        return False
    if t.shape[0] == 1:
        return True
    size = r.element_size()
    row, width = r.stride(0) * size, r.shape[1] * size
    if t.stride(1) == 1 and t.stride(0) * t.element_size() == row:
        return not (off % row >= width and off % row + t.shape[1] * t.element_size() <= row)
    return True


def _gate_rows(gate: torch.Tensor, shape):
    """(gate, row stride, per column) of a gate that broadcasts to ``shape``."""
    g = gate.expand(shape)
    rows, cols = shape
    if g.stride(1) == 0:                    # one value per row (or for all of them)
        return g, (g.stride(0) if rows > 1 else 0), 0
    if rows == 1 or g.stride(0) == 0:       # one row for all of them
        return rows16(g[:1])[0], 0, 1
    return *rows16(g), 1


def add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor],
                 weight: Optional[torch.Tensor], eps: float = 1e-6, *,
                 post_weight: Optional[torch.Tensor] = None,
                 gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0,
                 quantize: bool = False, inplace: bool = False, stream=None):
    """Per row of x, in fp32, with ``rms(v) = sqrt(mean v^2 + eps)``:

        b = x                      (post_weight * x / rms(x) with a post_weight)
        r = residual + residual_scale * gate * b
        y = weight * r / rms(r)

    x: bf16 or fp32 ``[rows, cols]``, cols a multiple of 8 up to 16384; residual of
    the same shape, or None for 0; weight and post_weight ``[cols]``; gate broadcasts
    to x's shape (``[cols]``, ``[rows, 1]``, ``[rows, cols]``, ...), bf16 or fp32 like
    every operand.

    Returns ``(y, r)``.  y has x's dtype, or with ``quantize`` is the pair
    ``(float8_e4m3fn values, fp32 scales)`` of ``quantize_blocks``; it is formed from
    r before r is rounded to the residual's dtype (x's without a residual).  Without
    a weight y is None.  ``inplace`` stores r over ``residual``, which must not share
    memory with another operand (x or a gate of its shape may be it).  Where r is x
    itself (no residual, gate, scale or post_weight), x is returned as r.  No gradients:
    operands that ask for one are refused while autograd records."""
    _native.refuse_gradients("add_rms_norm", x, residual, weight, post_weight, gate)
    if x.dim() != 2 or not x.is_cuda or x.dtype not in _VALUES:
        raise ValueError("add_rms_norm: x must be a 2-D bf16 or fp32 CUDA tensor")
    rows, cols = x.shape
    if cols == 0 or cols % 8:
        raise ValueError(f"add_rms_norm: {cols} columns (a positive multiple of 8)")
    if cols > MAX_COLS:
        raise NotImplementedError(f"add_rms_norm: {cols} columns (at most {MAX_COLS})")
    if quantize and weight is None:
        raise ValueError("add_rms_norm: quantize needs a weight")
    dev = x.device
    if weight is not None:
        _check("weight", weight, (cols,), dev)
    if post_weight is not None:
        _check("post_weight", post_weight, (cols,), dev)
    if residual is not None:
        _check("residual", residual, x.shape, dev)
    if inplace and (residual is None or rows16(residual)[0] is not residual):
        raise ValueError("add_rms_norm: in place, residual must be given, with dense 16-byte "
                         "aligned rows")
    if inplace and any(_clash(residual, t) for t in (x, gate, weight, post_weight)):
        raise ValueError("add_rms_norm: in place, residual must not share memory with another "
                         "operand (x or a gate of its shape may be residual itself)")
    if gate is not None and (gate.dtype not in _VALUES or gate.device != x.device):
        raise ValueError("add_rms_norm: gate must be bf16 or fp32 on x's device")
    scale = float(residual_scale)
    same = residual is None and gate is None and post_weight is None and scale == 1.0
    xt = rt = DTYPES[x.dtype]
    yt = DTYPES[torch.float8_e4m3fn] if quantize else xt
    with _native.launching(dev, stream):
        xr, xs = rows16(x)
        rp, rs, r, ros = 0, 0, x, cols
        if residual is not None:
            rr, rs = rows16(residual)
            rp, rt = rr.data_ptr(), DTYPES[residual.dtype]
        if inplace:
            r, ros = residual, rs
        elif not same:
            r = new_rows(rows, cols, x.dtype if residual is None else residual.dtype, dev)
        gp = gs = gt = gcols = wp = wt = pp = pt = yp = sp = 0
        if gate is not None:
            g, gs, gcols = _gate_rows(gate, x.shape)
            gp, gt = g.data_ptr(), DTYPES[g.dtype]
        if post_weight is not None:
            post_weight = _vector(post_weight)
            pp, pt = post_weight.data_ptr(), DTYPES[post_weight.dtype]
        y = ys = None
        if weight is not None:
            weight = _vector(weight)
            wp, wt = weight.data_ptr(), DTYPES[weight.dtype]
            y = new_rows(rows, cols, torch.float8_e4m3fn if quantize else x.dtype, dev)
            yp = y.data_ptr()
            if quantize:
                ys = new_scales(rows, cols, dev)
                sp = ys.data_ptr()
        if rows and not (same and y is None):
            _native.call("tf_add_rms_norm", xr.data_ptr(), xt, xs, rp, rt, rs, gp, gt, gs, gcols,
                         pp, pt, wp, wt, eps, scale, rows, cols, 0 if same else r.data_ptr(), ros,
                         yp, yt, cols, sp, rows, _native.current_stream(dev))
    if inplace:
        torch.autograd.graph.increment_version(residual)   # (written behind autograd's back)
    return ((y, ys) if quantize else y), r
