"""FP8 products with a scale for each block of 128 columns of the activations.

``fp8_linear`` quantises activations with one scale per tensor, as the reference's
linears do (``qwen3_8/fp8_triton.py:127-130``).  Here every row has a scale per
128 columns, the granularity of the weights' 128 x 128 blocks: no other row's
values change a row's result, an outlier costs precision only within its own block,
and no pass over the whole tensor comes first, so that the producer of the
activations can write them quantised (``add_rms_norm(..., quantize=True)``).  (The
number of rows does pick the kernel, and with it a result's last bits.)

* ``quantize_blocks(x)`` -> e4m3 rows and their scales
* ``block_scaled_linear(x, weight, weight_scale_inv, bias)``: the product with a
  checkpoint's block-FP8 weight (``Fp8Linear.weight`` / ``weight_scale_inv``)

Scales are fp32 ``[rows, ceil(cols / 128)]``, stored with a block's rows side by
side (``stride(0) == 1``).  There is no non-native path and no gradient: operands that
ask for one are refused while autograd records.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _native
from .fp8_linear import _ptr

BLOCK = 128
DTYPES = {torch.bfloat16: _native.TF_DTYPE_BF16, torch.float32: _native.TF_DTYPE_FP32,
          torch.float8_e4m3fn: _native.TF_DTYPE_FP8_E4M3}


def blocks(n: int) -> int:
    return -(-n // BLOCK)


def rows16(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """(rows, their stride): ``t`` itself if the kernels take its rows as they lie
    (dense columns, rows that do not overlap, 16-byte aligned), else a copy; the stride
    of one row is its width, whatever torch says.  Widths are multiples of 8, or 16 of
    e4m3 values."""
    rows, cols = t.shape
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t, cols
        if t.stride(1) == 1:
            stride = t.stride(0) if rows > 1 else cols
            if stride >= cols and stride % (16 if t.dtype == torch.float8_e4m3fn else 8) == 0:
                return t, stride
    return t.clone(memory_format=torch.contiguous_format), cols


def new_rows(rows: int, cols: int, dtype: torch.dtype, device) -> torch.Tensor:
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)


def new_scales(rows: int, cols: int, device) -> torch.Tensor:
    """Room for the scales of ``rows`` x ``cols`` values, a block's rows side by side."""
    return torch.empty_strided((rows, blocks(cols)), (1, rows), dtype=torch.float32,
                               device=device)


def quantize_blocks(x: torch.Tensor, stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Per row and 128 columns (the last block may be shorter): scale ``s = max(amax
    |x|, 1e-12) / 448`` in fp32, values ``e4m3(x / s)``, each rounded to nearest
    even.  x: bf16 or fp32 ``[rows, cols]``, cols a multiple of 8.  Returns
    float8_e4m3fn ``[rows, cols]`` and fp32 scales ``[rows, ceil(cols / 128)]``.
    A NaN or infinite value poisons its row's block (scale NaN or inf)."""
    _native.refuse_gradients("quantize_blocks", x)
    if x.dim() != 2 or not x.is_cuda or x.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("quantize_blocks: x must be a 2-D bf16 or fp32 CUDA tensor")
    rows, cols = x.shape
    if cols == 0 or cols % 8:
        raise ValueError(f"quantize_blocks: {cols} columns (a positive multiple of 8)")
    dev = x.device
    with _native.launching(dev, stream):
        x, stride = rows16(x)
        xq = new_rows(rows, cols, torch.float8_e4m3fn, dev)
        scale = new_scales(rows, cols, dev)
        _native.call("tf_block_quant", x.data_ptr(), DTYPES[x.dtype], rows, cols, stride,
                     xq.data_ptr(), cols, scale.data_ptr(), rows, _native.current_stream(dev))
    return xq, scale


def check_weight(fn: str, what: str, w: torch.Tensor, scale: torch.Tensor, k: int, device) -> tuple:
    """The fields of the ``tf_fp8_mat`` of a weight up to its bias."""
    n = w.shape[0] if w.dim() == 2 else 0
    if w.dtype != torch.float8_e4m3fn or n == 0 or w.shape[1] != k or w.device != device:
        raise ValueError(f"{fn}: {what} must be float8_e4m3fn [out, {k}] on x's device, not "
                         f"{w.dtype} {tuple(w.shape)}")
    ptr = w.data_ptr()
    stride = k if w.is_contiguous() or n == 1 else w.stride(0)
    if ptr % 16 or stride % 16 or stride < k or w.stride(1) != 1:
        raise ValueError(f"{fn}: {what} rows must be contiguous and 16-byte aligned")
    shape = (-(-n // BLOCK), -(-k // BLOCK))
    if scale.dtype != torch.float32 or scale.shape != shape or scale.device != device:
        raise ValueError(f"{fn}: scales of {what} must be fp32 {shape} on x's device, one per "
                         f"128 x 128 block")
    sn, sk = scale.stride()
    return ptr, stride, scale.data_ptr(), sn, sk


def check_input(fn: str, x: torch.Tensor, x_scale: Optional[torch.Tensor], k: int) -> int:
    """The rows of an x of ``k`` columns that the products take."""
    if not x.is_cuda or x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"{fn}: x {tuple(x.shape)} must be a CUDA tensor of {k} columns")
    if k == 0:
        raise ValueError(f"{fn}: no columns")
    if k % 16:
        raise NotImplementedError(f"{fn}: {k} columns (a multiple of 16)")
    if x.dtype not in DTYPES:
        raise ValueError(f"{fn}: x must be bf16, fp32 or float8_e4m3fn, not {x.dtype}")
    quantized = x.dtype == torch.float8_e4m3fn
    if quantized != (x_scale is not None):
        raise ValueError(f"{fn}: x_scale goes with a float8_e4m3fn x")
    if not quantized:
        return x.numel() // k
    if x.dim() != 2:
        raise ValueError(f"{fn}: a quantised x must be 2-D")
    if (x_scale.dtype != torch.float32 or x_scale.device != x.device
            or tuple(x_scale.shape) != (x.shape[0], blocks(k))):
        raise ValueError(f"{fn}: x_scale must be fp32 {(x.shape[0], blocks(k))} on x's device")
    return x.shape[0]


def input_rows(x: torch.Tensor, x_scale: Optional[torch.Tensor]):
    """(x's rows, their stride, scales, their stride) as the entry points take them;
    copies what lies otherwise, on the stream that is current."""
    x2d, stride = rows16(x if x.dim() == 2 else x.reshape(-1, x.shape[-1]))
    if x_scale is None:
        return x2d, stride, None, 0
    rows, nb = x_scale.shape
    s0, s1 = x_scale.stride()
    if not ((rows == 1 or s0 == 1) and (nb == 1 or s1 >= rows)):
        x_scale, s1 = x_scale.t().contiguous().t(), rows
    return x2d, stride, x_scale, rows if nb == 1 else s1


def workspace(name: str, device, *sizes):
    """(scratch or None, bytes) that entry point ``name`` asks for."""
    nbytes = _native.call(name, *sizes)
    if not nbytes:
        return None, 0
    return torch.empty_strided((nbytes,), (1,), dtype=torch.uint8, device=device), nbytes


_OneMat = _native.Fp8Mat * 1


def block_scaled_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale_inv: torch.Tensor,
                        bias: Optional[torch.Tensor] = None, *,
                        x_scale: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """``bf16(sum_kb x_scale[m, kb] * weight_scale_inv[n // 128, kb] * (xq w^T)[m, n] over
    block kb + bias)``.  Up to 16 rows the products are exact and added in fp32; with
    more the fp8 MFMA adds them, which of each 8 neighbouring columns cuts every product
    13 bits below the largest and adds the rest in fp32 (1.5e-5 of a sum of Gaussian
    values, below the rounding to bf16 unless the terms cancel).

    x: bf16 or fp32 ``[..., in]``, quantised here as ``quantize_blocks`` does, or
    float8_e4m3fn ``[rows, in]`` with its ``x_scale``; weight float8_e4m3fn
    ``[out, in]`` (in a multiple of 16) with fp32 scales per 128 x 128 block; bias
    bf16 ``[out]``.  Returns bf16 ``[..., out]``."""
    fn = "block_scaled_linear"
    _native.refuse_gradients(fn, x, x_scale, weight, weight_scale_inv, bias)
    rows = check_input(fn, x, x_scale, weight.shape[-1])
    dev, dtype = x.device, DTYPES[x.dtype]
    mat = check_weight(fn, "weight", weight, weight_scale_inv, x.shape[-1], dev)
    n, k = weight.shape
    if bias is not None and (bias.dtype != torch.bfloat16 or tuple(bias.shape) != (n,)
                             or bias.device != dev or not bias.is_contiguous()):
        raise ValueError(f"{fn}: bias must be a contiguous bf16 [{n}] on x's device")
    with _native.launching(dev, stream):
        out = new_rows(rows, n, torch.bfloat16, dev)
        if rows:
            xr, xs, sc, ss = input_rows(x, x_scale)
            ws, nbytes = workspace("tf_block_linear_workspace_bytes", dev, rows, n, k, dtype)
            _native.call("tf_block_linear", xr.data_ptr(), dtype, xs, _ptr(sc), ss,
                         _OneMat((*mat, _ptr(bias), n, out.data_ptr(), n)), rows, k, _ptr(ws),
                         nbytes, _native.current_stream(dev))
    return out if x.dim() == 2 else out.reshape(*x.shape[:-1], n)
