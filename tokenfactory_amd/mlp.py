"""The gated feed-forward block on block-FP8 weights.

``gated_mlp`` is ``down(silu(gate(x)) * up(x))`` (``qwen3_8/mlp.py:9-54``) with
activations quantised per row and 128 columns (``block_fp8``): the gate and up
products share a kernel whose output is the quantised hidden activations, formed
from the fp32 sums; the down product reads those.

``GatedMLP`` holds the block's weights under the reference's names, as
``Fp8Linear`` parameters, so a reference layer's state dict loads as is.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from . import _native
from .block_fp8 import (BLOCK, DTYPES, check_input, check_weight, input_rows, new_rows,
                        workspace)
from .fp8_linear import Fp8Linear, _ptr, _unaltered


_GateUpDown = _native.Fp8Mat * 3


def gated_mlp(x: torch.Tensor, gate_weight: torch.Tensor, gate_scale_inv: torch.Tensor,
              up_weight: torch.Tensor, up_scale_inv: torch.Tensor, down_weight: torch.Tensor,
              down_scale_inv: torch.Tensor, *, x_scale: Optional[torch.Tensor] = None,
              stream=None) -> torch.Tensor:
    """``bf16(h^ Wd^T)`` with ``h = silu(x^ Wg^T) * (x^ Wu^T)`` in fp32; ``^`` is
    ``quantize_blocks``' form.  Gate and up are added in fp32 up to 64 rows, the down
    product up to 16; with more rows the fp8 MFMA adds as in ``block_scaled_linear``, and
    what it cuts moves values of h next to a border of e4m3 by a step (the output is some
    0.23 % off in the norm, where its own rounding to bf16 is 0.17 %; 0.36 % was seen
    where a few channels of x are far larger than the rest).

    x: bf16 or fp32 ``[..., hidden]`` or float8_e4m3fn ``[rows, hidden]`` with its
    ``x_scale``; gate and up weights float8_e4m3fn ``[inter, hidden]``, down
    ``[out, inter]``, each with fp32 scales per 128 x 128 block; hidden and inter
    multiples of 16.  Returns bf16 ``[..., out]``; no gradients."""
    fn = "gated_mlp"
    _native.refuse_gradients(fn, x, x_scale, gate_weight, gate_scale_inv, up_weight, up_scale_inv,
                             down_weight, down_scale_inv)
    hidden = gate_weight.shape[-1]
    rows = check_input(fn, x, x_scale, hidden)
    dev = x.device
    gate = check_weight(fn, "gate_weight", gate_weight, gate_scale_inv, hidden, dev)
    up = check_weight(fn, "up_weight", up_weight, up_scale_inv, hidden, dev)
    inter = gate_weight.shape[0]
    if up_weight.shape[0] != inter:
        raise ValueError(f"{fn}: {inter} gate and {up_weight.shape[0]} up columns")
    down = check_weight(fn, "down_weight", down_weight, down_scale_inv, inter, dev)
    if inter % 16:
        raise NotImplementedError(f"{fn}: {inter} hidden activations (a multiple of 16)")
    n = down_weight.shape[0]
    dtype = DTYPES[x.dtype]
    with _native.launching(dev, stream):
        out = new_rows(rows, n, torch.bfloat16, dev)
        if rows:
            xr, xs, sc, ss = input_rows(x, x_scale)
            ws, nbytes = workspace("tf_gated_mlp_workspace_bytes", dev, rows, hidden, inter, n,
                                   dtype)
            mats = _GateUpDown((*gate, None, inter, None, inter), (*up, None, inter, None, inter),
                               (*down, None, n, out.data_ptr(), n))
            _native.call("tf_gated_mlp", xr.data_ptr(), dtype, xs, _ptr(sc), ss, mats, rows, hidden,
                         inter, ws.data_ptr(), nbytes, _native.current_stream(dev))
    return out if x.dim() == 2 else out.reshape(*x.shape[:-1], n)


class GatedMLP(nn.Module):
    """One TP rank's share of the gated feed-forward block (whole blocks of 128 columns):
    ``gate_proj`` and ``up_proj`` ``[intermediate_size / tp, hidden]`` and ``down_proj``,
    whose partial sums the caller adds over the ranks.  The three ``Fp8Linear``s hold
    weights and scales; ``forward`` reads them and does not call the modules, so that
    one that is more than that (a subclass, a hook, a bias) is refused."""

    def __init__(self, config):
        super().__init__()
        q = getattr(config, "quantization_config", None)
        if not isinstance(q, dict) or q.get("quant_method") != "fp8":
            raise NotImplementedError("GatedMLP: weights must be block-FP8 (quantization_config "
                                      "with quant_method fp8)")
        block = tuple(q.get("weight_block_size", [BLOCK, BLOCK]))
        if block != (BLOCK, BLOCK):
            raise NotImplementedError(f"GatedMLP: weight blocks of {block} (128 x 128)")
        act = getattr(config, "hidden_act", "silu")
        if act != "silu":
            raise NotImplementedError(f"GatedMLP: activation {act!r} (silu)")
        tp = getattr(config, "tp_size", 1)
        if config.intermediate_size % tp:
            raise ValueError("intermediate_size must divide by tp_size")
        inter = config.intermediate_size // tp
        if tp > 1 and inter % BLOCK:   # (no rows of the checkpoint's scales are the share's)
            raise NotImplementedError(f"GatedMLP: {inter} columns a rank cut a block of {BLOCK} "
                                      "columns that share a scale")
        if inter % 16 or config.hidden_size % 16:
            raise NotImplementedError(f"GatedMLP: {config.hidden_size} x {inter} (multiples of 16)")
        self.gate_proj = Fp8Linear(config.hidden_size, inter, block_size=block)
        self.up_proj = Fp8Linear(config.hidden_size, inter, block_size=block)
        self.down_proj = Fp8Linear(inter, config.hidden_size, block_size=block)

    def forward(self, x: torch.Tensor, x_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
        weights = []
        for name in ("gate_proj", "up_proj", "down_proj"):
            lin = self._modules[name]
            if not _unaltered(lin, Fp8Linear) or lin.bias is not None \
                    or (lin.block_h, lin.block_w) != (BLOCK, BLOCK):
                raise NotImplementedError(f"GatedMLP: {name} must be a plain Fp8Linear of 128 x 128 "
                                          "blocks without a bias: its call is passed by")
            weights += lin.weight, lin.weight_scale_inv
        return gated_mlp(x, *weights, x_scale=x_scale)
