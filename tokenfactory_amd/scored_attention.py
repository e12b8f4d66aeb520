"""Attention that also sums up how much every cached token is looked at.

``scored_attention`` is ``slot_based_attention`` with one more result: per request and
cached position, the softmax weight that the step's last ``window`` new tokens give it,
summed over them and over all query heads.  ``scores`` has ``req_to_token``'s layout
(``[max_reqs, max_context_len]``, a position's score beside its slot) and is shared by
the model's full-attention layers, whose weights add up in it, as the layers share the
slots; ``evict_tokens`` reads it.  There is no non-native path and no gradient.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _native
from .attention import (_KV_DTYPES, _check_inputs, _epilogue, _output, _pool_scales, _scratch,
                        slot_based_attention)
from .fp8_linear import _ptr


def check_scores(fn: str, scores: torch.Tensor, table: torch.Tensor) -> None:
    if scores.dtype != torch.float32 or scores.dim() != 2 or scores.device != table.device \
            or scores.shape[0] < table.shape[0] or scores.shape[1] < table.shape[1] \
            or scores.stride(1) != 1 or (scores.shape[0] > 1 and scores.stride(0) < scores.shape[1]):
        raise ValueError(f"{fn}: scores must be fp32 with req_to_token's rows and columns "
                         f"{tuple(table.shape)}, on its device, row-major")


MAX_ITEMS = 2048               # blocks of 16 heads of a kv head in one launch
MAX_KEPT_BYTES = 4 << 30       # scores kept between the two halves of a step


def _one_pass(bsz, n_q, n_kv, head_dim, kv_dtype, span) -> bool:
    """Whether a decode step keeps the attention's own scores for the weights (tf_attn_scored)
    instead of computing them again: 4 bytes per head and key, where K and V are head_dim /
    group times that (43 at 24 / 4 heads of 256, 32 at 32 / 8 of 128; half in fp8), unless
    the table is so wide that the longest context's room for every request is too much."""
    if n_q % n_kv or (kv_dtype == _native.TF_DTYPE_FP8_E4M3 and head_dim % 16):
        return False
    return (bsz * -(-(n_q // n_kv) // 16) <= MAX_ITEMS
            and 4 * bsz * n_q * span <= MAX_KEPT_BYTES)


def scored_attention(
    q: torch.Tensor,
    layer_k_buffer: torch.Tensor,
    layer_v_buffer: torch.Tensor,
    batch,
    scores: torch.Tensor,
    *,
    window: int = 32,
    add: bool = True,
    scaling: Optional[float] = None,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    gate: Optional[torch.Tensor] = None,
    out_amax: Optional[torch.Tensor] = None,
    stream: Optional[torch.cuda.Stream] = None,
) -> torch.Tensor:
    """``slot_based_attention(q, layer_k_buffer, layer_v_buffer, batch, ...)``, and
    ``scores[req_pool_indices[b], k] += w[b, k]`` for ``k < seq_lens[b]``, w the fp32 sum
    over the request's last ``min(window, extend_len)`` new tokens and all heads of
    their softmax weights (``add`` False: ``= w``, for a request's first step or scores of
    the last step alone).  Positions behind a request's length stay as they are.  A table
    row stands for one request of the batch at most.

    A captured call follows ``seq_lens`` (and ``extend_lens_tensor``) in place up to
    ``req_to_token``'s width; an eager one covers ``batch.max_seq_len`` keys, as the
    batch promises.  A batch of one has ``batch.max_seq_len`` keys in both, as in
    ``slot_based_attention``."""
    fn = "scored_attention"
    _native.refuse_gradients(fn, q, layer_k_buffer, layer_v_buffer, gate, scores)
    _check_inputs(q, layer_k_buffer, layer_v_buffer, batch)
    check_scores(fn, scores, batch.req_to_token)
    if window < 1:
        raise ValueError(f"{fn}: window {window}")
    rows = batch.req_pool_indices_list
    if rows is not None and len(set(rows)) != len(rows):
        raise ValueError(f"{fn}: a request row appears twice in one batch")
    n_tok, n_q, head_dim = q.shape
    n_slots, n_kv, _ = layer_k_buffer.shape
    bsz, device = batch.batch_size, q.device
    kv_dtype = _KV_DTYPES[layer_k_buffer.dtype]
    longest = int(batch.max_extend_len)
    ext_t = batch.extend_lens_tensor
    if longest > 1 and (ext_t is None or ext_t.device != device or ext_t.dtype != torch.long
                        or ext_t.numel() != bsz or not ext_t.is_contiguous()):
        raise ValueError(f"{fn}: batch.extend_lens_tensor must be contiguous int64 [batch_size] "
                         "on q's device")
    if n_tok and longest == 1 and (n_tok != bsz or len(batch.extend_lens) != bsz):
        raise ValueError(f"{fn}: {n_tok} tokens, {len(batch.extend_lens)} extend_lens of a "
                         f"decode batch of {bsz}")
    with _native.launching(device, stream):
        k_scale, v_scale = _pool_scales(q, kv_dtype, k_scale, v_scale)
        if q.stride(2) != 1 or q.stride(1) != head_dim:
            q = q.contiguous()
        rtt = batch.req_to_token
        span = (rtt.shape[1] if torch.cuda.is_current_stream_capturing()
                else max(1, int(batch.max_seq_len)))
        scale = head_dim ** -0.5 if scaling is None else float(scaling)
        override = int(batch.max_seq_len) if bsz == 1 else 0
        table = (rtt.data_ptr(), rtt.shape[0], rtt.stride(0), rtt.shape[1],
                 batch.req_pool_indices.data_ptr(), batch.seq_lens.data_ptr(), override)
        if n_tok and longest == 1 and _one_pass(bsz, n_q, n_kv, head_dim, kv_dtype, span):
            out = _output(q, out)
            ws, nbytes = _scratch("tf_attn_scored_workspace_bytes", device, bsz, span, n_q, n_kv,
                                  head_dim, kv_dtype)
            _native.call("tf_attn_scored", q.data_ptr(), q.stride(0), layer_k_buffer.data_ptr(),
                         layer_v_buffer.data_ptr(), n_slots, kv_dtype, _ptr(k_scale),
                         _ptr(v_scale), *table, bsz, span, n_q, n_kv, head_dim, scale,
                         out.data_ptr(), out.stride(0), scores.data_ptr(), scores.stride(0),
                         int(bool(add)), ws.data_ptr(), nbytes, *_epilogue(q, gate, out_amax),
                         _native.current_stream(device))
            return out
        out = slot_based_attention(q, layer_k_buffer, layer_v_buffer, batch, scaling=scaling,
                                   k_scale=k_scale, v_scale=v_scale, out=out, gate=gate,
                                   out_amax=out_amax)
        if n_tok == 0:
            return out
        window = min(int(window), longest)
        ws, nbytes = _scratch("tf_attn_weights_workspace_bytes", device, bsz, window, span, n_q,
                              n_kv, head_dim, kv_dtype)
        _native.call("tf_attn_weights", q.data_ptr(), q.stride(0), n_tok,
                     layer_k_buffer.data_ptr(), n_slots, kv_dtype, _ptr(k_scale), *table,
                     _ptr(ext_t) if longest > 1 else None, bsz, window, span, n_q, n_kv, head_dim,
                     scale, scores.data_ptr(), scores.stride(0), int(bool(add)), ws.data_ptr(),
                     nbytes, _native.current_stream(device))
    return out
