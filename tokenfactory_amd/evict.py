"""Eviction of cached tokens by the attention weight that ``scored_attention`` sums up.

A request's context is a row of slots; attention does not care which positions they were
written for (keys are stored rotated), so a token leaves the cache by leaving the row.
``evict_tokens`` shortens rows on the device, in order, and returns the slots for the
allocator.  There is no non-native path.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _native
from .attention import _scratch
from .fp8_linear import _ptr
from .scored_attention import check_scores


def evict_tokens(
    req_to_token: torch.Tensor,
    scores: torch.Tensor,
    req_pool_indices: torch.Tensor,
    seq_lens: torch.Tensor,
    keep: int,
    *,
    max_seq_len: int,
    first: Union[int, torch.Tensor] = 0,
    recent: int = 0,
    out_rows: Optional[torch.Tensor] = None,
    stream: Optional[torch.cuda.Stream] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Shortens the table rows of requests longer than ``max(keep, first + recent)`` tokens
    to that many: the first ``first`` stay (attention sinks, a shared prefix: an int, or
    int64 ``[B]`` on the device, a negative one counting as 0), the last ``recent`` stay,
    and of those between the ones with the largest score (equal scores: the earlier; NaN
    below every number), all in their order, their scores beside them.  The entries
    behind, up to the old length, become -1 with score 0.

    ``req_to_token`` int64 and ``scores`` fp32 ``[max_reqs, max_context_len]`` change in
    place; ``seq_lens`` (int64 ``[B]``, at most ``max_seq_len``) is read.  ``out_rows``
    (int64 ``[B]``): rows that receive the result instead, in the same layout, while the
    requests' own stay whole (for the prefix cache, say).  No row may be written for two
    requests, or written for one and read for another.

    Returns the new lengths, int64 ``[B]``, and the slots that left, int64
    ``[B, max(0, max_seq_len - keep)]``: in order, -1 behind them.  Slots that other
    requests share (the prefix) should lie in ``first``."""
    fn = "evict_tokens"
    table, device = req_to_token, req_to_token.device
    if not table.is_cuda:
        raise RuntimeError(f"{fn} runs only on ROCm devices")
    _native.refuse_gradients(fn, scores)
    if table.dtype != torch.int64 or table.dim() != 2 or table.stride(1) != 1 \
            or (table.shape[0] > 1 and table.stride(0) < table.shape[1]):
        raise ValueError(f"{fn}: req_to_token must be a row-major int64 [max_reqs, max_ctx] tensor")
    check_scores(fn, scores, table)
    bsz = req_pool_indices.numel()
    lists = [("req_pool_indices", req_pool_indices), ("seq_lens", seq_lens)]
    if out_rows is not None:
        lists.append(("out_rows", out_rows))
    if isinstance(first, torch.Tensor):
        lists.append(("first", first))
    for name, t in lists:
        if t.dtype != torch.int64 or t.device != device or t.numel() != bsz \
                or not t.is_contiguous():
            raise ValueError(f"{fn}: {name} must be contiguous int64 [{bsz}] on the table's device")
    first_n = 0 if isinstance(first, torch.Tensor) else int(first)
    keep, recent, max_seq_len = int(keep), int(recent), int(max_seq_len)
    if min(keep, recent, first_n) < 0:
        raise ValueError(f"{fn}: keep {keep}, first {first_n}, recent {recent}")
    if not 0 <= max_seq_len <= table.shape[1]:
        raise ValueError(f"{fn}: max_seq_len {max_seq_len} exceeds req_to_token width "
                         f"{table.shape[1]}")
    # (no row has more, and sums of theirs stay in 64 bits)
    keep, recent, first_n = (min(n, max_seq_len) for n in (keep, recent, first_n))
    width = max_seq_len - keep
    with _native.launching(device, stream):
        lens = torch.empty_strided((bsz,), (1,), dtype=torch.int64, device=device)
        freed = torch.empty_strided((bsz, width), (width, 1), dtype=torch.int64, device=device)
        if bsz:
            ws, nbytes = _scratch("tf_evict_workspace_bytes", device, max_seq_len,
                                  table.shape[1], bsz)
            _native.call("tf_evict_tokens", table.data_ptr(), table.shape[0], table.stride(0),
                         table.shape[1], scores.data_ptr(), scores.stride(0),
                         req_pool_indices.data_ptr(), _ptr(out_rows), seq_lens.data_ptr(),
                         first.data_ptr() if isinstance(first, torch.Tensor) else None, first_n,
                         recent, keep, max_seq_len, bsz, lens.data_ptr(),
                         freed.data_ptr() if width else None, width, _ptr(ws), nbytes,
                         _native.current_stream(device))
    return lens, freed
