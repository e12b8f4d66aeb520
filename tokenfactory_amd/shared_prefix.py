"""Attention of a step whose requests share prefixes.

Requests that hit the same radix-cache node hold the same slots in front
(``engine/scheduler.py:187-224``): samples of one prompt, a batch behind one system
prompt, branches of a conversation.  ``slot_based_attention`` reads every request's
whole context; ``shared_prefix_attention`` reads a group's shared keys and values once
for all of its requests, and each request's own behind them, and joins the two by their
softmax statistics.  Same inputs, output and semantics otherwise.  (Once for all at head_dim
256, and up to 128 of bf16 pools, where MFMA tiles take the shared part; elsewhere once per
32 query rows of a kv head, new tokens x query heads per kv head.)

``SharedPrefixes`` names the groups of a step.  It keeps the step's work lists on the
device, so that the layers of a model share them, as ``ForwardBatch`` carries those of
``slot_based_attention``.  There is no non-native path and no gradient.
"""
from __future__ import annotations

import threading
from typing import Dict, Iterable, List, Optional, Sequence, Tuple

import numpy as np
import torch

from . import _native
from .attention import (SHORT_ROWS, BatchLists, Route, _KV_DTYPES, _check_inputs, _cu_count,
                        _epilogue, _fork_join_events, _output, _plan_event, _pool_scales, _scratch,
                        _side_stream, _upload, _ws_lock, batch_lists, slot_based_attention)
from .fp8_linear import _ptr
from .planning import EXTEND_TILE_ROWS, plan_extend

MAX_PARTS = 2048          # parts of contexts in one launch
MAX_LAYOUTS = 64          # step layouts whose lists an object keeps
_captured: List[object] = []   # lists that captured graphs read


class SharedPrefixes:
    """The groups of a step: ``(members, length)`` each, members batch indices of
    requests whose table rows hold the same slots in their first ``length`` entries.  A
    request is in one group at most.  The lengths may exceed what a request sees (its
    rows mask the rest), so that one object serves a step's layers and, while the
    extend lengths stay the same, later steps too; ``seq_lens`` are read at launch, and
    lists are made again as ``max_seq_len`` grows (see ``planned_length``).

    A graph may capture calls once an eager call with the same layout has run (it
    uploads the lists; of several, those of the nearest ``max_seq_len`` are taken).  Its
    replays follow ``seq_lens``, but share out the CUs as for that length; lists that a
    graph reads stay allocated."""

    def __init__(self, groups: Iterable[Tuple[Sequence[int], int]]):
        self.groups: List[Tuple[List[int], int]] = []
        seen: set = set()
        for members, length in groups:
            members, length = [int(b) for b in members], int(length)
            if length < 0 or length > 0x7fffffff or any(b < 0 for b in members):
                raise ValueError(f"shared prefix of {length} tokens for requests {members[:8]}")
            if len(set(members)) != len(members) or seen.intersection(members):
                raise ValueError("a request appears twice in the groups")
            seen.update(members)
            if length and len(members) > 1:   # (nothing is shared otherwise)
                self.groups.append((members, length))
        self._last = max(seen, default=-1)
        self._longest = max((n for _, n in self.groups), default=0)
        self._lock = threading.Lock()
        self._plans: Dict[tuple, _Plan] = {}

    def _plan(self, batch, n_tok, n_q, n_kv, head_dim, kv_dtype, device) -> "_Plan":
        max_len = planned_length(int(batch.max_seq_len), self._longest)
        key = (device.index, batch.batch_size, n_tok, n_q, n_kv, head_dim, kv_dtype,
               batch.req_to_token.shape[1], tuple(batch.extend_lens), max_len)
        plan = self._plans.get(key)
        if plan is not None and plan.ready:
            return plan
        if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            # (lists cannot be made here: those of the layout that were made nearest by)
            with self._lock:
                made = [(abs(k[-1] - max_len), p) for k, p in self._plans.items()
                        if k[:-1] == key[:-1] and p.ready]
            if made:
                return min(made, key=lambda x: x[0])[1]
        elif plan is not None:
            return plan
        ext_lens = [int(e) for e in batch.extend_lens]
        if len(ext_lens) != batch.batch_size or sum(ext_lens) != n_tok \
                or min(ext_lens, default=1) < 1:
            raise ValueError(f"extend_lens {ext_lens[:8]}... do not match "
                             f"batch_size={batch.batch_size}, T={n_tok}")
        if self._last >= batch.batch_size:
            raise ValueError(f"request {self._last} of a batch of {batch.batch_size}")
        width = batch.req_to_token.shape[1]
        if any(n > width for _, n in self.groups):
            raise ValueError(f"a shared prefix exceeds req_to_token's width {width}")
        with self._lock:
            plan = self._plans.get(key)
            if plan is None:
                if len(self._plans) >= MAX_LAYOUTS:   # (calls under way hold their own)
                    del self._plans[next(iter(self._plans))]
                plan = self._plans[key] = _Plan(self.groups, ext_lens, n_q, n_kv, head_dim, device,
                                                _cu_count(device), max_len, kv_dtype)
            return plan


def _step_middle(n: int) -> int:
    """The middle of the step that holds n: steps of an eighth to a quarter of a length,
    the first of 64."""
    if n < 64:
        return 32
    shift = n.bit_length() - 3
    return ((n >> shift) << shift) + (1 << shift) // 2


def planned_length(max_len: int, longest: int) -> int:
    """The longest context that a plan is made for: a plan holds as long as what lies
    behind the longest shared part (or a context that does not reach its end) stays in one
    step of _step_middle, since the split of the CUs follows from the lengths (64 requests on
    8192 keys with 4096 of their own each: 211 us; 403 by the split of their first step,
    331 unshared)."""
    if max_len <= longest:
        return min(longest, _step_middle(max_len))
    return longest + _step_middle(max_len - longest)


KEYS_PER_STEP = 32   # of the extend kernel
MIN_STEPS = 2        # of a piece: 3 requests on 300 keys 18.3 us, with 8 18.5, with 16 21.9


def cut_units(steps: Sequence[int], cus: int) -> np.ndarray:
    """Pieces per unit, steps[i] steps of keys long: the shortest pieces of which there are
    no more than CUs (a piece more would be a round more), of MIN_STEPS at least."""
    steps = np.asarray(steps, dtype=np.int64)
    lo, hi = MIN_STEPS, max(MIN_STEPS, int(steps.max()))
    while lo < hi:
        mid = (lo + hi) // 2
        if (-(-steps // mid)).sum() <= cus:
            hi = mid
        else:
            lo = mid + 1
    return np.maximum(1, -(-steps // lo))


# Times in us that the split of a step is estimated with, by (narrow tiles, fp8 pool): of a
# streaming workgroup (8 waves) per unit and per 16 keys of it, of a step of 32 keys by MFMA
# tiles without and with all of their 256 rows.
_STEP_US = {(False, False): (3.0, 0.40, 0.45, 1.5), (False, True): (1.7, 0.21, 0.4, 1.9),
            (True, False): (2.0, 0.18, 0.3, 1.5)}


def _stream_share(steps: np.ndarray, rows: np.ndarray, own_units: np.ndarray,
                  own_keys: np.ndarray, n_kv: int, narrow: bool, fp8: bool, cus: int) -> int:
    """Workgroups, one per CU, that stream the requests' own parts beside the pieces of the
    shared ones: where both are estimated to end together.  steps, rows: of each MFMA unit;
    own_units (of 16 rows), own_keys: of each request's own part.  Measured with 64, 112,
    160 and 192 of 256: 64 requests on 8192 shared keys 75, 58, 52 and 63 us (two launches
    71), branches of 4 groups 74, 61, 54 and 51 (57), 96 on 2000 of 128 dims 84, 62, 51 and
    44 (62), 256 on 32768 of an fp8 pool 294, 318, 429 and 821 (330)."""
    unit, tile, step, full = _STEP_US[narrow, fp8]
    streams = n_kv * float((own_units * (unit + tile * own_keys / 16)).sum())
    total, longest = int(steps.sum()), int(steps.max())
    filled = np.minimum(rows, EXTEND_TILE_ROWS) / EXTEND_TILE_ROWS
    per_step = float((steps * (step + (full - step) * filled)).sum()) / total

    def end(n):   # (pieces are whole: the longest unit is cut into as many as it can)
        parts = max(1, (cus - n) * longest // total)
        rounds = max(1.0, len(steps) / (cus - n))
        return max(10 + streams / n, 12 + per_step * rounds * -(-longest // parts))

    return min(range(max(1, cus // 16), cus * 7 // 8 + 1, max(1, cus // 32)), key=end)


def _streams_all(rows: np.ndarray, keys: np.ndarray, own_keys: int, n_kv: int, cus: int) -> bool:
    """Whether the shared parts (rows and keys of each) are streamed as the requests' own are, in
    units of 16 rows, and not by MFMA tiles: where a unit holds a part's rows, so that its
    keys are still read once, and either the parts are many (32 groups of 2 on 500 keys 37
    us, 50 by tiles, 500 of 2 on 2000 964 and 1046) or own keys are nearly all (2 requests
    on 100 keys beside 62 of 4k: 119 and 128).  One group of 4 on 8000 keys, 16 rows of
    128 dims: 39 us streamed, whose merge joins hundreds of waves' partials, 22 by tiles."""
    return rows.max() <= 16 and (4 * n_kv * len(rows) >= cus or 8 * keys.sum() <= own_keys)


def _ragged(values: np.ndarray, counts: np.ndarray) -> Tuple[np.ndarray, np.ndarray]:
    """values[i] counts[i] times, and each one's number among those of its i."""
    ends = np.cumsum(counts)
    total = int(ends[-1]) if len(ends) else 0
    return np.repeat(values, counts), np.arange(total) - np.repeat(ends - counts, counts)


def _items(*columns) -> np.ndarray:
    return np.stack(np.broadcast_arrays(*columns), axis=1)


class _Plan:
    """The device lists of one step layout: parts of contexts and their tokens; the pieces of
    shared ones where MFMA tiles take them; and at head_dim 256 the extend kernel's
    entries of long prompts, which share nothing (MFMA-bound) and may be cut over their
    keys as in ``slot_based_attention``."""

    def __init__(self, groups, ext_lens, n_q, n_kv, head_dim, device, cus, max_len, kv_dtype):
        group = n_q // n_kv
        fp8 = kv_dtype == _native.TF_DTYPE_FP8_E4M3
        self.device, self.n_q, self.n_kv = device, n_q, n_kv
        ext = np.asarray(ext_lens, dtype=np.int64).reshape(-1)
        starts = np.cumsum(ext) - ext
        long_ = (ext * group > SHORT_ROWS) & (head_dim == 256)
        own = np.flatnonzero(~long_)   # requests with parts
        groups = [([b for b in m if not long_[b]], n) for m, n in groups]
        groups = [(m, n) for m, n in groups if len(m) > 1]
        self.shares = bool(groups)
        members = np.asarray([b for m, _ in groups for b in m], dtype=np.int64)
        first = np.asarray([m[0] for m, _ in groups], dtype=np.int64)
        sizes = np.asarray([len(m) for m, _ in groups], dtype=np.int64)
        lengths = np.asarray([n for _, n in groups], dtype=np.int64)
        group_of = np.repeat(np.arange(len(groups)), sizes)   # of members
        n_toks = np.bincount(group_of, weights=ext[members],
                             minlength=len(groups)).astype(np.int64)
        shared_rows, rows = n_toks * group, ext[own] * group
        prefix = np.zeros(len(ext), dtype=np.int64)
        prefix[members] = lengths[group_of]
        # (own parts are taken to be half full: the host knows the longest context alone)
        own_keys = np.maximum(0, max_len - prefix[own]) // 2
        mfma = self.shares and (head_dim == 256 or (head_dim <= 128 and not fp8)) \
            and not _streams_all(shared_rows, lengths, int(own_keys.sum()), n_kv, cus)
        # (Units of 16 rows stream beside the pieces, which outweighs that up to 64 rows read
        # their keys four times: 4 groups of 8 of 6 tokens on 4000 keys 58 us, 82 in units of
        # 32; 12 of 10 on 1000 35 and 51; with own parts of up to 2000 keys, 4 groups of 8
        # of 10, 149 and 132.)
        most = int(max([1, *rows.tolist(), *([] if mfma else shared_rows.tolist())]))
        self.row_groups = 2 if most > (64 if mfma else 16) else 1
        unit = 16 * self.row_groups
        self.slot_rows = min(unit, most)

        # Tokens: the groups', then the requests' own.
        reqs = np.concatenate([members, own])
        b, t = _ragged(reqs, ext[reqs])
        tokens = np.stack([starts[b] + t, b, ext[b] - 1 - t, np.zeros_like(b)], axis=1)
        tok0 = np.cumsum(ext[reqs]) - ext[reqs]
        group_tok0 = tok0[np.cumsum(sizes) - sizes] if len(groups) else lengths
        part = np.full(len(ext), -1, dtype=np.int64)      # a request's shared part
        part_tok = np.zeros(len(ext), dtype=np.int64)     # its first token among that one's
        part_tok[members] = tok0[:len(members)] - group_tok0[group_of]

        self.n_stream = self.n_shared = self.n_pieces = 0
        items, pieces, units = [], [], []
        if mfma:
            # Units: 256 rows of a group for a kv head each; pieces of their keys.
            blocks = -(-shared_rows // EXTEND_TILE_ROWS)
            g, hk = _ragged(np.arange(len(groups)), blocks * n_kv)
            row0, hk = EXTEND_TILE_ROWS * (hk // n_kv), hk % n_kv
            steps = -(-lengths[g] // KEYS_PER_STEP)
            if self.row_groups == 1:
                self.n_stream = _stream_share(steps, shared_rows[g] - row0, -(-rows // 16),
                                              own_keys, n_kv, head_dim != 256, fp8, cus)
            cuts = cut_units(steps, cus - self.n_stream)
            units = np.stack([np.cumsum(cuts) - cuts, cuts], axis=1)
            u, i = _ragged(np.arange(len(g)), cuts)
            g, k0, k1 = g[u], steps[u] * i // cuts[u], steps[u] * (i + 1) // cuts[u]
            pieces = np.stack([first[g], hk[u], row0[u], group_tok0[g], n_toks[g],
                               KEYS_PER_STEP * k0, np.minimum(KEYS_PER_STEP * k1, lengths[g]),
                               np.arange(1, len(u) + 1)], axis=1)
            self.n_pieces = len(pieces)
            part[members] = ((np.cumsum(blocks) - blocks) * n_kv)[group_of]
        elif self.shares:
            n_units = -(-shared_rows // unit)
            g, i = _ragged(np.arange(len(groups)), n_units)
            items = _items(first[g], group_tok0[g], n_toks[g], unit * i, 0, lengths[g], -1, 0)
            self.n_shared = len(items)
            part[members] = (np.cumsum(n_units) - n_units)[group_of]
        at, i = _ragged(np.arange(len(own)), -(-rows // unit))
        b = own[at]
        own_items = _items(b, tok0[len(members):][at], ext[b], unit * i, prefix[b], -1, part[b],
                           part_tok[b])
        items = np.concatenate([items, own_items]) if self.n_shared else own_items
        self.n_items = len(items)
        work, self.route = [], None
        if long_.any():
            work = plan_extend(ext_lens, n_q, n_kv, decode_to_decode_kernel=True)
            work = work[long_[work[:, 0]]]
            long_lens = ext[long_].tolist()
            self.route = Route(long_lens, sum(long_lens), n_q, n_kv, head_dim, kv_dtype, len(work),
                               exact=True, max_len=max_len, cus=cus)
        self.n_work = len(work)
        parts = [np.asarray(x, dtype=np.int32).reshape(-1)
                 for x in (items, work, pieces, tokens, units)]
        self._offsets = np.cumsum([0] + [4 * len(x) for x in parts])[:5].tolist()
        self._host = np.concatenate(parts)
        self._lock = threading.Lock()
        self._lists: Optional[torch.Tensor] = None
        self._users: set = set()
        self._event = None
        self._addresses: List[int] = []
        self._kept = False

    @property
    def ready(self) -> bool:
        """Whether a captured call finds its lists (or needs none)."""
        return self._lists is not None or not self.shares

    def lists(self) -> List[int]:
        """Addresses of (items, work, pieces, tokens, units) for launches on the current
        stream."""
        capturing = torch.cuda.is_current_stream_capturing()
        if not capturing and _native.current_stream(self.device) in self._users:
            return self._addresses
        stream = torch.cuda.current_stream(self.device)
        with self._lock:
            if self._lists is None:
                if capturing:
                    raise RuntimeError("shared prefixes cannot be planned in a graph capture: "
                                       "run the call once before it")
                self._lists = _upload(self._host, self.device, stream)
                self._addresses = [self._lists.data_ptr() + at for at in self._offsets]
                with _ws_lock:
                    self._event = _plan_event(self.device, stream)
                    self._event.record(stream)
                self._users.add(stream.cuda_stream)
            elif stream.cuda_stream not in self._users and not capturing:
                # (torch waits for the device before it captures)
                self._lists.record_stream(stream)
                stream.wait_event(self._event)
                self._users.add(stream.cuda_stream)
            if capturing and not self._kept:
                self._kept = True
                _captured.append(self._lists)
        return self._addresses

    def cut_prompts(self, batch, work: int) -> torch.Tensor:
        """The long prompts' entries (at ``work``) cut over their keys, by the batch's lengths: the
        batch keeps them for its other calls; a captured call cuts them in the graph."""
        stream = torch.cuda.current_stream(self.device)
        if torch.cuda.is_current_stream_capturing():
            cut = _PromptPieces(self, work)
            cut._launch(batch, stream)
        else:
            cut = batch_lists(batch, self, lambda: _PromptPieces(self, work))
            cut.ensure(batch, stream)
        return cut.lists


class _PromptPieces(BatchLists):
    def __init__(self, plan: _Plan, work: int):
        super().__init__(plan.device, None, plan.route.alloc(plan.device))
        self._plan, self._work = plan, work

    def _launch(self, batch, stream: torch.cuda.Stream) -> None:
        plan = self._plan
        plan.route.plan(self.lists, self._work, plan.n_work, None, None, 0, plan.n_q, plan.n_kv,
                        batch, stream)


def shared_prefix_attention(
    q: torch.Tensor,
    layer_k_buffer: torch.Tensor,
    layer_v_buffer: torch.Tensor,
    batch,
    shared: SharedPrefixes,
    *,
    scaling: Optional[float] = None,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    gate: Optional[torch.Tensor] = None,
    out_amax: Optional[torch.Tensor] = None,
    stream: Optional[torch.cuda.Stream] = None,
) -> torch.Tensor:
    """``slot_based_attention(q, layer_k_buffer, layer_v_buffer, batch)`` for a batch
    whose ``shared`` groups' keys and values are read once per group (head_dim 256, or up to
    128 with a bf16 pool), or once per 32 query rows of a kv head (other head dims: 64
    requests on 8192 keys, 32 / 8 heads of 128 in fp8, 172 us for 483 unshared; in bf16 58
    for 321); the first member's table row is the one read.  Arguments and result as there
    (sums are joined in another order, so bf16 results may differ in the last bit).

    Worth it where the shared part is most of what a step reads.  A few requests with little
    in common lose: 4 on 512 shared keys with up to 6000 of their own 37 us for 27.

    Steps in which nothing is shared run ``slot_based_attention`` itself: no group of two
    requests with few new tokens (prompts of more than 64 rows, new tokens x query heads
    per kv head, are bound by their products at head_dim 256, not by their keys' bytes),
    an fp8 pool whose head_dim is not a multiple of 16, more than 2048 parts, or a negative
    ``scaling`` (the tiles follow a row's largest product)."""
    fn = "shared_prefix_attention"
    _native.refuse_gradients(fn, q, layer_k_buffer, layer_v_buffer, gate)
    _check_inputs(q, layer_k_buffer, layer_v_buffer, batch)
    n_tok, n_q, head_dim = q.shape
    n_slots, n_kv, _ = layer_k_buffer.shape
    if n_q % n_kv:
        raise ValueError(f"num_q_heads {n_q} is not a multiple of num_kv_heads {n_kv}")
    kv_dtype = _KV_DTYPES[layer_k_buffer.dtype]
    with _native.launching(q.device, stream):
        plan = shared._plan(batch, n_tok, n_q, n_kv, head_dim, kv_dtype, q.device)
        if not plan.shares or plan.n_items > MAX_PARTS \
                or (scaling is not None and not scaling >= 0) \
                or (kv_dtype == _native.TF_DTYPE_FP8_E4M3 and head_dim % 16):
            return slot_based_attention(q, layer_k_buffer, layer_v_buffer, batch, scaling=scaling,
                                        k_scale=k_scale, v_scale=v_scale, out=out, gate=gate,
                                        out_amax=out_amax)
        scaling = head_dim ** -0.5 if scaling is None else float(scaling)
        k_scale, v_scale = _pool_scales(q, kv_dtype, k_scale, v_scale)
        if q.stride(2) != 1 or q.stride(1) != head_dim:
            q = q.contiguous()
        out = _output(q, out)
        epilogue = _epilogue(q, gate, out_amax)
        items, work, pieces, tokens, units = plan.lists()
        rtt = batch.req_to_token
        pool = (layer_k_buffer.data_ptr(), layer_v_buffer.data_ptr(), n_slots, kv_dtype,
                _ptr(k_scale), _ptr(v_scale), rtt.data_ptr(), rtt.shape[0], rtt.stride(0),
                rtt.shape[1], batch.req_pool_indices.data_ptr(), batch.seq_lens.data_ptr())
        ws, nbytes = _scratch("tf_attn_shared_workspace_bytes", q.device, plan.n_items,
                              plan.row_groups, plan.slot_rows, plan.n_pieces, plan.n_stream,
                              n_q, n_kv, head_dim, kv_dtype)

        def parts(handle):
            _native.call("tf_attn_shared", q.data_ptr(), q.stride(0), *pool, items, plan.n_items,
                         plan.n_shared, tokens, plan.row_groups, plan.slot_rows, pieces,
                         plan.n_pieces, units, plan.n_stream, n_q, n_kv, head_dim, scaling,
                         out.data_ptr(), out.stride(0), ws.data_ptr(), nbytes, *epilogue, handle)

        if not plan.n_work:
            parts(_native.current_stream(q.device))
            return out
        # Long prompts' entries, and the parts beside them on a second stream: they write
        # other rows of out, and take the CUs that the entries leave.
        main, side = torch.cuda.current_stream(q.device), _side_stream(q.device)
        fork, join = _fork_join_events(q.device, main)
        fork.record(main)
        if plan.route.split:
            cut = plan.cut_prompts(batch, work)
            work = cut.data_ptr()
            split_ws = torch.empty(_native.load().tf_attn_extend_split_workspace_bytes(),
                                   dtype=torch.uint8, device=q.device)
            _native.call("tf_attn_extend_split", q.data_ptr(), q.stride(0), *pool, 0, work,
                         plan.route.n_pieces, work + 32 * plan.route.n_pieces,
                         plan.route.n_merges, split_ws.data_ptr(), split_ws.numel(), n_q, n_kv,
                         scaling, out.data_ptr(), out.stride(0), *epilogue, main.cuda_stream)
        else:
            _native.call("tf_attn_extend", q.data_ptr(), q.stride(0), *pool, 0, work, plan.n_work,
                         n_q, n_kv, head_dim, scaling, out.data_ptr(), out.stride(0), *epilogue,
                         main.cuda_stream)
        side.wait_event(fork)
        parts(side.cuda_stream)
        join.record(side)
        main.wait_event(join)
    return out
