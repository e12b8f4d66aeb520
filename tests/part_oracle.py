"""Slot attention in 64 bits on the CPU, with what the bounds of the kernels' error need."""
from __future__ import annotations

import torch

from oracle.kv_quant import dequantize_e4m3


def pool64(pool, scale):
    if pool.dtype == torch.float8_e4m3fn:
        return dequantize_e4m3(pool.cpu(), scale.float().cpu().item()).double()
    return pool.double().cpu()


def attention64(wl, window=None, seq_lens=None):
    """(out, spread, weights) of a workload: out [T, Hq, D], spread = the softmax-weighted
    |V| of every output, and per request the weight that the last ``window`` new tokens
    give its keys, summed over heads ([len] each; None: of every new token)."""
    k_pool, v_pool = pool64(wl.k_pool, wl.k_scale), pool64(wl.v_pool, wl.v_scale)
    table, q = wl.batch.req_to_token.cpu(), wl.q.double().cpu()
    lens = list(seq_lens) if seq_lens is not None else wl.seq_lens
    group = wl.num_q_heads // wl.num_kv_heads
    out, spread, weights, at = torch.zeros_like(q), torch.zeros_like(q), [], 0
    for row, n, e in zip(wl.rows, lens, wl.ext_lens):
        slots = table[row, :n].clamp(min=0)
        k = k_pool[slots].repeat_interleave(group, dim=1)
        v = v_pool[slots].repeat_interleave(group, dim=1)
        w = torch.zeros(n, dtype=torch.float64)
        for t in range(e):
            seen = n - e + t + 1
            if seen <= 0:
                continue
            s = torch.einsum("hd,khd->hk", q[at + t], k[:seen]) * wl.scale
            p = torch.softmax(s, dim=1)
            out[at + t] = torch.einsum("hk,khd->hd", p, v[:seen])
            spread[at + t] = torch.einsum("hk,khd->hd", p, v[:seen].abs())
            if window is None or t >= e - window:
                w[:seen] += p.sum(dim=0)
        weights.append(w)
        at += e
    return out, spread, weights


def score_error(wl):
    """Bound of what a score's rounding does to 2^s, relatively: D exact products of bf16
    values are added in fp32 (every addition rounds by 2^-24 of at most the sum of
    |q k|, itself at most |q| |k|), the sum is scaled and exponentiated."""
    qn = wl.q.double().norm(dim=2).max().item()
    kn = pool64(wl.k_pool, wl.k_scale).nan_to_num(0.0).norm(dim=2).max().item()
    return (wl.head_dim + 3) * 2.0 ** -24 * qn * kn * abs(wl.scale) + 2.0 ** -21


def assert_attention(got, want, spread, wl, what=""):
    """|error| <= half a bf16 step of the output, plus the probabilities' own: half a bf16
    step each at head_dim 256 (P enters the MFMA as bf16), none elsewhere (24 bits),
    and the scores' error, both weighted by |V|.  Subnormal outputs round by 2^-134."""
    p_step = 2.0 ** -8 if wl.head_dim == 256 else 2.0 ** -23
    eps = p_step + 2.0 * score_error(wl)
    bound = 2.0 ** -8 * want.abs() * (1 + eps) + eps * spread * (1 + 2.0 ** -8) + 2.0 ** -133
    err = (got.double().cpu() - want).abs()
    assert torch.isfinite(got.float()).all(), what
    worst = (err / bound).max().item()
    assert worst <= 1, f"{what}: error {worst:.2f} of its bound"
