// The streaming kernels' tile work: 16 tokens of K and V per wave and step against up
// to two groups of 16 query rows (decode.hip describes the scheme, prefix_attn.hip
// runs it over parts of contexts).
#pragma once

#include <math.h>

#include "tf_common.h"

namespace tfa {

constexpr int kWaves = 4;
constexpr int kTile = 16;       // tokens per wave iteration
constexpr int kMaxChunk = 2048; // slot ids staged in LDS at a time
constexpr int kMaxItems = 2048; // requests per launch (per-item prefix lives in LDS)

// The kernels' shape.  DP: head dims in a row's tile (256, or 128 for head dims up
// to 128); NG: groups of 16 query rows a unit holds (1 or 2: four groups of 256 dims
// spill); OTHER: head dims that do not fill the tile (chunks past the head dim are
// read as zeros and not written) and probabilities split into three bf16 parts, all
// of their 24 bits, which the PV product takes one after the other, smallest first
// (the kernel these head dims ran before kept them in fp32; two parts are off by up
// to 2^-18 and 1 to 5 % faster).  BLK: items are row blocks (DecodeArgs::blocks);
// else one token each, and every row sees every key of its item.
template <int DP_, bool FP8_, int NG_, bool OTHER_, bool BLK_>
struct Cfg {
  static constexpr int DP = DP_;
  static constexpr bool FP8 = FP8_;
  static constexpr int NG = NG_;
  static constexpr bool OTHER = OTHER_;
  static constexpr bool BLK = BLK_;
  static_assert(DP == 256 || (DP == 128 && !FP8), "tile width");
  static constexpr int kAcc = DP / 16;                 // f32x4 accumulators per lane and group
  static constexpr int kChunks = FP8 ? 16 : DP / 8;    // 16-byte chunks per row of the tile
  static constexpr int kS = kChunks / 16;              // chunks per lane and token
  static constexpr int kSteps = DP / 32;               // 32-dim MFMA steps of QK^T
  static constexpr int kRows = 16 * NG;                // query rows per unit
  static constexpr int kRowFloats = DP;                // a partial row's O
  static constexpr bool kRowPlan = OTHER || BLK;       // DecodeArgs::by_owner and ipre are set
};

template <class C>
struct WaveState {
  float m[C::NG], l[C::NG];
  f32x4 acc[C::NG][C::kAcc];
};

// LDS slot for one group of one wave's state, element-major so lanes hit
// consecutive banks.
template <class C>
struct StateSlot {
  f32x4 acc[C::kAcc][kWave];
  float m[kWave];
  float l[kWave];
};

// Per-wave K staging tile: 16 token rows x kChunks 16-byte chunks; chunk c of
// row r sits at r * kChunks + (c ^ r) so that both the coalesced writes and the
// MFMA-layout reads are free of bank conflicts.
template <class C>
struct DecodeSmem {
  union {
    struct {
      int32_t slots[kMaxChunk];                     // slot id of each staged token
      u32x4 kstage[kWaves][kTile * C::kChunks];     // per-wave K tile
    } loop;
    StateSlot<C> merge[2];                          // wave-state exchange
  } u;
  u32x4 qfrag[C::NG][C::kSteps][kWave];             // Q^T B-operand fragments, lane-major
  int32_t ipre[kMaxItems + 1];                      // exclusive prefix of per-item tiles
  int32_t wsum[kWaves];
};

// Per-lane register slices of one 16-token tile: K (staged to LDS for the
// S^T = K Q^T MFMA) and V (transposed in registers for the PV MFMA).
template <class C>
struct KBuf {
  u32x4 k[4][C::kS];   // row of token 4g + j, chunk n + 16 s
};
template <class C>
struct VBuf {
  u32x4 v[4][C::kS];
};

template <class C>
__device__ __forceinline__ void merge_into(WaveState<C>& st, int q, float m2, float l2,
                                           const f32x4* acc2) {
  const float M = fmaxf(st.m[q], m2);
  const float a1 = (st.m[q] == -INFINITY) ? 0.f : fast_exp2(st.m[q] - M);
  const float a2 = (m2 == -INFINITY) ? 0.f : fast_exp2(m2 - M);
  st.l[q] = st.l[q] * a1 + l2 * a2;
#pragma unroll
  for (int i = 0; i < C::kAcc; ++i) st.acc[q][i] = st.acc[q][i] * a1 + acc2[i] * a2;
  st.m[q] = M;
}

template <class C>
__device__ __forceinline__ void reset_state(WaveState<C>& st) {
#pragma unroll
  for (int q = 0; q < C::NG; ++q) {
    st.m[q] = -INFINITY;
    st.l[q] = 0.f;
#pragma unroll
    for (int i = 0; i < C::kAcc; ++i) st.acc[q][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

template <class C>
__device__ __forceinline__ void put_state(StateSlot<C>* s, int lane, const WaveState<C>& st,
                                          int q) {
#pragma unroll
  for (int i = 0; i < C::kAcc; ++i) s->acc[i][lane] = st.acc[q][i];
  s->m[lane] = st.m[q];
  s->l[lane] = st.l[q];
}

template <class C>
__device__ __forceinline__ void take_state(const StateSlot<C>* s, int lane, WaveState<C>& st,
                                           int q) {
  f32x4 acc2[C::kAcc];
#pragma unroll
  for (int i = 0; i < C::kAcc; ++i) acc2[i] = s->acc[i][lane];
  merge_into<C>(st, q, s->m[lane], s->l[lane], acc2);
}

// Tree merge of the 4 wave states, group by group; wave 0 ends up holding the
// block state.
template <class C>
__device__ __forceinline__ void block_merge(StateSlot<C>* slots, int w, int lane,
                                            WaveState<C>& st, int n_groups) {
#pragma unroll
  for (int q = 0; q < C::NG; ++q) {
    if (C::NG > 1 && q >= n_groups) break;
    __syncthreads();
    if (w >= 2) put_state<C>(&slots[w - 2], lane, st, q);
    __syncthreads();
    if (w < 2) take_state<C>(&slots[w], lane, st, q);
    __syncthreads();
    if (w == 1) put_state<C>(&slots[0], lane, st, q);
    __syncthreads();
    if (w == 0) take_state<C>(&slots[0], lane, st, q);
  }
}
// Issue the loads of tile `it` (chunk tokens it*16 .. it*16+15, clamped to the
// chunk's last token so every address is a valid row): lane (g, n) reads chunk
// n (+ 16 s) of the rows of tokens 4g + j, the same row-contiguous pattern for
// K (the MFMA layout is produced through LDS) and V.  The loads are nontemporal:
// one-token units stream every row once.  Blocks of one request read its rows
// again, each for itself, and plain loads serve those better (2 prompts beside 12
// decodes at 128 dims 94.8 and 84.2 us, 20 requests of 6 tokens at 256 153 and 143),
// but cost steps of many rows that are read once more (64 decodes beside 3 tokens
// 211 and 240, 64 requests of 5 tokens 232 and 256).  n_chunks: chunks of a row
// (OTHER).
template <class C>
__device__ __forceinline__ void issue_rows(u32x4 (&x)[4][C::kS], const int32_t* slots, int it,
                                           int n_loc, int g, int n, const uint8_t* base,
                                           int64_t slot_bytes, int n_chunks) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t sl = slots[min(it * kTile + 4 * g + j, n_loc - 1)];
    const uint8_t* p = base + sl * slot_bytes;
#pragma unroll
    for (int s = 0; s < C::kS; ++s) {
      if (C::OTHER)
        x[j][s] = n + 16 * s < n_chunks ? ld_nt16(p + 16 * n + 256 * s) : u32x4{0u, 0u, 0u, 0u};
      else
        x[j][s] = ld_nt16(p + 16 * n + 256 * s);
    }
  }
}

// Writes the tile's K chunks to this wave's LDS staging tile (swizzled).
template <class C>
__device__ __forceinline__ void stage_k(const KBuf<C>& kb, u32x4* ks, int g, int n) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = 4 * g + j;
#pragma unroll
    for (int s = 0; s < C::kS; ++s) ks[r * C::kChunks + ((n + 16 * s) ^ r)] = kb.k[j][s];
  }
}

// The staged tile's K fragments, bf16: k-step kk of lane (g, n) is row n, dims
// 32kk + 8g .. (bf16: chunk 4kk + g) or, for fp8, dims 64u + 16g .. (chunk
// 4u + g, two k-steps).
template <class C>
__device__ __forceinline__ void k_frags(const u32x4* ks, int g, int n, u32x4 (&kf)[C::kSteps]) {
  if (C::FP8) {
#pragma unroll
    for (int u = 0; u < C::kSteps / 2; ++u) {
      const u32x4 x = ks[n * 16 + ((4 * u + g) ^ n)];
      kf[2 * u] = e4m3x8_to_bf16x8(x[0], x[1]);
      kf[2 * u + 1] = e4m3x8_to_bf16x8(x[2], x[3]);
    }
  } else {
#pragma unroll
    for (int kk = 0; kk < C::kSteps; ++kk) kf[kk] = ks[n * C::kChunks + ((4 * kk + g) ^ n)];
  }
}

// S^T = K Q^T for the tile, then the online-softmax update of group q's row n,
// whose visible tokens are those below lim (chunk-local); returns the tile's
// probabilities packed as the PV B operand (P^T, 4 tokens per lane), pl their
// lower parts, smallest first (OTHER).  scored(sc): called with the lane's four scores
// (log2 units, -inf where masked).
template <class C, class Scored>
__device__ __forceinline__ u32x2 qk_softmax(const u32x4 (&kf)[C::kSteps],
                                            const u32x4 (&qf)[C::kSteps], int it, int lim, int g,
                                            float sl2, WaveState<C>& st, int q,
                                            u32x2 (&pl)[2], const Scored& scored) {
  f32x4 sacc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int kk = 0; kk < C::kSteps; ++kk) sacc = mfma_16x16x32(kf[kk], qf[kk], sacc);
  float sc[4];
  float mx = -INFINITY;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int t = it * kTile + 4 * g + r;
    sc[r] = (t < lim) ? sacc[r] * sl2 : -INFINITY;
    mx = fmaxf(mx, sc[r]);
  }
  scored(sc);
  mx = wave_max_xor(mx, 16);
  mx = wave_max_xor(mx, 32);
  const float mnew = fmaxf(st.m[q], mx);
  // A causal row may not have seen a key yet: exponents relative to 0 then.
  const float mref = C::BLK && mnew == -INFINITY ? 0.f : mnew;
  const float alpha = fast_exp2(st.m[q] - mref);
  float p[4];
  float psum = 0.f;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    p[r] = fast_exp2(sc[r] - mref);
    psum += p[r];
  }
  st.l[q] = st.l[q] * alpha + psum;
  st.m[q] = mnew;
  if (__ballot(alpha != 1.f)) {
#pragma unroll
    for (int i = 0; i < C::kAcc; ++i) st.acc[q][i] *= alpha;
  }
  const u32x2 ph = {pack_bf16(p[0], p[1]), pack_bf16(p[2], p[3])};
  if (C::OTHER) {   // (the differences are exact)
#pragma unroll
    for (int r = 0; r < 4; ++r) p[r] -= r & 1 ? bf16_hi(ph[r >> 1]) : bf16_lo(ph[r >> 1]);
    pl[1] = u32x2{pack_bf16(p[0], p[1]), pack_bf16(p[2], p[3])};
#pragma unroll
    for (int r = 0; r < 4; ++r) p[r] -= r & 1 ? bf16_hi(pl[1][r >> 1]) : bf16_lo(pl[1][r >> 1]);
    pl[0] = u32x2{pack_bf16(p[0], p[1]), pack_bf16(p[2], p[3])};
  }
  return ph;
}

// O^T += V^T P^T for the tile, every group.
template <class C>
__device__ __forceinline__ void pv(const VBuf<C>& vb, const u32x2 (&pt)[C::NG],
                                   const u32x2 (&pl)[C::NG][2], WaveState<C>& st,
                                   int n_groups) {
  auto mma = [&](int i, u32x2 va) {
#pragma unroll
    for (int q = 0; q < C::NG; ++q) {
      if (C::NG > 1 && q >= n_groups) break;
      if (C::OTHER) {
#pragma unroll
        for (int k = 0; k < 2; ++k) st.acc[q][i] = mfma_16x16x16(va, pl[q][k], st.acc[q][i]);
      }
      st.acc[q][i] = mfma_16x16x16(va, pt[q], st.acc[q][i]);
    }
  };
  if (C::FP8) {
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      const int dw = e >> 2;
      const uint32_t b0 = e & 3;
      const uint32_t sel = b0 | ((4 + b0) << 8) | ((b0 + 1) << 16) | ((5 + b0) << 24);
      const uint32_t x = __builtin_amdgcn_perm(vb.v[1][0][dw], vb.v[0][0][dw], sel);
      const uint32_t y = __builtin_amdgcn_perm(vb.v[3][0][dw], vb.v[2][0][dw], sel);
      mma(e, u32x2{e4m3x2_to_bf16x2<false>(x), e4m3x2_to_bf16x2<false>(y)});
      mma(e + 1, u32x2{e4m3x2_to_bf16x2<true>(x), e4m3x2_to_bf16x2<true>(y)});
    }
  } else {
#pragma unroll
    for (int s = 0; s < C::kS; ++s) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int dw = e >> 1;
        const int hi = e & 1;
        mma(8 * s + e, u32x2{pair_sel(vb.v[1][s][dw], vb.v[0][s][dw], hi),
                             pair_sel(vb.v[3][s][dw], vb.v[2][s][dw], hi)});
      }
    }
  }
}

__device__ __forceinline__ bool not_finite(const f32x4& v) {
  float y = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) y = fmaf(v[e], 0.f, y);
  return y != y;
}

// Whether any of the lane's accumulators is NaN or infinite.
template <class C>
__device__ __forceinline__ bool any_odd(const WaveState<C>& st) {
  f32x4 x[2] = {};   // (eight short chains)
#pragma unroll
  for (int q = 0; q < C::NG; ++q)
#pragma unroll
    for (int i = 0; i < C::kAcc; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i & 1][e] = fmaf(st.acc[q][i][e], 0.f, x[i & 1][e]);
  const float y = (x[0][0] + x[0][1] + x[0][2] + x[0][3]) + (x[1][0] + x[1][1] + x[1][2] + x[1][3]);
  return y != y;
}
// ipre[i] = sum of tiles(i) of items < i, ipre[n_items] = total (block-wide scan).
template <int WAVES = kWaves, class Tiles>
__device__ __forceinline__ void item_prefix(int n_items, const Tiles& tiles, int32_t* ipre,
                                            int32_t* wsum) {
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int w = wave_id();
  constexpr int kPer = kMaxItems / (WAVES * kWave);
  int t[kPer];
  int sum = 0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int i = tid * kPer + k;
    t[k] = i < n_items ? tiles(i) : 0;
    sum += t[k];
  }
  int incl = sum;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const int v = __shfl_up(incl, off, kWave);
    if (lane >= off) incl += v;
  }
  if (lane == kWave - 1) wsum[w] = incl;
  __syncthreads();
  int excl = incl - sum;
  for (int k = 0; k < w; ++k) excl += wsum[k];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int i = tid * kPer + k;
    if (i <= n_items) ipre[i] = excl;
    excl += t[k];
  }
  if (tid == WAVES * kWave - 1 && n_items == kMaxItems) ipre[kMaxItems] = excl;
  __syncthreads();
}
// Workgroup that owns global tile x when N tiles are split over P workgroups.
__device__ __forceinline__ int owner_of(int64_t x, int64_t N, int P) {
  return (int)(((x + 1) * P - 1) / N);
}

}  // namespace tfa
