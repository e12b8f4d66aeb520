// The streaming half of the attention over parts of contexts: prefix_attn.hip describes the
// scheme and launches it, extend.hip beside its MFMA tiles.
#pragma once

#include "prefix_attn.h"
#include "stream_tile.h"
#include "tf_common.h"

namespace tfa {

// The context length of a request, clamped to its table row.
__device__ __forceinline__ int context_len(const PartArgs& a, int b) {
  const int64_t len =
      min(a.seq_override > 0 ? (int64_t)a.seq_override : a.seq_lens[b], a.rtt_cols);
  return len > 0 ? (int)len : 0;
}

__device__ __forceinline__ PartItem item_at(const PartArgs& a, int i) {
  if (a.items) return a.items[i];
  const int b = i / a.head_blocks;
  return PartItem{b, b, 1, (i - b * a.head_blocks) * a.unit_rows, 0, -1, -1, 0};
}
__device__ __forceinline__ PartTok tok_at(const PartArgs& a, int i) {
  return a.toks ? a.toks[i] : PartTok{i, i, 0, 0};
}

// Keys that token t of an item sees, counted from key 0.
__device__ __forceinline__ int token_seen(const PartArgs& a, const PartTok& t) {
  return context_len(a, t.b) - t.back;
}

// Keys of an item: a shared part's own bounds (a row of a shorter context masks what
// lies behind it), else up to the last key that its last row sees.
template <class C>
__device__ __forceinline__ int part_keys(const PartArgs& a, const PartItem& it) {
  if (it.b < 0) return 0;
  int end;
  if (it.k1 >= 0) {
    end = min((int64_t)it.k1, a.rtt_cols);
  } else {
    const int last = min(it.row0 + C::kRows, it.n_tok * a.group) - 1;
    end = token_seen(a, tok_at(a, it.tok0 + last / a.group));
  }
  return max(0, end - it.k0);
}

// What a unit costs beside its tiles (its slot ids, queries and partials), in tiles.
constexpr int kUnitTiles = 8;
constexpr int kHalfTiles = 8;                    // a wave stages slot ids for 8 tiles ahead,
constexpr int kHalf = kHalfTiles * kTile;        // in two halves by turns

// Positions of an item's units: its tiles behind kUnitTiles positions without work.
__device__ __forceinline__ int unit_span(int tiles) { return tiles ? tiles + kUnitTiles : 0; }

// Scores on their way to memory (SCORED) wait in LDS, as many tiles' as there is room for
// (28 KB a wave: 74 tiles of 6 rows), since loads issued after a store are waited for
// behind it: stored at every tile, or at every 8 tiles, they took a fifth of the kernel's
// time (64 requests of 1k to 8k keys 239 us, 201 without stores).
template <class C> constexpr int kKeptFloats = C::DP == 128 ? 12 << 8 : 28 << 8;

template <class C, bool SCORED, int WAVES>
struct StreamSmem {
  struct {
    int32_t slots[2 * kHalf];
    u32x4 kstage[kTile * C::kChunks];          // see stage_k
    u32x4 qfrag[C::NG > 1 ? C::NG : 0][C::kSteps][kWave];   // (one group's stay in registers)
    float kept[SCORED ? kKeptFloats<C> : 0];
  } wave[WAVES];
  int32_t ipre[kMaxItems + 1];                 // exclusive prefix of the items' spans
  int32_t wsum[WAVES];
};

// SCORED: the scores are kept (16 bytes per row and four keys, a few percent of the keys'
// own bytes), for the weights that follow.
template <class C, bool SCORED, int WAVES>
__device__ __forceinline__ void part_stream(const PartArgs& a,
                                            StreamSmem<C, SCORED, WAVES>& sm, int block) {
  static_assert(!SCORED || C::NG == 1, "scored items are the heads of one token");
  const int D = C::OTHER ? a.head_dim : C::DP;
  const int row_bytes = C::FP8 ? D : 2 * D;
  const int n_chunks = row_bytes / 16;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int w = wave_id();
  const int g = lane >> 4;
  const int n = lane & 15;

  // (every item by a thread of its own first: three loads in a row each)
  int32_t* spans = reinterpret_cast<int32_t*>(&sm.wave[0]);
  static_assert(sizeof(sm.wave) >= 4 * kMaxItems, "spans of the items");
  for (int i = tid; i < a.n_items; i += WAVES * kWave)
    spans[i] = unit_span((part_keys<C>(a, item_at(a, i)) + kTile - 1) / kTile);
  __syncthreads();
  item_prefix<WAVES>(a.n_items, [&](int i) { return spans[i]; }, sm.ipre, sm.wsum);
  if (block == 0)
    for (int i = tid; i <= a.n_items; i += WAVES * kWave) a.ipre[i] = sm.ipre[i];
  // Every wave is a worker of its own: what a unit costs in front of its tiles (loads in
  // a row) is then hidden by the other waves of the CU, and nothing is joined here.
  const int64_t N = (int64_t)a.hkv * sm.ipre[a.n_items];
  const int P = (int)min<int64_t>(a.n_workers, N);   // (owners of a unit are consecutive)
  const int me = block * WAVES + w;
  if (me >= P) return;
  const int64_t x_end = (int64_t)(me + 1) * N / P;
  int64_t x = (int64_t)me * N / P;

  const float sl2 = a.scale_log2 * (C::FP8 ? a.k_scale[0] : 1.f);
  const int64_t slot_bytes = (int64_t)a.hkv * row_bytes;
  int32_t* const slots = sm.wave[w].slots;
  u32x4* const ks = sm.wave[w].kstage;

  int item = 0;   // the first whose units reach x
  {
    int lo = 0, hi = a.n_items - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((int64_t)a.hkv * sm.ipre[mid] <= x) lo = mid; else hi = mid - 1;
    }
    item = lo;
  }

  while (x < x_end) {
    // ---- the segment: unit (item, hk), tiles [t0, t1)
    while ((int64_t)a.hkv * sm.ipre[item + 1] <= x) ++item;
    const int span = sm.ipre[item + 1] - sm.ipre[item];
    const int64_t r = x - (int64_t)a.hkv * sm.ipre[item];
    const int hk = (int)(r / span);
    const int v0 = (int)(r - (int64_t)hk * span);
    const int v1 = (int)min<int64_t>(span, v0 + (x_end - x));
    x += v1 - v0;
    const int t0 = max(0, v0 - kUnitTiles), t1 = v1 - kUnitTiles;
    if (t0 >= t1) continue;

    const PartItem im = item_at(a, item);
    const int L = part_keys<C>(a, im);
    const int n_rows = im.n_tok * a.group - im.row0;       // of kRows
    const int n_groups = min((n_rows + 15) / 16, C::NG);
    const int64_t row = clamp_i64(a.rpi[im.b], 0, a.rtt_rows - 1);
    const int64_t* rtt = a.rtt + row * a.rtt_stride + im.k0;
    const uint8_t* kbase = a.k_pool + (int64_t)hk * row_bytes;
    const uint8_t* vbase = a.v_pool + (int64_t)hk * row_bytes;
    // Row n of group q: its token and head, and how many of the part's keys it sees.
    auto row_of = [&](int q, int& qrow, int& hq, int& seen) {
      const int rho = im.row0 + min(16 * q + n, n_rows - 1);
      const int t = rho / a.group;
      const PartTok tok = tok_at(a, im.tok0 + t);
      qrow = tok.qrow;
      hq = hk * a.group + rho - t * a.group;
      seen = token_seen(a, tok) - im.k0;
      return 16 * q + n < n_rows;
    };
    u32x4 qf[C::kSteps];
    int seen[C::NG];
#pragma unroll
    for (int q = 0; q < C::NG; ++q) {
      int qrow, hq;
      const bool ok = row_of(q, qrow, hq, seen[q]);
      const __bf16* qp = a.q + (int64_t)qrow * a.q_stride + (int64_t)hq * D;
#pragma unroll
      for (int kk = 0; kk < C::kSteps; ++kk) {
        const int d0 = C::FP8 ? (64 * (kk >> 1) + 16 * g + 8 * (kk & 1)) : (32 * kk + 8 * g);
        qf[kk] = ok && (!C::OTHER || d0 < D) ? ld_g16(qp + d0) : u32x4{0u, 0u, 0u, 0u};
      }
      if constexpr (C::NG > 1) {
#pragma unroll
        for (int kk = 0; kk < C::kSteps; ++kk) sm.wave[w].qfrag[q][kk][lane] = qf[kk];
      }
    }

    WaveState<C> st;
    reset_state<C>(st);
    const int c0 = t0 * kTile;                    // keys below are counted from here
    const int n_loc = min(L, t1 * kTile) - c0;
    const int n_tiles = t1 - t0;
    // Slot ids of half h: key k's at slots[k % (2 kHalf)]; keys past the last repeat it.
    int64_t ids[kHalf / kWave];
    auto fetch_ids = [&](int h) {
#pragma unroll
      for (int i = 0; i < kHalf / kWave; ++i)
        ids[i] = rtt[c0 + min(h * kHalf + i * kWave + lane, n_loc - 1)];
    };
    auto stage_ids = [&](int h) {
#pragma unroll
      for (int i = 0; i < kHalf / kWave; ++i)
        slots[(h & 1) * kHalf + i * kWave + lane] =
            (int32_t)pool_row(ids[i], a.pool_slots, a.seq_override > 0);
      wave_lds_sync();
    };
    auto issue = [&](u32x4 (&x)[4][C::kS], int it, const uint8_t* base) {
      issue_rows<C>(x, slots, it & (2 * kHalfTiles - 1), 2 * kHalf, g, n, base, slot_bytes,
                    n_chunks);
    };
    wave_lds_sync();
    fetch_ids(0);
    stage_ids(0);

    // (rows of a multiple of 16 floats and 4: no two of a lane group on one bank)
    const int kept_tiles = SCORED ? (kKeptFloats<C> / min(n_rows, 16) - 4) / kTile : 0;
    const int kept_row = kept_tiles * kTile + 4;
    int kept_from = 0;

    // ---- the tiles, loads a tile ahead (see decode_kernel)
    KBuf<C> kb;
    VBuf<C> vb;
    auto scores = [&](int it, u32x2 (&pt)[C::NG], u32x2 (&pl)[C::NG][2]) {
      u32x4 kf[C::kSteps];
      k_frags<C>(ks, g, n, kf);
#pragma unroll
      for (int q = 0; q < C::NG; ++q) {
        if constexpr (C::NG > 1) {
          if (q >= n_groups) break;
#pragma unroll
          for (int kk = 0; kk < C::kSteps; ++kk) qf[kk] = sm.wave[w].qfrag[q][kk][lane];
        }
        const int lim = min(n_loc, seen[q] - c0);
        pt[q] = qk_softmax<C>(kf, qf, it, lim, g, sl2, st, q, pl[q], [&](const float (&sc)[4]) {
          if constexpr (SCORED) {
            if (n < n_rows)
              *reinterpret_cast<f32x4*>(
                  &sm.wave[w].kept[n * kept_row + (it - kept_from) * kTile + 4 * g]) =
                  f32x4{sc[0], sc[1], sc[2], sc[3]};
          }
        });
      }
    };
    // The kept scores of tiles kept_from .. it go out once there is no room for more, and
    // at the last tile.
    auto flush = [&](int it, bool last) {
      if constexpr (SCORED) {
        if (!last && it - kept_from + 1 < kept_tiles) return;
        const int64_t k0 = c0 + kept_from * kTile;
        const int keys = (int)min<int64_t>((it - kept_from + 1) * kTile, a.score_cap - k0);
        float* rows = a.row_scores + ((int64_t)a.hkv * im.b + hk) * a.group * a.score_cap +
                      im.row0 * a.score_cap + k0;
        wave_lds_sync();
        for (int r = 0; r < min(n_rows, 16); ++r)
          for (int k = 4 * lane; k < keys; k += 4 * kWave)
            *reinterpret_cast<f32x4*>(rows + r * a.score_cap + k) =
                *reinterpret_cast<const f32x4*>(&sm.wave[w].kept[r * kept_row + k]);
        wave_lds_sync();
        kept_from = it + 1;
      }
    };
    u32x2 pt[C::NG], pl[C::NG][2];
    issue(kb.k, 0, kbase);
    issue(vb.v, 0, vbase);
    int it = 0;
    for (; it + 1 < n_tiles; ++it) {
      // The ids of the next half, read while this one's tiles go by; its place held the
      // half before, whose last tile is issued.
      const int at = it & (kHalfTiles - 1);
      if (at == 0)
        fetch_ids(it / kHalfTiles + 1);
      else if (at == kHalfTiles / 2)
        stage_ids(it / kHalfTiles + 1);
      wave_lds_sync();
      stage_k<C>(kb, ks, g, n);
      wave_lds_sync();
      __builtin_amdgcn_sched_barrier(0);
      issue(kb.k, it + 1, kbase);
      __builtin_amdgcn_sched_barrier(0);
      scores(it, pt, pl);
      pv<C>(vb, pt, pl, st, n_groups);
      __builtin_amdgcn_sched_barrier(0);
      issue(vb.v, it + 1, vbase);
      __builtin_amdgcn_sched_barrier(0);
      flush(it, false);
    }
    wave_lds_sync();
    stage_k<C>(kb, ks, g, n);
    wave_lds_sync();
    scores(it, pt, pl);
    pv<C>(vb, pt, pl, st, n_groups);
    flush(it, true);

#pragma unroll
    for (int q = 0; q < C::NG; ++q) {
      st.l[q] += __shfl_xor(st.l[q], 16, kWave);
      st.l[q] += __shfl_xor(st.l[q], 32, kWave);
    }
    // Partials of (worker, unit), a row's dims side by side.  Lane (g, n) holds of
    // row n the dims 128 s + 32 g + 8 r + e (bf16: accumulator 8 s + e) or 64 g + 16 r
    // + e (fp8), four neighbours per store.
    const int64_t slot = (int64_t)me + (int64_t)item * a.hkv + hk;
#pragma unroll
    for (int q = 0; q < C::NG; ++q) {
      if (16 * q + n >= n_rows) continue;
      const int64_t pr = slot * a.slot_rows + 16 * q + n;
      float* po = a.part_o + pr * C::DP;
#pragma unroll
      for (int i = 0; i < C::kAcc; i += 4)
#pragma unroll
        for (int rr = 0; rr < 4; ++rr)
          *reinterpret_cast<f32x4*>(po + (C::FP8 ? 64 * g + 16 * rr + i
                                                 : 128 * (i >> 3) + 32 * g + 8 * rr + (i & 7))) =
              f32x4{st.acc[q][i][rr], st.acc[q][i + 1][rr], st.acc[q][i + 2][rr],
                    st.acc[q][i + 3][rr]};
      if (g == 0) a.part_ml[pr] = float2{st.m[q], st.l[q]};
    }
  }
}

}  // namespace tfa
