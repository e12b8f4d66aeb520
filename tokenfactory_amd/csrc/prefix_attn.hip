// Attention over parts of contexts, joined: steps whose requests share a prefix
// (tf_attn_shared), its keys read once for all of them (at some head dims once per 32 of
// their rows, see below).
//
// The softmax over a row's keys splits at any key: with m_i, l_i and o_i the maximum,
// the sum of 2^(s - m_i) and the sum of 2^(s - m_i) V over part i,
//   m = max m_i,  l = sum l_i 2^(m_i - m),  o = sum o_i 2^(m_i - m) / l.
// Part items are (query tokens, keys [k0, k1) of one request's table row): a group's
// shared keys are an item with the tokens of all of its requests, the keys behind them
// one item per request, or several where it has more rows than a unit.  Every item
// leaves fp32 partials, which part_merge_kernel joins.
//
// Shared parts go through MFMA tiles instead (but many parts of few rows, or where nearly all
// keys are own ones: shared_prefix.py has the rule and its figures), cut over their keys so that
// every CU has a piece: the extend kernel's at head_dim 256 (extend.hip, kPrefix),
// prefix_tiles.hip's up to 128 of bf16 pools.  Where the requests' own rows fit units of 16,
// up to four each, own parts are streamed by other workgroups of the same launch: the tiles
// keep the MFMA units busy, the streams wait for their loads, and at 256 dims a tile
// workgroup's LDS leaves no room for a stream's on its CU.
//
// At other head dims (fp8 pools up to 128, any from 129 to 255) shared parts are streamed in
// units of 16 or 32 rows, each of which reads the part's keys for itself: 64 requests on 8192
// keys, 32 / 8 heads of 128 in fp8, are 8 units, 172 us (unshared 483; in bf16 by tiles 58),
// 16 / 4 heads of 192 in bf16 112 (307).
//
// part_stream_kernel does the decode kernel's tile work (decode.hip) with waves that
// work alone: a persistent wave owns an equal share of all units' tiles (unit = (item, kv
// head)), and what it finds of a unit is a partial of its own.  With a unit's start
// counted as 8 tiles this is what short and ragged contexts need: 64 requests of 1 to
// 1024 keys (139 MB) take 30 us, 45 in the decode kernel, whose workgroups join their
// waves at the end of every unit; 64 of 4096 keys 165 us (6.5 TB/s) and 168.  Bound by
// HBM, or by the latency of a unit's first loads where contexts are short.
#include <math.h>

#include <algorithm>

#include "attn_row.h"
#include "part_stream.h"
#include "prefix_attn.h"
#include "stream_tile.h"
#include "tf_common.h"
#include "tf_internal.h"

namespace tfa {
namespace {

template <class C, bool SCORED>
__global__ void __launch_bounds__(kWaves * kWave,
                                  (C::NG == 1 && !SCORED) || C::DP == 128 ? 2 : 1)
part_stream_kernel(PartArgs a) {
  __shared__ StreamSmem<C, SCORED, kWaves> sm;
  part_stream<C, SCORED, kWaves>(a, sm, blockIdx.x);
}

// Joins the parts of every row: WPR waves per row take its partials in turn, kAhead of
// them in flight per wave, lane l dims 4 l .. 4 l + 3.  Bound by the latency of those
// reads (and by their bytes where a prefix is cut into many pieces).  A row whose sum
// is not finite is done again over the keys it sees: an MFMA multiplies V rows that a
// row does not see by zero, which is NaN for an infinite or NaN value there.  So is one
// whose sum is zero: its keys all score -inf (or below the tiles' first reference maximum),
// or it sees none, for which nothing is read again and zeros are written.
constexpr int kMergeWaves = 8;
constexpr int kAhead = 8;

// Owners of a streamed unit's partials: slots first .. first + count - 1.
struct Owners {
  int64_t first;
  int count;
};
__device__ __forceinline__ Owners unit_owners(const PartArgs& a, int item, int hk) {
  const int before = a.ipre[item], span = a.ipre[item + 1] - before;
  if (span == 0) return Owners{0, 0};
  const int64_t N = (int64_t)a.hkv * a.ipre[a.n_items];
  const int64_t p = (int64_t)a.hkv * before + (int64_t)hk * span;
  const int P = (int)min<int64_t>(a.n_workers, N);
  const int b0 = owner_of(p + kUnitTiles, N, P);
  return Owners{b0 + (int64_t)item * a.hkv + hk, owner_of(p + span - 1, N, P) - b0 + 1};
}

// The weights of a scored call: workgroups of the merge launch in front of the units'
// (neither reads what the other writes).  Each takes the sums of 2^score of its request's
// rows from the partials, then of kWeightKeys keys at a time
//   scores[row, k] (+)= sum over the heads of 2^(score - lse),
// four keys a thread, a quarter of the threads for every fourth head, added in a fixed
// order.  Bound by latency (of few keys) or by reading the scores: the whole launch takes
// 6.9 us for one request of 900 keys and 20 for 64 of 1k to 8k (28 MB of scores; twice and
// four times as many workgroups change nothing).
constexpr int kMergeThreads = kMergeWaves * kWave;
constexpr int kWeightHeads = kMergeThreads / 16;   // heads at a time
constexpr int kWeightKeys = kMergeThreads;

__device__ void add_weights(const PartArgs& a, int block) {
  __shared__ float lse[kWeightHeads];
  __shared__ f32x4 part[3][kWeightKeys / 4];
  const int lane = threadIdx.x & 63;
  const int quarter = wave_id() / 2, at = threadIdx.x % (kWeightKeys / 4);
  const int b = block / a.weight_blocks;
  const int hq = a.hkv * a.group;
  const int64_t len = min((int64_t)context_len(a, b), a.score_cap);
  const int64_t first = (int64_t)(block % a.weight_blocks) * kWeightKeys;
  if (first >= len) return;
  float* out = a.scores + clamp_i64(a.rpi[b], 0, a.rtt_rows - 1) * a.scores_stride;
  for (int h0 = 0; h0 < hq; h0 += kWeightHeads) {
    const int n_heads = min(kWeightHeads, hq - h0);
    __syncthreads();   // (the heads before are done with lse)
    {   // sixteen lanes per head, four partials in flight each
      const int i = threadIdx.x / 16, h = h0 + min(i, n_heads - 1);
      const int hk = h / a.group, r = h - hk * a.group;
      const Owners own = unit_owners(a, b * a.head_blocks + r / a.unit_rows, hk);
      float m = -INFINITY, l = 0.f;
      auto join = [&](float m2, float l2) {
        const float mn = fmaxf(m, m2);
        const float ref = mn == -INFINITY ? 0.f : mn;
        l = l * fast_exp2(m - ref) + l2 * fast_exp2(m2 - ref);
        m = mn;
      };
      for (int k = lane & 15; k < own.count; k += 64) {
        float2 ml[4];
#pragma unroll
        for (int c = 0; c < 4; ++c)
          ml[c] = a.part_ml[(own.first + min(k + 16 * c, own.count - 1)) * a.slot_rows +
                            r % a.unit_rows];
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (k + 16 * c < own.count) join(ml[c].x, ml[c].y);
      }
#pragma unroll
      for (int d = 8; d >= 1; d >>= 1)
        join(__shfl_xor(m, d, kWave), __shfl_xor(l, d, kWave));
      // (a NaN sum makes every weight of its row NaN, and so does -inf, of a row whose keys
      // all score -inf: every row sees one)
      if ((lane & 15) == 0) lse[i] = m + log2f(l);
    }
    const float* rows = a.row_scores + ((int64_t)b * hq + h0) * a.score_cap;
    for (int64_t k0 = first; k0 < len; k0 += (int64_t)a.weight_blocks * kWeightKeys) {
      const int64_t k = k0 + 4 * at;
      constexpr int kMine = kWeightHeads / 4;
      f32x4 s[kMine], sum = {0.f, 0.f, 0.f, 0.f};
      const bool live = k < len;
#pragma unroll
      for (int i = 0; i < kMine; ++i)
        if (live && quarter + 4 * i < n_heads)
          s[i] = *reinterpret_cast<const f32x4*>(rows + (quarter + 4 * i) * a.score_cap + k);
      __syncthreads();   // lse is there, and the keys before are done with part
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        if (quarter + 4 * i >= n_heads) break;
        const float off = lse[quarter + 4 * i];
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += fast_exp2(s[i][e] - off);
      }
      if (quarter) part[quarter - 1][at] = sum;
      __syncthreads();
      if (quarter == 0 && live) {
        for (int c = 0; c < 3; ++c) sum += part[c][at];
        const bool adds = a.add_scores || h0 > 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (k + e < len) out[k + e] = adds ? out[k + e] + sum[e] : sum[e];
      }
    }
  }
}

template <int DP, bool FP8, int WPR, bool SCORED>
__global__ void __launch_bounds__(kMergeWaves * kWave) part_merge_kernel(PartArgs a) {
  int unit = blockIdx.x;
  if constexpr (SCORED) {
    unit -= a.n_weights;
    if (unit < 0) {
      if (blockIdx.y == 0) add_weights(a, blockIdx.x);
      return;
    }
  }
  constexpr int kRows = kMergeWaves / WPR;   // rows of the unit side by side
  __shared__ f32x4 so[kMergeWaves][kWave];
  __shared__ float sm_m[kMergeWaves], sm_l[kMergeWaves];
  const int lane = threadIdx.x & 63;
  const int w = wave_id();
  const int item = a.own0 + unit / a.hkv;
  const int hk = unit % a.hkv;
  const PartItem im = item_at(a, item);
  const int n = (int)blockIdx.y * kRows + w / WPR;     // the wave's row of the unit
  const int n_rows = im.b < 0 ? 0 : min(im.n_tok * a.group - im.row0, a.unit_rows);
  if ((int)blockIdx.y * kRows >= n_rows) return;
  bool write = n < n_rows;

  const int rho = im.row0 + min(n, n_rows - 1);
  const int t = rho / a.group;
  const PartTok tok = tok_at(a, im.tok0 + t);
  const int hq = hk * a.group + rho - t * a.group;
  const int D = a.head_dim;
  const bool lane_in = 4 * lane < DP, lane_out = 4 * lane < D;
  u32x2 gv = {0u, 0u};
  if (write && a.gate && lane_out)
    gv = ld_g8(a.gate + (int64_t)tok.qrow * a.gate_stride + (int64_t)hq * a.gate_hstride +
               4 * lane);

  // Partials: the request's own part, then the shared one's.
  const Owners own = unit_owners(a, item, hk);
  Owners pre{0, 0};
  const float2* pre_ml = a.part_ml;   // of row `pre_row` of slot pre.first, and on
  const float* pre_o = a.part_o;
  int pre_rows = a.slot_rows, pre_row = 0;
  if (im.pfx >= 0) {
    const int rp = (im.pfx_tok + t) * a.group + rho - t * a.group;
    if (a.units) {
      const int2 u = a.units[im.pfx + rp / kExtendItemRows * a.hkv + hk];
      pre = Owners{u.x, u.y};
      pre_ml = a.piece_ml;
      pre_o = a.piece_o;
      pre_rows = kExtendItemRows;
    } else {
      pre = unit_owners(a, im.pfx + rp / a.unit_rows, hk);
    }
    pre_row = rp % (a.units ? kExtendItemRows : a.unit_rows);
  }
  float m = -INFINITY, l = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  const int parts = write ? own.count + pre.count : 0;
  for (int k0 = w % WPR; k0 < parts; k0 += WPR * kAhead) {
    f32x4 o[kAhead];
    float2 ml[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = min(k0 + WPR * k, parts - 1);
      const bool mine = i < own.count;
      const int64_t pr = mine ? (own.first + i) * a.slot_rows + n
                              : (pre.first + i - own.count) * pre_rows + pre_row;
      ml[k] = (mine ? a.part_ml : pre_ml)[pr];
      o[k] = lane_in ? reinterpret_cast<const f32x4*>((mine ? a.part_o : pre_o) + pr * DP)[lane]
                     : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    float mn = m;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (k0 + WPR * k >= parts) ml[k] = float2{-INFINITY, 0.f};   // a repeat of the last one
      mn = fmaxf(mn, ml[k].x);
    }
    // (NaN rows have a maximum of -inf and a NaN sum: the sum goes through)
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float a1 = fast_exp2(m - ref);
    acc *= a1;
    l *= a1;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const float a2 = fast_exp2(ml[k].x - ref);
      // (a part without a key for the row may not have written its O)
      if (k0 + WPR * k < parts && ml[k].y != 0.f) acc += o[k] * a2;
      l += ml[k].y * a2;
    }
    m = mn;
  }
  if (WPR > 1) {
    so[w][lane] = acc;
    if (lane == 0) {
      sm_m[w] = m;
      sm_l[w] = l;
    }
    __syncthreads();
    if (w % WPR) write = false;   // the row's first wave goes on alone
    if (write) {
#pragma unroll
      for (int k = 1; k < WPR; ++k) {
        const float m2 = sm_m[w + k], l2 = sm_l[w + k];
        const float mn = fmaxf(m, m2);
        const float ref = mn == -INFINITY ? 0.f : mn;
        const float a1 = fast_exp2(m - ref), a2 = fast_exp2(m2 - ref);
        acc = acc * a1 + so[w + k][lane] * a2;
        l = l * a1 + l2 * a2;
        m = mn;
      }
    }
  }

  uint32_t om = 0;
  const float vscale = FP8 ? a.v_scale[0] : 1.f;
  __bf16* orow = a.out + (int64_t)tok.qrow * a.out_stride + (int64_t)hq * D;
  if (write && (l == 0.f || __ballot(not_finite(acc)))) {
    const int row_bytes = FP8 ? D : 2 * D;
    const int seen = token_seen(a, tok);
    RowState rs;
    attend_row<FP8>(rs, a.q + (int64_t)tok.qrow * a.q_stride + (int64_t)hq * D,
                    reinterpret_cast<uint32_t*>(&so[w][0]), D,
                    a.rtt + clamp_i64(a.rpi[im.b], 0, a.rtt_rows - 1) * a.rtt_stride, 0, seen,
                    a.pool_slots, a.seq_override > 0, a.k_pool + (int64_t)hk * row_bytes,
                    a.v_pool + (int64_t)hk * row_bytes, (int64_t)a.hkv * row_bytes,
                    a.scale_log2 * (FP8 ? a.k_scale[0] : 1.f), lane);
    om = write_row(rs, seen > 0 ? vscale / rs.l : 0.f, D, orow,
                   a.gate ? a.gate + (int64_t)tok.qrow * a.gate_stride +
                                (int64_t)hq * a.gate_hstride
                          : nullptr,
                   lane);
    write = false;
  }
  if (write && lane_out) {
    const float inv = vscale / l;
    u32x2 o = {pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv)};
    if (a.gate) {
      o[0] = gate_pair(o[0], gv[0]);
      o[1] = gate_pair(o[1], gv[1]);
    }
    om = max(max(o[0] & 0x7fffu, (o[0] >> 16) & 0x7fffu),
             max(o[1] & 0x7fffu, (o[1] >> 16) & 0x7fffu));
    *reinterpret_cast<u32x2*>(orow + 4 * lane) = o;
  }
  amax_commit(a.amax, om);
}

constexpr int kStepWaves = 8;   // of a workgroup that streams beside MFMA pieces

// Kernel shape and workspace of a call.
struct PartPlan {
  bool fp8, narrow, other;
  int32_t unit_rows;    // 16 or 32
  int32_t n_workers;    // persistent waves
  int64_t ipre_bytes, ml_bytes, o_bytes, piece_ml_bytes, piece_o_bytes;
  int64_t total() const {
    return ipre_bytes + ml_bytes + o_bytes + piece_ml_bytes + piece_o_bytes;
  }
};

int make_part_plan(const char* fn, int32_t n_items, int32_t row_groups, int32_t slot_rows,
                   int32_t n_pieces, int32_t n_stream, int32_t num_q_heads,
                   int32_t num_kv_heads, int32_t head_dim, int32_t kv_dtype, PartPlan* p) {
  if (num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads)
    return fail(TF_ERR_INVALID, "%s: num_q_heads=%d not a multiple of num_kv_heads=%d", fn,
                num_q_heads, num_kv_heads);
  if (kv_dtype != TF_DTYPE_BF16 && kv_dtype != TF_DTYPE_FP8_E4M3)
    return fail(TF_ERR_UNSUPPORTED, "%s: kv_dtype=%d", fn, kv_dtype);
  p->fp8 = kv_dtype == TF_DTYPE_FP8_E4M3;
  if (head_dim < 8 || head_dim > 256 || head_dim % (p->fp8 ? 16 : 8))
    return fail(TF_ERR_UNSUPPORTED,
                "%s: head_dim=%d (a multiple of 8, for fp8 pools of 16, up to 256)", fn, head_dim);
  if (n_items < 0 || (row_groups != 1 && row_groups != 2) || slot_rows < 1 ||
      slot_rows > 16 * row_groups)
    return fail(TF_ERR_INVALID, "%s: n_items=%d row_groups=%d slot_rows=%d", fn, n_items,
                row_groups, slot_rows);
  if (n_items > kMaxItems)
    return fail(TF_ERR_UNSUPPORTED, "%s: %d parts in one call (at most %d)", fn, n_items,
                kMaxItems);
  if (n_stream < 0 || n_stream > 4096 || (n_stream && (!n_pieces || row_groups != 1)))
    return fail(TF_ERR_INVALID, "%s: n_stream=%d beside %d pieces, row_groups=%d", fn, n_stream,
                n_pieces, row_groups);
  p->other = head_dim != 256;
  p->narrow = head_dim <= 128 && !p->fp8;
  if (n_pieces < 0 || (n_pieces && p->other && !p->narrow))
    return fail(TF_ERR_INVALID, "%s: n_pieces=%d at head_dim=%d, kv_dtype=%d", fn, n_pieces,
                head_dim, kv_dtype);
  p->unit_rows = 16 * row_groups;
  // Four waves per CU, eight of the 128-dim ones (measured with half and twice as many:
  // 64 requests of 1 to 1024 keys 30 us, 42 with eight waves per CU; 16 of 1 to 2048 in
  // units of 32 rows 28 and 37 us with two; 96 of 1 to 700 at 32 / 8 heads of 128 56 us,
  // 83 with four).
  p->n_workers = kWaves * device_cu_count() * (p->narrow ? 2 : 1);
  if (n_stream) p->n_workers = kStepWaves * n_stream;
  const int64_t rows = (p->n_workers + (int64_t)n_items * num_kv_heads) * slot_rows;
  p->ipre_bytes = ((int64_t)(n_items + 1) * 4 + 255) / 256 * 256;
  p->ml_bytes = (rows * 8 + 255) / 256 * 256;
  p->o_bytes = rows * (p->narrow ? 128 : 256) * 4;
  p->piece_ml_bytes = (int64_t)n_pieces * kExtendItemRows * 8;
  p->piece_o_bytes = (int64_t)n_pieces * kExtendItemRows * (p->narrow ? 128 : 256) * 4;
  return TF_OK;
}

template <class C, bool SCORED>
void launch_stream(const PartArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((part_stream_kernel<C, SCORED>), dim3((unsigned)(a.n_workers / kWaves)),
                     dim3(kWaves * kWave), 0, s, a);
}

template <int NG, bool SCORED>
void launch_stream_groups(const PartArgs& a, const PartPlan& p, hipStream_t s) {
  if (p.narrow) return launch_stream<Cfg<128, false, NG, true, true>, SCORED>(a, s);
  if (p.other && p.fp8) return launch_stream<Cfg<256, true, NG, true, true>, SCORED>(a, s);
  if (p.other) return launch_stream<Cfg<256, false, NG, true, true>, SCORED>(a, s);
  if (p.fp8) return launch_stream<Cfg<256, true, NG, false, true>, SCORED>(a, s);
  return launch_stream<Cfg<256, false, NG, false, true>, SCORED>(a, s);
}

template <int WPR, bool SCORED>
void launch_merge_rows(const PartArgs& a, const PartPlan& p, hipStream_t s) {
  constexpr int kRows = kMergeWaves / WPR;
  const dim3 grid((unsigned)((a.n_items - a.own0) * a.hkv + a.n_weights),
                  (unsigned)((a.slot_rows + kRows - 1) / kRows));
  const dim3 block(kMergeWaves * kWave);
  if (p.narrow)
    hipLaunchKernelGGL((part_merge_kernel<128, false, WPR, SCORED>), grid, block, 0, s, a);
  else if (p.fp8)
    hipLaunchKernelGGL((part_merge_kernel<256, true, WPR, SCORED>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((part_merge_kernel<256, false, WPR, SCORED>), grid, block, 0, s, a);
}

// Four waves per row, one where the rows alone fill the CUs (72 rows 5.0 and 7.1 us, 1536
// rows 9.0 and 9.3, 96 x 32 rows of 128 dims 23.0 and 10.4, 6144 rows of 256 28.4 and 17.2).
template <bool SCORED>
void launch_merge(const PartArgs& a, const PartPlan& p, hipStream_t s) {
  if ((int64_t)(a.n_items - a.own0) * a.hkv * a.slot_rows > 2048)
    launch_merge_rows<1, SCORED>(a, p, s);
  else
    launch_merge_rows<4, SCORED>(a, p, s);
}

PartArgs part_args(const void* q, int64_t q_row_stride, const void* k_pool, const void* v_pool,
                   int64_t pool_slots, const float* k_scale, const float* v_scale,
                   const int64_t* req_to_token, int64_t rtt_rows, int64_t rtt_row_stride,
                   int64_t rtt_cols, const int64_t* req_pool_indices, const int64_t* seq_lens,
                   int32_t n_items, int32_t slot_rows, int32_t num_q_heads, int32_t num_kv_heads,
                   int32_t head_dim, float scale, void* out, int64_t out_row_stride,
                   void* workspace, const void* gate, int64_t gate_row_stride,
                   int64_t gate_head_stride, uint32_t* out_amax, const PartPlan& p) {
  PartArgs a = {};
  a.q = static_cast<const __bf16*>(q);
  a.q_stride = q_row_stride;
  a.k_pool = static_cast<const uint8_t*>(k_pool);
  a.v_pool = static_cast<const uint8_t*>(v_pool);
  a.pool_slots = pool_slots;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.rtt = req_to_token;
  a.rtt_rows = rtt_rows;
  a.rtt_stride = rtt_row_stride;
  a.rtt_cols = rtt_cols;
  a.rpi = req_pool_indices;
  a.seq_lens = seq_lens;
  a.n_items = n_items;
  a.unit_rows = p.unit_rows;
  a.slot_rows = slot_rows;
  a.hkv = num_kv_heads;
  a.group = num_q_heads / num_kv_heads;
  a.head_dim = head_dim;
  a.n_workers = p.n_workers;
  a.scale_log2 = scale * kLog2e;
  a.out = static_cast<__bf16*>(out);
  a.out_stride = out_row_stride;
  a.gate = static_cast<const __bf16*>(gate);
  a.gate_stride = gate_row_stride;
  a.gate_hstride = gate_head_stride;
  a.amax = out_amax;
  char* ws = static_cast<char*>(workspace);
  a.ipre = reinterpret_cast<int32_t*>(ws);
  a.part_ml = reinterpret_cast<float2*>(ws + p.ipre_bytes);
  a.part_o = reinterpret_cast<float*>(ws + p.ipre_bytes + p.ml_bytes);
  return a;
}

}  // namespace
}  // namespace tfa

extern "C" int64_t tf_attn_shared_workspace_bytes(int32_t n_items, int32_t row_groups,
                                                  int32_t slot_rows, int32_t n_pieces,
                                                  int32_t n_stream, int32_t num_q_heads,
                                                  int32_t num_kv_heads,
                                                  int32_t head_dim, int32_t kv_dtype) {
  using namespace tfa;
  clear_error();
  PartPlan p;
  const int rc = make_part_plan("shared", n_items, row_groups, slot_rows, n_pieces, n_stream,
                                num_q_heads, num_kv_heads, head_dim, kv_dtype, &p);
  return rc != TF_OK ? rc : p.total();
}

extern "C" int32_t tf_attn_shared(
    const void* q, int64_t q_row_stride, const void* k_pool, const void* v_pool,
    int64_t pool_slots, int32_t kv_dtype, const float* k_scale, const float* v_scale,
    const int64_t* req_to_token, int64_t rtt_rows, int64_t rtt_row_stride, int64_t rtt_cols,
    const int64_t* req_pool_indices, const int64_t* seq_lens, const int32_t* items,
    int32_t n_items, int32_t n_shared, const int32_t* tokens, int32_t row_groups,
    int32_t slot_rows, const int32_t* pieces, int32_t n_pieces, const int32_t* units,
    int32_t n_stream, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, float scale,
    void* out, int64_t out_row_stride, void* workspace, int64_t workspace_bytes, const void* gate,
    int64_t gate_row_stride, int64_t gate_head_stride, uint32_t* out_amax, tf_stream_t stream) {
  using namespace tfa;
  clear_error();
  PartPlan p;
  int rc = make_part_plan("shared", n_items, row_groups, slot_rows, n_pieces, n_stream, num_q_heads,
                          num_kv_heads, head_dim, kv_dtype, &p);
  if (rc != TF_OK) return rc;
  if (n_shared < 0 || n_shared > n_items || (n_shared && n_pieces))
    return fail(TF_ERR_INVALID, "shared: %d of %d parts are shared, and %d pieces", n_shared,
                n_items, n_pieces);
  if (n_pieces && !(scale >= 0.f))
    return fail(TF_ERR_UNSUPPORTED, "shared: scale=%g of pieces, whose rows follow their largest "
                "product", (double)scale);
  if (n_items == n_shared) return TF_OK;
  rc = check_slot_call("shared", q, q_row_stride, k_pool, v_pool, pool_slots, kv_dtype, k_scale,
                       v_scale, req_to_token, rtt_rows, rtt_row_stride, rtt_cols,
                       req_pool_indices, seq_lens, 0, num_q_heads, head_dim, out, out_row_stride,
                       gate, gate_row_stride, gate_head_stride, workspace, workspace_bytes,
                       p.total());
  if (rc != TF_OK) return rc;
  if (!items || !tokens || !aligned16(items) || !aligned16(tokens))
    return fail(TF_ERR_INVALID, "shared: items and tokens must be 16-byte aligned");
  if (n_pieces && (!pieces || !units || !aligned16(pieces) || !aligned8(units)))
    return fail(TF_ERR_INVALID, "shared: pieces and units must be 16- and 8-byte aligned");
  PartArgs a = part_args(q, q_row_stride, k_pool, v_pool, pool_slots, k_scale, v_scale,
                         req_to_token, rtt_rows, rtt_row_stride, rtt_cols, req_pool_indices,
                         seq_lens, n_items, slot_rows, num_q_heads, num_kv_heads, head_dim, scale,
                         out, out_row_stride, workspace, gate, gate_row_stride, gate_head_stride,
                         out_amax, p);
  a.items = reinterpret_cast<const PartItem*>(items);
  a.toks = reinterpret_cast<const PartTok*>(tokens);
  a.own0 = n_shared;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (n_pieces) {
    a.units = reinterpret_cast<const int2*>(units);
    char* at = static_cast<char*>(workspace) + p.ipre_bytes + p.ml_bytes + p.o_bytes;
    a.piece_ml = reinterpret_cast<float2*>(at);
    a.piece_o = reinterpret_cast<float*>(at + p.piece_ml_bytes);
    ExtendArgs e = {};
    e.q = a.q;
    e.q_stride = a.q_stride;
    e.k_pool = a.k_pool;
    e.v_pool = a.v_pool;
    e.pool_slots = a.pool_slots;
    e.k_scale = a.k_scale;
    e.v_scale = a.v_scale;
    e.rtt = a.rtt;
    e.rtt_rows = a.rtt_rows;
    e.rtt_stride = a.rtt_stride;
    e.rtt_cols = a.rtt_cols;
    e.rpi = a.rpi;
    e.seq_lens = a.seq_lens;
    e.work = pieces;
    e.hkv = a.hkv;
    e.group = a.group;
    e.scale_log2 = a.scale_log2;
    e.part_ml = reinterpret_cast<float*>(at);
    e.part_o = reinterpret_cast<float*>(at + p.piece_ml_bytes);
    e.toks = a.toks;
    const PartArgs* own = n_stream ? &a : nullptr;
    rc = p.narrow ? launch_prefix_tiles(e, head_dim, n_pieces, own, n_stream, s)
                  : launch_prefix_pieces(e, n_pieces, own, n_stream, p.fp8, s);
    if (rc != TF_OK) return rc;
  }
  if (!n_stream) {
    if (row_groups == 1)
      launch_stream_groups<1, false>(a, p, s);
    else
      launch_stream_groups<2, false>(a, p, s);
    rc = launch_status("tf_attn_shared stream launch");
    if (rc != TF_OK) return rc;
  }
  launch_merge<false>(a, p, s);
  return launch_status("tf_attn_shared merge launch");
}

namespace tfa {
namespace {

// tf_attn_scored: one new token per request.
struct ScoredPlan {
  PartPlan p;
  int32_t n_items, head_blocks, slot_rows;
  int64_t cap, scores_bytes;
  int64_t total() const { return p.total() + scores_bytes; }
};

int make_scored_plan(int32_t batch, int32_t max_len, int32_t num_q_heads, int32_t num_kv_heads,
                     int32_t head_dim, int32_t kv_dtype, ScoredPlan* r) {
  if (batch < 0 || max_len < 1 || num_kv_heads <= 0 || num_q_heads <= 0)
    return fail(TF_ERR_INVALID, "scored: batch=%d max_len=%d heads %d/%d", batch, max_len,
                num_q_heads, num_kv_heads);
  const int32_t group = num_q_heads / num_kv_heads;
  r->head_blocks = (group + 15) / 16;
  r->slot_rows = group < 1 ? 1 : group < 16 ? group : 16;
  if ((int64_t)batch * r->head_blocks > kMaxItems)
    return fail(TF_ERR_UNSUPPORTED, "scored: %d requests of %d head blocks (at most %d)", batch,
                r->head_blocks, kMaxItems);
  r->n_items = batch * r->head_blocks;
  const int rc = make_part_plan("scored", r->n_items, 1, r->slot_rows, 0, 0, num_q_heads,
                                num_kv_heads, head_dim, kv_dtype, &r->p);
  if (rc != TF_OK) return rc;
  r->p.o_bytes = (r->p.o_bytes + 255) / 256 * 256;
  r->cap = ((int64_t)max_len + kTile - 1) / kTile * kTile;
  r->scores_bytes = (int64_t)batch * num_q_heads * r->cap * 4;
  return TF_OK;
}

}  // namespace
}  // namespace tfa

extern "C" int64_t tf_attn_scored_workspace_bytes(int32_t batch_size, int32_t max_len,
                                                  int32_t num_q_heads, int32_t num_kv_heads,
                                                  int32_t head_dim, int32_t kv_dtype) {
  using namespace tfa;
  clear_error();
  ScoredPlan r;
  const int rc = make_scored_plan(batch_size, max_len, num_q_heads, num_kv_heads, head_dim,
                                  kv_dtype, &r);
  return rc != TF_OK ? rc : r.total();
}

extern "C" int32_t tf_attn_scored(
    const void* q, int64_t q_row_stride, const void* k_pool, const void* v_pool,
    int64_t pool_slots, int32_t kv_dtype, const float* k_scale, const float* v_scale,
    const int64_t* req_to_token, int64_t rtt_rows, int64_t rtt_row_stride, int64_t rtt_cols,
    const int64_t* req_pool_indices, const int64_t* seq_lens, int32_t seq_len_override,
    int32_t batch_size, int32_t max_len, int32_t num_q_heads, int32_t num_kv_heads,
    int32_t head_dim, float scale, void* out, int64_t out_row_stride, float* scores,
    int64_t scores_row_stride, int32_t add, void* workspace, int64_t workspace_bytes,
    const void* gate, int64_t gate_row_stride, int64_t gate_head_stride, uint32_t* out_amax,
    tf_stream_t stream) {
  using namespace tfa;
  clear_error();
  ScoredPlan r;
  int rc = make_scored_plan(batch_size, max_len, num_q_heads, num_kv_heads, head_dim, kv_dtype,
                            &r);
  if (rc != TF_OK) return rc;
  if (batch_size == 0) return TF_OK;
  rc = check_slot_call("scored", q, q_row_stride, k_pool, v_pool, pool_slots, kv_dtype, k_scale,
                       v_scale, req_to_token, rtt_rows, rtt_row_stride, rtt_cols,
                       req_pool_indices, seq_lens, seq_len_override, num_q_heads, head_dim, out,
                       out_row_stride, gate, gate_row_stride, gate_head_stride, workspace,
                       workspace_bytes, r.total());
  if (rc != TF_OK) return rc;
  if (!scores || scores_row_stride < rtt_cols)
    return fail(TF_ERR_INVALID, "scored: scores need rows of at least %lld", (long long)rtt_cols);
  PartArgs a = part_args(q, q_row_stride, k_pool, v_pool, pool_slots, k_scale, v_scale,
                         req_to_token, rtt_rows, rtt_row_stride, rtt_cols, req_pool_indices,
                         seq_lens, r.n_items, r.slot_rows, num_q_heads, num_kv_heads, head_dim,
                         scale, out, out_row_stride, workspace, gate, gate_row_stride,
                         gate_head_stride, out_amax, r.p);
  a.seq_override = seq_len_override;
  a.head_blocks = r.head_blocks;
  a.row_scores = reinterpret_cast<float*>(static_cast<char*>(workspace) + r.p.total());
  a.score_cap = r.cap;
  a.scores = scores;
  a.scores_stride = scores_row_stride;
  a.add_scores = add;
  const int64_t blocks = (r.cap + kWeightKeys - 1) / kWeightKeys;
  // (as many as CUs over all requests: each takes the sums of every row of its request)
  const int64_t most = std::max<int64_t>(1, device_cu_count() / batch_size);
  a.weight_blocks = (int32_t)std::min(blocks, most);
  a.n_weights = a.weight_blocks * batch_size;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  launch_stream_groups<1, true>(a, r.p, s);
  rc = launch_status("tf_attn_scored stream launch");
  if (rc != TF_OK) return rc;
  launch_merge<true>(a, r.p, s);
  return launch_status("tf_attn_scored launch");
}
