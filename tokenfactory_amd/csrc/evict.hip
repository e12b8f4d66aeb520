// Eviction of cached tokens by their attention weight (tf_evict_tokens): of each
// request's table row, the first tokens and the last ones stay, and of those between as
// many of the largest scores as the budget leaves room for; what stays moves together,
// in order, and the slots of the others are handed back.
//
// The room-th largest score is found digit by digit (radix selection over the scores'
// order-preserving integers, 11 bits at a time, counted in LDS), the entries above it
// stay and of the equal ones the first.  Then one ordered pass moves slots and scores:
// positions come from a scan over the workgroup and a running count.  In place: an entry
// moves to its own or an earlier position, a chunk is read before any of it is written,
// and no chunk is written before the ones in front of it.
#include <math.h>

#include "tf_common.h"
#include "tf_internal.h"

namespace tfa {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kPer = 4;                        // entries of a thread in a chunk
constexpr int kChunk = kThreads * kPer;
constexpr int kDigitBits = 11;
constexpr int kBins = 1 << kDigitBits;

struct EvictArgs {
  int64_t* table;
  int64_t table_rows, table_stride, table_cols;
  float* scores;
  int64_t scores_stride;
  const int64_t* rows;
  const int64_t* out_rows;    // NULL: in place
  const int64_t* seq_lens;
  const int64_t* first;       // per request; NULL: first_n for all
  int64_t first_n, recent, keep, max_len;
  int64_t* lens_out;
  int64_t* freed;
  int64_t freed_width;
};

// Integers in the order of the scores: -0 = +0, NaN below everything.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x);
  if ((u << 1) == 0) return 0x80000000u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// What stays of a request: [0, first), [end, n), and of [first, end) the `room` best.
struct Range {
  int n, first, end, room, left;   // left: entries that stay in all
};
__device__ __forceinline__ Range range_of(const EvictArgs& a, int b) {
  Range r;
  r.n = (int)clamp_i64(a.seq_lens[b], 0, min(a.table_cols, a.max_len));
  const int64_t first = max<int64_t>(0, a.first ? a.first[b] : a.first_n);
  r.first = (int)min<int64_t>(first, r.n);
  r.end = (int)max<int64_t>(r.first, r.n - min<int64_t>(a.recent, r.n));
  const int64_t budget = max<int64_t>(a.keep, r.first + a.recent);
  r.left = (int)min<int64_t>(r.n, budget);
  r.room = r.left - r.first - (r.n - r.end);
  return r;
}

__device__ __forceinline__ int wave_scan(int v, int lane) {   // inclusive
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const int o = __shfl_up(v, off, kWave);
    if (lane >= off) v += o;
  }
  return v;
}

__global__ void __launch_bounds__(kThreads) evict_kernel(EvictArgs a) {
  __shared__ int32_t bins[kBins];
  __shared__ int32_t wsum[2][kWaves];
  __shared__ uint32_t found[2];   // the digit of the room-th largest, and how many it needs
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = wave_id();
  const Range rg = range_of(a, b);
  const int64_t row = clamp_i64(a.rows[b], 0, a.table_rows - 1);
  const int64_t to = a.out_rows ? clamp_i64(a.out_rows[b], 0, a.table_rows - 1) : row;
  const int64_t* slots = a.table + row * a.table_stride;
  const float* scores = a.scores + row * a.scores_stride;
  int64_t* new_slots = a.table + to * a.table_stride;
  float* new_scores = a.scores + to * a.scores_stride;
  int64_t* freed = a.freed + (int64_t)b * a.freed_width;
  if (tid == 0) a.lens_out[b] = rg.left;

  // ---- the room-th largest: `cut`, of which `ties` stay
  uint32_t cut = 0;
  int ties = rg.room;
  const bool select = rg.room > 0 && rg.room < rg.end - rg.first;
  if (select) {
    uint32_t mask = 0;
    for (int shift = 32 - kDigitBits; ; shift -= kDigitBits) {
      const int lo = max(shift, 0);                  // 11, 11 and 10 bits
      const uint32_t digit = (1u << min(kDigitBits, shift + kDigitBits)) - 1;
      for (int i = tid; i < kBins; i += kThreads) bins[i] = 0;
      __syncthreads();
      for (int i = rg.first + tid; i < rg.end; i += kThreads) {
        const uint32_t k = order_of(scores[i]);
        if ((k & mask) == cut) atomicAdd(&bins[(k >> lo) & digit], 1);
      }
      __syncthreads();
      // Bins from the largest down, two a thread: where the count passes `ties`.
      const int i0 = kBins - 1 - 2 * tid;
      const int c0 = bins[i0], c1 = bins[i0 - 1];
      const int incl = wave_scan(c0 + c1, lane);
      if (lane == kWave - 1) wsum[0][w] = incl;
      __syncthreads();
      int before = incl - c0 - c1;
      for (int k = 0; k < w; ++k) before += wsum[0][k];
      if (before < ties && before + c0 >= ties) {
        found[0] = i0;
        found[1] = ties - before;
      } else if (before + c0 < ties && before + c0 + c1 >= ties) {
        found[0] = i0 - 1;
        found[1] = ties - before - c0;
      }
      __syncthreads();
      cut |= found[0] << lo;
      ties = (int)found[1];
      mask |= digit << lo;
      __syncthreads();
      if (lo == 0) break;
    }
  }

  // ---- the ordered pass
  const bool nothing = rg.left == rg.n;
  int gt0 = 0, eq0 = 0;   // entries before the chunk that stay for certain / that are ties
  const int start = nothing && to == row ? rg.n : 0;
  for (int c0 = start; c0 < rg.n; c0 += kChunk) {
    const int i0 = c0 + tid * kPer;
    int64_t s[kPer];
    float v[kPer];
    int sure = 0, tie = 0;   // bit per entry
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = i0 + j;
      if (i >= rg.n) continue;
      s[j] = slots[i];
      v[j] = scores[i];
      if (nothing || i < rg.first || i >= rg.end) {
        sure |= 1 << j;
      } else if (select) {
        const uint32_t k = order_of(v[j]);
        sure |= (k > cut) << j;
        tie |= (k == cut) << j;
      }
    }
    const int ns = __popc(sure), nt = __popc(tie);
    const int si = wave_scan(ns, lane), ti = wave_scan(nt, lane);
    if (lane == kWave - 1) {
      wsum[0][w] = si;
      wsum[1][w] = ti;
    }
    __syncthreads();   // (every entry of the chunk is read)
    int gt = gt0 + si - ns, eq = eq0 + ti - nt;
    int all_s = 0, all_t = 0;
    for (int k = 0; k < kWaves; ++k) {
      if (k < w) {
        gt += wsum[0][k];
        eq += wsum[1][k];
      }
      all_s += wsum[0][k];
      all_t += wsum[1][k];
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = i0 + j;
      if (i >= rg.n) continue;
      const bool is_tie = tie >> j & 1;
      const int at = gt + min(eq, ties);
      if ((sure >> j & 1) || (is_tie && eq < ties)) {
        new_slots[at] = s[j];
        new_scores[at] = v[j];
      } else if (i - at < a.freed_width) {
        freed[i - at] = s[j];
      }
      gt += sure >> j & 1;
      eq += is_tie;
    }
    gt0 += all_s;
    eq0 += all_t;
    __syncthreads();
  }
  // ---- behind what stays: empty entries without weight
  for (int i = rg.left + tid; i < rg.n; i += kThreads) {
    new_slots[i] = -1;
    new_scores[i] = 0.f;
  }
  for (int64_t i = rg.n - rg.left + tid; i < a.freed_width; i += kThreads) freed[i] = -1;
}

}  // namespace
}  // namespace tfa

extern "C" int32_t tf_evict_tokens(
    int64_t* req_to_token, int64_t rtt_rows, int64_t rtt_row_stride, int64_t rtt_cols,
    float* scores, int64_t scores_row_stride, const int64_t* rows, const int64_t* out_rows,
    const int64_t* seq_lens, const int64_t* first, int64_t first_n, int64_t recent, int64_t keep,
    int64_t max_len, int32_t batch_size, int64_t* new_lens, int64_t* freed, int64_t freed_width,
    tf_stream_t stream) {
  using namespace tfa;
  clear_error();
  if (batch_size < 0 || rtt_rows < 1 || rtt_cols < 1 || rtt_row_stride < rtt_cols ||
      scores_row_stride < rtt_cols || rtt_cols > INT32_MAX)
    return fail(TF_ERR_INVALID, "evict: bad batch or req_to_token extents");
  if (batch_size == 0) return TF_OK;
  if (!req_to_token || !scores || !rows || !seq_lens || !new_lens || (freed_width > 0 && !freed))
    return fail(TF_ERR_INVALID, "evict: null pointer argument");
  if (first_n < 0 || recent < 0 || keep < 0 || max_len < 0 || freed_width < 0)
    return fail(TF_ERR_INVALID, "evict: negative size");
  const int64_t need = (max_len < rtt_cols ? max_len : rtt_cols) - keep;
  if (freed_width < need)
    return fail(TF_ERR_INVALID, "evict: freed needs room for %lld slots a request",
                (long long)need);
  EvictArgs a = {};
  a.table = req_to_token;
  a.table_rows = rtt_rows;
  a.table_stride = rtt_row_stride;
  a.table_cols = rtt_cols;
  a.scores = scores;
  a.scores_stride = scores_row_stride;
  a.rows = rows;
  a.out_rows = out_rows;
  a.seq_lens = seq_lens;
  a.first = first;
  a.first_n = first_n;
  a.recent = recent;
  a.keep = keep;
  a.max_len = max_len;
  a.lens_out = new_lens;
  a.freed = freed;
  a.freed_width = freed_width;
  hipLaunchKernelGGL(evict_kernel, dim3((unsigned)batch_size), dim3(kThreads), 0,
                     reinterpret_cast<hipStream_t>(stream), a);
  return launch_status("tf_evict_tokens launch");
}
