// Eviction of cached tokens by their attention weight (tf_evict_tokens): of each
// request's table row, the first tokens and the last ones stay, and of those between as
// many of the largest scores as the budget leaves room for; what stays moves together,
// in order, and the slots of the others are handed back.
//
// One workgroup per request, or for rows that may be longer than 16384 five launches of
// one per 8192 entries: the same digits counted per run, each launch deriving a digit from
// the counts of the one before (kernel boundaries order them: no atomics, nothing to
// clear), then the moves into scratch and back.  Bound by latency: 3 rows of
// up to 1500 entries 6.2 us on the device, 64 of up to 8192 13.6 (9.4 MB), a call on 8 rows
// of 16384 23.6 us, of 24576 29.5, of 131072 39.7 (183 by a workgroup each, whose CU moves
// 25 GB/s).
//
// The room-th largest score is found digit by digit (radix selection over the scores'
// order-preserving integers, 11 bits at a time, counted in LDS), the entries above it
// stay and of the equal ones the first.  Every wave takes consecutive entries, 64 at a
// time, so that an entry's place is what the waves before it keep (one sum per wave
// through LDS), what its own wave kept so far, and a count over the lanes below.
#include <math.h>

#include <algorithm>

#include "tf_common.h"
#include "tf_internal.h"

namespace tfa {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
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
  // Long rows: per request and run of kRunEntries entries of the range between, counts of
  // the digits ([3][kBins]) and of entries above all that the third pass counts.
  int32_t* counts;
  int32_t* above;
  int2* cuts;              // [batch][3]: the digits found so far, and what they need
  int32_t n_runs;          // runs that a row of max_len takes
  int64_t* moved_slots;    // [batch][max_len]: what stays, on its way
  float* moved_scores;
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

// Inclusive sums over the lanes: within rows of 16, then over the rows, by lane moves of
// the vector unit (a shuffle goes through LDS: the three digits' scans took 1.5 us so).
template <int CTRL, int ROWS>
__device__ __forceinline__ int moved(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_scan(int v) {
  v += moved<0x111, 0xf>(v);   // from 1, 2, 4 and 8 lanes below in the row
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);   // the row's last lane to the next row (1 and 3)
  v += moved<0x143, 0xc>(v);   // lane 31 to rows 2 and 3
  return v;
}

// Sum over the waves in front of this one, and over all, of each wave's `mine`: through
// wsum, which the caller guards with barriers on both sides.
struct WaveSums {
  int before, all;
};
__device__ __forceinline__ WaveSums sum_waves(const int32_t* wsum, int lane, int w) {
  const int v = wave_scan(lane < kWaves ? wsum[lane] : 0);
  return WaveSums{w ? __builtin_amdgcn_readlane(v, w - 1) : 0,
                  __builtin_amdgcn_readlane(v, kWaves - 1)};
}

// One count for the lane's bin; a wave whose (active) lanes share one, as equal scores do,
// adds once.
__device__ __forceinline__ void count(int32_t* bins, uint32_t bin) {
  const uint32_t first = __builtin_amdgcn_readfirstlane(bin);
  const uint64_t others = __ballot(bin != first), all = __ballot(true);
  if (others == 0) {
    if ((int)(threadIdx.x & 63) == __ffsll((unsigned long long)all) - 1)
      atomicAdd(&bins[first], __popcll(all));
  } else {
    atomicAdd(&bins[bin], 1);
  }
}

// A barrier for LDS alone: loads and stores of global memory stay in flight.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// The digit of the ties-th largest in `bins` (by keys): found[0], and how many of that
// digit it needs: found[1].  Bins from the largest down, two a thread.
__device__ __forceinline__ void find_digit(const int32_t* bins, int ties, int32_t* wsum,
                                           uint32_t* found, int lane, int w) {
  const int i0 = kBins - 1 - 2 * (int)threadIdx.x;
  const int c0 = bins[i0], c1 = bins[i0 - 1];
  const int incl = wave_scan(c0 + c1);
  if (lane == kWave - 1) wsum[w] = incl;
  lds_barrier();
  const int before = sum_waves(wsum, lane, w).before + incl - c0 - c1;
  if (before < ties && before + c0 >= ties) {
    found[0] = i0;
    found[1] = ties - before;
  } else if (before + c0 < ties && before + c0 + c1 >= ties) {
    found[0] = i0 - 1;
    found[1] = ties - before - c0;
  }
  lds_barrier();
}

// Digits of the order integers: 11, 11 and 10 bits.
__device__ __forceinline__ int digit_shift(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }
__device__ __forceinline__ uint32_t digit_mask(int pass) { return pass == 2 ? 1023u : 2047u; }

// The entries that stay (`sure`, a bit per entry of the lane) and the ties of a wave so far.
struct Kept {
  int gt, eq;
};
// How many entries of the wave stay for certain and how many are ties.
template <int PER>
__device__ __forceinline__ Kept wave_kept(int sure, int tie) {
  Kept k{0, 0};
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    k.gt += __popcll(__ballot(sure >> j & 1));
    k.eq += __popcll(__ballot(tie >> j & 1));
  }
  return k;
}
// Where the lane's entry j goes: how many entries before it stay, of which `before` those of
// the waves (and runs) in front, which is moved past the wave's entries j; and whether it
// stays itself.
__device__ __forceinline__ bool place(Kept& before, int sure, int tie, int j, int ties, int& at) {
  const uint64_t ms = __ballot(sure >> j & 1), mt = __ballot(tie >> j & 1);
  const int gt = before.gt + __builtin_amdgcn_mbcnt_hi((uint32_t)(ms >> 32),
                                 __builtin_amdgcn_mbcnt_lo((uint32_t)ms, 0));
  const int eq = before.eq + __builtin_amdgcn_mbcnt_hi((uint32_t)(mt >> 32),
                                 __builtin_amdgcn_mbcnt_lo((uint32_t)mt, 0));
  before.gt += __popcll(ms);
  before.eq += __popcll(mt);
  at = gt + min(eq, ties);
  return (sure >> j & 1) || ((tie >> j & 1) && eq < ties);
}

// PER: entries of a thread.
template <int PER>
__global__ void __launch_bounds__(kThreads) evict_kernel(EvictArgs a) {
  __shared__ int32_t bins[kBins];
  __shared__ int32_t wsum[kWaves];
  __shared__ int32_t kept[2][kWaves];
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

  const bool nothing = rg.left == rg.n;
  if (nothing && to == row) {
    for (int64_t i = tid; i < a.freed_width; i += kThreads) freed[i] = -1;
    return;
  }
  // The row, read once: entry j of a lane is number i0 + 64 j.  Every load has returned
  // before the barrier that lets anything be written.
  const int i0 = w * kWave * PER + lane;
  float v[PER];
  int64_t s[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) v[j] = i0 + j * kWave < rg.n ? scores[i0 + j * kWave] : 0.f;
#pragma unroll
  for (int j = 0; j < PER; ++j) s[j] = i0 + j * kWave < rg.n ? slots[i0 + j * kWave] : 0;

  // ---- the room-th largest: `cut`, of which `ties` stay
  uint32_t cut = 0;
  int ties = rg.room;
  const bool select = rg.room > 0 && rg.room < rg.end - rg.first;
  if (select) {
    uint32_t mask = 0;
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = digit_shift(pass);
      const uint32_t digit = digit_mask(pass);
      for (int i = tid; i < kBins; i += kThreads) bins[i] = 0;
      lds_barrier();
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int i = i0 + j * kWave;
        if (PER == 16) asm volatile("" : "+v"(v[j]));   // (k is made again: 128 registers)
        const uint32_t k = order_of(v[j]);
        if (i >= rg.first && i < rg.end && (k & mask) == cut) count(bins, (k >> shift) & digit);
      }
      lds_barrier();
      find_digit(bins, ties, wsum, found, lane, w);
      cut |= found[0] << shift;
      ties = (int)found[1];
      mask |= digit << shift;
    }
  }

  // ---- what stays moves together, the rest goes out
  int sure = 0, tie = 0;   // bit per entry
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = i0 + j * kWave;
    const uint32_t k = order_of(v[j]);
    const bool outside = nothing || i < rg.first || i >= rg.end;
    sure |= (i < rg.n && (outside || (select && k > cut))) << j;
    tie |= (i < rg.n && !outside && select && k == cut) << j;
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) asm volatile("" ::"v"(s[j]));   // (see above)
  const Kept mine = wave_kept<PER>(sure, tie);
  if (lane == 0) {
    kept[0][w] = mine.gt;
    kept[1][w] = mine.eq;
  }
  lds_barrier();
  Kept before{sum_waves(kept[0], lane, w).before, sum_waves(kept[1], lane, w).before};
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = i0 + j * kWave;
    int at;
    const bool stays = place(before, sure, tie, j, ties, at);
    if (i >= rg.n) continue;
    if (stays) {
      new_slots[at] = s[j];
      new_scores[at] = v[j];
    } else if (i - at < a.freed_width) {
      freed[i - at] = s[j];
    }
  }
  // ---- behind what stays: empty entries without weight
  for (int i = rg.left + tid; i < rg.n; i += kThreads) {
    new_slots[i] = -1;
    new_scores[i] = 0.f;
  }
  for (int64_t i = rg.n - rg.left + tid; i < a.freed_width; i += kThreads) freed[i] = -1;
}

// ---------------------------------------------------------------- long rows
constexpr int kRunPer = 8;
constexpr int kRunEntries = kRunPer * kThreads;

struct Found {
  uint32_t cut;   // the digits of the passes so far
  int ties;       // entries with them that stay
};

// The digits of passes 0 .. passes - 1: those before the last from the launch before, the
// last from the runs' counts, by every workgroup for itself.  front: of the last pass, how
// many entries of the runs before `run` have digits 2 thread and 2 thread + 1.
__device__ Found find_cut(const EvictArgs& a, const Range& rg, int b, int passes, int32_t* bins,
                          int32_t* wsum, uint32_t* found, int run, int2& front) {
  front = int2{0, 0};
  if (passes == 0) return Found{0u, rg.room};
  const int lane = threadIdx.x & 63, w = wave_id();
  const int pass = passes - 1;
  const int runs = (rg.end - rg.first + kRunEntries - 1) / kRunEntries;
  Found f{0u, rg.room};
  if (pass > 0) {
    const int2 c = a.cuts[b * 3 + pass - 1];
    f = Found{(uint32_t)c.x, c.y};
  }
  const int32_t* counts = a.counts + ((int64_t)b * 3 + pass) * a.n_runs * kBins;
  const int i = 2 * (int)threadIdx.x;
  int c0 = 0, c1 = 0;
#pragma unroll 8
  for (int r = 0; r < runs; ++r) {
    const int2 c = *reinterpret_cast<const int2*>(counts + (int64_t)r * kBins + i);
    c0 += c.x;
    c1 += c.y;
    if (r < run) {
      front.x += c.x;
      front.y += c.y;
    }
  }
  bins[i] = c0;
  bins[i + 1] = c1;
  lds_barrier();
  find_digit(bins, f.ties, wsum, found, lane, w);
  f.cut |= found[0] << digit_shift(pass);
  f.ties = (int)found[1];
  if (blockIdx.x == 0 && threadIdx.x == 0) a.cuts[b * 3 + pass] = int2{(int)f.cut, f.ties};
  lds_barrier();
  return f;
}

// Counts a run's digits of one pass, among the entries that share the digits before.
template <int PASS>
__global__ void __launch_bounds__(kThreads) evict_count_kernel(EvictArgs a) {
  __shared__ int32_t bins[kBins];
  __shared__ int32_t wsum[kWaves];
  __shared__ uint32_t found[2];
  const int b = blockIdx.y, run = blockIdx.x, tid = threadIdx.x;
  const Range rg = range_of(a, b);
  const int mid = rg.end - rg.first, from = run * kRunEntries;
  if (rg.room <= 0 || rg.room >= mid || from >= mid) return;   // (nothing to choose)
  const int64_t row = clamp_i64(a.rows[b], 0, a.table_rows - 1);
  const float* scores = a.scores + row * a.scores_stride + rg.first + from;
  float v[kRunPer];
#pragma unroll
  for (int j = 0; j < kRunPer; ++j) {
    const int i = j * kThreads + tid;
    v[j] = from + i < mid ? scores[i] : 0.f;
  }
  int2 front;
  const Found f = find_cut(a, rg, b, PASS, bins, wsum, found, 0, front);
  constexpr uint32_t mask = PASS == 0 ? 0u : PASS == 1 ? 0xffe00000u : 0xfffffc00u;
  for (int i = tid; i < kBins; i += kThreads) bins[i] = 0;
  if (tid < kWaves) wsum[tid] = 0;
  lds_barrier();
  int above = 0;   // entries that the digits before put above the cut
#pragma unroll
  for (int j = 0; j < kRunPer; ++j) {
    if (from + j * kThreads + tid >= mid) continue;
    const uint32_t k = order_of(v[j]);
    if ((k & mask) == f.cut) count(bins, (k >> digit_shift(PASS)) & digit_mask(PASS));
    if (PASS == 2) above += (k & mask) > f.cut;
  }
  if (PASS == 2) {
    above = wave_scan(above);
    if ((tid & 63) == kWave - 1) wsum[wave_id()] = above;
  }
  lds_barrier();
  int32_t* counts = a.counts + (((int64_t)b * 3 + PASS) * a.n_runs + run) * kBins;
  for (int i = tid; i < kBins; i += kThreads) counts[i] = bins[i];
  if (PASS == 2 && tid == 0) {
    int sum = 0;
    for (int k = 0; k < kWaves; ++k) sum += wsum[k];
    a.above[(int64_t)b * a.n_runs + run] = sum;
  }
}

// Moves what stays of a run into scratch, in order, and the slots of the others out.  The
// entries in front of the range and behind it go with its first and last run.
__global__ void __launch_bounds__(kThreads) evict_move_kernel(EvictArgs a) {
  __shared__ int32_t bins[kBins];
  __shared__ int32_t wsum[2][kWaves];
  __shared__ int32_t kept[2][kWaves];
  __shared__ uint32_t found[2];
  const int b = blockIdx.y, run = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = wave_id();
  const Range rg = range_of(a, b);
  const int mid = rg.end - rg.first, from = run * kRunEntries;
  if (run == 0 && tid == 0) a.lens_out[b] = rg.left;
  const int64_t row = clamp_i64(a.rows[b], 0, a.table_rows - 1);
  const int64_t* slots = a.table + row * a.table_stride;
  const float* scores = a.scores + row * a.scores_stride;
  int64_t* new_slots = a.moved_slots + (int64_t)b * a.max_len;
  float* new_scores = a.moved_scores + (int64_t)b * a.max_len;
  int64_t* freed = a.freed + (int64_t)b * a.freed_width;
  // (every workgroup of the row takes a share of what does not depend on scores)
  const int stride = gridDim.x * kThreads, at0 = run * kThreads + tid;
  for (int i = at0; i < rg.first; i += stride) {
    new_slots[i] = slots[i];
    new_scores[i] = scores[i];
  }
  for (int i = at0; i < rg.n - rg.end; i += stride) {
    new_slots[rg.left - (rg.n - rg.end) + i] = slots[rg.end + i];
    new_scores[rg.left - (rg.n - rg.end) + i] = scores[rg.end + i];
  }
  for (int64_t i = rg.n - rg.left + at0; i < a.freed_width; i += stride) freed[i] = -1;
  if (from >= mid) return;

  const bool select = rg.room > 0 && rg.room < mid, all = rg.room >= mid;
  int64_t s[kRunPer];
  float v[kRunPer];
  const int i0 = from + w * kWave * kRunPer + lane;   // entry j of the lane is i0 + 64 j
#pragma unroll
  for (int j = 0; j < kRunPer; ++j) {
    const int i = i0 + j * kWave;
    s[j] = i < mid ? slots[rg.first + i] : 0;
    v[j] = i < mid ? scores[rg.first + i] : 0.f;
  }
  Found f{0u, 0};
  int gt0 = 0, eq0 = 0;   // of the runs before: above the cut, equal to it
  if (select) {
    int g = 0;   // (counted above by the launch before)
    for (int r = tid; r < run; r += kThreads) g += a.above[(int64_t)b * a.n_runs + r];
    int2 front;
    f = find_cut(a, rg, b, 3, bins, wsum[0], found, run, front);
    const int digit = (int)(f.cut & digit_mask(2));
    g += (2 * tid > digit ? front.x : 0) + (2 * tid + 1 > digit ? front.y : 0);
    const int e = 2 * tid == digit ? front.x : 2 * tid + 1 == digit ? front.y : 0;
    const int gi = wave_scan(g), ei = wave_scan(e);
    if (lane == kWave - 1) {
      wsum[0][w] = gi;
      wsum[1][w] = ei;
    }
    lds_barrier();
    gt0 = sum_waves(wsum[0], lane, w).all;
    eq0 = sum_waves(wsum[1], lane, w).all;
    lds_barrier();
  } else if (all) {
    gt0 = from;
  }
  int sure = 0, tie = 0;
#pragma unroll
  for (int j = 0; j < kRunPer; ++j) {
    const uint32_t k = order_of(v[j]);
    const bool in = i0 + j * kWave < mid;
    sure |= (in && (all || (select && k > f.cut))) << j;
    tie |= (in && select && k == f.cut) << j;
  }
  const Kept mine = wave_kept<kRunPer>(sure, tie);
  if (lane == 0) {
    kept[0][w] = mine.gt;
    kept[1][w] = mine.eq;
  }
  lds_barrier();
  Kept before{gt0 + sum_waves(kept[0], lane, w).before, eq0 + sum_waves(kept[1], lane, w).before};
#pragma unroll
  for (int j = 0; j < kRunPer; ++j) {
    const int i = i0 + j * kWave;
    int at;
    const bool stays = place(before, sure, tie, j, f.ties, at);
    if (i >= mid) continue;
    if (stays) {
      new_slots[rg.first + at] = s[j];
      new_scores[rg.first + at] = v[j];
    } else if (i - at < a.freed_width) {
      freed[i - at] = s[j];
    }
  }
}

// What stayed comes back, with empty entries behind it.
__global__ void __launch_bounds__(kThreads) evict_return_kernel(EvictArgs a) {
  const int b = blockIdx.y;
  const Range rg = range_of(a, b);
  const int64_t row = clamp_i64(a.rows[b], 0, a.table_rows - 1);
  const int64_t to = a.out_rows ? clamp_i64(a.out_rows[b], 0, a.table_rows - 1) : row;
  int64_t* slots = a.table + to * a.table_stride;
  float* scores = a.scores + to * a.scores_stride;
  const int64_t* from_slots = a.moved_slots + (int64_t)b * a.max_len;
  const float* from_scores = a.moved_scores + (int64_t)b * a.max_len;
  if (to == row && rg.left == rg.n) return;
  for (int i = blockIdx.x * kThreads + threadIdx.x; i < rg.n; i += gridDim.x * kThreads) {
    const bool there = i < rg.left;
    slots[i] = there ? from_slots[i] : -1;
    scores[i] = there ? from_scores[i] : 0.f;
  }
}

struct SplitPlan {
  int32_t n_runs;
  int64_t counts_bytes, above_bytes, cuts_bytes, slots_bytes, scores_bytes;
  int64_t total() const {
    return counts_bytes + above_bytes + cuts_bytes + slots_bytes + scores_bytes;
  }
};
SplitPlan split_plan(int64_t max_len, int32_t batch) {
  SplitPlan p;
  p.n_runs = (int32_t)((max_len + kRunEntries - 1) / kRunEntries);
  p.counts_bytes = (int64_t)batch * 3 * p.n_runs * kBins * 4;
  p.above_bytes = ((int64_t)batch * p.n_runs * 4 + 255) / 256 * 256;
  p.cuts_bytes = ((int64_t)batch * 3 * 8 + 255) / 256 * 256;
  p.slots_bytes = (int64_t)batch * max_len * 8;
  p.scores_bytes = (int64_t)batch * max_len * 4;
  return p;
}
// Rows that may be this long are split (see the top).
constexpr int64_t kSplitLen = 16 * kThreads + 1;

// With as few entries a thread as hold the row: what the kernel does not need it does not
// fetch (its unrolled code is read once, by every CU's first wave).
template <int PER>
void launch_evict(const EvictArgs& a, int32_t batch, hipStream_t s) {
  if constexpr (PER < 16)
    if (a.max_len > PER * kThreads) return launch_evict<2 * PER>(a, batch, s);
  hipLaunchKernelGGL(evict_kernel<PER>, dim3((unsigned)batch), dim3(kThreads), 0, s, a);
}

}  // namespace
}  // namespace tfa

extern "C" int64_t tf_evict_workspace_bytes(int64_t max_len, int64_t rtt_cols,
                                            int32_t batch_size) {
  using namespace tfa;
  clear_error();
  if (max_len < 0 || rtt_cols < 1 || batch_size < 0)
    return fail(TF_ERR_INVALID, "evict: max_len=%lld rtt_cols=%lld batch_size=%d",
                (long long)max_len, (long long)rtt_cols, batch_size);
  const int64_t len = max_len < rtt_cols ? max_len : rtt_cols;
  return len < kSplitLen ? 0 : split_plan(len, batch_size).total();
}

extern "C" int32_t tf_evict_tokens(
    int64_t* req_to_token, int64_t rtt_rows, int64_t rtt_row_stride, int64_t rtt_cols,
    float* scores, int64_t scores_row_stride, const int64_t* rows, const int64_t* out_rows,
    const int64_t* seq_lens, const int64_t* first, int64_t first_n, int64_t recent, int64_t keep,
    int64_t max_len, int32_t batch_size, int64_t* new_lens, int64_t* freed, int64_t freed_width,
    void* workspace, int64_t workspace_bytes, tf_stream_t stream) {
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
  if (max_len > rtt_cols) max_len = rtt_cols;
  if (freed_width < max_len - keep)
    return fail(TF_ERR_INVALID, "evict: freed needs room for %lld slots a request",
                (long long)(max_len - keep));
  if (batch_size > 65535) return fail(TF_ERR_UNSUPPORTED, "evict: batch_size=%d", batch_size);
  const int64_t need = tf_evict_workspace_bytes(max_len, rtt_cols, batch_size);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(TF_ERR_INVALID, "evict: workspace needs %lld bytes, got %lld", (long long)need,
                (long long)workspace_bytes);
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
  a.first_n = std::min(first_n, max_len);   // (no row has more, and no sum of theirs overflows)
  a.recent = std::min(recent, max_len);
  a.keep = std::min(keep, max_len);
  a.max_len = max_len;
  a.lens_out = new_lens;
  a.freed = freed;
  a.freed_width = freed_width;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (need == 0) {
    launch_evict<2>(a, batch_size, s);
    return launch_status("tf_evict_tokens launch");
  }
  const SplitPlan p = split_plan(max_len, batch_size);
  char* ws = static_cast<char*>(workspace);
  a.n_runs = p.n_runs;
  a.counts = reinterpret_cast<int32_t*>(ws);
  a.above = reinterpret_cast<int32_t*>(ws += p.counts_bytes);
  a.cuts = reinterpret_cast<int2*>(ws += p.above_bytes);
  a.moved_slots = reinterpret_cast<int64_t*>(ws += p.cuts_bytes);
  a.moved_scores = reinterpret_cast<float*>(ws += p.slots_bytes);
  const dim3 grid((unsigned)p.n_runs, (unsigned)batch_size), block(kThreads);
  hipLaunchKernelGGL(evict_count_kernel<0>, grid, block, 0, s, a);
  hipLaunchKernelGGL(evict_count_kernel<1>, grid, block, 0, s, a);
  hipLaunchKernelGGL(evict_count_kernel<2>, grid, block, 0, s, a);
  hipLaunchKernelGGL(evict_move_kernel, grid, block, 0, s, a);
  hipLaunchKernelGGL(evict_return_kernel, grid, block, 0, s, a);
  return launch_status("tf_evict_tokens launch");
}
