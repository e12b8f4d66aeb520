// Eviction of cached tokens by their attention weight (tf_evict_tokens): of each
// request's table row, the first tokens and the last ones stay, and of those between as
// many of the largest scores as the budget leaves room for; what stays moves together,
// in order, and the slots of the others are handed back.
//
// One workgroup per request, or for rows that may be longer than 16384 five launches of
// one per 8192 entries: the same digits counted per run, each launch deriving a digit from
// the counts of the one before (kernel boundaries order them: no atomics, nothing to
// clear), then the moves into scratch and back.  Bound by latency: 8 rows of 131072 take
// 183 us by a workgroup each, whose CU moves 25 GB/s, and 44 in launches; of 24576 42 and
// 34; of 16384 27 and 33 (longer ones are no longer read once for all three digits).
//
// The room-th largest score is found digit by digit (radix selection over the scores'
// order-preserving integers, 11 bits at a time, counted in LDS), the entries above it
// stay and of the equal ones the first.  Then one ordered pass moves slots and scores:
// positions come from a scan over the workgroup and a running count.  In place: an entry
// moves to its own or an earlier position, a chunk is read before any of it is written,
// and no chunk is written before the ones in front of it.
#include <math.h>

#include <algorithm>

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
constexpr int kAhead = 16;                     // scores of a thread in flight

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

__device__ __forceinline__ int wave_scan(int v, int lane) {   // inclusive
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const int o = __shfl_up(v, off, kWave);
    if (lane >= off) v += o;
  }
  return v;
}

// Sum over the waves in front of this one, and over all, of each wave's `mine`: through
// wsum, which the caller guards with barriers on both sides.
struct WaveSums {
  int before, all;
};
__device__ __forceinline__ WaveSums sum_waves(const int32_t* wsum, int lane, int w) {
  const int v = wave_scan(lane < kWaves ? wsum[lane] : 0, lane);
  return WaveSums{w ? __shfl(v, w - 1, kWave) : 0, __shfl(v, kWaves - 1, kWave)};
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
  const int incl = wave_scan(c0 + c1, lane);
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

// Places of PER entries a thread, entry j being number j * kThreads + thread: how many
// before it stay for certain (sure), and how many are ties, from counts per wave in LDS.
template <int PER>
struct Places {
  int32_t counts[2][PER * kWaves];
};
template <int PER>
__device__ __forceinline__ void places(Places<PER>& lds, int sure, int tie, int lane, int w,
                                       int (&gt)[PER], int (&eq)[PER], int& all_gt, int& all_eq) {
  static_assert(PER * kWaves == kWave || PER * kWaves == 2 * kWave, "one or two counts a lane");
  constexpr int kEach = PER * kWaves / kWave;
  int own[2][PER];   // before the entry within its wave
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const uint64_t below = (1ull << lane) - 1;
    const uint64_t ms = __ballot(sure >> j & 1), mt = __ballot(tie >> j & 1);
    own[0][j] = __popcll(ms & below);
    own[1][j] = __popcll(mt & below);
    if (lane == 0) {
      lds.counts[0][j * kWaves + w] = __popcll(ms);
      lds.counts[1][j * kWaves + w] = __popcll(mt);
    }
  }
  lds_barrier();
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    int n[kEach], sum = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) sum += n[e] = lds.counts[c][lane * kEach + e];
    const int incl = wave_scan(sum, lane);
    (c ? all_eq : all_gt) = __shfl(incl, kWave - 1, kWave);
    int before[kEach];   // the lane's counts
    before[0] = incl - sum;
    if (kEach == 2) before[kEach - 1] = incl - n[kEach - 1];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int at = j * kWaves + w;
      const int v = __shfl(before[0], at / kEach, kWave);
      const int u = kEach == 2 ? __shfl(before[kEach - 1], at / kEach, kWave) : v;
      (c ? eq : gt)[j] = own[c][j] + (at % kEach ? u : v);
    }
  }
}

__global__ void __launch_bounds__(kThreads) evict_kernel(EvictArgs a) {
  __shared__ int32_t bins[kBins];
  __shared__ int32_t wsum[kWaves];
  __shared__ Places<kPer> order;
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
  const int mid = rg.end - rg.first;
  const bool select = rg.room > 0 && rg.room < mid;
  if (select) {
    // Scores kAhead at a time: those of a short range are read once and stay.
    uint32_t key[kAhead];
    auto load = [&](int base) {
      float v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int i = base + j * kThreads + tid;
        v[j] = i < mid ? scores[rg.first + i] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) key[j] = order_of(v[j]);
    };
    constexpr int kRun = kAhead * kThreads;
    if (mid <= kRun) load(0);
    uint32_t mask = 0;
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = digit_shift(pass);
      const uint32_t digit = digit_mask(pass);
      for (int i = tid; i < kBins; i += kThreads) bins[i] = 0;
      lds_barrier();
      for (int base = 0; base < mid; base += kRun) {
        if (mid > kRun) load(base);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          if (base + j * kThreads >= mid) break;
          if (base + j * kThreads + tid < mid && (key[j] & mask) == cut)
            count(bins, (key[j] >> shift) & digit);
        }
      }
      lds_barrier();
      find_digit(bins, ties, wsum, found, lane, w);
      cut |= found[0] << shift;
      ties = (int)found[1];
      mask |= digit << shift;
    }
  }

  // ---- the ordered pass, a chunk's entries read while the one before it moves
  const bool nothing = rg.left == rg.n;
  int gt0 = 0, eq0 = 0;   // entries before the chunk that stay for certain / that are ties
  const int start = nothing && to == row ? rg.n : 0;
  int64_t s[kPer];
  float v[kPer];
  auto read = [&](int c0) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = c0 + j * kThreads + tid;
      if (i < rg.n) {
        s[j] = slots[i];
        v[j] = scores[i];
      }
    }
  };
  if (start < rg.n) read(start);
  for (int c0 = start; c0 < rg.n; c0 += kChunk) {
    int64_t my_s[kPer];
    float my_v[kPer];
    int sure = 0, tie = 0;   // bit per entry
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = c0 + j * kThreads + tid;
      my_s[j] = s[j];
      my_v[j] = v[j];
      if (i >= rg.n) continue;
      if (nothing || i < rg.first || i >= rg.end) {
        sure |= 1 << j;
      } else if (select) {
        const uint32_t k = order_of(my_v[j]);
        sure |= (k > cut) << j;
        tie |= (k == cut) << j;
      }
    }
    // (the chunk's loads have returned before the barrier that lets others write there)
#pragma unroll
    for (int j = 0; j < kPer; ++j) asm volatile("" ::"v"(my_s[j]), "v"(my_v[j]));
    if (c0 + kChunk < rg.n) read(c0 + kChunk);
    int gt[kPer], eq[kPer], all_gt, all_eq;
    places<kPer>(order, sure, tie, lane, w, gt, eq, all_gt, all_eq);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = c0 + j * kThreads + tid;
      if (i >= rg.n) continue;
      const int at = gt0 + gt[j] + min(eq0 + eq[j], ties);
      if ((sure >> j & 1) || ((tie >> j & 1) && eq0 + eq[j] < ties)) {
        new_slots[at] = my_s[j];
        new_scores[at] = my_v[j];
      } else if (i - at < a.freed_width) {
        freed[i - at] = my_s[j];
      }
    }
    gt0 += all_gt;
    eq0 += all_eq;
    lds_barrier();
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
// last from the runs' counts, by every workgroup for itself.
__device__ Found find_cut(const EvictArgs& a, const Range& rg, int b, int passes, int32_t* bins,
                          int32_t* wsum, uint32_t* found) {
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
  const Found f = find_cut(a, rg, b, PASS, bins, wsum, found);
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
    above = wave_scan(above, tid & 63);
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
  __shared__ Places<kRunPer> order;
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
#pragma unroll
  for (int j = 0; j < kRunPer; ++j) {
    const int i = from + j * kThreads + tid;
    if (i >= mid) continue;
    s[j] = slots[rg.first + i];
    v[j] = scores[rg.first + i];
  }
  Found f{0u, 0};
  int gt0 = 0, eq0 = 0;   // of the runs before: above the cut, equal to it
  if (select) {
    f = find_cut(a, rg, b, 3, bins, wsum[0], found);
    const int32_t* counts = a.counts + ((int64_t)b * 3 + 2) * a.n_runs * kBins;
    const uint32_t digit = f.cut & digit_mask(2);
    int g = 0, e = 0;
#pragma unroll 8
    for (int r = 0; r < run; ++r) {
      const int c = counts[(int64_t)r * kBins + tid];   // (the pass has kThreads digits)
      g += (uint32_t)tid > digit ? c : 0;
      e += (uint32_t)tid == digit ? c : 0;
    }
    for (int r = tid; r < run; r += kThreads) g += a.above[(int64_t)b * a.n_runs + r];
    const int gi = wave_scan(g, lane), ei = wave_scan(e, lane);
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
    if (from + j * kThreads + tid >= mid) continue;
    const uint32_t k = order_of(v[j]);
    sure |= (all || (select && k > f.cut)) << j;
    tie |= (select && k == f.cut) << j;
  }
  int gt[kRunPer], eq[kRunPer], all_gt, all_eq;
  places<kRunPer>(order, sure, tie, lane, w, gt, eq, all_gt, all_eq);
#pragma unroll
  for (int j = 0; j < kRunPer; ++j) {
    const int i = from + j * kThreads + tid;
    if (i >= mid) continue;
    const int at = gt0 + gt[j] + min(eq0 + eq[j], f.ties);
    if ((sure >> j & 1) || ((tie >> j & 1) && eq0 + eq[j] < f.ties)) {
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
constexpr int64_t kSplitLen = kAhead * kThreads + 1;

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
    hipLaunchKernelGGL(evict_kernel, dim3((unsigned)batch_size), dim3(kThreads), 0, s, a);
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
