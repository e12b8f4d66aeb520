// How much attention every cached token gets (tf_attn_weights): the softmax weights that
// the last `window` new tokens of each request give its keys, summed over those tokens
// and all query heads.  For steps with prompts; a decode step's come with its attention
// (prefix_attn.hip, SCORED).
//
//   w[b, k] = sum_{t, h} 2^(s[t, h, k] - lse[t, h]),  s = q . k scale log2 e,
//   lse = log2 sum_k 2^s over the keys that (t, h) sees.
// Only K is read, twice: the weights need every row's lse first, and the scores cost less
// to compute again (MFMA) than to keep: a row's scores are 4 bytes a key, 32 tokens of 24
// heads 3 KB a key, where the K row of 4 heads of 256 is 2 KB.
//
// row_stats_kernel: workgroup (128 keys, request, kv head), 32 keys per wave, the wave's
// K rows in registers as MFMA operands; the rows (t, h) of the kv head's group pass by in
// blocks of 32 through LDS.  S^T[key, row] = K Q^T leaves a row's scores in lanes n and
// n + 32, whose maximum and sum of 2^(s - max) are joined over the waves and written per
// (row, 128 keys).  row_lse_kernel joins those.  key_sums_kernel is the same loop with
// 2^(s - lse) summed per key over the rows, per kv head, in a fixed order; add_sums_kernel
// adds the heads' sums (no atomics: results do not depend on timing) into the scores.
//
// Bound by latency.  4 prompts of 2048 new tokens on contexts of up to 10000, 24 / 4 heads of
// 256, window 32 (192 rows): 43 us of statistics and 45 of sums, 11 GFLOP and 58 MB of K
// each, 5 for either small launch, where the attention itself takes 1100; a workgroup takes
// 1.6 us for its window, 4 to 7 for its keys and 2 per block of rows.  No faster: waves of
// 64 keys, blocks of 64 rows, one barrier per block, three waves per SIMD in place of two.
// Where keys are few, workgroups share a window's row blocks (3 prompts of 174 tokens on 190:
// 14 and 16 us by one, 7 and 9.5 by six).
#include <math.h>

#include <algorithm>

#include "tf_common.h"
#include "tf_internal.h"

namespace tfa {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kKeys = 32 * kWaves;   // keys of a workgroup
constexpr int kBlock = 32;           // query rows per step

struct WeightArgs {
  const __bf16* q;
  int64_t q_stride, q_rows;
  const uint8_t* k_pool;
  int64_t pool_slots;
  const float* k_scale;
  const int64_t* rtt;
  int64_t rtt_rows, rtt_stride, rtt_cols;
  const int64_t* rpi;
  const int64_t* seq_lens;
  int32_t seq_override;
  const int64_t* extend_lens;   // NULL: one new token each
  int32_t batch, window, hkv, group, head_dim;
  int32_t cap;                  // keys that the workspace has room for (a multiple of 128)
  int32_t rows_cap;             // rows of a kv head it has room for
  int32_t splits;               // workgroups that share the row blocks of 128 keys
  float scale_log2;
  float2* stats;                // [b][hk][row][cap / 128]
  float* lse;                   // [b][hk][row]
  float* sums;                  // [b][hk][split][cap]
  float* scores;
  int64_t scores_stride;
  int32_t add;
};

__device__ __forceinline__ int context_len(const WeightArgs& a, int b) {
  const int64_t len = min(min(a.seq_override > 0 ? (int64_t)a.seq_override : a.seq_lens[b],
                              a.rtt_cols), (int64_t)a.cap);
  return len > 0 ? (int)len : 0;
}

// The request's window: its tokens, and the q row of the first of them.  Every thread of
// the workgroup calls it.
struct Window {
  int n_tok;
  int64_t qrow;
};
__device__ Window window_of(const WeightArgs& a, int b, int64_t* red) {
  if (!a.extend_lens) return Window{1, b};
  int64_t before = 0;
  for (int i = threadIdx.x; i < b; i += blockDim.x) before += a.extend_lens[i];
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) before += __shfl_xor(before, m, kWave);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = before;
  __syncthreads();
  before = 0;
  for (int i = 0; i < (int)blockDim.x / kWave; ++i) before += red[i];
  const int64_t ext = a.extend_lens[b];
  const int n = (int)max<int64_t>(0, min(min<int64_t>(ext, a.window),
                                         (int64_t)a.rows_cap / a.group));
  return Window{n, before + ext - n};
}

// The row blocks of a workgroup: its share of the window's.
struct Blocks {
  int first, end;
};
__device__ __forceinline__ Blocks blocks_of(const WeightArgs& a, const Window& win, int split) {
  const int n = (win.n_tok * a.group + kBlock - 1) / kBlock;
  const int each = (n + a.splits - 1) / a.splits;
  return Blocks{min(n, split * each), min(n, (split + 1) * each)};
}

// One request's kv head against 128 keys, as the two passes share it.
template <int DP, bool FP8>
struct Tile {
  static constexpr int kSteps = DP / 16;
  static constexpr int kChunks = DP / 8;   // 16-byte chunks of a staged q row
  static constexpr int kLoads = kBlock * kChunks / kThreads;   // per thread and block
  static_assert(kLoads >= 1, "block loads");
  u32x4 kf[kSteps];

  // K^T operand: lane (g, n) holds dims 16 kk + 8 g .. + 7 of the wave's key n; keys past
  // the last repeat it (their scores are masked).
  __device__ __forceinline__ void load_keys(const WeightArgs& a, const int64_t* rtt, int key0,
                                            int len, int hk, int lane) {
    const int g = lane >> 5, n = lane & 31;
    const int64_t slot = pool_row(rtt[min(key0 + n, len - 1)], a.pool_slots, a.seq_override > 0);
    const int row_bytes = FP8 ? a.head_dim : 2 * a.head_dim;
    const uint8_t* p = a.k_pool + (slot * a.hkv + hk) * row_bytes;
#pragma unroll
    for (int kk = 0; kk < kSteps; ++kk) {
      const int d = 16 * kk + 8 * g;
      if (d >= a.head_dim) {
        kf[kk] = u32x4{0u, 0u, 0u, 0u};
      } else if (FP8) {
        const u32x2 x = ld_g8(p + d);
        kf[kk] = e4m3x8_to_bf16x8(x[0], x[1]);
      } else {
        kf[kk] = ld_g16(p + 2 * d);
      }
    }
  }

  // Rows block * 32 .. + 31 (past the last one: repeats of it).
  __device__ __forceinline__ void fetch(const WeightArgs& a, const Window& win, int hk, int block,
                                        u32x4 (&x)[kLoads]) const {
    const int n_rows = win.n_tok * a.group;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = i * kThreads + threadIdx.x;
      const int c = at % kChunks;
      const int rho = min(block * kBlock + at / kChunks, n_rows - 1);
      const int t = rho / a.group, h = rho - t * a.group;
      x[i] = 8 * c < a.head_dim
                 ? ld_g16(a.q + clamp_i64(win.qrow + t, 0, a.q_rows - 1) * a.q_stride +
                          (int64_t)(hk * a.group + h) * a.head_dim + 8 * c)
                 : u32x4{0u, 0u, 0u, 0u};
    }
  }
  // Chunk c of row r at c ^ r, free of bank conflicts for the operand reads.
  __device__ __forceinline__ void stage(u32x4* lds, const u32x4 (&x)[kLoads]) const {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = i * kThreads + threadIdx.x;
      const int c = at % kChunks, r = at / kChunks;
      lds[r * kChunks + ((c ^ r) & (kChunks - 1))] = x[i];
    }
  }
  // S^T[key 8 (r / 4) + 4 g + r % 4][row n] of the staged block, raw.
  __device__ __forceinline__ f32x16 scores(const u32x4* lds, int lane) const {
    const int g = lane >> 5, n = lane & 31;
    f32x16 s = {};
#pragma unroll
    for (int kk = 0; kk < kSteps; ++kk)
      s = mfma_32x32x16(kf[kk], lds[n * kChunks + (((2 * kk + g) ^ n) & (kChunks - 1))], s);
    return s;
  }
};

// Keys that the row at position n of a block sees, counted from the wave's first key.
__device__ __forceinline__ int row_seen(const WeightArgs& a, const Window& win, int rho, int len,
                                        int key0) {
  const int t = min(rho / a.group, win.n_tok - 1);
  return len - (win.n_tok - 1 - t) - key0;
}

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, kWave); }

template <int DP, bool FP8>
__global__ void __launch_bounds__(kThreads) row_stats_kernel(WeightArgs a) {
  using T = Tile<DP, FP8>;
  __shared__ u32x4 qs[kBlock * T::kChunks];
  __shared__ float2 part[2][kWaves][kBlock];
  __shared__ int64_t red[kWaves];
  const int b = blockIdx.y, hk = blockIdx.z / a.splits;
  const int lane = threadIdx.x & 63, w = wave_id(), g = lane >> 5, n = lane & 31;
  const int len = context_len(a, b);
  const Window win = window_of(a, b, red);
  const int n_rows = win.n_tok * a.group;
  const Blocks blocks = blocks_of(a, win, blockIdx.z % a.splits);
  if (len == 0 || blocks.first >= blocks.end) return;
  const int64_t* rtt = a.rtt + clamp_i64(a.rpi[b], 0, a.rtt_rows - 1) * a.rtt_stride;
  const float sl2 = a.scale_log2 * (FP8 ? a.k_scale[0] : 1.f);
  const int tiles = a.cap / kKeys;
  float2* stats = a.stats + ((int64_t)b * a.hkv + hk) * a.rows_cap * tiles;

  for (int tile = blockIdx.x; tile * kKeys < len; tile += gridDim.x) {
    const int key0 = tile * kKeys + 32 * w;
    T tl;
    u32x4 x[T::kLoads];
    tl.fetch(a, win, hk, blocks.first, x);
    tl.load_keys(a, rtt, key0, len, hk, lane);
    for (int i = blocks.first; i < blocks.end; ++i) {
      __syncthreads();   // the block before is read
      tl.stage(qs, x);
      __syncthreads();
      if (i + 1 < blocks.end) tl.fetch(a, win, hk, i + 1, x);
      f32x16 s = tl.scores(qs, lane);
      const int seen = row_seen(a, win, i * kBlock + n, len, key0);
      float m = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = 8 * (r >> 2) + 4 * g + (r & 3) < seen ? s[r] * sl2 : -INFINITY;
        m = fmaxf(m, s[r]);
      }
      m = fmaxf(m, other_half(m));
      const float ref = m == -INFINITY ? 0.f : m;
      float l = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) l += fast_exp2(s[r] - ref);
      l += other_half(l);
      if (g == 0) part[i & 1][w][n] = float2{m, l};
      __syncthreads();
      if (w == 0 && g == 0 && i * kBlock + n < n_rows) {
        float2 ml = part[i & 1][0][n];
#pragma unroll
        for (int k = 1; k < kWaves; ++k) {
          const float2 o = part[i & 1][k][n];
          const float mn = fmaxf(ml.x, o.x);
          const float rf = mn == -INFINITY ? 0.f : mn;
          ml = float2{mn, ml.y * fast_exp2(ml.x - rf) + o.y * fast_exp2(o.x - rf)};
        }
        stats[(int64_t)(i * kBlock + n) * tiles + tile] = ml;
      }
    }
  }
}

// One wave per row: lse over the tiles of 128 keys (-inf where the row sees none).
template <int kRowsWg>
__global__ void __launch_bounds__(kRowsWg * kWave) row_lse_kernel(WeightArgs a) {
  __shared__ int64_t red[kRowsWg];
  const int b = blockIdx.y, hk = blockIdx.z;
  const int lane = threadIdx.x & 63;
  const int row = blockIdx.x * kRowsWg + wave_id();
  const int len = context_len(a, b);
  const Window win = window_of(a, b, red);
  if (len == 0 || row >= win.n_tok * a.group) return;
  const int tiles = a.cap / kKeys, used = (len + kKeys - 1) / kKeys;
  const int64_t at = ((int64_t)b * a.hkv + hk) * a.rows_cap + row;
  float m = -INFINITY, l = 0.f;
  for (int i = lane; i < used; i += kWave) {
    const float2 o = a.stats[at * tiles + i];
    const float mn = fmaxf(m, o.x);
    const float rf = mn == -INFINITY ? 0.f : mn;
    l = l * fast_exp2(m - rf) + o.y * fast_exp2(o.x - rf);
    m = mn;
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    const float m2 = __shfl_xor(m, d, kWave), l2 = __shfl_xor(l, d, kWave);
    const float mn = fmaxf(m, m2);
    const float rf = mn == -INFINITY ? 0.f : mn;
    l = l * fast_exp2(m - rf) + l2 * fast_exp2(m2 - rf);
    m = mn;
  }
  // (NaN scores: a NaN sum, whose logarithm passes on to every weight of the row; so does the
  // -inf of a row whose keys all score -inf)
  if (lane == 0) a.lse[at] = m + log2f(l);
}

template <int DP, bool FP8>
__global__ void __launch_bounds__(kThreads) key_sums_kernel(WeightArgs a) {
  using T = Tile<DP, FP8>;
  __shared__ u32x4 qs[kBlock * T::kChunks];
  __shared__ int64_t red[kWaves];
  const int b = blockIdx.y, hk = blockIdx.z / a.splits;
  const int lane = threadIdx.x & 63, w = wave_id(), g = lane >> 5, n = lane & 31;
  const int len = context_len(a, b);
  const Window win = window_of(a, b, red);
  const int n_rows = win.n_tok * a.group;
  const Blocks blocks = blocks_of(a, win, blockIdx.z % a.splits);
  if (len == 0) return;
  const int64_t* rtt = a.rtt + clamp_i64(a.rpi[b], 0, a.rtt_rows - 1) * a.rtt_stride;
  const float sl2 = a.scale_log2 * (FP8 ? a.k_scale[0] : 1.f);
  const float* lse = a.lse + ((int64_t)b * a.hkv + hk) * a.rows_cap;
  // (a share without rows writes zeros)
  float* sums = a.sums + ((int64_t)b * a.hkv * a.splits + blockIdx.z) * a.cap;

  for (int tile = blockIdx.x; tile * kKeys < len; tile += gridDim.x) {
    const int key0 = tile * kKeys + 32 * w;
    T tl;
    u32x4 x[T::kLoads];
    if (blocks.first < blocks.end) {
      tl.fetch(a, win, hk, blocks.first, x);
      tl.load_keys(a, rtt, key0, len, hk, lane);
    }
    f32x16 acc = {};
    for (int i = blocks.first; i < blocks.end; ++i) {
      const int rho = i * kBlock + n;
      const float off = rho < n_rows ? lse[rho] : INFINITY;   // (repeats of the last row)
      __syncthreads();
      tl.stage(qs, x);
      __syncthreads();
      if (i + 1 < blocks.end) tl.fetch(a, win, hk, i + 1, x);
      const f32x16 s = tl.scores(qs, lane);
      const int seen = rho < n_rows ? row_seen(a, win, rho, len, key0) : 0;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        acc[r] += 8 * (r >> 2) + 4 * g + (r & 3) < seen ? fast_exp2(fmaf(s[r], sl2, -off)) : 0.f;
    }
    __syncthreads();
    // Sums over the 32 rows: lanes hand each other the half of their keys that they give up,
    // until lane n is left with register n / 2.
#pragma unroll
    for (int half = 8; half >= 1; half /= 2) {
      const bool up = n & (2 * half);
#pragma unroll
      for (int r = 0; r < half; ++r) {
        const float kept = up ? acc[r + half] : acc[r], given = up ? acc[r] : acc[r + half];
        acc[r] = kept + __shfl_xor(given, 2 * half, kWave);
      }
    }
    const float v = acc[0] + __shfl_xor(acc[0], 1, kWave);
    const int r = n >> 1;
    if (!(n & 1)) sums[key0 + 8 * (r >> 2) + 4 * g + (r & 3)] = v;
  }
}

// scores[row, k] (+)= the sums of the kv heads and splits, for the keys of each request.
__global__ void __launch_bounds__(kThreads) add_sums_kernel(WeightArgs a) {
  const int b = blockIdx.y;
  const int len = context_len(a, b);
  float* out = a.scores + clamp_i64(a.rpi[b], 0, a.rtt_rows - 1) * a.scores_stride;
  const int parts = a.hkv * a.splits;
  const float* sums = a.sums + (int64_t)b * parts * a.cap;
  for (int k = blockIdx.x * kThreads + threadIdx.x; k < len; k += gridDim.x * kThreads) {
    float v = 0.f;
#pragma unroll 8
    for (int h = 0; h < parts; ++h) v += sums[(int64_t)h * a.cap + k];
    out[k] = a.add ? out[k] + v : v;
  }
}

struct WeightPlan {
  int32_t cap, rows_cap, splits;
  int64_t stats_bytes, lse_bytes, sums_bytes;
  int64_t total() const { return stats_bytes + lse_bytes + sums_bytes; }
};

int make_weight_plan(int32_t batch, int32_t window, int32_t max_len, int32_t num_q_heads,
                     int32_t num_kv_heads, int32_t head_dim, int32_t kv_dtype, WeightPlan* p) {
  if (batch < 0 || batch > 65535 || window < 1 || max_len < 1)
    return fail(TF_ERR_INVALID, "weights: batch=%d window=%d max_len=%d", batch, window, max_len);
  if (num_kv_heads <= 0 || num_kv_heads > 65535 || num_q_heads <= 0 || num_q_heads % num_kv_heads)
    return fail(TF_ERR_INVALID, "weights: num_q_heads=%d not a multiple of num_kv_heads=%d",
                num_q_heads, num_kv_heads);
  if (kv_dtype != TF_DTYPE_BF16 && kv_dtype != TF_DTYPE_FP8_E4M3)
    return fail(TF_ERR_UNSUPPORTED, "weights: kv_dtype=%d", kv_dtype);
  if (head_dim < 8 || head_dim > 256 || head_dim % 8)
    return fail(TF_ERR_UNSUPPORTED, "weights: head_dim=%d (a multiple of 8 up to 256)", head_dim);
  const int64_t rows = (int64_t)window * (num_q_heads / num_kv_heads);
  const int64_t cap = ((int64_t)max_len + kKeys - 1) / kKeys * kKeys;
  if (rows > (1 << 20) || cap > INT32_MAX - kKeys)
    return fail(TF_ERR_UNSUPPORTED, "weights: %lld rows of %lld keys", (long long)rows,
                (long long)cap);
  p->cap = (int32_t)cap;
  p->rows_cap = (int32_t)rows;
  const int64_t units = (int64_t)batch * num_kv_heads;
  // Row blocks are shared by several workgroups where there are fewer than CUs without.
  const int64_t wgs = std::max<int64_t>(1, units * (cap / kKeys));
  p->splits = (int32_t)std::max<int64_t>(
      1, std::min<int64_t>({(rows + kBlock - 1) / kBlock, device_cu_count() / wgs,
                            65535 / num_kv_heads, 64}));
  p->stats_bytes = (units * rows * (cap / kKeys) * 8 + 255) / 256 * 256;
  p->lse_bytes = (units * rows * 4 + 255) / 256 * 256;
  p->sums_bytes = units * p->splits * cap * 4;
  return TF_OK;
}

template <int DP, bool FP8>
void launch_tiles(const WeightArgs& a, hipStream_t s) {
  const dim3 tiles((unsigned)(a.cap / kKeys), (unsigned)a.batch, (unsigned)(a.hkv * a.splits));
  constexpr int kRowsWg = 4;
  const dim3 rows((unsigned)((a.rows_cap + kRowsWg - 1) / kRowsWg), (unsigned)a.batch,
                  (unsigned)a.hkv);
  hipLaunchKernelGGL((row_stats_kernel<DP, FP8>), tiles, dim3(kThreads), 0, s, a);
  hipLaunchKernelGGL((row_lse_kernel<kRowsWg>), rows, dim3(kRowsWg * kWave), 0, s, a);
  hipLaunchKernelGGL((key_sums_kernel<DP, FP8>), tiles, dim3(kThreads), 0, s, a);
}

template <bool FP8>
void launch_dims(const WeightArgs& a, hipStream_t s) {
  if (a.head_dim <= 64) return launch_tiles<64, FP8>(a, s);
  if (a.head_dim <= 128) return launch_tiles<128, FP8>(a, s);
  return launch_tiles<256, FP8>(a, s);
}

}  // namespace
}  // namespace tfa

extern "C" int64_t tf_attn_weights_workspace_bytes(int32_t batch_size, int32_t window,
                                                   int32_t max_len, int32_t num_q_heads,
                                                   int32_t num_kv_heads, int32_t head_dim,
                                                   int32_t kv_dtype) {
  using namespace tfa;
  clear_error();
  WeightPlan p;
  const int rc = make_weight_plan(batch_size, window, max_len, num_q_heads, num_kv_heads,
                                  head_dim, kv_dtype, &p);
  return rc != TF_OK ? rc : p.total();
}

extern "C" int32_t tf_attn_weights(
    const void* q, int64_t q_row_stride, int64_t q_rows, const void* k_pool, int64_t pool_slots,
    int32_t kv_dtype, const float* k_scale, const int64_t* req_to_token, int64_t rtt_rows,
    int64_t rtt_row_stride, int64_t rtt_cols, const int64_t* req_pool_indices,
    const int64_t* seq_lens, int32_t seq_len_override, const int64_t* extend_lens, int32_t batch_size, int32_t window,
    int32_t max_len, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, float scale,
    float* scores, int64_t scores_row_stride, int32_t add, void* workspace,
    int64_t workspace_bytes, tf_stream_t stream) {
  using namespace tfa;
  clear_error();
  if (!extend_lens) window = 1;
  WeightPlan p;
  int rc = make_weight_plan(batch_size, window, max_len, num_q_heads, num_kv_heads, head_dim,
                            kv_dtype, &p);
  if (rc != TF_OK) return rc;
  if (batch_size == 0) return TF_OK;
  if (q_rows < 1) return fail(TF_ERR_INVALID, "weights: q_rows=%lld", (long long)q_rows);
  // (the pool stands for V, q for the output: neither is used here)
  rc = check_slot_call("weights", q, q_row_stride, k_pool, k_pool, pool_slots, kv_dtype, k_scale,
                       k_scale, req_to_token, rtt_rows, rtt_row_stride, rtt_cols,
                       req_pool_indices, seq_lens, seq_len_override, num_q_heads, head_dim, q,
                       q_row_stride, nullptr, 0, 0, workspace, workspace_bytes, p.total());
  if (rc != TF_OK) return rc;
  if (!scores || scores_row_stride < rtt_cols)
    return fail(TF_ERR_INVALID, "weights: scores need rows of at least %lld", (long long)rtt_cols);
  WeightArgs a = {};
  a.q = static_cast<const __bf16*>(q);
  a.q_stride = q_row_stride;
  a.q_rows = q_rows;
  a.k_pool = static_cast<const uint8_t*>(k_pool);
  a.pool_slots = pool_slots;
  a.k_scale = k_scale;
  a.rtt = req_to_token;
  a.rtt_rows = rtt_rows;
  a.rtt_stride = rtt_row_stride;
  a.rtt_cols = rtt_cols;
  a.rpi = req_pool_indices;
  a.seq_lens = seq_lens;
  a.seq_override = seq_len_override;
  a.extend_lens = extend_lens;
  a.batch = batch_size;
  a.window = window;
  a.hkv = num_kv_heads;
  a.group = num_q_heads / num_kv_heads;
  a.head_dim = head_dim;
  a.cap = p.cap;
  a.rows_cap = p.rows_cap;
  a.splits = p.splits;
  a.scale_log2 = scale * kLog2e;
  char* ws = static_cast<char*>(workspace);
  a.stats = reinterpret_cast<float2*>(ws);
  a.lse = reinterpret_cast<float*>(ws + p.stats_bytes);
  a.sums = reinterpret_cast<float*>(ws + p.stats_bytes + p.lse_bytes);
  a.scores = scores;
  a.scores_stride = scores_row_stride;
  a.add = add;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (kv_dtype == TF_DTYPE_FP8_E4M3)
    launch_dims<true>(a, s);
  else
    launch_dims<false>(a, s);
  const int64_t blocks = ((int64_t)p.cap + kThreads - 1) / kThreads;
  const dim3 grid((unsigned)std::min<int64_t>(blocks, 64), (unsigned)batch_size);
  hipLaunchKernelGGL(add_sums_kernel, grid, dim3(kThreads), 0, s, a);
  return launch_status("tf_attn_weights launch");
}
