// FP8 products with a scale for each block of 128, and the gated feed-forward
// block built from them.
//
// A matrix held in 8 bits is e4m3 values with one fp32 scale per row and 128
// columns (activations) or per 128 x 128 block (weights):
//   quantise   s = fl32(max(amax|x|, 1e-12) / 448),  q = e4m3(fl32(x / s))
//   product    out[m][n] = sum_kb xs[m][kb] ws[n / 128][kb] (xq w^T)[m][n] over block kb
//   gated MLP  h = silu(x Wg^T) (x Wu^T) in fp32, quantised, times Wd^T
// The weights are the reference's block-FP8 linears' (qwen3_8/fp8_linear.py:12-212),
// the block its Qwen3_8MLP (qwen3_8/mlp.py:9-54).  A scale per block instead of
// one per tensor (fp8_linear.hip) keeps a row's result free of the other rows' values
// and needs no pass over the whole tensor before the first value is written, so
// the quantisation folds into whatever produces the values.
#include <algorithm>

#include "block_plan.h"
#include "block_quant.h"
#include "fp8_tile.h"
#include "tf_common.h"
#include "tf_internal.h"

namespace tfa {
namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------- quantisation
// One wave: kQuantRows rows x 4 blocks of 128 columns, a row's 512 at a time; 16
// lanes hold a block's columns, 8 each.  All of a lane's loads are issued before
// the first is used.  Scales are stored [block][row].  HBM-bound: 8192 x 17408 bf16
// 84 us = 5.1 TB/s, as fast as a copy; 48 x 6144 3.8, a launch and a load.
constexpr int kQuantCols = 4 * kQBlock;
constexpr int kQuantRows = 4;
constexpr int kQuantWgRows = kQuantRows * (kThreads / kWave);

struct BlockQuantArgs {
  const uint8_t* x;
  int64_t xs;              // row stride, elements
  int64_t rows;
  int32_t cols, out_cols;  // out_cols: cols, or more to write zeros behind them
  uint8_t* xq;
  int64_t qs;
  float* scale;
  int64_t ss;              // scale of (row, block) at block * ss + row
  int32_t col_groups;
};

template <bool F32>
__global__ void __launch_bounds__(kThreads) block_quant_kernel(BlockQuantArgs a) {
  const int64_t rg = blockIdx.x / a.col_groups;
  const int cg = (int)(blockIdx.x - rg * a.col_groups);
  const int l = threadIdx.x & 63;
  const int64_t row0 = rg * kQuantWgRows + wave_id() * kQuantRows;
  const int c = cg * kQuantCols + 8 * l;
  float v[kQuantRows][8];
#pragma unroll
  for (int r = 0; r < kQuantRows; ++r) {
    if (row0 + r < a.rows && c < a.cols) {
      load8<F32>(a.x, (row0 + r) * a.xs + c, v[r]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[r][j] = 0.f;
    }
  }
#pragma unroll
  for (int r = 0; r < kQuantRows; ++r) {
    const int64_t row = row0 + r;
    if (row >= a.rows) break;   // (a wave's rows are its own)
    const float s = block_scale(amax_lanes16(amax_bits8(v[r])));
    if (c < a.out_cols)
      *reinterpret_cast<u32x2*>(a.xq + row * a.qs + c) = quant8(v[r], block_div(s));
    if ((l & 15) == 0 && c < a.cols) a.scale[(int64_t)(c / kQBlock) * a.ss + row] = s;
  }
}

// Quantised rows whose last block is short, with zeros behind them (a.x and a.xq in
// bytes, a.cols a multiple of 16): what the tiles stage.  16 bytes a thread.
__global__ void __launch_bounds__(kThreads) block_pad_kernel(BlockQuantArgs a) {
  const int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int per = a.out_cols / 16;
  const int64_t row = e / per;
  if (row >= a.rows) return;
  const int c = 16 * (int)(e - row * per);
  *reinterpret_cast<u32x4*>(a.xq + row * a.qs + c) =
      c < a.cols ? ld_g16(a.x + row * a.xs + c) : u32x4{0u, 0u, 0u, 0u};
}

// ---------------------------------------------------------------- GEMM
constexpr int kSpread = 2, kAtStep = 4;   // staging instructions per row of MFMAs; see below
constexpr int kGroupM = 8;            // m-tiles per group of the XCD tile order

// As fp8_linear.hip's tile: a workgroup of 2 x WN waves owns 32 MT activation
// rows x 64 WN weight rows, a wave 16 MT x 64 of them in 4 x MT 16x16 tiles of
// the transposed product D[n][m].  Large products (8192 rows times 5120 x 2 x 17408:
// 1265 us in a kernel trace = 2.31 PFLOP/s) have the MFMA busy 58 % of the time at the
// 1.9 GHz that the power allows: of an earlier build's 1273 us MFMA and fold alone took
// 763, with the operands' way from LDS 985, the staging alone 955 (81 % of its requests
// hit L2).  Small ones are bound by the 36 to 60 GB/s that a CU's loads into LDS bring
// in, whatever their depth: 48 rows 48.7 us for 178 MB of weights, 3.7 TB/s on the 136
// CUs that have a tile.
template <int MT, int WN, int STAGES>
struct BlockTile {
  static constexpr int kThreads = 2 * kWave * WN;
  static constexpr int kBM = 32 * MT;
  static constexpr int kBN = 64 * WN;
  static constexpr int kXBytes = kBM * kKSlice;
  static constexpr int kWBytes = kBN * kKSlice;
  static constexpr int kScales = kBM + 2;       // row scales, then two column blocks'
  static constexpr int kSInst = (kScales + kThreads - 1) / kThreads;
  static constexpr int kStage = kXBytes + kWBytes + kSInst * kThreads * 4;
  static constexpr int kRowsPerInst = kThreads / 8;
  static constexpr int kXInst = kBM / kRowsPerInst;
  static constexpr int kWInst = kBN / kRowsPerInst;
  static constexpr int kLoads = kXInst + kWInst + kSInst;   // per thread per slice
  static_assert(kBM % kRowsPerInst == 0 && kBN % kRowsPerInst == 0, "staging rows");
};

struct BlockMat {
  const uint8_t* w;       // e4m3 [N, K], row stride wrs bytes
  int64_t wrs;
  const float* wsc;       // scale of column block n / 128, K block kb at nb * sn + kb * sk
  int64_t sn, sk;
  int32_t N;
};

// Output tiles [0, full) are computed whole, by a workgroup each; the rest, which
// would leave CUs idle, by `splits` workgroups each over parts of K, whose fp32
// partial tiles a second kernel adds in split order (the result does not depend on
// timing).  Gate and up products that leave the kernel unfused (n_mats == 2) are all
// partials: their tiles are those of both matrices side by side.
struct BlockGemmArgs {
  const uint8_t* xq;      // e4m3 [M, 128 KB], zeros behind K, row stride xs bytes (few
                          // rows: [M, K], nothing is read behind K)
  int64_t xs;
  const float* xsc;       // scale of (row, block) at block * xss + row
  int64_t xss;
  BlockMat mat[2];        // linear: the weight; gated: gate and up
  int32_t n_mats, tn1;    // tn1: first n-tile of mat[1] where n_mats is 2
  int32_t M, KB;
  int32_t tail;           // bytes of the last K slice that the weights have
  int32_t tiles_m, tiles, full, splits;
  int32_t bm, bn;         // rows and (weight) rows of a tile
  float* part;            // fp32 [tiles - full][splits][bm][bn]
  const uint16_t* bias;
  uint16_t* out;          // bf16 [M, N]
  int64_t os;
  uint8_t* hq;            // gated: e4m3 [M, 128 HB], and its scales
  int64_t hqs;
  float* hsc;
  int64_t hss;
};

__device__ __forceinline__ float silu(float g) {
  return g * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-g * kLog2e));
}

// A lane's 32 e4m3 bytes as bf16, 8 a step of the bf16 MFMA.
__device__ __forceinline__ void widen_frag(const i32x8& f, u32x4* w) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
    w[e] = e4m3x8_to_bf16x8((uint32_t)f[2 * e], (uint32_t)f[2 * e + 1]);
}

__device__ __forceinline__ void store_out(const BlockGemmArgs& a, int64_t m, int n, int N,
                                          f32x4 v) {
  if (a.bias) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n + r < N) v[r] += __uint_as_float((uint32_t)a.bias[n + r] << 16);
  }
  uint16_t* o = a.out + m * a.os + n;
  const u32x2 pk = {pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
  if (n + 3 < N && a.os % 4 == 0) {
    *reinterpret_cast<u32x2*>(o) = pk;
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n + r < N) o[r] = (uint16_t)(pk[r >> 1] >> (16 * (r & 1)));
  }
}

// GATED: the workgroup's 64 WN = 256 weight rows are 128 rows of the gate and
// the same 128 of the up projection: of a wave's 64, the first 32 are gate rows
// and the last 32 the up rows of the same columns, so g and u of one column
// meet in one lane, and the workgroup holds whole 128-blocks of h.
// WIDE: the operands widened to bf16, exactly, for MFMAs that add in fp32.
template <int MT, int WN, int STAGES, bool GATED, bool WIDE>
__global__ void __launch_bounds__(2 * kWave * WN)
block_gemm_kernel(BlockGemmArgs a) {
  using T = BlockTile<MT, WN, STAGES>;
  static_assert(!GATED || (WN == 4 && kGatedCols == kQBlock),
                "a gated tile holds one 128-block of h");
  __shared__ __attribute__((aligned(16))) uint8_t smem[STAGES * T::kStage];
  const int t = threadIdx.x, w = wave_id(), l = t & 63;
  const int wm = w / WN, wn = w % WN;
  const bool whole = GATED || (int)blockIdx.x < a.full;
  int lin, split = 0, slot = 0;
  if (whole) {
    lin = xcd_order(blockIdx.x, a.full);
  } else {
    const int i = blockIdx.x - a.full, rest = a.tiles - a.full;
    split = i / rest;
    const int o = xcd_order(i - split * rest, rest);
    lin = a.full + o;
    slot = o * a.splits + split;
  }
  int tm_i, tn_i;
  tile_at(lin, a.tiles, a.tiles_m, kGroupM, &tm_i, &tn_i);
  const int second = GATED ? (w >= WN) : (a.n_mats > 1 && tn_i >= a.tn1);
  const BlockMat mat = a.mat[second];   // gated: the matrix whose rows this wave stages
  const int m0 = tm_i * T::kBM;
  const int n0 = GATED ? tn_i * kQBlock : (tn_i - (second ? a.tn1 : 0)) * T::kBN;
  const int parts = whole ? 1 : a.splits;
  const int kb0 = (int)((int64_t)a.KB * split / parts);
  const int KB = (int)((int64_t)a.KB * (split + 1) / parts) - kb0;

  // Staging as in fp8_linear.hip: thread t moves 16-byte chunk t % 8 of row
  // kRowsPerInst i + t / 8 (instruction i), fetched from chunk (t % 8) ^ swz(row);
  // rows past the matrix repeat its last row.  Chunks behind the weights' last
  // column repeat the slice's first: the activations are zero there.
  const int srow = t >> 3;
  const uint32_t cb = 16 * ((t & 7) ^ swz(srow));
  const uint32_t over = cb >= (uint32_t)a.tail ? cb : 0;
  const uint8_t* xbase = a.xq + (int64_t)m0 * a.xs;
  const uint8_t* wbase = mat.w + (int64_t)n0 * mat.wrs;
  uint32_t xo[T::kXInst], wo[T::kWInst];
#pragma unroll
  for (int i = 0; i < T::kXInst; ++i)
    xo[i] = (uint32_t)min(T::kRowsPerInst * i + srow, a.M - 1 - m0) * (uint32_t)a.xs + cb;
#pragma unroll
  for (int i = 0; i < T::kWInst; ++i) {
    const int r = GATED ? 32 * i + (srow & 31) : T::kRowsPerInst * i + srow;
    wo[i] = (uint32_t)min(r, mat.N - 1 - n0) * (uint32_t)mat.wrs + cb;
  }
  // Scales: element e = i threads + t of a slice's list, the 32 MT rows' and then
  // those of two column blocks (gated: of gate and up).
  const uint8_t* sp0[T::kSInst];
  uint32_t sstep[T::kSInst];
#pragma unroll
  for (int i = 0; i < T::kSInst; ++i) {
    const int e = i * T::kThreads + t;
    if (e < T::kBM) {
      sp0[i] = reinterpret_cast<const uint8_t*>(a.xsc + min(m0 + e, a.M - 1));
      sstep[i] = (uint32_t)a.xss * 4u;
    } else {
      const int two = min(e - T::kBM, 1);
      const BlockMat& sm = GATED ? a.mat[two] : mat;
      const int nb = GATED ? tn_i : min(n0 / kQBlock + two, (sm.N - 1) / kQBlock);
      sp0[i] = reinterpret_cast<const uint8_t*>(sm.wsc + nb * sm.sn);
      sstep[i] = (uint32_t)sm.sk * 4u;
    }
  }
  const uint32_t lds0 = lds_addr(smem);

  auto issue_one = [&](int kb, int st, int idx) {
    const uint32_t sb = lds0 + st * T::kStage + w * 1024;
    if (idx < T::kXInst) {
      dma16(xbase + (int64_t)kb * kKSlice, xo[idx], sb + idx * 16 * T::kThreads);
    } else if (idx < T::kXInst + T::kWInst) {
      const int i = idx - T::kXInst;
      dma16(wbase + (int64_t)kb * kKSlice, wo[i], sb + T::kXBytes + i * 16 * T::kThreads);
    } else {
      const int i = idx - T::kXInst - T::kWInst;
      dma4_at(sp0[i] + (uint64_t)(uint32_t)kb * sstep[i],
              lds0 + st * T::kStage + T::kXBytes + T::kWBytes + i * 4 * T::kThreads + w * 256);
    }
  };
  // Before slice kb is staged: from the last on, chunks that the weights lack.
  bool cut = false;
  auto enter = [&](int kb) {
    if (kb == a.KB - 1 && !cut) {
      cut = true;
#pragma unroll
      for (int i = 0; i < T::kWInst; ++i) wo[i] -= over;
    }
  };

  const int rr = l & 15, g = l >> 4;
  const int o0 = 16 * ((2 * g) ^ swz(rr)), o1 = 16 * ((2 * g + 1) ^ swz(rr));
  const int xrow = wm * 16 * MT + rr;   // + 16 tm
  const int wrow = wn * 64 + rr;        // + 16 tn

  f32x4 acc[MT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // A slice's loads start at the step that frees its stage: kAtStep of x there,
  // kSpread per row after it (5120 x 2 x 17408 columns at 8192 rows, timed beside each
  // other: 1217 us; all three a row from the next slice on 1273, two barriers a slice to
  // free the weights' part of a stage sooner 1231).
  constexpr int kInLast = MT > 1 ? (kAtStep < T::kXInst ? kAtStep : T::kXInst) : T::kLoads;
  int kfill;
  // Slices past the last are never used; their stage is refilled with the last
  // slice so that every step issues (and waits for) the same loads.
#pragma unroll
  for (int i = 0; i < STAGES; ++i) {
    kfill = kb0 + min(i, KB - 1);
    if (i < STAGES - 1 || MT == 1) enter(kfill);
#pragma unroll
    for (int idx = 0; idx < (i < STAGES - 1 ? T::kLoads : kInLast); ++idx) issue_one(kfill, i, idx);
  }
  vm_wait<(STAGES - 2) * T::kLoads + kInLast>();
  __syncthreads();

  // A slice is MT rows of four MFMAs.  Each MFMA starts from zero; its product is
  // folded into the accumulators with the row's and the column block's scale, one
  // FMA per element, between the next row's MFMAs (the last row's during the next
  // slice).  A row's operand is read one row ahead, and the step to the next slice
  // is taken before the last row: by then every wave has read all of this slice,
  // and the next one's weights are read each behind the last MFMA that uses their
  // registers, so that no wave starts a slice by waiting for twelve reads.
  i32x8 wf[4], xf[2];
  f32x4 p[2][4];
  u32x4 ww[4][4];
  float xr[2], w0, w1, s0 = 0.f, s1 = 0.f;   // s0, s1: scales of the row before
#pragma unroll
  for (int tn = 0; tn < 4; ++tn) p[0][tn] = p[1][tn] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto scales_of = [&](int st) {
    return reinterpret_cast<const float*>(smem + st * T::kStage + T::kXBytes + T::kWBytes);
  };
  auto read_x = [&](int st, int tm, int slot) {
    xf[slot] = frag(smem + st * T::kStage + (xrow + 16 * tm) * kKSlice, o0, o1);
    xr[slot] = scales_of(st)[xrow + 16 * tm];
  };
  auto read_w = [&](int st, int tn) {
    wf[tn] = frag(smem + st * T::kStage + T::kXBytes + (wrow + 16 * tn) * kKSlice, o0, o1);
  };
  auto read_ws = [&](int st) {
    w0 = scales_of(st)[T::kBM + (GATED ? 0 : wn >> 1)];
    w1 = GATED ? scales_of(st)[T::kBM + 1] : w0;
  };
  read_x(0, 0, 0);
#pragma unroll
  for (int tn = 0; tn < 4; ++tn) read_w(0, tn);
  read_ws(0);
  int st = 0;
  for (int j = 0; j < KB; ++j) {
    const int st1 = st == STAGES - 1 ? 0 : st + 1;   // the next slice's stage
    if constexpr (MT > 1) enter(kfill);
#pragma unroll
    for (int tm = 0; tm < MT; ++tm) {
      // The stage of the slice before is free: slice j - 1 + STAGES goes there.
      if (tm < MT - 1) {
        const int from = kInLast + tm * kSpread;
        const int to = tm == MT - 2 ? T::kLoads : min(from + kSpread, T::kLoads);
#pragma unroll
        for (int idx = from; idx < to; ++idx)
          issue_one(kfill, st == 0 ? STAGES - 1 : st - 1, idx);
      }
      const float c0 = xr[tm & 1] * w0, c1 = GATED ? xr[tm & 1] * w1 : c0;
      if (tm == MT - 1) {
        vm_wait<(STAGES - 2) * T::kLoads>();
        __syncthreads();
        kfill = kb0 + min(j + STAGES, KB - 1);
        if constexpr (MT == 1) enter(kfill);
#pragma unroll
        for (int q = 0; q < kInLast; ++q) issue_one(kfill, st, q);
        read_x(st1, 0, MT & 1);
        read_ws(st1);
      } else {
        read_x(st, tm + 1, (tm + 1) & 1);
      }
      if constexpr (!WIDE) __builtin_amdgcn_sched_barrier(0);
      // products of the row before: of this slice, or the last one's
      u32x4 xw[4];
      if constexpr (WIDE) widen_frag(xf[tm & 1], xw);
#pragma unroll
      for (int tn = 0; tn < 4; ++tn) {
        const int back = tm > 0 ? tm - 1 : MT - 1;
        f32x4 q = p[back & 1][tn];
        if constexpr (WIDE) {
          if (tm == 0) widen_frag(wf[tn], ww[tn]);
          p[tm & 1][tn] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int e = 0; e < 4; ++e) p[tm & 1][tn] = mfma_16x16x32(ww[tn][e], xw[e], p[tm & 1][tn]);
        } else {
          p[tm & 1][tn] = mfma_fp8(wf[tn], xf[tm & 1]);
        }
        if (tm == MT - 1) read_w(st1, tn);
        acc[back][tn] += q * (GATED && tn >= 2 ? s1 : s0);
      }
      if constexpr (!WIDE) {
      if (tm == MT - 1)
        __builtin_amdgcn_sched_group_barrier(0x100, GATED ? 5 : 4, 0);   // LDS reads
      else
        __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
      for (int tn = 0; tn < 4; ++tn) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);   // 1 MFMA
        if (tm == MT - 1) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);   // 4 VALU
      }
      __builtin_amdgcn_sched_barrier(0);
      }
      s0 = c0;
      s1 = c1;
    }
    if constexpr (MT & 1) {   // (an even MT has read it into the first slot)
      xf[0] = xf[1];
      xr[0] = xr[1];
    }
    st = st1;
  }
  vm_wait<0>();   // the refills of the last steps land before the stages are reused
#pragma unroll
  for (int tn = 0; tn < 4; ++tn)
    acc[MT - 1][tn] += p[(MT - 1) & 1][tn] * (GATED && tn >= 2 ? s1 : s0);

  // Lane holds D[wn 64 + 16 tn + 4 g + r][m0 + wm 16 MT + 16 tm + rr].
  if (!whole) {   // (never where gated)
    float* part = a.part + (int64_t)slot * T::kBM * T::kBN + wn * 64 + 4 * g;
#pragma unroll
    for (int tm = 0; tm < MT; ++tm) {
      const int row = xrow + 16 * tm;
      if (m0 + row >= a.M) continue;
#pragma unroll
      for (int tn = 0; tn < 4; ++tn)
        *reinterpret_cast<f32x4*>(part + row * T::kBN + 16 * tn) = acc[tm][tn];
    }
    return;
  }
  if constexpr (!GATED) {
#pragma unroll
    for (int tn = 0; tn < 4; ++tn) {
      const int n = n0 + wn * 64 + 16 * tn + 4 * g;
      if (n >= mat.N) continue;
#pragma unroll
      for (int tm = 0; tm < MT; ++tm) {
        const int m = m0 + xrow + 16 * tm;
        if (m < a.M) store_out(a, m, n, mat.N, acc[tm][tn]);
      }
    }
  } else {
    // h of this lane: columns 32 wn + 16 j + 4 g + r of the block, j = 0, 1.  A
    // row's amax crosses the four lane groups and the four waves of a row.
    constexpr int kPitch = kQBlock + 16;   // bytes per row of the output tile
    uint8_t* tile = smem;
    uint32_t* amax = reinterpret_cast<uint32_t*>(smem + T::kBM * kPitch);
    static_assert(T::kBM * (kPitch + 16) <= STAGES * T::kStage, "epilogue fits the stages");
    __syncthreads();
#pragma unroll
    for (int tm = 0; tm < MT; ++tm) {
      uint32_t mx = 0;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int n = n0 + 32 * wn + 16 * j + 4 * g;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float h = n + r < mat.N ? silu(acc[tm][j][r]) * acc[tm][2 + j][r] : 0.f;
          acc[tm][j][r] = h;
          mx = max(mx, __float_as_uint(h) & 0x7fffffffu);
        }
      }
      mx = max(mx, (uint32_t)__shfl_xor((int)mx, 16, kWave));
      mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32, kWave));
      if (g == 0) amax[4 * (xrow + 16 * tm) + wn] = mx;
    }
    __syncthreads();
#pragma unroll
    for (int tm = 0; tm < MT; ++tm) {
      const int row = xrow + 16 * tm;
      const u32x4 m4 = ld_s16(amax + 4 * row);
      const float s = block_scale(max(max(m4[0], m4[1]), max(m4[2], m4[3])));
      if (wn == 0 && g == 0 && m0 + row < a.M)
        a.hsc[(int64_t)tn_i * a.hss + m0 + row] = s;
      const BlockDiv d = block_div(s);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const f32x4 h = acc[tm][j];
        *reinterpret_cast<uint32_t*>(tile + row * kPitch + 32 * wn + 16 * j + 4 * g) =
            quant4(h[0], h[1], h[2], h[3], d);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < T::kBM * 8 / T::kThreads; ++i) {
      const int row = i * (T::kThreads / 8) + (t >> 3), c = 16 * (t & 7);
      if (m0 + row < a.M)
        *reinterpret_cast<u32x4*>(a.hq + (m0 + row) * a.hqs + (int64_t)tn_i * kQBlock + c) =
            ld_s16(tile + row * kPitch + c);
    }
  }
}

// Sum of the splits' partials of four columns, in split order.  Every partial is
// loaded before the first add, so the loads' latencies overlap.
__device__ __forceinline__ f32x4 sum_splits(const BlockGemmArgs& a, const float* p) {
  const int64_t step = (int64_t)a.bm * a.bn;
  f32x4 v[kMaxSplits];
#pragma unroll
  for (int sp = 0; sp < kMaxSplits; ++sp)
    if (sp < a.splits) v[sp] = *reinterpret_cast<const f32x4*>(p + sp * step);
#pragma unroll
  for (int sp = 1; sp < kMaxSplits; ++sp)
    if (sp < a.splits) v[0] += v[sp];
  return v[0];
}

// The split tiles of a product (blockIdx.y): out = bf16(sum of the partials + bias),
// four columns per thread, rows in order.
__global__ void __launch_bounds__(kThreads) block_reduce_kernel(BlockGemmArgs a) {
  const int o = blockIdx.y;
  int tm, tn;
  tile_at(a.full + o, a.tiles, a.tiles_m, kGroupM, &tm, &tn);
  const int quads = a.bn == 256 ? 6 : 5;   // log2(bn / 4)
  const int in = blockIdx.x * kThreads + threadIdx.x;
  const int row = in >> quads, col = 4 * (in & ((1 << quads) - 1));
  const int64_t m = (int64_t)tm * a.bm + row;
  const int n = tn * a.bn + col;
  if (m >= a.M || n >= a.mat[0].N) return;
  const float* p = a.part + ((int64_t)o * a.splits * a.bm + row) * a.bn + col;
  store_out(a, m, n, a.mat[0].N, sum_splits(a, p));
}

// h = silu(g) u from the partials of both projections, quantised: 32 lanes hold a
// block's 128 columns of one row, four each.
__global__ void __launch_bounds__(kThreads) gated_finish_kernel(BlockGemmArgs a) {
  const int hb = (a.mat[0].N + kQBlock - 1) / kQBlock;
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (unit >= (int64_t)a.M * hb) return;   // (all 32 lanes of a unit together)
  const int m = (int)(unit / hb), b = (int)(unit - (int64_t)m * hb);
  const int c = b * kQBlock + 4 * (threadIdx.x & 31);
  f32x4 h = {0.f, 0.f, 0.f, 0.f};
  uint32_t mx = 0;
  if (c < a.mat[0].N) {   // N is a multiple of 16: four columns in or out together
    const int tm = m / a.bm, tn = c / a.bn;
    const int og = tile_index(tm, tn, a.tiles, a.tiles_m, kGroupM);
    const int ou = tile_index(tm, a.tn1 + tn, a.tiles, a.tiles_m, kGroupM);
    const float* p = a.part + (int64_t)(m - tm * a.bm) * a.bn + c - tn * a.bn;
    const int64_t step = (int64_t)a.splits * a.bm * a.bn;
    const f32x4 gt = sum_splits(a, p + og * step), up = sum_splits(a, p + ou * step);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      h[r] = silu(gt[r]) * up[r];
      mx = max(mx, __float_as_uint(h[r]) & 0x7fffffffu);
    }
  }
  mx = amax_lanes16(mx);
  mx = max(mx, (uint32_t)__shfl_xor((int)mx, 16, kWave));
  const float s = block_scale(mx);
  if ((threadIdx.x & 31) == 0) a.hsc[b * a.hss + m] = s;
  *reinterpret_cast<uint32_t*>(a.hq + m * a.hqs + c) =
      quant4(h[0], h[1], h[2], h[3], block_div(s));
}

// ---------------------------------------------------------------- few rows
// Products of at most 16 rows: bound by the weights' way from memory, which one
// launch has to ask for at once.  A workgroup of 8 waves owns 16 columns (gated:
// of both projections); the waves take the K slices in turn, load them into
// registers a few slices ahead, and add their sums through LDS at the end, in
// wave order (1 row of 5120 times 2 x 17408 columns: 30.3 us = 5.9 TB/s).  A
// load covers whole 128-byte lines (8 lanes a row; 16 rows of 64
// bytes read the same matrix at 3.4 TB/s instead of 5.1), so the operands, which
// want a lane per row, pass through LDS of the wave's own.  They are widened to
// bf16, exactly: the bf16 MFMA adds in fp32, where the fp8 one cuts each product
// 13 bits below the largest of its eight, and there is time for it.
// XK: x is e4m3 rows with scales (kXRows), or bf16 / fp32 rows that every
// workgroup quantises into LDS while its first weights are on their way: no
// launch of its own, free while the blocks are few and all workgroups run at once
// (1 row of 6144 times 5120 columns 11.1 us against 11.4 for quantised rows alone;
// the 1088 workgroups of 5120 x 2 x 17408 lost 13 us, a launch takes 4).
// Gated: h = silu(g) u is written in fp32; the next product quantises it.
enum { kXRows = 0, kXBf16 = 1, kXF32 = 2 };
constexpr int kRowsMax = 16;
constexpr int kRowsWaves = 8;

struct RowsArgs {
  const uint8_t* x;       // rows, stride xs elements
  int64_t xs;
  const float* xsc;       // e4m3 rows: scale of (row, block) at block * xss + row
  int64_t xss;
  BlockMat mat[2];
  int32_t M, K, KB, tail;
  const uint16_t* bias;
  uint16_t* out;          // bf16 [M, N]
  int64_t os;
  float* h;               // gated: [M, N]
};

// Row pitch of x in LDS (bytes) and the LDS that M rows take with their scales.
__host__ __device__ constexpr int64_t rows_pitch(int64_t kb) { return kb * kQBlock + 16; }
__host__ __device__ constexpr int64_t rows_lds(int64_t m, int64_t kb) {
  return m * (rows_pitch(kb) + 4 * kb);
}

struct RowsSlice {        // one K slice of 16 weight rows (and of x), as loaded
  u32x4 w[2][2], x[2];
  float ws[2], xs;
};

template <bool GATED, int XK>
__global__ void __launch_bounds__(kRowsWaves * kWave, 4) block_rows_kernel(RowsArgs a) {
  constexpr int kMats = GATED ? 2 : 1;
  constexpr int kTiles = kMats + (XK == kXRows);          // 2 KB of LDS each, per wave
  constexpr int kDepth = GATED ? 2 : 4;   // (128 VGPRs: two workgroups per CU)
  static_assert(!GATED || XK == kXRows, "a gated product's x comes quantised");
  __shared__ __attribute__((aligned(16))) uint8_t tiles[kRowsWaves][kTiles][16 * kKSlice];
  extern __shared__ __attribute__((aligned(16))) uint8_t xlds[];
  const int t = threadIdx.x, w = wave_id(), l = t & 63, rr = l & 15, g = l >> 4;
  const int n0 = blockIdx.x * 16;
  const int row = min(rr, a.M - 1);
  const int64_t pitch = rows_pitch(a.KB);
  float* xscale = reinterpret_cast<float*>(xlds + a.M * pitch);

  // Loads: lane l has chunk l % 8 of row l / 8, and of row l / 8 + 8.
  const int lr = l >> 3, lc = 16 * (l & 7);
  const uint8_t* wp[kMats][2];
  const uint8_t* wsp[kMats];
#pragma unroll
  for (int i = 0; i < kMats; ++i) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      wp[i][h] = a.mat[i].w + (int64_t)min(n0 + lr + 8 * h, a.mat[i].N - 1) * a.mat[i].wrs;
    wsp[i] = reinterpret_cast<const uint8_t*>(a.mat[i].wsc + (n0 / kQBlock) * a.mat[i].sn);
  }
  const uint8_t* xp[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) xp[h] = a.x + min(lr + 8 * h, a.M - 1) * a.xs;
  const int n_slices = (a.KB - w + kRowsWaves - 1) / kRowsWaves;   // of this wave

  auto load = [&](RowsSlice& s, int i) {
    const int kb = w + i * kRowsWaves;
    const int64_t k = (int64_t)kb * kQBlock;
    // chunks behind the last column: the slice's first, times zeros for x
    const bool gone = kb == a.KB - 1 && lc >= a.tail;
    const int c = gone ? 0 : lc;
#pragma unroll
    for (int m = 0; m < kMats; ++m) {
#pragma unroll
      for (int h = 0; h < 2; ++h) s.w[m][h] = ld_nt16(wp[m][h] + k + c);
      s.ws[m] = *reinterpret_cast<const float*>(wsp[m] + (int64_t)kb * a.mat[m].sk * 4);
    }
    if constexpr (XK == kXRows) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s.x[h] = ld_g16(xp[h] + k + c);
        if (gone) s.x[h] = u32x4{0u, 0u, 0u, 0u};
      }
      s.xs = a.xsc[kb * a.xss + row];
    }
  };
  // A tile in LDS: row r's chunk c at chunk c ^ swz(r), so that neither the rows'
  // writes nor the operands' reads (16 rows of a chunk) meet in a bank.
  const int put0 = lr * kKSlice + (lc ^ (16 * swz(lr)));
  const int put1 = (lr + 8) * kKSlice + (lc ^ (16 * swz(lr + 8)));
  const int get0 = rr * kKSlice + 16 * (g ^ swz(rr)), get1 = rr * kKSlice + 16 * ((g + 4) ^ swz(rr));
  f32x4 acc[kMats];
#pragma unroll
  for (int m = 0; m < kMats; ++m) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto use = [&](const RowsSlice& s, int i) {
    const int kb = w + i * kRowsWaves;
#pragma unroll
    for (int m = 0; m < kMats; ++m) {
      st_s16(tiles[w][m] + put0, s.w[m][0]);
      st_s16(tiles[w][m] + put1, s.w[m][1]);
    }
    if constexpr (XK == kXRows) {
      st_s16(tiles[w][kMats] + put0, s.x[0]);
      st_s16(tiles[w][kMats] + put1, s.x[1]);
    }
    wave_lds_sync();
    // Operands: lane l has chunks l / 16 and l / 16 + 4 of row l % 16, of both sides.
    u32x4 wf[kMats][2], xf[2];
#pragma unroll
    for (int m = 0; m < kMats; ++m) {
      wf[m][0] = ld_s16(tiles[w][m] + get0);
      wf[m][1] = ld_s16(tiles[w][m] + get1);
    }
    float xs;
    if constexpr (XK == kXRows) {
      xf[0] = ld_s16(tiles[w][kMats] + get0);
      xf[1] = ld_s16(tiles[w][kMats] + get1);
      xs = s.xs;
    } else {
      const uint8_t* p = xlds + row * pitch + kb * kQBlock + 16 * g;
      xf[0] = ld_s16(p);
      xf[1] = ld_s16(p + 64);
      xs = xscale[row * a.KB + kb];
    }
    wave_lds_sync();   // (before the next slice's writes)
    f32x4 p[kMats];
#pragma unroll
    for (int m = 0; m < kMats; ++m) p[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int c = q >> 1, d = 2 * (q & 1);
      const u32x4 xb = e4m3x8_to_bf16x8(xf[c][d], xf[c][d + 1]);
#pragma unroll
      for (int m = 0; m < kMats; ++m)
        p[m] = mfma_16x16x32(e4m3x8_to_bf16x8(wf[m][c][d], wf[m][c][d + 1]), xb, p[m]);
    }
#pragma unroll
    for (int m = 0; m < kMats; ++m) acc[m] += p[m] * (xs * s.ws[m]);
  };

  RowsSlice ring[kDepth];
#pragma unroll
  for (int j = 0; j < kDepth; ++j)
    if (j < n_slices) load(ring[j], j);
  if constexpr (XK != kXRows) {
    // 16 lanes quantise a block, four blocks' loads in flight
    constexpr int kAtOnce = 4;
    const int units = a.M * a.KB;
    for (int u0 = t >> 4; u0 < units; u0 += kAtOnce * kRowsWaves * 4) {
      float v[kAtOnce][8];
#pragma unroll
      for (int b = 0; b < kAtOnce; ++b) {
        const int u = u0 + b * kRowsWaves * 4, m = u / a.KB, c = (u - m * a.KB) * kQBlock + 8 * rr;
        if (u < units && c < a.K) {
          load8<XK == kXF32>(a.x, m * a.xs + c, v[b]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[b][j] = 0.f;
        }
      }
#pragma unroll
      for (int b = 0; b < kAtOnce; ++b) {
        const int u = u0 + b * kRowsWaves * 4, m = u / a.KB, kb = u - m * a.KB;
        if (u >= units) break;   // (16 lanes together)
        const float s = block_scale(amax_lanes16(amax_bits8(v[b])));
        *reinterpret_cast<u32x2*>(xlds + m * pitch + kb * kQBlock + 8 * rr) = quant8(v[b], block_div(s));
        if (rr == 0) xscale[m * a.KB + kb] = s;
      }
    }
    __syncthreads();
  }
  int i = 0;
  for (; i + 2 * kDepth <= n_slices; i += kDepth) {
#pragma unroll
    for (int j = 0; j < kDepth; ++j) {
      use(ring[j], i + j);
      load(ring[j], i + kDepth + j);
    }
  }
#pragma unroll
  for (int j = 0; j < kDepth; ++j) {
    if (i + j < n_slices) use(ring[j], i + j);
    if (i + kDepth + j < n_slices) load(ring[j], i + kDepth + j);
  }
#pragma unroll
  for (int j = 0; j < kDepth; ++j)
    if (i + kDepth + j < n_slices) use(ring[j], i + kDepth + j);

  // Lane holds D[4 g + r][rr]: row rr, columns 4 g + r.  A wave's sums take its own
  // tiles' place.
#pragma unroll
  for (int m = 0; m < kMats; ++m)
    *reinterpret_cast<f32x4*>(&tiles[w][m][4 * (16 * rr + 4 * g)]) = acc[m];
  __syncthreads();
  if (t >= 256) return;
  const int m = t >> 4, n = n0 + (t & 15);
  float sum[kMats];
#pragma unroll
  for (int q = 0; q < kMats; ++q) {
    sum[q] = 0.f;
#pragma unroll
    for (int v = 0; v < kRowsWaves; ++v)
      sum[q] += *reinterpret_cast<const float*>(&tiles[v][q][4 * t]);
  }
  if (m >= a.M || n >= a.mat[0].N) return;
  if constexpr (GATED) {
    a.h[(int64_t)m * a.mat[0].N + n] = silu(sum[0]) * sum[1];
  } else {
    if (a.bias) sum[0] += __uint_as_float((uint32_t)a.bias[n] << 16);
    a.out[(int64_t)m * a.os + n] = (uint16_t)(pack_bf16(sum[0], 0.f) & 0xffffu);
  }
}

// ---------------------------------------------------------------- launches
template <int MT, int WN, int STAGES, bool GATED, bool WIDE = false>
void launch_gemm(BlockGemmArgs a, hipStream_t stream) {
  using T = BlockTile<MT, WN, STAGES>;
  a.bm = T::kBM;
  a.bn = T::kBN;
  a.tiles_m = (int)ceil_div(a.M, T::kBM);
  a.tn1 = (int)ceil_div(a.mat[0].N, GATED ? kQBlock : T::kBN);
  a.tiles = a.tiles_m * a.tn1 * (GATED ? 1 : a.n_mats);
  const int rest = a.tiles - a.full;
  hipLaunchKernelGGL((block_gemm_kernel<MT, WN, STAGES, GATED, WIDE>),
                     dim3((uint32_t)(a.full + rest * a.splits)), dim3(T::kThreads), 0, stream, a);
  if (rest == 0) return;
  if (a.n_mats == 2)
    hipLaunchKernelGGL(gated_finish_kernel,
                       dim3((uint32_t)ceil_div(a.M * ceil_div(a.mat[0].N, kQBlock),
                                               kThreads / 32)),
                       dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL(block_reduce_kernel,
                       dim3(T::kBM * T::kBN / 4 / kThreads, (uint32_t)rest), dim3(kThreads), 0,
                       stream, a);
}

// The tiles of a product, or with two matrices of a gated one, and the kernel that
// finishes the partials where there are any.
void launch_tiles(BlockGemmArgs a, const BlockPlan& p, int n_mats, float* part, hipStream_t s) {
  a.n_mats = n_mats;
  a.full = p.full;
  a.splits = p.splits;
  a.part = part;
  const Shape sh = p.shape;
  const bool wide = n_mats == 2 && wide_gated(a.M);
  if (p.fused) {
    if (sh.mt == 2)
      wide ? launch_gemm<2, 4, 3, true, true>(a, s) : launch_gemm<2, 4, 3, true>(a, s);
    else if (sh.mt == 4)
      launch_gemm<4, 4, 3, true>(a, s);
    else if (sh.mt == 6)
      launch_gemm<6, 4, 2, true>(a, s);
    else
      launch_gemm<8, 4, 2, true>(a, s);
  } else if (sh.mt == 1) {
    wide ? launch_gemm<1, 2, 3, false, true>(a, s) : launch_gemm<1, 2, 3, false>(a, s);
  } else if (sh.mt == 2) {
    wide ? launch_gemm<2, 2, 3, false, true>(a, s) : launch_gemm<2, 2, 3, false>(a, s);
  } else if (sh.mt == 4 && sh.wn == 2) {
    launch_gemm<4, 2, 3, false>(a, s);
  } else if (sh.mt == 6 && sh.wn == 2) {
    launch_gemm<6, 2, 3, false>(a, s);
  } else if (sh.mt == 4) {
    launch_gemm<4, 4, 3, false>(a, s);
  } else if (sh.mt == 6) {
    launch_gemm<6, 4, 2, false>(a, s);
  } else {
    launch_gemm<8, 4, 2, false>(a, s);
  }
}

// Whether a product of M rows runs on the kernel of few rows, and whether that
// quantises its x itself: at most two rows (4 rows of 6144 times 5120 columns: 17.9 us,
// 12.6 and a launch of 4 from quantised rows), of a length whose e4m3 values fit
// beside the tiles of two workgroups, in workgroups that all run at once (two per CU).
constexpr int64_t kRowsOwn = 2, kRowsLds = 40 << 10;
bool few_rows(int64_t m) { return m <= kRowsMax; }
bool rows_quantise(int64_t m, int64_t n, int64_t kb) {
  return m <= kRowsOwn && rows_lds(m, kb) <= kRowsLds &&
         ceil_div(n, 16) <= 2 * device_cu_count();
}

void launch_rows(const RowsArgs& a, int xk, hipStream_t s) {
  const dim3 grid((uint32_t)ceil_div(a.mat[0].N, 16)), block(kRowsWaves * kWave);
  const size_t lds = xk == kXRows ? 0 : (size_t)rows_lds(a.M, a.KB);
  if (xk == kXRows && a.h)
    hipLaunchKernelGGL((block_rows_kernel<true, kXRows>), grid, block, lds, s, a);
  else if (xk == kXRows)
    hipLaunchKernelGGL((block_rows_kernel<false, kXRows>), grid, block, lds, s, a);
  else if (xk == kXBf16)
    hipLaunchKernelGGL((block_rows_kernel<false, kXBf16>), grid, block, lds, s, a);
  else
    hipLaunchKernelGGL((block_rows_kernel<false, kXF32>), grid, block, lds, s, a);
}

// ---------------------------------------------------------------- arguments
constexpr int64_t kMaxDim = 1 << 24;   // columns of a matrix: 32-bit offsets inside a tile
constexpr int64_t kMaxRows = 1 << 24;

int32_t check_rows(const char* fn, int64_t rows, int64_t cols, int64_t multiple) {
  if (rows < 0 || cols <= 0 || cols % multiple)
    return fail(TF_ERR_INVALID, "%s: rows=%lld cols=%lld (cols a positive multiple of %lld)", fn,
                (long long)rows, (long long)cols, (long long)multiple);
  if (rows > kMaxRows || cols > kMaxDim)
    return fail(TF_ERR_UNSUPPORTED, "%s: %lld x %lld is too large", fn, (long long)rows,
                (long long)cols);
  return TF_OK;
}

int32_t quant_setup(const char* fn, const void* x, int32_t x_dtype, int64_t rows, int64_t cols,
                    int64_t x_row_stride, void* xq, int64_t xq_row_stride, float* x_scale,
                    int64_t x_scale_stride, int64_t out_cols, BlockQuantArgs* a) {
  int32_t rc = check_rows(fn, rows, cols, 8);
  if (rc != TF_OK) return rc;
  if (x_dtype != TF_DTYPE_BF16 && x_dtype != TF_DTYPE_FP32)
    return fail(TF_ERR_UNSUPPORTED, "%s: x must be bf16 or fp32 (dtype %d)", fn, x_dtype);
  if (x_row_stride < cols || x_row_stride % 8 || xq_row_stride < out_cols || xq_row_stride % 8 ||
      x_scale_stride < rows || x_scale_stride > kMaxRows)
    return fail(TF_ERR_INVALID, "%s: strides %lld/%lld/%lld (rows multiples of 8; scales from the "
                "number of rows up)", fn, (long long)x_row_stride, (long long)xq_row_stride,
                (long long)x_scale_stride);
  if (rows > 0 && (!x || !xq || !x_scale)) return fail(TF_ERR_INVALID, "%s: null pointer", fn);
  if (!aligned16(x) || !aligned8(xq) || (reinterpret_cast<uintptr_t>(x_scale) & 3u))
    return fail(TF_ERR_INVALID, "%s: x 16-byte, xq 8-byte, scales 4-byte aligned", fn);
  a->x = static_cast<const uint8_t*>(x);
  a->xs = x_row_stride;
  a->rows = rows;
  a->cols = (int32_t)cols;
  a->out_cols = (int32_t)out_cols;
  a->xq = static_cast<uint8_t*>(xq);
  a->qs = xq_row_stride;
  a->scale = x_scale;
  a->ss = x_scale_stride;
  a->col_groups = (int32_t)ceil_div(out_cols, kQuantCols);
  if (ceil_div(rows, kQuantWgRows) * a->col_groups > UINT32_MAX / kThreads)   // (of one launch)
    return fail(TF_ERR_UNSUPPORTED, "%s: too large", fn);
  return TF_OK;
}

void launch_quant(const BlockQuantArgs& a, bool f32, hipStream_t s) {
  const dim3 grid((uint32_t)(ceil_div(a.rows, kQuantWgRows) * a.col_groups));
  if (f32)
    hipLaunchKernelGGL(block_quant_kernel<true>, grid, dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL(block_quant_kernel<false>, grid, dim3(kThreads), 0, s, a);
}

// Checks one weight and describes it (out and bias are the caller's).
int32_t weight_setup(const char* fn, const char* what, const tf_fp8_mat* t, int64_t n, int64_t k,
                     BlockMat* b) {
  if (t->n != n || n <= 0)
    return fail(TF_ERR_INVALID, "%s: %s has %lld columns, expected %lld", fn, what,
                (long long)t->n, (long long)n);
  if (n > kMaxDim) return fail(TF_ERR_UNSUPPORTED, "%s: %s is too large", fn, what);
  if (!t->w || !t->w_scale) return fail(TF_ERR_INVALID, "%s: %s: null pointer", fn, what);
  if (!aligned16(t->w) || (reinterpret_cast<uintptr_t>(t->w_scale) & 3u))
    return fail(TF_ERR_INVALID, "%s: %s 16-byte, its scales 4-byte aligned", fn, what);
  if (t->w_row_stride < k || t->w_row_stride % 16 || t->w_row_stride > kMaxDim ||
      t->w_scale_row_stride < 0 || t->w_scale_col_stride < 0 || t->w_scale_col_stride > kMaxDim)
    return fail(TF_ERR_INVALID, "%s: %s strides %lld/%lld/%lld (rows 16-byte multiples)", fn, what,
                (long long)t->w_row_stride, (long long)t->w_scale_row_stride,
                (long long)t->w_scale_col_stride);
  b->w = static_cast<const uint8_t*>(t->w);
  b->wrs = t->w_row_stride;
  b->wsc = t->w_scale;
  b->sn = t->w_scale_row_stride;
  b->sk = t->w_scale_col_stride;
  b->N = (int32_t)n;
  return TF_OK;
}

int32_t out_setup(const char* fn, const tf_fp8_mat* t, BlockGemmArgs* a) {
  if (!t->out) return fail(TF_ERR_INVALID, "%s: null output", fn);
  if (t->out_row_stride < t->n)
    return fail(TF_ERR_INVALID, "%s: out row stride %lld for %lld columns", fn,
                (long long)t->out_row_stride, (long long)t->n);
  if (!aligned8(t->out) || (reinterpret_cast<uintptr_t>(t->bias) & 1u))
    return fail(TF_ERR_INVALID, "%s: out must be 8-byte aligned", fn);
  a->bias = static_cast<const uint16_t*>(t->bias);
  a->out = static_cast<uint16_t*>(t->out);
  a->os = t->out_row_stride;
  return TF_OK;
}

// Workspace of both products' calls: x quantised (where it comes unquantised),
// the quantised hidden activations (gated), the partials.
struct Layout {
  int64_t xsc, hq, hsc, part, bytes;
};
// Whether a product copies its quantised x to have zeros behind a short last block.
bool pads(int64_t m, int64_t k) { return k % kQBlock != 0 && !few_rows(m); }

Layout layout(int64_t m, int64_t k, int64_t inter, bool quantized, int64_t parts) {
  Layout l;
  l.xsc = quantized && !pads(m, k) ? 0 : round_up(m * round_up(k, kQBlock), 256);
  l.hq = l.xsc + (quantized ? 0 : round_up(4 * m * ceil_div(k, kQBlock), 256));
  l.hsc = l.hq + round_up(m * round_up(inter, kQBlock), 256);
  l.part = l.hsc + round_up(4 * m * ceil_div(inter, kQBlock), 256);
  l.bytes = l.part + 4 * parts;
  return l;
}

// x of a product: quantised rows as they come or padded into the workspace, or
// others quantised into it.
int32_t input_setup(const char* fn, const void* x, int32_t x_dtype, int64_t x_row_stride,
                    const float* x_scale, int64_t x_scale_stride, int64_t m, int64_t k,
                    uint8_t* ws, const Layout& l, BlockGemmArgs* g, BlockQuantArgs* q) {
  g->M = (int32_t)m;
  g->KB = (int32_t)ceil_div(k, kQBlock);
  g->tail = (int32_t)(k - (int64_t)(g->KB - 1) * kQBlock);
  if (x_dtype != TF_DTYPE_FP8_E4M3) {
    float* sc = reinterpret_cast<float*>(ws + l.xsc);
    const int64_t kp = (int64_t)g->KB * kQBlock;
    g->xq = ws;
    g->xs = kp;
    g->xsc = sc;
    g->xss = m;
    return quant_setup(fn, x, x_dtype, m, k, x_row_stride, ws, kp, sc, m, kp, q);
  }
  if (!x || !x_scale) return fail(TF_ERR_INVALID, "%s: null pointer", fn);
  if (!aligned16(x) || (reinterpret_cast<uintptr_t>(x_scale) & 3u))
    return fail(TF_ERR_INVALID, "%s: x 16-byte, its scales 4-byte aligned", fn);
  if (x_row_stride < k || x_row_stride % 16 || x_row_stride > kMaxDim || x_scale_stride < m ||
      x_scale_stride > kMaxRows)
    return fail(TF_ERR_INVALID, "%s: quantised x strides %lld/%lld (rows a multiple of 16 from "
                "their width up, scales from the number of rows up)", fn, (long long)x_row_stride,
                (long long)x_scale_stride);
  g->xq = static_cast<const uint8_t*>(x);
  g->xs = x_row_stride;
  g->xsc = x_scale;
  g->xss = x_scale_stride;
  if (pads(m, k)) {
    if (m * (g->KB * kQBlock / 16) > UINT32_MAX)   // (threads of one launch)
      return fail(TF_ERR_UNSUPPORTED, "%s: too large", fn);
    q->x = g->xq;
    q->xs = x_row_stride;
    q->rows = m;
    q->cols = (int32_t)k;
    q->out_cols = g->KB * kQBlock;
    q->xq = ws;
    q->qs = q->out_cols;
    g->xq = ws;
    g->xs = q->qs;
  }
  return TF_OK;
}

void launch_pad(const BlockQuantArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(block_pad_kernel,
                     dim3((uint32_t)ceil_div(a.rows * (a.out_cols / 16), kThreads)),
                     dim3(kThreads), 0, s, a);
}

bool bad_workspace(const void* ws, int64_t bytes, int64_t need) {
  return need > 0 && (!ws || !aligned16(ws) || bytes < need);
}

// The product of few rows; xk: of g.xq, or of the rows that q describes.
RowsArgs rows_args(const BlockGemmArgs& g, int64_t k, int xk, const BlockQuantArgs& q) {
  RowsArgs r{};
  r.x = xk == kXRows ? g.xq : q.x;
  r.xs = xk == kXRows ? g.xs : q.xs;
  r.xsc = g.xsc;
  r.xss = g.xss;
  r.mat[0] = g.mat[0];
  r.mat[1] = g.mat[1];
  r.M = g.M;
  r.K = (int32_t)k;
  r.KB = g.KB;
  r.tail = g.tail;
  r.bias = g.bias;
  r.out = g.out;
  r.os = g.os;
  return r;
}

// Makes the x of g's one product in a launch of its own unless it comes quantised or the
// kernel of few rows quantises it; says what that kernel's x is.
int prepare_input(int32_t dtype, int64_t k, const BlockGemmArgs& g, const BlockQuantArgs& q,
                  hipStream_t s) {
  if (dtype == TF_DTYPE_FP8_E4M3) {
    if (pads(g.M, k)) launch_pad(q, s);
    return kXRows;
  }
  const bool f32 = dtype == TF_DTYPE_FP32;
  if (rows_quantise(g.M, g.mat[0].N, g.KB)) return f32 ? kXF32 : kXBf16;
  launch_quant(q, f32, s);
  return kXRows;
}

// fp32 elements that a product, or the first half of a gated block (partials, or the
// unquantised h of the kernel of few rows), passes through the workspace.
int64_t linear_parts(int64_t m, int64_t n, int64_t k) {
  if (few_rows(m)) return 0;
  return plan_linear(m, n, 1, ceil_div(k, kQBlock), false, device_cu_count()).part;
}
int64_t gated_parts(int64_t m, int64_t inter, int64_t hidden) {
  if (few_rows(m)) return m * inter;
  return plan_gated(m, inter, ceil_div(hidden, kQBlock), device_cu_count()).part;
}

int32_t check_product(const char* fn, int64_t m, int64_t n, int64_t k) {
  const int32_t rc = check_rows(fn, m, k, 16);
  if (rc != TF_OK) return rc;
  if (n <= 0) return fail(TF_ERR_INVALID, "%s: %lld columns", fn, (long long)n);
  // a launch has 2^32 threads: 128 for 32 x 64 outputs where tiles are smallest
  if (n > kMaxDim || ceil_div(m, 32) * ceil_div(n, 64) > UINT32_MAX / 128)
    return fail(TF_ERR_UNSUPPORTED, "%s: %lld x %lld is too large", fn, (long long)m,
                (long long)n);
  return TF_OK;
}

}  // namespace
}  // namespace tfa

extern "C" {

int32_t tf_block_quant(const void* x, int32_t x_dtype, int64_t rows, int64_t cols,
                       int64_t x_row_stride, void* xq, int64_t xq_row_stride, float* x_scale,
                       int64_t x_scale_stride, tf_stream_t stream) {
  using namespace tfa;
  clear_error();
  BlockQuantArgs a;
  const int32_t rc = quant_setup("block_quant", x, x_dtype, rows, cols, x_row_stride, xq,
                                 xq_row_stride, x_scale, x_scale_stride, cols, &a);
  if (rc != TF_OK || rows == 0) return rc;
  launch_quant(a, x_dtype == TF_DTYPE_FP32, reinterpret_cast<hipStream_t>(stream));
  return launch_status("tf_block_quant launch");
}

int64_t tf_block_linear_workspace_bytes(int64_t m, int64_t n, int64_t k, int32_t x_dtype) {
  using namespace tfa;
  clear_error();
  const int32_t rc = check_product("block_linear", m, n, k);
  if (rc != TF_OK) return rc;
  if (m == 0) return 0;
  return layout(m, k, 0, x_dtype == TF_DTYPE_FP8_E4M3, linear_parts(m, n, k)).bytes;
}

int32_t tf_block_linear(const void* x, int32_t x_dtype, int64_t x_row_stride,
                        const float* x_scale, int64_t x_scale_stride, const tf_fp8_mat* mat,
                        int64_t m, int64_t k, void* workspace, int64_t workspace_bytes,
                        tf_stream_t stream) {
  using namespace tfa;
  clear_error();
  if (!mat) return fail(TF_ERR_INVALID, "block_linear: no weight");
  int32_t rc = check_product("block_linear", m, mat->n, k);
  if (rc != TF_OK || m == 0) return rc;
  const int64_t n = mat->n;
  const bool quantized = x_dtype == TF_DTYPE_FP8_E4M3;
  const Layout l = layout(m, k, 0, quantized, linear_parts(m, n, k));
  if (bad_workspace(workspace, workspace_bytes, l.bytes))
    return fail(TF_ERR_INVALID, "block_linear: workspace of %lld bytes (needs %lld, 16-byte "
                "aligned)", (long long)workspace_bytes, (long long)l.bytes);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  BlockGemmArgs g{};
  BlockQuantArgs q;
  if ((rc = weight_setup("block_linear", "weight", mat, n, k, &g.mat[0])) != TF_OK) return rc;
  if ((rc = out_setup("block_linear", mat, &g)) != TF_OK) return rc;
  rc = input_setup("block_linear", x, x_dtype, x_row_stride, x_scale, x_scale_stride, m, k, ws, l,
                   &g, &q);
  if (rc != TF_OK) return rc;   // nothing is launched for arguments that any part refuses
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int xk = prepare_input(x_dtype, k, g, q, s);
  if (few_rows(m))
    launch_rows(rows_args(g, k, xk, q), xk, s);
  else
    launch_tiles(g, plan_linear(m, n, 1, g.KB, false, device_cu_count()), 1,
                 reinterpret_cast<float*>(ws + l.part), s);
  return launch_status("tf_block_linear launch");
}

int64_t tf_gated_mlp_workspace_bytes(int64_t m, int64_t hidden, int64_t inter, int64_t n_out,
                                     int32_t x_dtype) {
  using namespace tfa;
  clear_error();
  int32_t rc = check_product("gated_mlp", m, inter, hidden);
  if (rc == TF_OK) rc = check_product("gated_mlp", m, n_out, inter);
  if (rc != TF_OK) return rc;
  if (m == 0) return 0;
  return layout(m, hidden, inter, x_dtype == TF_DTYPE_FP8_E4M3,
                std::max(gated_parts(m, inter, hidden), linear_parts(m, n_out, inter)))
      .bytes;
}

int32_t tf_gated_mlp(const void* x, int32_t x_dtype, int64_t x_row_stride, const float* x_scale,
                     int64_t x_scale_stride, const tf_fp8_mat* mats, int64_t m, int64_t hidden,
                     int64_t inter, void* workspace, int64_t workspace_bytes,
                     tf_stream_t stream) {
  using namespace tfa;
  if (!mats) {
    clear_error();
    return fail(TF_ERR_INVALID, "gated_mlp: no weights");
  }
  const tf_fp8_mat *gate = mats, *up = mats + 1, *down = mats + 2;
  const int64_t n_out = down->n;
  const int64_t need = tf_gated_mlp_workspace_bytes(m, hidden, inter, n_out, x_dtype);
  if (need < 0) return (int32_t)need;   // (it cleared and set the error)
  if (m == 0) return TF_OK;
  if (bad_workspace(workspace, workspace_bytes, need))
    return fail(TF_ERR_INVALID, "gated_mlp: workspace of %lld bytes (needs %lld, 16-byte aligned)",
                (long long)workspace_bytes, (long long)need);
  const bool quantized = x_dtype == TF_DTYPE_FP8_E4M3;
  const Layout l = layout(m, hidden, inter, quantized, 0);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  float* part = reinterpret_cast<float*>(ws + l.part);
  BlockGemmArgs g{}, d{};
  BlockQuantArgs q;
  int32_t rc;
  if ((rc = weight_setup("gated_mlp", "gate weight", gate, inter, hidden, &g.mat[0])) != TF_OK ||
      (rc = weight_setup("gated_mlp", "up weight", up, inter, hidden, &g.mat[1])) != TF_OK ||
      (rc = weight_setup("gated_mlp", "down weight", down, n_out, inter, &d.mat[0])) != TF_OK ||
      (rc = out_setup("gated_mlp", down, &d)) != TF_OK ||
      (rc = input_setup("gated_mlp", x, x_dtype, x_row_stride, x_scale, x_scale_stride, m, hidden,
                        ws, l, &g, &q)) != TF_OK)
    return rc;
  d.M = (int32_t)m;
  d.KB = (int32_t)ceil_div(inter, kQBlock);
  d.tail = (int32_t)(inter - (int64_t)(d.KB - 1) * kQBlock);
  d.xq = g.hq = ws + l.hq;
  d.xs = g.hqs = (int64_t)d.KB * kQBlock;
  d.xsc = g.hsc = reinterpret_cast<float*>(ws + l.hsc);
  d.xss = g.hss = m;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (!quantized)
    launch_quant(q, x_dtype == TF_DTYPE_FP32, s);
  else if (pads(m, hidden))
    launch_pad(q, s);
  if (few_rows(m)) {
    RowsArgs r = rows_args(g, hidden, kXRows, q);
    r.h = part;
    launch_rows(r, kXRows, s);
    rc = quant_setup("gated_mlp", part, TF_DTYPE_FP32, m, inter, inter, ws + l.hq, d.xs,
                     g.hsc, m, d.xs, &q);
    if (rc != TF_OK) return rc;
    const int xk = prepare_input(TF_DTYPE_FP32, inter, d, q, s);
    launch_rows(rows_args(d, inter, xk, q), xk, s);
    return launch_status("tf_gated_mlp launch");
  }
  const int64_t cus = device_cu_count();
  launch_tiles(g, plan_gated(m, inter, g.KB, cus), 2, part, s);
  launch_tiles(d, plan_linear(m, n_out, 1, d.KB, false, cus), 1, part, s);
  return launch_status("tf_gated_mlp launch");
}

}  // extern "C"
