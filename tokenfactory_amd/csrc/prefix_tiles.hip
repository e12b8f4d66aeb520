// Pieces of shared prefixes at head dims up to 128 (bf16 pools): what extend.hip's tiles do
// at 256 for tf_attn_shared (prefix_attn.hip), with rows of 128 dims.
//
// A workgroup takes 256 query rows (32 per wave) of a group's tokens over a piece of the
// shared keys, 64 keys at a time: K and V rows go through registers into one of two LDS
// buffers a tile ahead (one barrier per tile), chunks swizzled so that both operand reads
// are free of bank conflicts.  Per tile a wave computes with v_mfma_f32_32x32x16_bf16
//   S^T[key, row] = K Q^T   (Q^T in registers, read once),
//   O^T[dim, row] += V^T P^T (V^T by ds_read_b64_tr_b16),
// a lane owning one row's half of the scores and of the dims.  P enters as three bf16
// parts, all of its 24 bits, smallest first, as in the streaming kernel at these head dims
// (decode.hip): that triples the PV products, which these steps have to spare: they are
// bound by their launch, their first loads and the partials (96 requests on 2000 keys, 32 /
// 8 heads: 3.1 GFLOP, 38 us beside the streams of 700 own keys each at most, 113 MB).
#include <math.h>

#include "part_stream.h"
#include "prefix_attn.h"
#include "tf_common.h"
#include "tf_internal.h"

namespace tfa {
namespace {

typedef __attribute__((address_space(3))) void lds_void;
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

constexpr int kDims = 128;                     // of a staged row; dims past the head's are zeros
constexpr int kTileWaves = 8;
constexpr int kThreads = kTileWaves * kWave;
constexpr int kRowsPerWave = 32;
static_assert(kTileWaves * kRowsPerWave == kExtendItemRows, "rows of an entry");
constexpr int kBN = 64;                        // keys per tile
constexpr int kRowBytes = 2 * kDims;
constexpr int kRowChunks = kRowBytes / 16;     // 16
constexpr int kPerThread = kBN * kRowChunks / kThreads;   // 16-byte chunks of K (and V): 2
constexpr int kQSteps = kDims / 16;
constexpr float kNoKeys = -1e30f;              // reference maximum of a row before its first key
constexpr float kRescaleLog2 = 8.f;            // it is raised when outgrown by more than 2^8

struct __attribute__((aligned(16))) Smem {
  uint8_t k[2][kBN * kRowBytes];   // chunk c of key n at c ^ (n & 15)
  uint8_t v[2][kBN * kRowBytes];   // chunk c of key n at c ^ 4 (n & 3)
};

struct OwnParts {
  PartArgs a;
  int32_t n_stream;
};

// V^T operand of dims 32 mt + n for the 16 keys at `p` (see extend.hip, v_frag).
__device__ __forceinline__ u32x4 v_frag(const uint8_t* p) {
  const u32x2 lo = __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p)));
  const u32x2 hi = __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p + 8 * kRowBytes)));
  return u32x4{lo[0], lo[1], hi[0], hi[1]};
}

template <class... Beside>
__global__ void __launch_bounds__(kThreads) prefix_tiles_kernel(ExtendArgs a, int32_t head_dim,
                                                                Beside... beside) {
  __shared__ Smem sm;
  int entry = blockIdx.x;
  if constexpr (sizeof...(Beside) > 0) {
    const OwnParts& own = (beside, ...);
    if (entry < own.n_stream) {
      using C = Cfg<128, false, 1, true, true>;
      static_assert(sizeof(StreamSmem<C, false, kTileWaves>) <= sizeof(sm), "LDS");
      part_stream<C, false, kTileWaves>(
          own.a, reinterpret_cast<StreamSmem<C, false, kTileWaves>&>(sm), entry);
      return;
    }
    entry -= own.n_stream;
  }
  const int32_t* wk = a.work + 8 * (int64_t)entry;
  const int b = wk[0], hk = wk[1], row0 = wk[2], tok0 = wk[3], key0 = wk[5], slot = wk[7] - 1;
  const int G = a.group, rows_total = wk[4] * G;
  const int tid = threadIdx.x, lane = tid & 63, w = wave_id();
  const int g = lane >> 5, n = lane & 31;
  const int L = (int)min<int64_t>(wk[6], a.rtt_cols) - key0;   // keys of the piece
  const int w_first = row0 + kRowsPerWave * w;
  const bool idle = w_first >= rows_total;      // a wave without rows stages only
  const int rho = min(w_first + n, rows_total - 1);
  const int64_t pr = (int64_t)slot * kExtendItemRows + kRowsPerWave * w + n;
  if (L <= 0) {
    if (g == 0 && w_first + n < rows_total)
      reinterpret_cast<float2*>(a.part_ml)[pr] = float2{kNoKeys, 0.f};
    return;
  }

  // The lane's row: its Q^T fragments (dims 16 kk + 8 g ..) and the keys it sees.
  const PartTok tok = a.toks[tok0 + rho / G];
  const int seen = (int)min<int64_t>(L, min(a.seq_lens[tok.b], a.rtt_cols) - tok.back - key0);
  const __bf16* qp = a.q + (int64_t)tok.qrow * a.q_stride +
                     (int64_t)(hk * G + rho % G) * head_dim + 8 * g;
  u32x4 qf[kQSteps];
#pragma unroll
  for (int kk = 0; kk < kQSteps; ++kk)
    qf[kk] = 16 * kk + 8 * g < head_dim ? ld_g16(qp + 16 * kk) : u32x4{0u, 0u, 0u, 0u};
  int all_seen = seen;   // keys that every row of the wave sees
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) all_seen = min(all_seen, __shfl_xor(all_seen, m, kWave));

  // Staging: thread tid moves chunk tid % 16 of keys tid / 16 and tid / 16 + 32.
  const int64_t* rtt = a.rtt + clamp_i64(a.rpi[b], 0, a.rtt_rows - 1) * a.rtt_stride + key0;
  const int chunk = tid % kRowChunks, key = tid / kRowChunks;
  const bool live = 8 * chunk < head_dim;
  const int64_t row_bytes = 2 * (int64_t)head_dim, slot_bytes = a.hkv * row_bytes;
  const uint8_t* kb = a.k_pool + hk * row_bytes + 16 * chunk;
  const uint8_t* vb = a.v_pool + hk * row_bytes + 16 * chunk;
  const int n_tiles = (L + kBN - 1) / kBN;
  int64_t ids[kPerThread];
  u32x4 kx[kPerThread], vx[kPerThread];
  auto fetch_ids = [&](int tile) {   // (keys past the last repeat it: masked below)
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) ids[i] = rtt[min(tile * kBN + key + 32 * i, L - 1)];
  };
  auto fetch_rows = [&]() {
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int64_t off = pool_row(ids[i], a.pool_slots, false) * slot_bytes;
      kx[i] = live ? ld_g16(kb + off) : u32x4{0u, 0u, 0u, 0u};
      vx[i] = live ? ld_g16(vb + off) : u32x4{0u, 0u, 0u, 0u};
    }
  };
  auto stage = [&](int buf) {
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int k = key + 32 * i;
      st_s16(sm.k[buf] + k * kRowBytes + 16 * (chunk ^ (k & 15)), kx[i]);
      st_s16(sm.v[buf] + k * kRowBytes + 16 * (chunk ^ (4 * (k & 3))), vx[i]);
    }
  };

  // LDS read offsets of the lane: K row n, V as the transposing reads take it.
  const int r = (lane & 15) >> 2;
  const int vlow = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const int vbase = (4 * g + r) * kRowBytes + 16 * vlow + 8 * (lane & 1);
  int vaddr[4];
#pragma unroll
  for (int mt = 0; mt < 4; ++mt) vaddr[mt] = vbase + 64 * (mt ^ r);

  const float sl2 = a.scale_log2;
  float m = kNoKeys, l = 0.f;
  f32x16 acc[4];
#pragma unroll
  for (int mt = 0; mt < 4; ++mt) acc[mt] = f32x16{};

  fetch_ids(0);
  fetch_rows();
  fetch_ids(min(1, n_tiles - 1));
  for (int j = 0; j < n_tiles; ++j) {
    // Buffer j & 1 was read last at tile j - 2, whose readers are past barrier j - 1.
    stage(j & 1);
    __syncthreads();
    if (j + 1 < n_tiles) {
      fetch_rows();
      fetch_ids(min(j + 2, n_tiles - 1));
    }
    if (idle) continue;
    const uint8_t* ks = sm.k[j & 1];
    const uint8_t* vs = sm.v[j & 1];
    f32x16 s[2] = {f32x16{}, f32x16{}};
#pragma unroll
    for (int kk = 0; kk < kQSteps; ++kk)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        s[h] = mfma_32x32x16(
            ld_s16(ks + (32 * h + n) * kRowBytes + 16 * ((2 * kk + g) ^ (n & 15))), qf[kk], s[h]);
    const int k0 = j * kBN;
    if (k0 + kBN > all_seen) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (k0 + 32 * h + 8 * (i >> 2) + 4 * g + (i & 3) >= seen) s[h][i] = -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[h][i]);
    mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
    const bool grow = (mx - m) * sl2 > kRescaleLog2;
    if (__ballot(grow)) {
      const float mnew = grow ? mx : m;
      const float alpha = grow ? fast_exp2((m - mnew) * sl2) : 1.f;
      m = mnew;
      l *= alpha;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) acc[mt] *= alpha;
    }
    const float moff = m * sl2;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int q = 0; q < 2; ++q) {   // 16 keys: 8 a lane
        u32x4 pt[3];                  // parts of P^T, largest first
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float p0 = fast_exp2(fmaf(s[h][8 * q + 2 * i], sl2, -moff));
          float p1 = fast_exp2(fmaf(s[h][8 * q + 2 * i + 1], sl2, -moff));
          l += p0 + p1;
#pragma unroll
          for (int c = 0; c < 3; ++c) {   // (the differences are exact)
            pt[c][i] = pack_bf16(p0, p1);
            p0 -= bf16_lo(pt[c][i]);
            p1 -= bf16_hi(pt[c][i]);
          }
        }
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          const u32x4 vf = v_frag(vs + vaddr[mt] + (32 * h + 16 * q) * kRowBytes);
#pragma unroll
          for (int c = 2; c >= 0; --c) acc[mt] = mfma_32x32x16(vf, pt[c], acc[mt]);
        }
      }
  }
  l += __shfl_xor(l, 32, kWave);
  if (w_first + n < rows_total) {   // a row's dims side by side, for the merge by rows
#pragma unroll
    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4*>(a.part_o + pr * kDims + 32 * mt + 8 * i + 4 * g) =
            f32x4{acc[mt][4 * i], acc[mt][4 * i + 1], acc[mt][4 * i + 2], acc[mt][4 * i + 3]};
    if (g == 0) reinterpret_cast<float2*>(a.part_ml)[pr] = float2{m * sl2, l};
  }
}

}  // namespace

int launch_prefix_tiles(const ExtendArgs& a, int32_t head_dim, int32_t n_pieces,
                        const PartArgs* own, int32_t n_stream, hipStream_t s) {
  if (own)
    hipLaunchKernelGGL((prefix_tiles_kernel<OwnParts>), dim3((unsigned)(n_stream + n_pieces)),
                       dim3(kThreads), 0, s, a, head_dim, OwnParts{*own, n_stream});
  else
    hipLaunchKernelGGL((prefix_tiles_kernel<>), dim3((unsigned)n_pieces), dim3(kThreads), 0, s, a,
                       head_dim);
  return launch_status("tf_attn_shared prefix launch");
}

}  // namespace tfa
