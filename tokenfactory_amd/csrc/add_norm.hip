// Norms before and after a block, fused with the block's gate, the residual sum
// and the quantisation for the next product.  Per row of x (a block's output):
//   b  = x                                         or wp * x / rms(x)
//   r' = r + alpha * (gate * b)                    the residual stream
//   y  = w * r' / rms(r')                          the next block's input
// with rms(v) = sqrt(mean v^2 + eps), all of it in fp32; r' is rounded to the
// residual's type when it is stored, and y is formed from r' before that
// rounding.  y leaves in x's type or as e4m3 with a scale per 128 columns
// (block_quant.h).  The decoder layer's residual sums and norms
// (qwen3_8/decoder_layer.py:57-81, qwen3_8/rms_norm.py:19-24), with the forms
// around them: a norm of the block's output, a gate (per row, per column or per
// element) and a residual multiplier.
//
// HBM-bound: a row is read once into registers and written once.  A workgroup
// owns a row, a thread NV groups of 8 columns, one wave-wide and one LDS step per
// sum; 16 neighbouring lanes hold the 128 columns of a scale.  8192 x 5120 bf16 with
// a residual, quantised: 66 us = 4.5 TB/s (a copy of its 294 MB takes 57); rows kept
// in flight by a workgroup for the next one, rows in order per XCD and non-temporal
// accesses took 72 to 82.  777 x 2560 with an fp32 residual, post norm and gate: 8.1;
// 48 x 5120: 4.2, a launch and two dependent sums.

#include "block_quant.h"
#include "tf_common.h"
#include "tf_internal.h"

namespace tfa {
namespace {

constexpr int kMaxWaves = 16;

struct Operand {          // bf16 or fp32 rows; NULL: absent
  const uint8_t* p;
  int64_t stride;         // elements between rows
  int32_t f32;
};

struct AddNormArgs {
  Operand x, res, gate, post, w;
  int32_t gate_cols;      // gate: 8 columns of a row side by side (else one value per row)
  float eps, alpha;
  int64_t rows;
  int32_t cols;
  uint8_t* res_out;       // r' (NULL: not stored)
  int64_t ros;
  int32_t ro_f32;
  uint8_t* y;             // NULL: no norm of r'
  int64_t ys;
  int32_t y_dtype;
  float* ysc;             // e4m3: scale of (row, block) at block * yss + row
  int64_t yss;
};

// Eight elements as they lie in memory; converted where they are used, so that a
// thread's loads stay in flight together whatever their types.
struct Raw8 {
  u32x4 a, b;
};
__device__ __forceinline__ Raw8 fetch(const Operand& o, int64_t elem) {
  Raw8 r;
  const uint8_t* p = o.p + elem * (o.f32 ? 4 : 2);
  r.a = ld_g16(p);
  r.b = o.f32 ? ld_g16(p + 16) : u32x4{0u, 0u, 0u, 0u};
  return r;
}
__device__ __forceinline__ void widen(const Raw8& r, int f32, float* v) {
  if (f32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = __uint_as_float(r.a[j]);
      v[4 + j] = __uint_as_float(r.b[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = bf16_lo(r.a[j]);
      v[2 * j + 1] = bf16_hi(r.a[j]);
    }
  }
}
__device__ __forceinline__ void store8(uint8_t* p, int64_t elem, int f32, const float* v) {
  if (f32) {
    f32x4* q = reinterpret_cast<f32x4*>(p + elem * 4);
    q[0] = f32x4{v[0], v[1], v[2], v[3]};
    q[1] = f32x4{v[4], v[5], v[6], v[7]};
  } else {
    *reinterpret_cast<u32x4*>(p + elem * 2) =
        u32x4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]),
              pack_bf16(v[6], v[7])};
  }
}

// Sum over the workgroup, in 64 bits from the waves' sums on (a value next to a
// border of e4m3 moves by a step for an error in the last bits); every thread gets
// the same bits.
__device__ __forceinline__ double block_sum(float v, float* red) {
  v = sum_lanes16(v);
  v += __shfl_xor(v, 16, kWave);
  v += __shfl_xor(v, 32, kWave);
  const int n = blockDim.x / kWave;
  if (n == 1) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = red[0];
  for (int i = 1; i < n; ++i) s += red[i];
  return s;
}

// 1 / rms of a row from its sum of squares.
__device__ __forceinline__ float inverse_rms(double sum, const AddNormArgs& a) {
  return 1.f / sqrtf((float)(sum / a.cols + a.eps));
}

template <int NV>
__global__ void __launch_bounds__(kMaxWaves * kWave, NV == 1 ? 8 : 4) add_norm_kernel(AddNormArgs a) {
  __shared__ float red[2][kMaxWaves];
  const int64_t row = blockIdx.x;
  const int t = threadIdx.x;
  Raw8 xr[NV], rr[NV], gr[NV], pr[NV], wr[NV];
  int col[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    col[i] = 8 * (t + i * (int)blockDim.x);
    if (col[i] >= a.cols) continue;
    xr[i] = fetch(a.x, row * a.x.stride + col[i]);
    if (a.res.p) rr[i] = fetch(a.res, row * a.res.stride + col[i]);
    if (a.gate_cols) gr[i] = fetch(a.gate, row * a.gate.stride + col[i]);
    if (a.post.p) pr[i] = fetch(a.post, col[i]);
    if (a.w.p) wr[i] = fetch(a.w, col[i]);
  }
  float g0 = 1.f;   // a gate value of the whole row
  if (a.gate.p && !a.gate_cols)
    g0 = a.gate.f32 ? reinterpret_cast<const float*>(a.gate.p)[row * a.gate.stride]
                    : bf16_lo(reinterpret_cast<const uint16_t*>(a.gate.p)[row * a.gate.stride]);

  float v[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (col[i] < a.cols) {
      widen(xr[i], a.x.f32, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    }
  }
  if (a.post.p) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += v[i][j] * v[i][j];
    const float rstd = inverse_rms(block_sum(ss, red[0]), a);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (col[i] >= a.cols) continue;
      float p[8];
      widen(pr[i], a.post.f32, p);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * rstd * p[j];
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (col[i] >= a.cols) continue;
    if (a.gate_cols) {
      float g[8];
      widen(gr[i], a.gate.f32, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] *= g[j];
    } else if (a.gate.p) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] *= g0;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] *= a.alpha;
    if (a.res.p) {
      float r[8];
      widen(rr[i], a.res.f32, r);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] += r[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += v[i][j] * v[i][j];
    if (a.res_out) store8(a.res_out, row * a.ros + col[i], a.ro_f32, v[i]);
  }
  if (!a.y) return;
  const float rstd = inverse_rms(block_sum(ss, red[1]), a);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (col[i] < a.cols) {
      widen(wr[i], a.w.f32, y);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = v[i][j] * rstd * y[j];
    }
    if (a.y_dtype == DT_FP8_E4M3) {   // (the 16 lanes of a block take this path together)
      const float s = block_scale(amax_lanes16(amax_bits8(y)));
      if (col[i] < a.cols) {
        *reinterpret_cast<u32x2*>(a.y + row * a.ys + col[i]) = quant8(y, block_div(s));
        if (col[i] % kQBlock == 0) a.ysc[(int64_t)(col[i] / kQBlock) * a.yss + row] = s;
      }
    } else if (col[i] < a.cols) {
      store8(a.y, row * a.ys + col[i], a.y_dtype == DT_FP32, y);
    }
  }
}

constexpr int64_t kMaxCols = 8 * kWave * kMaxWaves * 2;   // (NV = 4 would spill)

// An operand of the call: rows (or one row) of bf16 or fp32 in 16-byte pieces.
int32_t operand(const char* what, const void* p, int32_t dtype, int64_t stride, int64_t min_stride,
                Operand* o) {
  *o = Operand{static_cast<const uint8_t*>(p), stride, dtype == TF_DTYPE_FP32};
  if (!p) return TF_OK;
  if (dtype != TF_DTYPE_BF16 && dtype != TF_DTYPE_FP32)
    return fail(TF_ERR_UNSUPPORTED, "add_rms_norm: %s must be bf16 or fp32 (dtype %d)", what,
                dtype);
  if (!aligned16(p) || stride % 8 || stride < min_stride)
    return fail(TF_ERR_INVALID, "add_rms_norm: %s rows must be 16-byte aligned, %lld apart at "
                "least (stride %lld)", what, (long long)min_stride, (long long)stride);
  return TF_OK;
}

}  // namespace
}  // namespace tfa

extern "C" int32_t tf_add_rms_norm(
    const void* x, int32_t x_dtype, int64_t x_row_stride, const void* residual,
    int32_t residual_dtype, int64_t residual_row_stride, const void* gate, int32_t gate_dtype,
    int64_t gate_row_stride, int32_t gate_per_column, const void* post_weight,
    int32_t post_weight_dtype, const void* weight, int32_t weight_dtype, float eps,
    float residual_scale, int64_t rows, int64_t cols, void* residual_out,
    int64_t residual_out_row_stride, void* y, int32_t y_dtype, int64_t y_row_stride,
    float* y_scale, int64_t y_scale_stride, tf_stream_t stream) {
  using namespace tfa;
  clear_error();
  if (rows < 0 || cols <= 0 || cols % 8)
    return fail(TF_ERR_INVALID, "add_rms_norm: rows=%lld cols=%lld (a positive multiple of 8)",
                (long long)rows, (long long)cols);
  if (cols > kMaxCols || rows > INT32_MAX)
    return fail(TF_ERR_UNSUPPORTED, "add_rms_norm: %lld x %lld (at most %lld columns)",
                (long long)rows, (long long)cols, (long long)kMaxCols);
  if (rows == 0) return TF_OK;
  if (!x || (!y && !residual_out) || (y && !weight))
    return fail(TF_ERR_INVALID, "add_rms_norm: null pointer");
  AddNormArgs a{};
  int32_t rc;
  if ((rc = operand("x", x, x_dtype, x_row_stride, cols, &a.x)) != TF_OK ||
      (rc = operand("residual", residual, residual_dtype, residual_row_stride, cols, &a.res)) !=
          TF_OK ||
      (rc = operand("post_weight", post_weight, post_weight_dtype, 0, 0, &a.post)) != TF_OK ||
      (rc = operand("weight", y ? weight : nullptr, weight_dtype, 0, 0, &a.w)) != TF_OK)
    return rc;
  if (gate_per_column) {
    rc = operand("gate", gate, gate_dtype, gate_row_stride, 0, &a.gate);
    if (rc != TF_OK) return rc;
    if (gate && gate_row_stride != 0 && gate_row_stride < cols)
      return fail(TF_ERR_INVALID, "add_rms_norm: gate row stride %lld",
                  (long long)gate_row_stride);
    a.gate_cols = gate != nullptr;
  } else if (gate) {
    const uintptr_t mask = gate_dtype == TF_DTYPE_FP32 ? 3u : 1u;
    if (gate_dtype != TF_DTYPE_BF16 && gate_dtype != TF_DTYPE_FP32)
      return fail(TF_ERR_UNSUPPORTED, "add_rms_norm: gate must be bf16 or fp32 (dtype %d)",
                  gate_dtype);
    if (gate_row_stride < 0 || (reinterpret_cast<uintptr_t>(gate) & mask))
      return fail(TF_ERR_INVALID, "add_rms_norm: gate row stride %lld or alignment",
                  (long long)gate_row_stride);
    a.gate = Operand{static_cast<const uint8_t*>(gate), gate_row_stride,
                     gate_dtype == TF_DTYPE_FP32};
  }
  if (residual_out) {
    if (!aligned16(residual_out) || residual_out_row_stride < cols || residual_out_row_stride % 8)
      return fail(TF_ERR_INVALID, "add_rms_norm: residual_out rows must be 16-byte aligned "
                  "(stride %lld)", (long long)residual_out_row_stride);
    a.res_out = static_cast<uint8_t*>(residual_out);
    a.ros = residual_out_row_stride;
    a.ro_f32 = (residual ? residual_dtype : x_dtype) == TF_DTYPE_FP32;
  }
  if (y) {
    if (y_dtype != TF_DTYPE_BF16 && y_dtype != TF_DTYPE_FP32 && y_dtype != TF_DTYPE_FP8_E4M3)
      return fail(TF_ERR_UNSUPPORTED, "add_rms_norm: y dtype %d", y_dtype);
    if (!aligned16(y) || y_row_stride < cols || y_row_stride % 8)
      return fail(TF_ERR_INVALID, "add_rms_norm: y rows must be 16-byte aligned (stride %lld)",
                  (long long)y_row_stride);
    if (y_dtype == TF_DTYPE_FP8_E4M3 &&
        (!y_scale || (reinterpret_cast<uintptr_t>(y_scale) & 3u) || y_scale_stride < rows))
      return fail(TF_ERR_INVALID, "add_rms_norm: quantised y needs scales, %lld apart at least "
                  "(stride %lld)", (long long)rows, (long long)y_scale_stride);
    a.y = static_cast<uint8_t*>(y);
    a.ys = y_row_stride;
    a.y_dtype = y_dtype;
    a.ysc = y_scale;
    a.yss = y_scale_stride;
  }
  a.eps = eps;
  a.alpha = residual_scale;
  a.rows = rows;
  a.cols = (int32_t)cols;
  const int64_t chunks = cols / 8;
  const int nv = chunks > kWave * kMaxWaves ? 2 : 1;
  const int threads = (int)((chunks + (int64_t)nv * kWave - 1) / ((int64_t)nv * kWave)) * kWave;
  if (rows * threads > UINT32_MAX)   // (of one launch)
    return fail(TF_ERR_UNSUPPORTED, "add_rms_norm: %lld x %lld is too large", (long long)rows,
                (long long)cols);
  const dim3 grid((uint32_t)rows), block(threads);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (nv == 1)
    hipLaunchKernelGGL(add_norm_kernel<1>, grid, block, 0, s, a);
  else
    hipLaunchKernelGGL(add_norm_kernel<2>, grid, block, 0, s, a);
  return launch_status("tf_add_rms_norm launch");
}
