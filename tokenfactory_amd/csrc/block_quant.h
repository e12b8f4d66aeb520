// Device side of the block quantisation: e4m3 values with one fp32 scale per 128
// columns of a row,
//   s = fl32(max(amax|x|, 1e-12) / 448),  q = e4m3(fl32(x / s)),
// both roundings as torch's tensor operations make them.  amax travels as the
// bits of |x|: for them integer order is float order and NaN sorts above inf, so
// a NaN (or inf) anywhere in a block makes its scale NaN (inf) and with it every
// product of the block, and no other row's.
#pragma once

#include "tf_common.h"

namespace tfa {

constexpr int kQBlock = 128;

// Eight consecutive elements (16-byte aligned) of a bf16 or fp32 array.
template <bool F32>
__device__ __forceinline__ void load8(const uint8_t* p, int64_t elem, float* v) {
  if constexpr (F32) {
    const u32x4 a = ld_g16(p + elem * 4), b = ld_g16(p + elem * 4 + 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = __uint_as_float(a[j]);
      v[4 + j] = __uint_as_float(b[j]);
    }
  } else {
    const u32x4 a = ld_g16(p + elem * 2);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = bf16_lo(a[j]);
      v[2 * j + 1] = bf16_hi(a[j]);
    }
  }
}

__device__ __forceinline__ uint32_t amax_bits8(const float* v) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
  return m;
}
// v of another of the 16 lanes of a row (a DPP control), without a way through LDS.
template <int CTRL>
__device__ __forceinline__ int dpp(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, false);
}
// The steps of a reduction over 16 lanes: lanes 1 and 2 away, then the mirrored lane
// of 8 and of 16, whose group's value by then is the same in all its lanes.
constexpr int kDppXor1 = 0xB1, kDppXor2 = 0x4E, kDppMirror8 = 0x141, kDppMirror16 = 0x140;
// Maximum over the 16 lanes that hold a block (all of them call it).
__device__ __forceinline__ uint32_t amax_lanes16(uint32_t m) {
  m = max(m, (uint32_t)dpp<kDppXor1>((int)m));
  m = max(m, (uint32_t)dpp<kDppXor2>((int)m));
  m = max(m, (uint32_t)dpp<kDppMirror8>((int)m));
  return max(m, (uint32_t)dpp<kDppMirror16>((int)m));
}
__device__ __forceinline__ float sum_lanes16(float v) {
  v += __int_as_float(dpp<kDppXor1>(__float_as_int(v)));
  v += __int_as_float(dpp<kDppXor2>(__float_as_int(v)));
  v += __int_as_float(dpp<kDppMirror8>(__float_as_int(v)));
  return v + __int_as_float(dpp<kDppMirror16>(__float_as_int(v)));
}

__device__ __forceinline__ float block_scale(uint32_t amax_bits) {
  const uint32_t floor_bits = __float_as_uint(1e-12f);
  return __uint_as_float(max(amax_bits, floor_bits)) / 448.f;
}

// Divisor of a block: s, and 1 / s.  The quotient fl32(x / s) of a value is its
// approximation x * inv corrected once by its exact remainder (the ten
// instructions of a division per value made the quantisation of 8192 x 17408 bf16
// values VALU-bound: 117 us).  That is the rounded quotient wherever the quotient
// is a number of 24 bits, ties of e4m3 among them, and otherwise unless it lies
// within 2^-23 ulp of the middle of two.  An infinite s gives 0 and, for infinite
// values, NaN, as the division does; a NaN s NaN.
struct BlockDiv {
  float s, inv;
};
__device__ __forceinline__ BlockDiv block_div(float s) {
  return {s == __builtin_inff() ? 0.f : s, 1.f / s};
}
__device__ __forceinline__ float quotient(float x, BlockDiv d) {
  const float q = x * d.inv;
  return __builtin_copysignf(__builtin_fmaf(__builtin_fmaf(-q, d.s, x), d.inv, q), x);   // (-0)
}

// (|x / s| is at most 448 and a rounding, which rounds to 448: no clamp.)
__device__ __forceinline__ uint32_t quant4(float a, float b, float c, float e, BlockDiv d) {
  const uint32_t r = __builtin_amdgcn_cvt_pk_fp8_f32(quotient(a, d), quotient(b, d), 0u, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(quotient(c, d), quotient(e, d), r, true);
}
__device__ __forceinline__ u32x2 quant8(const float* v, BlockDiv d) {
  return u32x2{quant4(v[0], v[1], v[2], v[3], d), quant4(v[4], v[5], v[6], v[7], d)};
}

}  // namespace tfa
