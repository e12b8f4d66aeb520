// Pieces shared by the FP8 tile GEMMs (fp8_linear.hip, block_fp8.hip): staging of
// 128-byte operand rows straight from global memory into swizzled LDS, the MFMA
// operand fragments read from there, and the order in which output tiles are
// dealt to the XCDs.
#pragma once

#include "tf_common.h"

namespace tfa {

typedef int32_t i32x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kKSlice = 128;          // K per slice = one weight-scale block

__device__ __forceinline__ int swz(int r) { return (r & 7) ^ ((r >> 3) & 1); }

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(const lds_void*)p;
}
// global_load_lds_dword{,x4} with a scalar base and a 32-bit per-lane offset:
// lane l's 4 / 16 bytes from sbase + voff land at LDS address M0 + 4 l / 16 l.
// Invisible to the compiler's wait counting: readers wait with an explicit
// s_waitcnt vmcnt and a barrier.
__device__ __forceinline__ void dma4(const void* sbase, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1"
               :: "v"(voff), "s"(sbase), "s"(lds) : "m0");
}
__device__ __forceinline__ void dma16(const void* sbase, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :: "v"(voff), "s"(sbase), "s"(lds) : "m0");
}

// The same with a 64-bit address per lane.
__device__ __forceinline__ void dma4_at(const void* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off"
               :: "v"(p), "s"(lds) : "m0");
}

template <int N>
__device__ __forceinline__ void vm_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory");
}

// Operand fragment of 16 rows x 128 bytes: lane l holds row l % 16, bytes
// 32 (l / 16) .. + 31 (chunks 2 (l / 16) and 2 (l / 16) + 1, stored swizzled).
// The f8f6f4 MFMA sums over (lane group, byte) pairs in the same way for both
// operands, so any k order shared by the two operands gives the same product.
__device__ __forceinline__ i32x8 frag(const uint8_t* row, int o0, int o1) {
  const u32x4 a = ld_s16(row + o0), b = ld_s16(row + o1);
  i32x8 f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[j] = (int32_t)a[j];
    f[4 + j] = (int32_t)b[j];
  }
  return f;
}

__device__ __forceinline__ f32x4 mfma_fp8(const i32x8& w, const i32x8& x) {
  // e4m3 x e4m3 (format 0 for both operands), no block exponents: an
  // unscaled v_mfma_f32_16x16x128_f8f6f4 from zero.
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, f32x4{0.f, 0.f, 0.f, 0.f}, 0,
                                                          0, 0, 0, 0, 0);
}

// Tile order.  Workgroup b of a grid runs on XCD b % 8 (workgroups are dealt to
// the 8 XCDs round-robin), and each XCD takes its workgroups in launch order.
// XCD x gets the contiguous range [x T / 8, (x + 1) T / 8) (rounded) of a
// grouped order in which gm_max consecutive m-tiles share each n-tile, so the
// workgroups one XCD runs at once cover a compact block of tiles (8 m-tiles x
// 4 n-tiles for 32 CUs) whose X and W slices its L2 serves once to all of
// them.  Under split-K (grid = splits x T) the same permutation is applied to
// each split's tiles.
__device__ __forceinline__ int xcd_order(int b, int tiles) {
  const int x = b & 7, i = b >> 3, q = tiles >> 3, r = tiles & 7;
  return x * q + min(x, r) + i;
}
__device__ __forceinline__ void tile_at(int lin, int tiles, int tiles_m, int gm_max, int* tm,
                                        int* tn) {
  const int tiles_n = tiles / tiles_m;
  const int group = gm_max * tiles_n;
  const int gid = lin / group, in = lin - gid * group;
  const int gm = min(tiles_m - gid * gm_max, gm_max);
  *tm = gid * gm_max + in % gm;
  *tn = in / gm;
}
// The place of a tile in that order.
__device__ __forceinline__ int tile_index(int tm, int tn, int tiles, int tiles_m, int gm_max) {
  const int gid = tm / gm_max, gm = min(tiles_m - gid * gm_max, gm_max);
  return gid * gm_max * (tiles / tiles_m) + tn * gm + tm - gid * gm_max;
}
__device__ __forceinline__ void xcd_tile(int b, int tiles, int tiles_m, int gm_max, int* tm,
                                         int* tn) {
  tile_at(xcd_order(b, tiles), tiles, tiles_m, gm_max, tm, tn);
}

}  // namespace tfa
