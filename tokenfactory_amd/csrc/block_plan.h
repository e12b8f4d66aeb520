// Which tiles a block-scaled product of more than 16 rows runs on (block_fp8.hip).
// Host code alone, a function of the sizes and the number of CUs.
#pragma once

#include <math.h>
#include <stdint.h>

namespace tfa {

// A tile shape (MT, WN) and its estimated time: a workgroup takes fixed +
// per_slice x K slices microseconds, workgroups run in rounds of one per CU (two
// of the small ones share a CU and take 1.5 times as long), a split adds a
// launch and its partials' way through memory.  Fitted to a sweep of every shape
// and 1 to 16 splits over 24 numbers of rows from 17 to 8192 at six products (640
// to 12288 columns, K 2176 to 17408) and four gated ones; with the present kernels
// the same sweep finds the choice 1.3 % behind the best of 144 products on average and
// 13 % at most (3000 x 5120 x 2592: 57.4 us for 50.8), 0.2 % and 8 % for 96 gated
// ones.  The estimates only rank the shapes: the wide forms take longer than theirs
// (48 x 5120 x 2 x 17408 33 us, measured 48).  What the rarer shapes are for: without 192 rows x 128 columns 333 x 5120 x 12288 takes 49.9 us for 37.6,
// without 128 x 256 1500 x 5120 x 17408 149.8 for 131.7.  A split is taken of the
// tiles behind the last full round only: with every tile whole 4096 x 5120 x 17408
// takes 357 us for 318 (256 tiles whole, 64 by 4 workgroups each), 1300 x 12288 x
// 4096 100 for 91.
struct Shape {
  int mt, wn;
};
struct ShapeCost {
  Shape shape;
  float fixed, per_slice;
  bool two;        // two workgroups per CU
};
constexpr ShapeCost kShapes[] = {{{1, 2}, 2.48f, 0.470f, true},  {{2, 2}, 2.80f, 0.493f, true},
                                 {{4, 2}, 3.15f, 0.708f, false}, {{6, 2}, 2.28f, 0.888f, false},
                                 {{4, 4}, 1.45f, 0.938f, false}, {{6, 4}, 1.79f, 1.374f, false},
                                 {{8, 4}, 2.96f, 1.550f, false}};
constexpr ShapeCost kGatedShapes[] = {{{2, 4}, 3.04f, 0.750f, false},
                                      {{4, 4}, 4.39f, 1.090f, false},
                                      {{6, 4}, 1.93f, 1.572f, false},
                                      {{8, 4}, 4.67f, 1.771f, false}};
constexpr int kMaxSplits = 16;        // split-K factor limit
constexpr int64_t kGatedCols = 128;   // columns of h of a gated tile: a block of its scales
constexpr float kReduceUs = 2.8f, kPartialBytesPerUs = 2.8e6f;   // written, then read

struct BlockPlan {
  Shape shape;
  int full, splits;   // tiles computed whole; workgroups per tile of the others
  int64_t part;       // fp32 elements of partials
  bool fused;         // gated: h leaves the product's kernel quantised
  float us;
};

inline float rounds(const ShapeCost& c, int64_t wgs, int64_t cus) {
  if (!c.two) return (float)((wgs + cus - 1) / cus);
  const int64_t full = wgs / (2 * cus), rem = wgs - full * 2 * cus;
  return 1.5f * (float)full + (rem == 0 ? 0.f : rem <= cus ? 1.f : 1.5f);
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// Whether gate and up products run on the bf16 MFMA.  The fp8 one cuts each product
// 13 bits below the largest of its eight (1.5e-5 of a sum of Gaussian values, 1e-4
// where a few channels are large), which rounding h to e4m3 turns into whole steps
// of the values next to a border: the block's output is 0.23 % off instead of 0.17 %
// (the bf16 rounding alone), single rows 0.4 %.  Up to 64 rows the staging hides most
// of the wider MFMAs (block of 5120 x 17408 at 48 rows 76.3 us for 74.0, at 64 78.1 for
// 76.3; of 5120 x 2176 at 48 25.5 for 23.2).  Above, they would take 112 us for 84 at 65
// rows of 5120 x 17408, 37 for 31 at 200 of 5120 x 2176.
constexpr int64_t kWideRows = 64;
inline bool wide_gated(int64_t m) { return m <= kWideRows; }

// n_mats matrices of n columns over kb K slices, on cus CUs; parts: every tile leaves
// as partials, split or not.
inline BlockPlan plan_linear(int64_t m, int64_t n, int n_mats, int64_t kb, bool parts,
                             int64_t cus) {
  BlockPlan best{kShapes[0].shape, 0, 1, 0, false, INFINITY};
  for (const ShapeCost& c : kShapes) {
    if (n_mats == 2 && wide_gated(m) && c.shape.mt > 2) continue;   // (no wide form)
    const int64_t bm = 32 * c.shape.mt, bn = 64 * c.shape.wn;
    const int64_t tiles = ceil_div(m, bm) * ceil_div(n, bn) * n_mats;
    const int64_t round = c.two ? 2 * cus : cus;
    const float filled = (float)(m * n * n_mats) / (float)(tiles * bm * bn);
    for (int64_t sp = 1; sp <= kMaxSplits; ++sp) {
      const int64_t full = parts ? 0 : sp == 1 ? tiles : tiles / round * round;
      const int64_t rest = tiles - full;   // split, or partials
      if (sp > 1 && (kb / sp < 2 || rest == 0 || rest * sp > 2 * cus)) break;
      float us = rounds(c, full, cus) * (c.fixed + c.per_slice * (float)kb);
      if (rest > 0)
        us += rounds(c, rest * sp, cus) * (c.fixed + c.per_slice * (float)ceil_div(kb, sp)) +
              kReduceUs + filled * (float)(rest * sp * bm * bn) * 8.f / kPartialBytesPerUs;
      if (us < best.us) best = {c.shape, (int)full, (int)sp, rest * sp * bm * bn, false, us};
    }
  }
  return best;
}

inline BlockPlan plan_gated(int64_t m, int64_t inter, int64_t kb, int64_t cus) {
  BlockPlan best = plan_linear(m, inter, 2, kb, true, cus);
  // (a launch has 2^32 threads; the one that finishes partials 32 per row and block)
  if (m * ceil_div(inter, kGatedCols) * 32 > UINT32_MAX) best.us = INFINITY;
  for (const ShapeCost& c : kGatedShapes) {
    if (wide_gated(m) && c.shape.mt > 2) continue;
    const int64_t tiles = ceil_div(m, 32 * c.shape.mt) * ceil_div(inter, kGatedCols);
    const float us = rounds(c, tiles, cus) * (c.fixed + c.per_slice * (float)kb);
    if (us < best.us) best = {c.shape, (int)tiles, 1, 0, true, us};
  }
  return best;
}

}  // namespace tfa
