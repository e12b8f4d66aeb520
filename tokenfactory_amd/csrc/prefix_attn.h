// Lists and arguments of the attention over parts of contexts (prefix_attn.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tfa {

// Query rows row0 .. of the n_tok tokens at tokens[tok0] (row = t * G + head of the kv
// head's group) over keys [k0, k1) of request b's table row; k1 < 0: up to what the
// rows see.  pfx: of a request's own part, the shared part before it (-1: none): its
// first item, or its first unit in PartArgs::units; pfx_tok: where the request's tokens
// start among that part's.
struct PartItem {
  int32_t b, tok0, n_tok, row0, k0, k1, pfx, pfx_tok;
};

// A query token: its row of q, its request, and how many tokens of that follow it.
struct PartTok {
  int32_t qrow, b, back, pad;
};

struct PartArgs {
  const __bf16* q;
  int64_t q_stride;
  const uint8_t* k_pool;
  const uint8_t* v_pool;
  int64_t pool_slots;
  const float* k_scale;
  const float* v_scale;
  const int64_t* rtt;
  int64_t rtt_rows, rtt_stride, rtt_cols;
  const int64_t* rpi;
  const int64_t* seq_lens;
  int32_t seq_override;
  // Shared parts, then the requests' own (from own0).  NULL (and toks): one new token per
  // request, item i the i % head_blocks-th block of its heads.
  const PartItem* items;
  const PartTok* toks;
  int32_t head_blocks;
  int32_t n_items, own0;
  int32_t unit_rows;       // query rows of a unit
  int32_t slot_rows;       // of them that any unit uses: rows of a partial slot
  int32_t hkv, group, head_dim;
  int32_t n_workers;       // waves that stream the items
  float scale_log2;
  __bf16* out;
  int64_t out_stride;
  const __bf16* gate;
  int64_t gate_stride, gate_hstride;
  uint32_t* amax;
  int32_t* ipre;           // prefix of the items' spans, for the merge
  float2* part_ml;         // partials of (worker + unit) slots
  float* part_o;
  // Shared parts that MFMA tiles took in pieces (NULL: they are items): unit
  // pfx + (row / 256) * hkv + kv head is {first slot, slots}.
  const int2* units;
  const float2* piece_ml;  // [slot][256], [slot][256][256 or 128]
  const float* piece_o;
  // Scored calls: every row's scores (log2 units, -inf where masked) of its first
  // score_cap keys, row q_row * q heads + head, and the table that their weights go to.
  float* row_scores;
  int64_t score_cap;
  float* scores;
  int64_t scores_stride;
  int32_t add_scores;
  int32_t weight_blocks, n_weights;   // workgroups for them: per request, and in all
};

}  // namespace tfa
