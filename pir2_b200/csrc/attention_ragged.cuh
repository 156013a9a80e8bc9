// Causal grouped-query attention of ragged batches: packed prompts of
// different lengths (pir2b_prompt_attention) and new tokens over the paged
// K/V cache (pir2b_cache_attention).
//
// out[t, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale (q_t . k_j) - m),
// over the keys j that query t sees: those of its own sequence up to its own
// position, m their largest score.  A query that sees no key gives zeros.
#pragma once
#include "kv_cache.cuh"

namespace pir2b {

struct RaggedArgs {
  const __nv_bfloat16 *q;   // [rows, hq, D] view
  int64_t q_row, q_head;
  const __nv_bfloat16 *k, *v;   // packed rows (prompts), [rows, hk, D] views
  int64_t k_row, k_head, v_row, v_head;
  CachePages c;                 // pages (cache)
  const int *starts, *lengths;
  __nv_bfloat16 *out;           // [rows, hq * D]
  int64_t ldo;
  int64_t rows;
  int batch, hq, hk;
  int group;                    // hq / hk
  uint32_t inverse;             // floor(2^32 / group), 2^32 - 1 for 1
  float scale_log2;             // scale * log2(e)
  int q_by_tma, out_by_tma;     // q tiles (output rows of a warp) are whole boxes: the group divides 128 (32)
  int splits;                   // CTAs along the keys of a unit, at most 32
  float *part_o;                // [splits, rows, hq, D] sums, where splits > 1,
  float2 *part_ml;              // [splits, rows, hq] and their (maximum, sum of weights)
  int sms;                      // of the device
  int ordered;                  // longer sequences first
  int cluster;                  // few-row kernel: CTAs of a unit, as a cluster; 0: as pieces of a list
  // Few-row kernel: CTAs wanted and launched, and per unit of rows its first piece and how
  // many; part_o and part_ml are then [CTAs, unit rows].
  int pieces, parts;
  int2 *part_units;
};

// x / group, x >= 0: the product falls short of the quotient by one at most.
__device__ __forceinline__ int over_group(const RaggedArgs &a, int x) {
  const int q = int(__umulhi(uint32_t(x), a.inverse));
  return q + (x - q * a.group >= a.group);
}

} // namespace pir2b
