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
  float scale_log2;             // scale * log2(e)
  int splits;                   // CTAs along the keys of a unit, at most 32
  float *part_o;                // [splits, rows, hq, D] sums, where splits > 1,
  float2 *part_ml;              // [splits, rows, hq] and their (maximum, sum of weights)
};

// The plain form: a warp per (row, head), D / 32 dimensions per lane, one key
// at a time with the running maximum and sum.
template <int D>
__global__ void __launch_bounds__(128) prompt_simple_kernel(const RaggedArgs a) {
  constexpr int E = D / 32;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t item = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int64_t row = item / a.hq;
  const int h = int(item % a.hq), kvh = h / (a.hq / a.hk);
  if (row >= a.rows)
    return;
  const int b = sequence_of(a.starts, a.batch, row);
  if (b < 0)
    return;
  const int64_t begin = max(__ldg(a.starts + b), 0);
  const int64_t keys = row - begin + 1;
  float q[E], o[E];
  const __nv_bfloat16 *qp = a.q + row * a.q_row + h * a.q_head + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = __bfloat162float(qp[e]);
    o[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int64_t j = 0; j < keys; ++j) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e)
      s += q[e] * __bfloat162float(a.k[(begin + j) * a.k_row + kvh * a.k_head + lane * E + e]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1)
      s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= a.scale_log2;
    const float top = fmaxf(m, s);
    const float keep = m == -INFINITY ? 1.f : exp2f(m - top);   // nothing summed yet: keep 0 (or a NaN)
    const float p = s == -INFINITY ? 0.f : exp2f(s - top);   // NaN and +inf scores give NaN
    m = top;
    l = l * keep + p;
#pragma unroll
    for (int e = 0; e < E; ++e)
      o[e] = o[e] * keep + p * __bfloat162float(a.v[(begin + j) * a.v_row + kvh * a.v_head + lane * E + e]);
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e)
    a.out[row * a.ldo + h * D + lane * E + e] = __float2bfloat16(o[e] * inv);
}

} // namespace pir2b
