// Paged K/V cache of the text layers: quantised rows written as they come
// from the projections, and read back as bf16.
//
// A cache is a pool of pages; page p holds `page` consecutive tokens of one
// sequence for every kv head, k_pages / v_pages [pages, hk, page, D] as bf16,
// int8 or E4M3, the two 8-bit formats with one fp32 scale per token and head
// ([pages, hk, page]).  table[b, i] is the page of positions
// [i * page, (i + 1) * page) of sequence b.  Rows are quantised as the
// activation packs are (symmetric-row-v1, quant.cuh): s = max|v| * f32(1/L),
// 1 for a row of zeros, L = 127 or 448; code = rint(v / s) clamped, or the
// nearest E4M3 number.  An infinity becomes the largest code.  A row with a
// NaN gets codes of 0 and the NaN as its scale, so every reader of the row
// sees it and the codes themselves are always numbers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cstdint>
#include "args.cuh"
#include "ptx.cuh"

namespace pir2b {

constexpr int kCacheBf16 = 16, kCacheInt8 = 8, kCacheE4m3 = 9;

// Codes of bad device-side indices (a page outside the pool, a position
// outside the table): the access is skipped and the status word records it.
constexpr int kStatusBadPage = 0x201;

__device__ __forceinline__ void record_status(int code) { atomicCAS(&g_device_status, 0, code); }

struct CachePages {
  void *k, *v;             // [pages, hk, page, D] codes
  float *ks, *vs;          // [pages, hk, page] scales (8-bit formats)
  int64_t k_page, v_page;  // elements from one page to the next
  int64_t ks_page, vs_page;
  const int *table;        // [batch, width] page of each block of positions
  int64_t ldt;             // table row stride
  int width;               // table columns
  int pages;
  int shift;               // log2(tokens per page)
  int hk;
};

struct CacheRowsArgs {
  CachePages c;
  const __nv_bfloat16 *k, *v;    // new rows (write), [rows, hk, D] views
  __nv_bfloat16 *k_out, *v_out;  // packed rows (read), [rows, hk, D]
  int64_t k_row, k_head, v_row, v_head;
  const int *starts;   // [batch + 1] packed rows of each sequence
  const int *lengths;  // [batch] tokens of each sequence, the new ones last
  int batch;
  int64_t rows;
};

// Sequence of packed row r: the last b with starts[b] <= r, -1 if none.
__device__ __forceinline__ int sequence_of(const int *starts, int batch, int64_t r) {
  int lo = 0, hi = batch;   // starts[lo] <= r < starts[hi] wherever r belongs to a sequence
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(starts + mid) <= r)
      lo = mid;
    else
      hi = mid;
  }
  return (__ldg(starts + lo) <= r && r < __ldg(starts + lo + 1)) ? lo : -1;
}

// Page of position `pos` of sequence b, or -1 (recorded) when the position
// lies outside the table or the table names no page of the pool.
__device__ __forceinline__ int page_of(const CachePages &c, int b, int64_t pos) {
  const int64_t block = pos >> c.shift;
  int page = -1;
  if (pos >= 0 && block < c.width)
    page = __ldg(c.table + b * c.ldt + block);
  if (page < 0 || page >= c.pages) {
    record_status(kStatusBadPage);
    return -1;
  }
  return page;
}

// Largest magnitude of eight bf16 as its bits: magnitudes order as integers,
// infinity (0x7f80) above the finite ones and NaNs above that.
__device__ __forceinline__ uint32_t magnitude8(const uint4 &x) {
  const uint32_t m = __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
  return max(m & 0xffffu, m >> 16);
}

// The same with infinities left out.
__device__ __forceinline__ uint32_t magnitude8_finite(const uint4 &x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t e = (w[i >> 1] >> ((i & 1) * 16)) & 0x7fffu;
    m = max(m, e == 0x7f80u ? 0u : e);
  }
  return m;
}

// Quotients x / s of a pair, y being 1 / s correctly rounded: a product and one
// step by the remainder, which an FMA gives exactly (Markstein's division).
// For a bf16 x and a scale that is f32(1/127) or f32(1/448) times a bf16 the
// result is the correctly rounded quotient: there are 2^14 pairs of
// significands, and all were compared.
__device__ __forceinline__ float2 quotients(float2 x, float2 minus_s, float2 y) {
  const float2 q = __fmul2_rn(x, y);
  return __ffma2_rn(__ffma2_rn(q, minus_s, x), y, q);
}

__device__ __forceinline__ float2 bf16_pair(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi) {
  uint16_t e;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(e) : "f"(hi), "f"(lo));
  return e;
}

// Eight finite bf16 -> eight codes under scale s = 1 / y, 2^-80 < s < 2^100 (so that no
// step over- or underflows): quotients rounded to nearest even.  int8: adding
// 1.5 * 2^23 rounds to an integer and leaves it in the low byte; a quotient is
// at most 127 (1 + 2^-22), so there is nothing to clamp.
template <int kFormat>
__device__ __forceinline__ uint2 quantise8(const uint4 &x, float s, float y) {
  const float2 minus_s = make_float2(-s, -s), yy = make_float2(y, y);
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t pair[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 q = quotients(bf16_pair(w[i]), minus_s, yy);
    if constexpr (kFormat == kCacheInt8) {
      const float2 r = __fadd2_rn(q, make_float2(12582912.f, 12582912.f));
      pair[i] = __byte_perm(__float_as_uint(r.x), __float_as_uint(r.y), 0x0040);
    } else {
      pair[i] = e4m3_pair(q.x, q.y);
    }
  }
  return make_uint2(__byte_perm(pair[0], pair[1], 0x5410), __byte_perm(pair[2], pair[3], 0x5410));
}

// The same for any row: infinities become the largest code, and under a NaN
// scale every code is 0.
template <int kFormat>
__device__ __noinline__ uint2 quantise8_any(uint4 x, float s) {
  constexpr float kLimit = kFormat == kCacheInt8 ? 127.f : 448.f;
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t out[2] = {0, 0};
  for (int i = 0; i < 4; ++i) {
    const float2 v = bf16_pair(w[i]);
    float2 q = make_float2(__fdiv_rn(v.x, s), __fdiv_rn(v.y, s));
    q.x = q.x == q.x ? fminf(fmaxf(q.x, -kLimit), kLimit) : 0.f;
    q.y = q.y == q.y ? fminf(fmaxf(q.y, -kLimit), kLimit) : 0.f;
    uint32_t pair;
    if constexpr (kFormat == kCacheInt8)
      pair = (uint32_t(__float2int_rn(q.x)) & 0xffu) | ((uint32_t(__float2int_rn(q.y)) & 0xffu) << 8);
    else
      pair = e4m3_pair(q.x, q.y);
    out[i >> 1] |= pair << ((i & 1) * 16);
  }
  return make_uint2(out[0], out[1]);
}

// Two 8-bit codes (the low 16 bits of `pair`) as fp32 values.
template <int kFormat>
__device__ __forceinline__ float2 code_values(uint32_t pair) {
  if constexpr (kFormat == kCacheInt8) {
    return make_float2(float(int8_t(pair & 0xff)), float(int8_t((pair >> 8) & 0xff)));
  } else {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(pair)));
    return __half22float2(*reinterpret_cast<__half2 *>(&h));
  }
}

// The same search by a whole warp, 128 candidates at a time.
__device__ __forceinline__ int sequence_of_warp(const int *starts, int batch, int64_t r) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = batch;
  do {
    const int step = (hi - lo + 127) >> 7;
    int count = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = lo + (i * 32 + lane) * step;
      count += __popc(__ballot_sync(0xffffffffu, at < hi && __ldg(starts + min(at, hi)) <= r));
    }
    if (count == 0)
      return -1;
    lo += (count - 1) * step;
    hi = min(hi, lo + step);
  } while (hi - lo > 1);
  return r < __ldg(starts + lo + 1) ? lo : -1;
}

constexpr int kCacheWarps = 4;

// A warp per token and 32 kFlight / (D / 16) of its (head, k or v) rows: D / 16
// lanes per row, each with two 16-byte pieces of it, 2 kFlight loads in flight;
// the row maximum comes by shuffles.  HBM-bound in bytes (2 D in, D + 4 out per
// row of an 8-bit cache), but instructions for the scale of a row weigh as
// much, so a lane takes as many of its values as keeps the loads coalesced.
// 33910 tokens of 8 kv heads of 128 to int8: 38 us, 5520 GB/s, 84 % of a copy's
// rate, 2.8 instructions a cycle and SM.
// The rows are fetched before the token's sequence and page are known.
template <int kFormat, int D, int kFlight>
__global__ void __launch_bounds__(kCacheWarps * 32) cache_write_kernel(const CacheRowsArgs a) {
  constexpr int kLanes = D / 16, kRows = 32 / kLanes;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = int64_t(blockIdx.x) * kCacheWarps + (threadIdx.x >> 5);
  if (row >= a.rows)
    return;
  const int lane = threadIdx.x & 31, l = lane % kLanes, hk = a.c.hk;
  const int r0 = blockIdx.y * kRows * kFlight + lane / kLanes;   // k rows of all heads, then v rows
  uint4 x[kFlight][2];
#pragma unroll
  for (int i = 0; i < kFlight; ++i) {
    const int r = r0 + i * kRows, head = r < hk ? r : r - hk;
    x[i][0] = x[i][1] = make_uint4(0, 0, 0, 0);
    if (r < 2 * hk) {
      const uint4 *src = reinterpret_cast<const uint4 *>(r < hk ? a.k + row * a.k_row + head * a.k_head
                                                                : a.v + row * a.v_row + head * a.v_head) + l;
      x[i][0] = __ldg(src);
      x[i][1] = __ldg(src + kLanes);
    }
  }
  const int b = sequence_of_warp(a.starts, a.batch, row);
  if (b < 0)
    return;
  const int64_t pos = int64_t(__ldg(a.lengths + b)) - __ldg(a.starts + b + 1) + row;
  const int page = page_of(a.c, b, pos);
  if (page < 0)
    return;
  const int in_page = int(pos & ((1 << a.c.shift) - 1));
  const int64_t k_at = page * a.c.k_page, v_at = page * a.c.v_page;
  float *k_scale = a.c.ks + page * a.c.ks_page, *v_scale = a.c.vs + page * a.c.vs_page;
#pragma unroll
  for (int i = 0; i < kFlight; ++i) {
    const int r = r0 + i * kRows, head = r < hk ? r : r - hk;
    const int slot = (head << a.c.shift) + in_page;          // below 2^17
    const int64_t at = (r < hk ? k_at : v_at) + (slot * D + l * 8);
    if constexpr (kFormat == kCacheBf16) {
      if (r < 2 * hk) {
        __nv_bfloat16 *to = static_cast<__nv_bfloat16 *>(r < hk ? a.c.k : a.c.v) + at;
        *reinterpret_cast<uint4 *>(to) = x[i][0];
        *reinterpret_cast<uint4 *>(to + kLanes * 8) = x[i][1];
      }
    } else {
      uint32_t m = max(magnitude8(x[i][0]), magnitude8(x[i][1]));
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1)
        m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      const bool odd = __any_sync(0xffffffffu, m >= 0x7f80u);   // an infinity or a NaN in some row
      if (odd) {
        m = max(magnitude8_finite(x[i][0]), magnitude8_finite(x[i][1]));
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1)
          m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      }
      const float most = __uint_as_float(m << 16);
      const float s = m == 0 ? 1.f : __fmul_rn(most, kFormat == kCacheInt8 ? 1.0f / 127.0f : 1.0f / 448.0f);
      uint2 q[2];
      if (!odd && s > 0x1p-80f && s < 0x1p100f) {
        const float y = __frcp_rn(s);
        q[0] = quantise8<kFormat>(x[i][0], s, y);
        q[1] = quantise8<kFormat>(x[i][1], s, y);
      } else {
        q[0] = quantise8_any<kFormat>(x[i][0], s);
        q[1] = quantise8_any<kFormat>(x[i][1], s);
      }
      if (r < 2 * hk) {
        uint8_t *to = static_cast<uint8_t *>(r < hk ? a.c.k : a.c.v) + at;
        *reinterpret_cast<uint2 *>(to) = q[0];
        *reinterpret_cast<uint2 *>(to + kLanes * 8) = q[1];
        if (l == 0)
          (r < hk ? k_scale : v_scale)[slot] = s;
      }
    }
  }
}

// The other way: positions 0 .. n-1 of each sequence to packed bf16 rows
// [rows, hk, D], bf16(code * scale).  A position without a page reads as 0.
// HBM-bound; the same tokens back from int8: 36 us, 5790 GB/s.
template <int kFormat, int D>
__global__ void __launch_bounds__(kCacheWarps * 32) cache_read_kernel(const CacheRowsArgs a) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes, kFlight = 4;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = int64_t(blockIdx.x) * kCacheWarps + (threadIdx.x >> 5);
  if (row >= a.rows)
    return;
  const int lane = threadIdx.x & 31, l = lane % kLanes, hk = a.c.hk;
  const int b = sequence_of_warp(a.starts, a.batch, row);
  if (b < 0)
    return;
  const int64_t pos = row - __ldg(a.starts + b);
  const int page = page_of(a.c, b, pos);
  const int64_t in_page = pos & ((1 << a.c.shift) - 1);
  for (int r0 = 0; r0 < 2 * hk; r0 += kRows * kFlight) {
    uint4 x[kFlight];
    float s[kFlight];
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      const int r = r0 + i * kRows + lane / kLanes, head = r < hk ? r : r - hk;
      const int64_t slot = (int64_t(head) << a.c.shift) + in_page;
      const int64_t at = page * (r < hk ? a.c.k_page : a.c.v_page) + slot * D + l * 8;
      x[i] = make_uint4(0, 0, 0, 0);
      s[i] = 0.f;
      if (r < 2 * hk && page >= 0) {
        const void *codes = r < hk ? a.c.k : a.c.v;
        if constexpr (kFormat == kCacheBf16) {
          x[i] = __ldg(reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(codes) + at));
        } else {
          const uint2 q = __ldg(reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(codes) + at));
          x[i].x = q.x, x[i].y = q.y;
          s[i] = __ldg((r < hk ? a.c.ks + page * a.c.ks_page : a.c.vs + page * a.c.vs_page) + slot);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      const int r = r0 + i * kRows + lane / kLanes, head = r < hk ? r : r - hk;
      uint4 y = x[i];
      if constexpr (kFormat != kCacheBf16) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = code_values<kFormat>((e < 2 ? x[i].x : x[i].y) >> ((e & 1) * 16));
          const __nv_bfloat162 h = __floats2bfloat162_rn(__fmul_rn(f.x, s[i]), __fmul_rn(f.y, s[i]));
          w[e] = *reinterpret_cast<const uint32_t *>(&h);
        }
        y = make_uint4(w[0], w[1], w[2], w[3]);
      }
      if (r < 2 * hk)
        *reinterpret_cast<uint4 *>((r < hk ? a.k_out : a.v_out) + (row * hk + head) * D + l * 8) = y;
    }
  }
}

} // namespace pir2b
