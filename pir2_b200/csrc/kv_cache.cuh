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

__device__ __forceinline__ float max_nan(float x, float y) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(x), "f"(y));
  return m;
}

// Largest |value| of eight bf16, infinities aside; a NaN where one is.
__device__ __forceinline__ float row_max8(const uint4 &x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float lo = fabsf(__uint_as_float(w[i] << 16)), hi = fabsf(__uint_as_float(w[i] & 0xffff0000u));
    m = max_nan(m, lo == INFINITY ? 0.f : lo);
    m = max_nan(m, hi == INFINITY ? 0.f : hi);
  }
  return m;
}

// Eight bf16 -> eight codes under scale s (0 under a NaN).
template <int kFormat>
__device__ __forceinline__ uint2 quantise8(const uint4 &x, float s) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t out[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo = __fdiv_rn(__uint_as_float(w[i] << 16), s);
    float hi = __fdiv_rn(__uint_as_float(w[i] & 0xffff0000u), s);
    lo = lo != lo ? 0.f : lo;
    hi = hi != hi ? 0.f : hi;
    uint32_t pair;
    if constexpr (kFormat == kCacheInt8) {
      const int a = __float2int_rn(fminf(fmaxf(lo, -127.f), 127.f));
      const int b = __float2int_rn(fminf(fmaxf(hi, -127.f), 127.f));
      pair = (uint32_t(a) & 0xffu) | ((uint32_t(b) & 0xffu) << 8);
    } else {
      uint16_t e;
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(e) : "f"(hi), "f"(lo));
      pair = e;
    }
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

constexpr int kCacheThreads = 256;

// One group of D / 8 lanes per (row, head, k or v): a 16-byte load per lane,
// the row maximum by shuffles inside the group, an 8-byte store per lane.
// HBM-bound: 2 D bytes in, D + 4 out per row of an 8-bit cache.
template <int kFormat, int D>
__global__ void __launch_bounds__(kCacheThreads) cache_write_kernel(const CacheRowsArgs a) {
  constexpr int kLanes = D / 8;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t item = (int64_t(blockIdx.x) * kCacheThreads + threadIdx.x) / kLanes;
  const int l = threadIdx.x % kLanes;
  const int hk = a.c.hk;
  const int64_t row = item / (2 * hk);
  const int which = int(item % (2 * hk)) / hk, head = int(item % hk);   // k rows of all heads, then v rows
  const bool active = row < a.rows;
  int page = -1;
  int64_t pos = 0;
  if (active) {
    const int b = sequence_of(a.starts, a.batch, row);
    if (b >= 0) {
      pos = int64_t(__ldg(a.lengths + b)) - __ldg(a.starts + b + 1) + row;
      page = page_of(a.c, b, pos);
    }
  }
  uint4 x = make_uint4(0, 0, 0, 0);
  if (page >= 0) {
    const __nv_bfloat16 *src = which ? a.v + row * a.v_row + head * a.v_head : a.k + row * a.k_row + head * a.k_head;
    x = *reinterpret_cast<const uint4 *>(src + l * 8);
  }
  const int64_t slot = (int64_t(head) << a.c.shift) + (pos & ((1 << a.c.shift) - 1));
  const int64_t at = int64_t(page) * (which ? a.c.v_page : a.c.k_page) + slot * D + l * 8;
  void *codes = which ? a.c.v : a.c.k;
  if constexpr (kFormat == kCacheBf16) {
    if (page >= 0)
      *reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(codes) + at) = x;
  } else {
    float m = row_max8(x);
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1)
      m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float s = m == 0.f ? 1.f : __fmul_rn(m, kFormat == kCacheInt8 ? 1.0f / 127.0f : 1.0f / 448.0f);
    if (page >= 0) {
      *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(codes) + at) = quantise8<kFormat>(x, s);
      if (l == 0)
        (which ? a.c.vs + page * a.c.vs_page : a.c.ks + page * a.c.ks_page)[slot] = s;
    }
  }
}

// The other way: positions 0 .. n-1 of each sequence to packed bf16 rows
// [rows, hk, D], bf16(code * scale).  A position without a page reads as 0.
template <int kFormat, int D>
__global__ void __launch_bounds__(kCacheThreads) cache_read_kernel(const CacheRowsArgs a) {
  constexpr int kLanes = D / 8;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t item = (int64_t(blockIdx.x) * kCacheThreads + threadIdx.x) / kLanes;
  const int l = threadIdx.x % kLanes;
  const int hk = a.c.hk;
  const int64_t row = item / (2 * hk);
  const int which = int(item % (2 * hk)) / hk, head = int(item % hk);
  if (row >= a.rows)
    return;
  const int b = sequence_of(a.starts, a.batch, row);
  if (b < 0)
    return;
  const int64_t pos = row - __ldg(a.starts + b);
  const int page = page_of(a.c, b, pos);
  uint4 y = make_uint4(0, 0, 0, 0);
  if (page >= 0) {
    const int64_t slot = (int64_t(head) << a.c.shift) + (pos & ((1 << a.c.shift) - 1));
    const int64_t at = int64_t(page) * (which ? a.c.v_page : a.c.k_page) + slot * D + l * 8;
    const void *codes = which ? a.c.v : a.c.k;
    if constexpr (kFormat == kCacheBf16) {
      y = *reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(codes) + at);
    } else {
      const uint2 q = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(codes) + at);
      const float s = which ? a.c.vs[page * a.c.vs_page + slot] : a.c.ks[page * a.c.ks_page + slot];
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = code_values<kFormat>((i < 2 ? q.x : q.y) >> ((i & 1) * 16));
        const __nv_bfloat162 h = __floats2bfloat162_rn(__fmul_rn(f.x, s), __fmul_rn(f.y, s));
        w[i] = *reinterpret_cast<const uint32_t *>(&h);
      }
      y = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  *reinterpret_cast<uint4 *>((which ? a.v_out : a.k_out) + (row * hk + head) * D + l * 8) = y;
}

} // namespace pir2b
