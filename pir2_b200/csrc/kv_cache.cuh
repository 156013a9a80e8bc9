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
//
// int4 rows are codes of -7..7, two to a byte (the even channel in the low
// bits, two's complement), an E4M3 factor for every 32 channels and the row's
// fp32 scale: value = code * factor * scale, the first product exact in bf16.
// With m the row's largest finite magnitude, s = 2^(floor(log2 m) - 10), at
// least 2^-126, 1 for a row of zeros; f = E4M3(m_group / s / 7); code = v / s /
// f rounded to nearest even and clamped, 0 where f is 0.  s is a power of two
// so that the quotients are those of numbers of 8 and of 4 bits, which lie on a
// border of the rounding or far from it: any exact division gives these codes.
// m / s is below 2048, so f is below 304.  An infinity counts as m (as 0 where
// no other value but zeros is finite); a row with a NaN gets codes and factors of 0
// and the NaN as its scale.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cstdint>
#include <type_traits>
#include "args.cuh"
#include "attention.cuh"
#include "ptx.cuh"

namespace pir2b {

constexpr int kCacheBf16 = 16, kCacheInt8 = 8, kCacheE4m3 = 9, kCacheInt4 = 24;
constexpr int kFactorGroup = 32;   // channels of an int4 row that share a factor

// Bytes of d channels' codes.
__host__ __device__ constexpr int code_bytes(int format, int d) {
  return format == kCacheBf16 ? 2 * d : format == kCacheInt4 ? d / 2 : d;
}

// Codes of bad device-side indices (a page outside the pool, a position
// outside the table): the access is skipped and the status word records it.
constexpr int kStatusBadPage = 0x201;

__device__ __forceinline__ void record_status(int code) { atomicCAS(&g_device_status, 0, code); }

struct CachePages {
  void *k, *v;             // [pages, hk, page, D] codes
  float *ks, *vs;          // [pages, hk, page] scales (quantised formats)
  uint8_t *kf, *vf;        // [pages, hk, page, D / 32] factors (int4)
  int64_t k_page, v_page;  // elements (int4: bytes) from one page to the next
  int64_t ks_page, vs_page, kf_page, vf_page;
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

// Scale of an int4 row whose largest finite magnitude has the bits m (a bf16's;
// a NaN's give a NaN).
__device__ __forceinline__ float int4_scale(uint32_t m) {
  if (m > 0x7f80u)
    return __uint_as_float(m << 16);
  return m == 0 ? 1.f : __uint_as_float(uint32_t(max(int(m >> 7) - 10, 1)) << 23);
}

// E4M3 factor of a group whose largest magnitude has the bits m, in the low byte.
// (The division as in quotients(): of a bf16 by 7 it is the correctly rounded one.)
__device__ __forceinline__ uint32_t int4_factor(uint32_t m, float inverse) {
  const float x = __uint_as_float(m << 16) * inverse, q = __fmul_rn(x, 1.0f / 7.0f);
  return e4m3_pair(__fmaf_rn(__fmaf_rn(q, -7.f, x), 1.0f / 7.0f, q), 0.f) & 0xffu;
}

__device__ __forceinline__ float e4m3_value(uint32_t code) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(code)));
  return __half2float(__ushort_as_half(uint16_t(h)));
}

// Four finite bf16 -> four 4-bit codes.  quotients() is exact here: all 2^10
// pairs of significands give the integer of the true quotient (a test compares
// them).  A pair of codes, 8 added to each, is one small number's low byte.
__device__ __forceinline__ uint32_t quantise4_int4(uint32_t x, uint32_t y, float inverse, float f) {
  const float rf = f == 0.f ? 0.f : __frcp_rn(f);
  const float2 inv = make_float2(inverse, inverse), minus_f = make_float2(-f, -f), rr = make_float2(rf, rf);
  uint32_t pair[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float2 q = quotients(__fmul2_rn(bf16_pair(i ? y : x), inv), minus_f, rr);
    q.x = fminf(fmaxf(q.x, -7.f), 7.f), q.y = fminf(fmaxf(q.y, -7.f), 7.f);
    // 1.5 * 2^23 + 8: rounds to an integer, to even as it is even itself.
    q = __fadd2_rn(__fadd2_rn(q, make_float2(12582920.f, 12582920.f)), make_float2(-12582912.f, -12582912.f));
    pair[i] = __float_as_uint(__fmaf_rn(q.y, 16.f, q.x) + 12582912.f);
  }
  return (__byte_perm(pair[0], pair[1], 0x0040) & 0xffffu) ^ 0x8888u;
}

// The same for a row of ordinary scale and a group of ordinary factor (or none but
// zeros), where no code passes 7 before it is rounded: straight by the product fs
// of the two, with an approximate reciprocal, which quotients() makes up for (a
// test takes reciprocals off by three places).
__device__ __forceinline__ bool int4_ordinary(uint32_t factor) { return factor == 0 || factor >= 8; }   // E4M3's subnormal ones are below 8

__device__ __forceinline__ float reciprocal_of_factor(float fs) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fs));
  return fs == 0.f ? 0.f : y;
}

__device__ __forceinline__ uint32_t ordinary8_int4(const uint4 &x, float fs, float r) {
  const float2 minus = make_float2(-fs, -fs), rr = make_float2(r, r), up = make_float2(12582920.f, 12582920.f);
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t pair[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 q = __fadd2_rn(quotients(bf16_pair(w[i]), minus, rr), up);
    pair[i] = (__float_as_uint(q.y) << 4) + __float_as_uint(q.x);
  }
  return __byte_perm(__byte_perm(pair[0], pair[1], 0x0040), __byte_perm(pair[2], pair[3], 0x0040), 0x5410) ^ 0x88888888u;
}

// Infinities of a piece as the magnitude m with their sign.
__device__ __noinline__ uint4 bounded8(uint4 x, uint32_t m) {
  uint32_t w[4] = {x.x, x.y, x.z, x.w};
  for (int i = 0; i < 8; ++i) {
    const int at = (i & 1) * 16;
    if (((w[i >> 1] >> at) & 0x7fffu) == 0x7f80u)
      w[i >> 1] = (w[i >> 1] & ~(0x7fffu << at)) | (m << at);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Eight 4-bit codes times their factor as fp32 values.
__device__ __forceinline__ void int4_values(uint32_t w, float f, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    v[i] = float(int32_t(w << (28 - 4 * i)) >> 28) * f;
}

__device__ __forceinline__ uint32_t bf162_fma(uint32_t x, uint32_t y, uint32_t z) {
  uint32_t w;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(w) : "r"(x), "r"(y), "r"(z));
  return w;
}

// Places kAt and kAt + 4 of a word's codes times f: a nibble t (two's complement, t
// = u ^ 8 with u = code + 8) in bits 3-6 of a bf16 16 makes 16 + u, and an FMA takes
// 24 f away.
template <int kAt>
__device__ __forceinline__ uint32_t int4_pair_bf16(uint32_t w, uint32_t f, uint32_t minus_24f) {
  const uint32_t t = kAt == 0 ? w << 3 : w >> (kAt == 0 ? 0 : 4 * kAt - 3);
  return bf162_fma((t & 0x00780078u) ^ 0x41c041c0u, f, minus_24f);
}

// Eight codes times f in order, exact where f is a number of four bits far from
// bf16's limits.
__device__ __forceinline__ uint4 int4_to_bf16x8(uint32_t w, float f) {
  const uint32_t ff = pack_bf16x2(f, f), m = pack_bf16x2(-24.f * f, -24.f * f);
  const uint32_t p0 = int4_pair_bf16<0>(w, ff, m), p1 = int4_pair_bf16<1>(w, ff, m);
  const uint32_t p2 = int4_pair_bf16<2>(w, ff, m), p3 = int4_pair_bf16<3>(w, ff, m);
  return make_uint4(__byte_perm(p0, p1, 0x5410), __byte_perm(p2, p3, 0x5410), __byte_perm(p0, p1, 0x7632), __byte_perm(p2, p3, 0x7632));
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

// What keep_row needs of rows with an infinity or a NaN among them, and of groups
// with small factors: out of the way of the others.
struct BoundedRow {
  uint4 x0, x1;
  uint32_t m, mg;       // largest finite magnitude (or a NaN's), the groups'
};

template <int kLanes>
__device__ __noinline__ BoundedRow bounded_row(uint4 x0, uint4 x1) {
  uint32_t m = max(magnitude8_finite(x0), magnitude8_finite(x1));
  for (int o = kLanes / 2; o > 0; o >>= 1)
    m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (m > 0x7f80u)
    x0 = x1 = make_uint4(0, 0, 0, 0);
  x0 = bounded8(x0, m), x1 = bounded8(x1, m);
  uint32_t mg = magnitude8(x0) | (magnitude8(x1) << 16);
  mg = __vmaxu2(mg, __shfl_xor_sync(0xffffffffu, mg, 1));
  mg = __vmaxu2(mg, __shfl_xor_sync(0xffffffffu, mg, 2));
  return {x0, x1, m, mg};
}

__device__ __noinline__ uint32_t quantise8_int4_any(uint4 x, float inverse, float f) {
  return quantise4_int4(x.x, x.y, inverse, f) | (quantise4_int4(x.z, x.w, inverse, f) << 16);
}

// A row to its slot: D / 16 lanes of it with 16 bytes of either half each (x0 from
// l * 8 on, x1 from D / 2 + l * 8 on); `codes`, `factors` and `scale` are the lane's
// places.  All lanes of the warp come here.
template <int kFormat, int D>
__device__ __forceinline__ void keep_row(uint4 x0, uint4 x1, int l, bool kept, uint8_t *codes, uint8_t *factors, float *scale) {
  constexpr int kLanes = D / 16;
  if constexpr (kFormat == kCacheBf16) {
    if (kept) {
      *reinterpret_cast<uint4 *>(codes) = x0;
      *reinterpret_cast<uint4 *>(codes + D) = x1;
    }
    return;
  }
  const uint32_t m0 = magnitude8(x0), m1 = magnitude8(x1);
  if constexpr (kFormat == kCacheInt4) {
    // Four lanes' pieces are a group; the halves of a word are the two groups'.
    uint32_t mg = m0 | (m1 << 16);
    mg = __vmaxu2(mg, __shfl_xor_sync(0xffffffffu, mg, 1));
    mg = __vmaxu2(mg, __shfl_xor_sync(0xffffffffu, mg, 2));
    uint32_t m = max(mg & 0xffffu, mg >> 16);
    if (kLanes == 8)
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 4));
    if (__any_sync(0xffffffffu, m >= 0x7f80u)) {      // an infinity or a NaN in some row
      const BoundedRow bounded = bounded_row<kLanes>(x0, x1);
      x0 = bounded.x0, x1 = bounded.x1, m = bounded.m, mg = bounded.mg;
    }
    const float s = int4_scale(m), inverse = m > 0x7f80u ? 1.f : __uint_as_float(0x7f000000u - __float_as_uint(s));   // 1 / s
    // Two lanes of a group make its first factor, two its second.
    const uint32_t mine = int4_factor(l & 2 ? mg >> 16 : mg & 0xffffu, inverse);
    const uint32_t other = __shfl_xor_sync(0xffffffffu, mine, 2);
    const uint32_t f0 = l & 2 ? other : mine, f1 = l & 2 ? mine : other;
    const float a = e4m3_value(f0), b = e4m3_value(f1);
    uint32_t q0, q1;
    if (__all_sync(0xffffffffu, s >= 0x1p-100f && int4_ordinary(f0) && int4_ordinary(f1))) {
      const float as = a * s, bs = b * s, ra = reciprocal_of_factor(as), rb = reciprocal_of_factor(bs);
      q0 = ordinary8_int4(x0, as, ra);
      q1 = ordinary8_int4(x1, bs, rb);
    } else {
      q0 = quantise8_int4_any(x0, inverse, a);
      q1 = quantise8_int4_any(x1, inverse, b);
    }
    if (kept) {
      *reinterpret_cast<uint32_t *>(codes) = q0;
      *reinterpret_cast<uint32_t *>(codes + D / 4) = q1;
      if ((l & 1) == 0)                               // two lanes of a group, one factor each
        factors[l & 2 ? D / 2 / kFactorGroup : 0] = uint8_t(mine);
      if (l == 0)
        *scale = s;
    }
  } else {
    uint32_t m = max(m0, m1);
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1)
      m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const bool odd = __any_sync(0xffffffffu, m >= 0x7f80u);   // an infinity or a NaN in some row
    if (odd) {
      m = max(magnitude8_finite(x0), magnitude8_finite(x1));
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1)
        m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    }
    const float most = __uint_as_float(m << 16);
    const float s = m == 0 ? 1.f : __fmul_rn(most, kFormat == kCacheInt8 ? 1.0f / 127.0f : 1.0f / 448.0f);
    uint2 q[2];
    if (!odd && s > 0x1p-80f && s < 0x1p100f) {
      const float y = __frcp_rn(s);
      q[0] = quantise8<kFormat>(x0, s, y);
      q[1] = quantise8<kFormat>(x1, s, y);
    } else {
      q[0] = quantise8_any<kFormat>(x0, s);
      q[1] = quantise8_any<kFormat>(x1, s);
    }
    if (kept) {
      *reinterpret_cast<uint2 *>(codes) = q[0];
      *reinterpret_cast<uint2 *>(codes + D / 2) = q[1];
      if (l == 0)
        *scale = s;
    }
  }
}

constexpr int kCacheWarps = 4;

// A warp per token and 32 kFlight / (D / 16) of its (head, k or v) rows: D / 16
// lanes per row, each with two 16-byte pieces of it, 2 kFlight loads in flight;
// the row maximum comes by shuffles.  HBM-bound in bytes (2 D in, D + 4 out per
// row of an 8-bit cache), but instructions for the scale of a row weigh as
// much, so a lane takes as many of its values as keeps the loads coalesced.
// 33910 tokens of 8 kv heads of 128 to int8: 38 us, 5520 GB/s, 84 % of a copy's
// rate, 2.8 instructions a cycle and SM.  To int4 45 us (bytes 27), to bf16 46 (42).
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
  constexpr int kUnit = kFormat == kCacheBf16 ? 2 : 1;       // bytes that page strides count
  const int64_t k_at = int64_t(kUnit) * page * a.c.k_page, v_at = int64_t(kUnit) * page * a.c.v_page;
  float *k_scale = a.c.ks + page * a.c.ks_page, *v_scale = a.c.vs + page * a.c.vs_page;
#pragma unroll
  for (int i = 0; i < kFlight; ++i) {
    const int r = r0 + i * kRows, head = r < hk ? r : r - hk;
    const int slot = (head << a.c.shift) + in_page;          // below 2^17
    uint8_t *codes = static_cast<uint8_t *>(r < hk ? a.c.k : a.c.v) +
                     ((r < hk ? k_at : v_at) + (slot * code_bytes(kFormat, D) + l * code_bytes(kFormat, 8)));
    uint8_t *factor = nullptr;
    if constexpr (kFormat == kCacheInt4)
      factor = (r < hk ? a.c.kf + page * a.c.kf_page : a.c.vf + page * a.c.vf_page) + slot * (D / kFactorGroup) + l / 4;
    keep_row<kFormat, D>(x[i][0], x[i][1], l, r < 2 * hk, codes, factor, (r < hk ? k_scale : v_scale) + slot);
  }
}

// Position of a new token outside the rotation's table.
constexpr int kStatusBadPosition = 0x202;

struct CacheAppendArgs {
  CachePages c;
  const __nv_bfloat16 *qkv;      // [rows, hq + 2 hk, D] view
  int64_t row, head;
  const __nv_bfloat16 *q_weight, *k_weight;   // [D] of the heads' norms, or null
  float eps;
  const float *cos, *sin;        // [turns, D / 2]
  int64_t turns;
  const int *positions;          // [rows] rows of the table, or null: positions in the cache
  __nv_bfloat16 *q_out, *k_out;  // [rows, hq, D], [rows, hk, D] or null
  int64_t q_row, k_row;
  const int *starts, *lengths;
  int batch, hq;
  int64_t rows;
};

// Norm, rotation and cache write of new tokens in one pass: for each head row x
// of q and k
//   y = x / sqrt(mean x^2 + eps) w            (where there is a weight)
//   z = (y_a cos - y_b sin, y_b cos + y_a sin), a and b the halves of the head,
// in fp32, each operation rounded by itself (no contraction: the values next to
// borders of codes are then those of the same operations anywhere else), the
// squares added within a lane, then by halves of the lanes.  z is rounded to
// bf16; q leaves in it, and k and v are quantised from it as cache_write does.
//
// D / 16 lanes per head row, each with eight channels of either half, so that a
// rotation's pairs meet in a lane; a warp per token takes kFlight passes over 32 /
// (D / 16) head rows each at a time, the first loaded before the token's place is
// known, first of q, then of k and v.  (With few tokens blockIdx.y names the
// passes that a warp takes.)  The square root and division of kFlight passes'
// norms are made at once, each in lanes of its own.
//
// 64 prompts of 280-816 tokens, 16 query and 8 kv heads of 128: to int4 pages 110 us
// (int8 99, E4M3 101, bf16 89), of which bytes take 70.  The schedulers issue in 67 %
// of the cycles; of the time of the 19 warps of an SM 24 % goes to the result before,
// 16 % to loads, 16 % to other warps' turns and 10 % to busy math pipes.  Five CTAs of
// 96 registers spill 8 to 36 bytes of each thread.  With 16 channels in a row per lane, which hands half of them to a partner
// for the rotation, and codes by exact reciprocals, this and the read back took 194
// us together, now 143; rows asked into L2 before the token's place is known are 2 of
// that.
template <int kFormat, int D, int kFlight>
__global__ void __launch_bounds__(kCacheWarps * 32, 5) cache_append_kernel(const CacheAppendArgs a) {
  constexpr int kLanes = D / 16, kRows = 32 / kLanes, kTaken = kRows * kFlight;
  static_assert(kFlight <= kLanes);
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = int64_t(blockIdx.x) * kCacheWarps + (threadIdx.x >> 5);
  if (row >= a.rows)
    return;
  const int lane = threadIdx.x & 31, l = lane % kLanes, of = lane / kLanes, hk = a.c.hk;
  const __nv_bfloat16 *source = a.qkv + row * a.row + of * a.head + l * 8;
  const int64_t apart = kRows * a.head;              // from pass to pass
  // The rows of kFlight passes from head `first` of `heads` on.
  auto fetch = [&](const __nv_bfloat16 *from, int first, int heads, uint4 (&x)[kFlight][2]) {
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      x[i][0] = x[i][1] = make_uint4(0, 0, 0, 0);
      if (first + i * kRows + of < heads) {
        const uint4 *src = reinterpret_cast<const uint4 *>(from + i * apart);
        x[i][0] = *src;
        x[i][1] = src[D / 16];
      }
    }
  };
  // This warp's passes: all, or those of one kFlight of one kind.
  int kind = 0, begin = 0, stop = 3;
  bool one = false;
  if (gridDim.y > 1) {
    const int q_parts = (a.hq + kTaken - 1) / kTaken, kv_parts = (hk + kTaken - 1) / kTaken, part = blockIdx.y;
    kind = part < q_parts ? 0 : part < q_parts + kv_parts ? 1 : 2;
    begin = (part - (kind == 0 ? 0 : kind == 1 ? q_parts : q_parts + kv_parts)) * kTaken;
    stop = kind + 1;
    one = true;
  }
  auto start_of = [&](int which, int first) { return source + int64_t((which == 0 ? 0 : which == 1 ? a.hq : a.hq + hk) + first) * a.head; };
  uint4 x[kFlight][2];
  fetch(start_of(kind, begin), begin, kind == 0 ? a.hq : hk, x);
  if (!one)                                           // the rest of the token's rows on their way to L2
    for (int head = lane; head < a.hq + 2 * hk; head += 32) {
      const __nv_bfloat16 *at = a.qkv + row * a.row + head * a.head;
      asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
      if (D == 128)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(at + 64));
    }
  const int b = sequence_of_warp(a.starts, a.batch, row);
  if (b < 0)
    return;
  const int64_t pos = int64_t(__ldg(a.lengths + b)) - __ldg(a.starts + b + 1) + row;
  int64_t turn = a.positions ? int64_t(__ldg(a.positions + row)) : pos;
  const bool turned = turn >= 0 && turn < a.turns;
  if (!turned) {
    record_status(kStatusBadPosition);
    turn = 0;
  }
  float2 cos[4], sin[4];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float4 c = __ldg(reinterpret_cast<const float4 *>(a.cos + turn * (D / 2)) + 2 * l + j);
    const float4 s = __ldg(reinterpret_cast<const float4 *>(a.sin + turn * (D / 2)) + 2 * l + j);
    cos[2 * j] = make_float2(c.x, c.y), cos[2 * j + 1] = make_float2(c.z, c.w);
    sin[2 * j] = make_float2(s.x, s.y), sin[2 * j + 1] = make_float2(s.z, s.w);
  }
  const int found = turned ? page_of(a.c, b, pos) : -1;
  const int64_t page = max(found, 0);
  const int in_page = int(pos & ((1 << a.c.shift) - 1));

  // All passes of one kind: 0 q, 1 k, 2 v.
  auto take = [&](auto which) {
    constexpr int kKind = which.value;
    constexpr bool kTurned = kKind < 2, kKept = kKind > 0;
    const int heads = kKind == 0 ? a.hq : hk;
    // This lane's places for head `begin + of`, and from pass to pass.
    const int slot = ((begin + of) << a.c.shift) + in_page, slots = kRows << a.c.shift;
    uint8_t *codes = nullptr, *factors = nullptr;
    float *scales = nullptr;
    if constexpr (kKept) {
      codes = static_cast<uint8_t *>(kKind == 1 ? a.c.k : a.c.v) +
              (kFormat == kCacheBf16 ? 2 : 1) * page * (kKind == 1 ? a.c.k_page : a.c.v_page) +
              int64_t(slot) * code_bytes(kFormat, D) + l * code_bytes(kFormat, 8);
      if constexpr (kFormat != kCacheBf16)
        scales = (kKind == 1 ? a.c.ks + page * a.c.ks_page : a.c.vs + page * a.c.vs_page) + slot;
      if constexpr (kFormat == kCacheInt4)
        factors = (kKind == 1 ? a.c.kf + page * a.c.kf_page : a.c.vf + page * a.c.vf_page) + slot * (D / kFactorGroup) + l / 4;
    }
    __nv_bfloat16 *out = nullptr;
    if constexpr (kTurned) {
      out = kKind == 0 ? a.q_out + row * a.q_row : a.k_out == nullptr ? nullptr : a.k_out + row * a.k_row;
      if (out != nullptr)
        out += (begin + of) * D + l * 8;
    }
    const __nv_bfloat16 *weight = kKind == 0 ? a.q_weight : kKind == 1 ? a.k_weight : nullptr;
    uint4 wl, wh;
    if (kTurned && weight != nullptr) {
      wl = __ldg(reinterpret_cast<const uint4 *>(weight) + l), wh = __ldg(reinterpret_cast<const uint4 *>(weight) + l + D / 16);
    }
    const __nv_bfloat16 *from = start_of(kKind, begin);
    for (int first = begin;;) {
      float inverse[kFlight];
      if (kTurned && weight != nullptr) {
        float mine = 0.f;
#pragma unroll
        for (int i = 0; i < kFlight; ++i) {
          // Sums of four channels and their partners, two of them per lane.
          auto sum_of = [&](uint32_t p0, uint32_t p1, uint32_t q0, uint32_t q1) {
            const float2 u0 = bf16_pair(p0), u1 = bf16_pair(p1), v0 = bf16_pair(q0), v1 = bf16_pair(q1);
            const float2 p = __fadd2_rn(__fmul2_rn(u0, u0), __fmul2_rn(v0, v0)), q = __fadd2_rn(__fmul2_rn(u1, u1), __fmul2_rn(v1, v1));
            const float2 pq = __fadd2_rn(p, q);
            return __fadd_rn(pq.x, pq.y);
          };
          float s0 = sum_of(x[i][0].x, x[i][0].y, x[i][1].x, x[i][1].y), s1 = sum_of(x[i][0].z, x[i][0].w, x[i][1].z, x[i][1].w);
#pragma unroll
          for (int o = kLanes / 2; o > 0; o >>= 1) {
            s0 = __fadd_rn(s0, __shfl_xor_sync(0xffffffffu, s0, o));
            s1 = __fadd_rn(s1, __shfl_xor_sync(0xffffffffu, s1, o));
          }
          mine = l % kFlight == i ? __fadd_rn(s0, s1) : mine;
        }
        mine = __fdiv_rn(1.f, __fsqrt_rn(__fadd_rn(mine * (1.f / D), a.eps)));
#pragma unroll
        for (int i = 0; i < kFlight; ++i)
          inverse[i] = __shfl_sync(0xffffffffu, mine, of * kLanes + i);
      }
#pragma unroll
      for (int i = 0; i < kFlight; ++i) {
        if (first + i * kRows >= heads)
          break;
        const bool there = first + i * kRows + of < heads;
        uint4 y0 = x[i][0], y1 = x[i][1];
        if constexpr (kTurned) {
          const uint32_t lo[4] = {y0.x, y0.y, y0.z, y0.w}, hi[4] = {y1.x, y1.y, y1.z, y1.w};
          const uint32_t wlo[4] = {wl.x, wl.y, wl.z, wl.w}, whi[4] = {wh.x, wh.y, wh.z, wh.w};
          uint32_t z[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float2 u = bf16_pair(lo[j]), v = bf16_pair(hi[j]);
            if (weight != nullptr) {
              const float2 inv2 = make_float2(inverse[i], inverse[i]);
              u = __fmul2_rn(__fmul2_rn(u, inv2), bf16_pair(wlo[j]));
              v = __fmul2_rn(__fmul2_rn(v, inv2), bf16_pair(whi[j]));
            }
            // Single sums: a pair's would be joined with the products into FMAs.
            const float2 uc = __fmul2_rn(u, cos[j]), vs = __fmul2_rn(v, sin[j]);
            const float2 vc = __fmul2_rn(v, cos[j]), us = __fmul2_rn(u, sin[j]);
            z[j] = pack_bf16x2(__fsub_rn(uc.x, vs.x), __fsub_rn(uc.y, vs.y));
            z[4 + j] = pack_bf16x2(__fadd_rn(vc.x, us.x), __fadd_rn(vc.y, us.y));
          }
          y0 = make_uint4(z[0], z[1], z[2], z[3]), y1 = make_uint4(z[4], z[5], z[6], z[7]);
          if (there && (kKind == 0 || out != nullptr)) {
            *reinterpret_cast<uint4 *>(out) = y0;
            *reinterpret_cast<uint4 *>(out + D / 2) = y1;
          }
          out = kKind == 0 || out != nullptr ? out + kRows * D : out;
        }
        if constexpr (kKept) {
          keep_row<kFormat, D>(y0, y1, l, there && found >= 0, codes, factors, scales);
          codes += slots * code_bytes(kFormat, D);
          factors += slots * (D / kFactorGroup);
          scales += slots;
        }
      }
      first += kTaken;
      if (one || first >= heads)
        break;
      from += kFlight * apart;
      fetch(from, first, heads, x);
    }
  };
  for (; kind < stop; ++kind) {
    if (kind == 0)
      take(std::integral_constant<int, 0>{});
    else if (kind == 1)
      take(std::integral_constant<int, 1>{});
    else
      take(std::integral_constant<int, 2>{});
    if (kind + 1 < stop)
      fetch(start_of(kind + 1, 0), 0, hk, x);
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

// The same of int4 pages: D / 16 lanes per row with eight channels of either half
// each (so that stores of a row lie side by side), k and v at once.  The same 64
// prompts back: 33 us, of which 27 are bytes, most of them the bf16 rows that leave.
template <int D>
__global__ void __launch_bounds__(kCacheWarps * 32) cache_read_int4_kernel(const CacheRowsArgs a) {
  constexpr int kLanes = D / 16, kRows = 32 / kLanes;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = int64_t(blockIdx.x) * kCacheWarps + (threadIdx.x >> 5);
  if (row >= a.rows)
    return;
  const int lane = threadIdx.x & 31, l = lane % kLanes, of = lane / kLanes, hk = a.c.hk;
  const int b = sequence_of_warp(a.starts, a.batch, row);
  if (b < 0)
    return;
  const int64_t pos = row - __ldg(a.starts + b);
  const int found = page_of(a.c, b, pos);
  const int64_t page = max(found, 0);
  // This lane's places, of k and of v, and from pass to pass.
  const int slot = (of << a.c.shift) + int(pos & ((1 << a.c.shift) - 1)), slots = kRows << a.c.shift;
  const uint8_t *codes[2] = {static_cast<const uint8_t *>(a.c.k) + page * a.c.k_page + slot * (D / 2) + l * 4,
                             static_cast<const uint8_t *>(a.c.v) + page * a.c.v_page + slot * (D / 2) + l * 4};
  const uint8_t *factors[2] = {a.c.kf + page * a.c.kf_page + slot * (D / kFactorGroup) + l / 4,
                               a.c.vf + page * a.c.vf_page + slot * (D / kFactorGroup) + l / 4};
  const float *scales[2] = {a.c.ks + page * a.c.ks_page + slot, a.c.vs + page * a.c.vs_page + slot};
  __nv_bfloat16 *out[2] = {a.k_out + (row * hk + of) * D + l * 8, a.v_out + (row * hk + of) * D + l * 8};
  for (int head = of; head - of < hk; head += kRows) {
    const bool there = head < hk;
    uint32_t x[2][2], f8[2][2];
    float s[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x[i][0] = x[i][1] = f8[i][0] = f8[i][1] = 0;
      s[i] = 0.f;
      if (there && found >= 0) {
        x[i][0] = __ldg(reinterpret_cast<const uint32_t *>(codes[i]));
        x[i][1] = __ldg(reinterpret_cast<const uint32_t *>(codes[i] + D / 4));
        f8[i][0] = __ldg(factors[i]), f8[i][1] = __ldg(factors[i] + D / 2 / kFactorGroup);
        s[i] = __ldg(scales[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint4 y[2];
      const float f[2] = {e4m3_value(f8[i][0]), e4m3_value(f8[i][1])};
      // A power of two (or 0), as cache_write makes them, changes no bits of the products.
      if (__all_sync(0xffffffffu, (__float_as_uint(s[i]) & 0x807fffffu) == 0 && s[i] < 0x1p100f && (s[i] == 0.f || s[i] > 0x1p-100f) &&
                                      f[0] == f[0] && f[1] == f[1])) {
        y[0] = int4_to_bf16x8(x[i][0], f[0] * s[i]);
        y[1] = int4_to_bf16x8(x[i][1], f[1] * s[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float v[8];
          int4_values(x[i][j], f[j], v);
          y[j] = make_uint4(pack_bf16x2(v[0] * s[i], v[1] * s[i]), pack_bf16x2(v[2] * s[i], v[3] * s[i]),
                            pack_bf16x2(v[4] * s[i], v[5] * s[i]), pack_bf16x2(v[6] * s[i], v[7] * s[i]));
        }
      }
      if (there) {
        *reinterpret_cast<uint4 *>(out[i]) = y[0];
        *reinterpret_cast<uint4 *>(out[i] + D / 2) = y[1];
      }
      codes[i] += slots * (D / 2), factors[i] += slots * (D / kFactorGroup), scales[i] += slots, out[i] += kRows * D;
    }
  }
}

} // namespace pir2b
