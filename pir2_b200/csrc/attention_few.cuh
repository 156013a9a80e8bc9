// Attention of a few new rows per sequence over the paged K/V cache.
//
// A unit is up to 8 kNT rows (query token x head of one kv head's group) of
// one sequence; a CTA streams a range of the unit's keys once, four warps
// taking 16-key steps in turn.  Few rows cannot fill a 128-row tensor tile
// and the work is reading the cache, so the products run on warp-level MMAs
// (m16n8k16, fp32 sums) with the keys as the M rows:
//   S^T [16 keys x 8 rows]  = K [16 x D] Q^T,
//   O^T [D x 8 rows]       += V^T [D x 16 keys] P^T.
// Each warp has a ring of its own: its first lane keeps the TMA copies of the
// next steps in flight, and all lanes read the step at hand into MMA
// fragments.  Which key is which M row, and the order of D inside a product,
// are free: each lane takes whole 16-byte pieces, and rows are dealt so that
// the swizzled tiles are read without bank conflicts.  8-bit codes become fp16
// (K, the cheaper conversion; q is scaled to fit) and bf16 (V: the weights need
// its range) exactly in registers; the scales multiply scores and weights in
// fp32.  P is transposed between the products by movmatrix.  The running maximum of a row
// moves only when a score passes it by more than 8 (in log2), so that most
// steps have one vote and no rescaling; sums and maxima are fp32.  The weights, times
// V's scales, are rounded to bf16 for their product (error against 64 bits 0.0018 to
// 0.0023 of the result, with weights in fp32 0.0017, bf16's own rounding): a second
// product for what the rounding leaves would double V's MMAs.
//
// What bounds it, one new token per sequence, 16 query and 8 kv heads of 128,
// replayed from a graph (called in a loop): bf16 over four histories of
// 29000-32700, 85 us (87), 6150 GB/s, 94 % of a copy's rate.  int8 over 64
// histories of 500-4000, 62 us (65), 4710 GB/s: instructions, a third of them the
// conversion of codes, which no warp-level MMA takes beside 16-bit weights.  int4
// over the same, 47 us (48), 23 of them bytes: 391 instructions per 16 keys and a
// quarter as many at starts and ends issue in 54 % of the cycles; for 14 % of the time
// an SM has no CTA yet or none any more; in the rest its 15 warps all wait, for a busy
// math pipe or its dispatch (24 % of a warp's time), for the result before (17 %), at
// barriers and for loads (6 % each).  Its steps are of 32 keys, whose six small pieces all lanes copy by 16 bytes (copies of
// one lane in bulk: 67 us), with the hidden positions' steps apart; q's fragments
// are read from shared memory, for which four CTAs of 128 registers stay on an SM
// (three, with q in registers: four histories of 29000-32700 42 us for 45, the 64
// histories 55 for 47).
#pragma once
#include <cuda.h>
#include <type_traits>
#include "attention_ragged.cuh"

namespace pir2b {

constexpr int kFewWarps = 4;

// Two bf16 pairs from a word of four 8-bit codes, exactly.
// int8: with u the low seven bits and s the sign bit of a byte, 0x43'u is
// 128 + u and 0x43's0 is 128 or 256, so their difference is u - 128 s.
// E4M3: sign and magnitude bits moved to bf16's places hold value * 2^-120
// (subnormals included).  The pool holds no E4M3 NaN (cache_write puts a NaN
// into the scale).
template <int kFormat>
__device__ __forceinline__ void codes_to_bf16(uint32_t w, uint32_t &lo, uint32_t &hi) {
  auto sub = [](uint32_t x, uint32_t y) {
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<__nv_bfloat162 *>(&x), *reinterpret_cast<__nv_bfloat162 *>(&y));
    return *reinterpret_cast<const uint32_t *>(&d);
  };
  if constexpr (kFormat == kCacheInt8) {
    const uint32_t a = __byte_perm(w, 0x43434343u, 0x4140), b = __byte_perm(w, 0x43434343u, 0x4342);
    lo = sub(a & 0xff7fff7fu, a & 0xff80ff80u);
    hi = sub(b & 0xff7fff7fu, b & 0xff80ff80u);
  } else {
    const __nv_bfloat162 up = __halves2bfloat162(__ushort_as_bfloat16(0x7b80), __ushort_as_bfloat16(0x7b80));  // 2^120
    const uint32_t a = __byte_perm(w, 0, 0x1404), b = __byte_perm(w, 0, 0x3424);
    uint32_t x = (a & 0x80008000u) | ((a & 0x7f007f00u) >> 4), y = (b & 0x80008000u) | ((b & 0x7f007f00u) >> 4);
    const __nv_bfloat162 m = __hmul2(*reinterpret_cast<__nv_bfloat162 *>(&x), up);
    const __nv_bfloat162 n = __hmul2(*reinterpret_cast<__nv_bfloat162 *>(&y), up);
    lo = *reinterpret_cast<const uint32_t *>(&m);
    hi = *reinterpret_cast<const uint32_t *>(&n);
  }
}

// Two fp16 pairs from a word of four 8-bit codes, exactly: 0x64'(code + 128) is
// 1024 + 128 + code; E4M3 converts.
template <int kFormat>
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t &lo, uint32_t &hi) {
  if constexpr (kFormat == kCacheInt8) {
    const uint32_t x = w ^ 0x80808080u, offset = 0x64806480u;   // 1152
    const uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
    asm("sub.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(offset));
    asm("sub.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(offset));
  } else {
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"(uint16_t(w)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"(uint16_t(w >> 16)));
  }
}

// int4: a nibble t (two's complement, t = u ^ 8 with u = code + 8) moved to the
// mantissa of a constant makes a small number of u there, and one FMA takes u's
// offset away and applies the factor, exactly: (c + u / n) f - (c + 8 / n) f.
// K's fp16 pairs come a quarter as large (66 times the largest factor must not
// overflow): from bits 2-5 64 + u / 4, from bits 6-9 4 + u / 4.
struct Int4Factors {
  uint32_t f, minus_66f, minus_6f;    // fp16 pairs of one factor
};

__device__ __forceinline__ uint32_t half2_mul(uint32_t x, uint32_t y) {
  uint32_t z;
  asm("mul.f16x2 %0, %1, %2;" : "=r"(z) : "r"(x), "r"(y));
  return z;
}

__device__ __forceinline__ uint32_t half2_fma(uint32_t x, uint32_t y, uint32_t z) {
  uint32_t w;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(w) : "r"(x), "r"(y), "r"(z));
  return w;
}

__device__ __forceinline__ Int4Factors int4_factors(uint32_t pair) {   // of an fp16 pair of one factor
  return {pair, half2_mul(pair, 0xd420d420u), half2_mul(pair, 0xc600c600u)};
}

// (x & mask) ^ kBits in one instruction: of its operands one may be a constant, so
// the mask has to be in a register that the compiler does not see through.
template <uint32_t kBits>
__device__ __forceinline__ uint32_t masked_xor(uint32_t x, uint32_t mask) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0x6c;" : "=r"(y) : "r"(x), "n"(kBits), "r"(mask));
  return y;
}

struct Int4Masks {
  uint32_t low, high, mantissa;     // bits 2-5, 6-9 and 3-6 of each half
};

__device__ __forceinline__ Int4Masks int4_masks() {
  Int4Masks m;
  asm volatile("mov.b32 %0, 0x003c003c;" : "=r"(m.low));
  asm volatile("mov.b32 %0, 0x03c003c0;" : "=r"(m.high));
  asm volatile("mov.b32 %0, 0x00780078;" : "=r"(m.mantissa));
  return m;
}

// A word's codes 2 kHalf, 2 kHalf + 1 with those four places on, as fp16 pairs times f / 4.
template <int kHalf>
__device__ __forceinline__ void int4_to_half(uint32_t w, const Int4Factors &f, const Int4Masks &m, uint32_t &even, uint32_t &odd) {
  const uint32_t t = kHalf ? w >> 6 : w << 2;
  even = half2_fma(masked_xor<0x54205420u>(t, m.low), f.f, f.minus_66f);
  odd = half2_fma(masked_xor<0x46004600u>(t, m.high), f.f, f.minus_6f);
}

// Code kAt of each half of a word as a bf16 pair times the halves' factors:
// bits 3-6 of 16 + u.
template <int kAt>
__device__ __forceinline__ uint32_t int4_to_bf16(uint32_t w, uint32_t f, uint32_t minus_24f, const Int4Masks &m) {
  const uint32_t t = kAt == 0 ? w << 3 : w >> (kAt == 0 ? 0 : 4 * kAt - 3);
  return bf162_fma(masked_xor<0x41c041c0u>(t, m.mantissa), f, minus_24f);
}

// Two factors as a bf16 pair, and -24 times it.  Any byte gives a number.
__device__ __forceinline__ uint32_t factor_pair_bf16(uint32_t lo, uint32_t hi, uint32_t &minus_24f) {
  const uint32_t zero = 0x80008000u, x = ((lo | (hi << 16)) & 0x007f007fu) << 4;
  const uint32_t f = bf162_fma(x, 0x7b807b80u, zero);            // 2^120, as for E4M3 codes
  minus_24f = bf162_fma(f, 0xc1c0c1c0u, zero);
  return f;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ void mma_half_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Whether a packed bf16 pair holds a NaN or an infinity.
__device__ __forceinline__ bool pair_not_finite(uint32_t w) {
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

// Tokens of sequence b in the cache, at most what the table names.
__device__ __forceinline__ int cache_length(const CachePages &c, const int *lengths, int b) {
  const int64_t length = __ldg(lengths + b), capacity = int64_t(c.width) << c.shift;
  if (length > capacity)
    record_status(kStatusBadPage);
  return int(max(int64_t(0), min(length, capacity)));
}

// Position of the first of its n new rows (negative when it has fewer tokens).
__device__ __forceinline__ int first_new_position(const int *lengths, int b, int n) {
  return int(max(int64_t(__ldg(lengths + b)) - n, -(int64_t(1) << 30)));
}

// The unit of a slot: sequences are given floor(starts[b] * group / tile) + b
// as their first slot, which leaves each of them ceil(rows * group / tile) at
// least and takes floor(rows * group / tile) + batch in all, so the host can
// size the grid without the lengths.  Returns the sequence, or -1.
// All lanes of a warp search together, 128 candidates at a time; s0 and s1 are
// the sequence's first row and the one after its last.
__device__ __forceinline__ int unit_of(const RaggedArgs &a, int tile_log2, int slot, int &tile, int &s0, int &s1) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = a.batch, first[4], after[4], count = 0, step;
  do {
    step = (hi - lo + 127) >> 7;
    count = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = min(lo + (i * 32 + lane) * step, a.batch);
      first[i] = max(__ldg(a.starts + at), 0);
      after[i] = __ldg(a.starts + min(at + 1, a.batch));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = lo + (i * 32 + lane) * step;
      const bool before = at < hi && ((int64_t(first[i]) * a.group) >> tile_log2) + at <= slot;
      count += __popc(__ballot_sync(0xffffffffu, before));
    }
    if (count == 0)
      return -1;
    lo += (count - 1) * step;
    hi = min(hi, lo + step);
  } while (hi - lo > 1);
  const int which = (count - 1) >> 5, of = (count - 1) & 31;
  s0 = __shfl_sync(0xffffffffu, which & 2 ? (which & 1 ? first[3] : first[2]) : (which & 1 ? first[1] : first[0]), of);
  s1 = __shfl_sync(0xffffffffu, which & 2 ? (which & 1 ? after[3] : after[2]) : (which & 1 ? after[1] : after[0]), of);
  s1 = int(min(int64_t(s1), a.rows));
  tile = slot - int((int64_t(s0) * a.group) >> tile_log2) - lo;
  return (tile >= 0 && (int64_t(tile) << tile_log2) < int64_t(s1 - s0) * a.group) ? lo : -1;
}

// Sequences that can be put in order of their length, four to a lane.
constexpr int kOrdered = 128;

// The same with the units of longer sequences first (batch <= kOrdered): where
// CTAs wait for others to end, long ones started last would run alone.
// Sequences are taken by sixteenths of the longest's length, and as they come
// within a sixteenth.  `index` counts the units of one kv head without gaps.
__device__ __forceinline__ int unit_by_length(const RaggedArgs &a, int tile_log2, int index, int &tile, int &s0, int &s1) {
  const int lane = threadIdx.x & 31;
  int first[4], rows[4], length[4], units[4], most = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int b = min(i * 32 + lane, a.batch - 1);
    first[i] = max(__ldg(a.starts + b), 0);
    rows[i] = i * 32 + lane < a.batch ? int(max(int64_t(0), min(int64_t(__ldg(a.starts + b + 1)), a.rows) - first[i])) : 0;
    length[i] = max(__ldg(a.lengths + b), 0);
    units[i] = int((int64_t(rows[i]) * a.group + (1 << tile_log2) - 1) >> tile_log2);
    if (rows[i] > 0)
      most = max(most, length[i]);
  }
  const float part = 15.99f / float(max(1, int(__reduce_max_sync(0xffffffffu, most))));
#pragma unroll
  for (int i = 0; i < 4; ++i)
    length[i] = int(float(length[i]) * part);
  int before = 0, mine = 0, which = -1;
#pragma unroll
  for (int c = 15; c >= 0; --c) {
    int here = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      here += length[i] == c ? units[i] : 0;
    const int all = __reduce_add_sync(0xffffffffu, here);
    if (which < 0) {
      if (index - before < all) {
        which = c;
        mine = here;
      } else {
        before += all;
      }
    }
  }
  if (which < 0)
    return -1;
  int upto = mine;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, upto, x);
    if (lane >= x)
      upto += y;
  }
  const int owner = __ffs(__ballot_sync(0xffffffffu, upto > index - before)) - 1;
  int at = index - before - (upto - mine), b = -1;
  s0 = s1 = tile = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (length[i] == which && b < 0) {
      if (at < units[i])
        b = i * 32 + lane, tile = at, s0 = first[i], s1 = first[i] + rows[i];
      at -= units[i];
    }
  }
  b = __shfl_sync(0xffffffffu, b, owner);
  tile = __shfl_sync(0xffffffffu, tile, owner);
  s0 = __shfl_sync(0xffffffffu, s0, owner);
  s1 = __shfl_sync(0xffffffffu, s1, owner);
  return b;
}

// CTAs that the registers and shared memory of an SM take.
constexpr int few_ctas(int format, int d, int nt) { return nt == 2 || (format == kCacheBf16 && d == 128) ? 2 : 4; }

// Shared memory of the few-row kernel: each warp's ring of K and V tiles of 16
// rows, their scales, factors and barriers; at the end the warps' partial sums.
template <int kFormat, int D, int kNT>
struct FewShape {
  static constexpr int kRowBytes = code_bytes(kFormat, D);
  static constexpr int kBoxes = kRowBytes > 128 ? 2 : 1;          // a swizzled row has at most 128 bytes
  static constexpr int kTile = 16 * kRowBytes;
  static constexpr bool kInt4 = kFormat == kCacheInt4;
  static constexpr int kSub = kInt4 ? 2 : 1;                      // tiles of 16 keys in a step
  static constexpr int kStages = kInt4 ? 2 : 3;
  static constexpr int kCtas = few_ctas(kFormat, D, kNT);   // on an SM
  static constexpr int kRing = kFewWarps * kStages * 2 * kSub * kTile;
  // int4: of 16 keys, K's factors, V's factors, K's scales, V's scales, 64 bytes for each.
  static constexpr int kBeside = 256;
  static constexpr int kScales = kFewWarps * kStages * (kInt4 ? kSub * kBeside : 2 * 16 * 4);
  // int4: q's fragments, which its longer conversions leave no registers for.
  static constexpr int kQuery = kInt4 ? kFewWarps * kNT * (D / 16) * 2 * 32 * 4 : 0;
  static constexpr int kCopied = kRing + kScales + kQuery;
  static constexpr int kSums = kFewWarps * kNT * 8 * (D + 4 + 2) * 4 + kNT * 8 * (D + 4) * 4;
  // The barriers lie behind both: their memory may hold nothing else (sums
  // written over them were seen to turn back into barriers).
  static constexpr int kBarriers = kCopied > kSums ? kCopied : kSums;
  static constexpr int kSmem = kInt4 ? kBarriers : 1024 /* alignment */ + kBarriers + kFewWarps * kStages * 8;
};

// 4-D tiled load into this CTA's shared memory.
__device__ __forceinline__ void tma_load_4d(void *dst, const void *tmap, uint64_t *bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::
          "r"(smem_u32(dst)),
      "l"(tmap), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// Offset of 16-byte piece `c` (below 8) of row `r` in a swizzled tile of
// kRowBytes rows (of 256 bytes: in the first of two boxes of 128-byte halves).
template <int kRowBytes>
__device__ __forceinline__ int offset_of(int r, int c) {
  return kRowBytes >= 128 ? r * 128 + ((c ^ (r & 7)) << 4)
         : kRowBytes == 64 ? r * 64 + ((c ^ ((r >> 1) & 3)) << 4) : r * 32 + (c << 4);   // rows of 32 lie plain
}

// Where sequences and kv heads are few, the work of a call is cut into pieces
// that fill the SMs: pieces of about equal length, however the
// lengths of the sequences differ: with s_b 16-key steps for each of a
// sequence's units, W steps in all and `pieces` CTAs wanted, T is a little over
// W / (pieces - units), at least 16, and each unit has ceil(s_b / T) pieces, W /
// T + units at most in all.  They are numbered sequence, kv head, unit, piece.
struct FewPiece {
  int b, kvh, tile;      // sequence (-1: none), kv head, unit of its rows
  int index, count;      // piece of the unit
};

// Units of sequence b and the steps of each (one at least, to write zeros).
__device__ __forceinline__ void units_of(const RaggedArgs &a, int group, int rows_log2, int b, uint32_t &units,
                                         uint32_t &steps) {
  const int64_t s0 = max(__ldg(a.starts + b), 0), s1 = min(int64_t(__ldg(a.starts + b + 1)), a.rows);
  const int64_t length = min(int64_t(__ldg(a.lengths + b)), int64_t(a.c.width) << a.c.shift);
  units = uint32_t((max(s1 - s0, int64_t(0)) * group + (1 << rows_log2) - 1) >> rows_log2);
  steps = uint32_t(max(int64_t(1), (length + 15) >> 4));
}

// The block's piece: every warp searches by itself, a lane over every 32nd part
// of the sequences.
__device__ __forceinline__ FewPiece piece_of_block(const RaggedArgs &a, int group, int rows_log2) {
  const int lane = threadIdx.x & 31, each = (a.batch + 31) >> 5;
  const int b0 = lane * each, b1 = min(a.batch, b0 + each);
  uint32_t units = 0, steps = 1;
  float work = 0.f, whole = 0.f;
  for (int b = b0; b < b1; ++b) {
    units_of(a, group, rows_log2, b, units, steps);
    work += float(units) * float(steps);
    whole += float(units);
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) {
    work += __shfl_xor_sync(0xffffffffu, work, x);
    whole += __shfl_xor_sync(0xffffffffu, whole, x);
  }
  const float cuts = fmaxf(a.pieces - whole * a.c.hk, 0.5f * a.pieces);
  const uint32_t length = max(uint32_t(4 * kFewWarps), uint32_t(work * 1.0001f * a.c.hk / cuts) + 1);
  uint32_t mine = 0;
  for (int b = b0; b < b1; ++b) {
    if (each > 1)
      units_of(a, group, rows_log2, b, units, steps);
    mine += units * a.c.hk * ((steps + length - 1) / length);
  }
  uint32_t upto = mine;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, upto, x);
    if (lane >= x)
      upto += y;
  }
  const uint32_t owners = __ballot_sync(0xffffffffu, blockIdx.x < upto);
  FewPiece p = {-1, 0, 0, 0, 1};
  if (owners == 0)
    return p;
  const int owner = __ffs(owners) - 1;
  uint32_t at = upto - mine, count = 1;
  int found = b0;
  if (lane == owner) {
    for (;; ++found) {
      units_of(a, group, rows_log2, found, units, steps);
      count = (steps + length - 1) / length;
      const uint32_t pieces = units * a.c.hk * count;
      if (blockIdx.x < at + pieces || found + 1 >= b1)
        break;
      at += pieces;
    }
  }
  p.b = __shfl_sync(0xffffffffu, found, owner);
  p.count = int(__shfl_sync(0xffffffffu, count, owner));
  units = __shfl_sync(0xffffffffu, units, owner);
  const uint32_t rest = blockIdx.x - __shfl_sync(0xffffffffu, at, owner), unit = rest / uint32_t(p.count);
  p.index = int(rest - unit * uint32_t(p.count));
  p.kvh = int(unit / units);
  p.tile = int(unit - uint32_t(p.kvh) * units);
  return p;
}

// A lane's values of an output row, divided by the sum of the weights.
template <int E>
__device__ __forceinline__ void store_row(__nv_bfloat16 *out, const float (&sum)[E], float total) {
  const float inv = total == 0.f ? 0.f : 1.f / total;
  uint32_t w[E / 2];
#pragma unroll
  for (int e = 0; e < E; e += 2)
    w[e / 2] = pack_bf16x2(sum[e] * inv, sum[e + 1] * inv);
  if constexpr (E == 4)
    *reinterpret_cast<uint2 *>(out) = make_uint2(w[0], w[1]);
  else
    *reinterpret_cast<uint32_t *>(out) = w[0];
}

template <int kFormat, int D, int kNT>
__global__ void __launch_bounds__(kFewWarps * 32, FewShape<kFormat, D, kNT>::kCtas)
    attention_few_kernel(const RaggedArgs a, const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v) {
  using Shape = FewShape<kFormat, D, kNT>;
  constexpr bool kBf16 = kFormat == kCacheBf16, kInt4 = kFormat == kCacheInt4;
  constexpr int kRows = 8 * kNT, kRowsLog2 = kNT == 1 ? 3 : 4;
  constexpr int KS = D / 16;                       // K steps of S, and M tiles of O
  constexpr int KW = Shape::kRowBytes / 16;        // words of a lane's quarter of a K row
  constexpr int VW = Shape::kRowBytes / 32;        // words of a lane's eighth of a V row
  constexpr int kRowBytes = Shape::kRowBytes, kStages = Shape::kStages, kTile = Shape::kTile;
  extern __shared__ __align__(16) uint8_t few_raw[];
  uint8_t *few_sm =
      kInt4 ? few_raw : reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(few_raw) + 1023) & ~uintptr_t(1023));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q4 = lane & 3;
  const int group = a.group;
  uint8_t *ring = few_sm + warp * kStages * 2 * Shape::kSub * kTile;                      // [kStages][K, V][kSub]
  float *scales = reinterpret_cast<float *>(few_sm + Shape::kRing) + warp * kStages * 32;   // [kStages][K, V][16]
  uint64_t *full = reinterpret_cast<uint64_t *>(few_sm + Shape::kBarriers) + warp * kStages;
  if (!kInt4 && lane == 0) {
    for (int i = 0; i < kStages; ++i)
      mbar_init(&full[i], 1);
    fence_barrier_init();
  }
  __syncwarp();
  pdl_wait();
  pdl_launch_dependents();
  FewPiece piece;
  if (a.cluster > 0) {                              // a unit's pieces are the CTAs of a cluster
    const int unit = int(blockIdx.x) / a.cluster;
    piece.kvh = unit % a.hk;
    int s0, s1;
    piece.b = a.ordered ? unit_by_length(a, kRowsLog2, unit / a.hk, piece.tile, s0, s1)
                        : unit_of(a, kRowsLog2, unit / a.hk, piece.tile, s0, s1);
    piece.index = int(blockIdx.x) % a.cluster;
    piece.count = a.cluster;
  } else {
    piece = piece_of_block(a, group, kRowsLog2);
  }
  const int b = piece.b, kvh = piece.kvh, tile = piece.tile;
  if (b < 0)
    return;
  const int64_t begin = max(__ldg(a.starts + b), 0);
  const int n = int(min(int64_t(__ldg(a.starts + b + 1)), a.rows) - begin);
  const int r0 = tile << kRowsLog2;
  const int r1 = min(r0 + kRows, n * group);       // the unit's rows: r = token * group + head
  // Row r sees positions 0 .. first_new + r / group.
  const int length = cache_length(a.c, a.lengths, b);
  const int first_new = first_new_position(a.lengths, b, n);
  const int keys = max(0, min(length, first_new + (r1 - 1) / group + 1));
  const int all_see = min(length, first_new + r0 / group + 1);   // every row sees positions below this
  // This piece's steps of 16 (int4: 32) keys, as equal as the pieces of the unit can be.
  constexpr int kStepLog2 = kInt4 ? 5 : 4;
  const int steps = (keys + (1 << kStepLog2) - 1) >> kStepLog2;
  const int step_begin = int(int64_t(steps) * piece.index / piece.count);
  const int step_end = int(int64_t(steps) * (piece.index + 1) / piece.count);

  // The warp's steps: every kFewWarps-th from `step0` on.
  const int step0 = step_begin + warp;
  const int count = step_end > step0 ? (step_end - step0 + kFewWarps - 1) / kFewWarps : 0;
  const int page_mask = (1 << a.c.shift) - 1;
  int pages_of_lane = 0;                            // the pages of the next 32 steps to copy
  auto copy = [&](int i) {
    const int step = step0 + i * kFewWarps, stage = i % kStages;
    if ((i & 31) == 0 && i + lane < count)          // a bad page reads page 0: any values do
      pages_of_lane = max(0, page_of(a.c, b, int64_t(step + lane * kFewWarps) << 4));
    const int page = __shfl_sync(0xffffffffu, pages_of_lane, i & 31);
    if (lane == 0) {
      uint8_t *to = ring + stage * 2 * kTile;
      const int in_page = (step << 4) & page_mask;
      mbar_arrive_expect_tx(&full[stage], 2 * kTile + (kBf16 ? 0 : 128));
#pragma unroll
      for (int h = 0; h < Shape::kBoxes; ++h) {
        tma_load_4d(to + h * 2048, &tm_k, &full[stage], h * 64, in_page, kvh, page);
        tma_load_4d(to + kTile + h * 2048, &tm_v, &full[stage], h * 64, in_page, kvh, page);
      }
      if constexpr (!kBf16) {
        const int64_t slot = (int64_t(kvh) << a.c.shift) + in_page;
        bulk_load(scales + stage * 32, a.c.ks + page * a.c.ks_page + slot, 64, &full[stage]);
        bulk_load(scales + stage * 32 + 16, a.c.vs + page * a.c.vs_page + slot, 64, &full[stage]);
      }
    }
  };
  // int4: small pieces of six arrays, copied by all lanes, 16 bytes each (a lane
  // that issues six bulk copies per 16 keys spends more instructions on them than
  // the warp on the products).  Lane i of 16 keys' codes has piece i of 32; of
  // what lies beside them, 16 lanes for each half of the step.
  uint8_t *beside = few_sm + Shape::kRing + warp * kStages * Shape::kSub * Shape::kBeside;   // [kStages][kSub][kBeside]
  constexpr int kHeadUnit = D / kFactorGroup;           // bytes of a row's factors
  const int which = (lane >> 2) & 3, unit = which < 2 ? kHeadUnit : 4;
  const int64_t of_head = int64_t(kvh) << a.c.shift;
  const uint8_t *k_src = static_cast<const uint8_t *>(a.c.k) + of_head * kRowBytes + lane * 16;
  const uint8_t *v_src = static_cast<const uint8_t *>(a.c.v) + of_head * kRowBytes + lane * 16;
  const Int4Masks masks = int4_masks();
  const uint8_t *beside_src = (which == 0   ? a.c.kf
                               : which == 1 ? a.c.vf
                               : which == 2 ? reinterpret_cast<const uint8_t *>(a.c.ks)
                                            : reinterpret_cast<const uint8_t *>(a.c.vs)) + of_head * unit + (lane & 3) * 16;
  // From page to page in units of 16 bytes, below 2^32: one product of 32 bits each.
  const uint32_t beside_page = uint32_t((which == 0   ? a.c.kf_page
                                         : which == 1 ? a.c.vf_page
                                         : which == 2 ? a.c.ks_page * 4
                                                      : a.c.vs_page * 4) >> 4);
  const uint32_t k_page = uint32_t(a.c.k_page >> 4), v_page = uint32_t(a.c.v_page >> 4);
  auto at_page = [](const uint8_t *p, int page, uint32_t stride, int beyond) { return p + (uint64_t(uint32_t(page)) * stride << 4) + beyond; };
  const bool beside_mine = (lane & 3) * 16 < 16 * unit;
  const int piece_at = kRowBytes == 64 ? (lane >> 2) * 64 + (((lane & 3) ^ ((lane >> 3) & 3)) << 4) : lane * 16;
  auto copy4 = [&](int i, int stage) {
    if (i < count) {
      const int key0 = (step0 + i * kFewWarps) << 5, in_page = key0 & page_mask;
      uint8_t *to = ring + stage * 4 * kTile + piece_at, *beside_to = beside + stage * 512 + lane * 16;
      if (a.c.shift > 4) {                          // 32 keys of a page
        if ((i & 31) == 0)                          // the pages of the next 32 steps
          pages_of_lane = i + lane < count ? max(0, page_of(a.c, b, key0 + lane * (32 * kFewWarps))) : 0;
        const int page = __shfl_sync(0xffffffffu, pages_of_lane, i & 31);
        const uint8_t *k_at = at_page(k_src, page, k_page, in_page * kRowBytes), *v_at = at_page(v_src, page, v_page, in_page * kRowBytes);
#pragma unroll
        for (int j = 0; j < 2 * kTile / 512; ++j) {
          cp_async_16(to + j * 512, k_at + j * 512);
          cp_async_16(to + 2 * kTile + j * 512, v_at + j * 512);
        }
        if (beside_mine)
          cp_async_16(beside_to, at_page(beside_src, page, beside_page, (in_page + (lane & 16)) * unit));
      } else {                                      // 16 keys each of two pages
        if ((i & 15) == 0) {
          const int key = key0 + (lane >> 1) * (32 * kFewWarps) + (lane & 1) * 16;
          pages_of_lane = i + (lane >> 1) < count && key < keys ? max(0, page_of(a.c, b, key)) : 0;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int page = __shfl_sync(0xffffffffu, pages_of_lane, (2 * i + h) & 31);
          const uint8_t *k_at = at_page(k_src, page, k_page, 0), *v_at = at_page(v_src, page, v_page, 0);
#pragma unroll
          for (int j = 0; j < kTile / 512; ++j) {
            cp_async_16(to + h * kTile + j * 512, k_at + j * 512);
            cp_async_16(to + (2 + h) * kTile + j * 512, v_at + j * 512);
          }
          if (lane >> 4 == h && beside_mine)
            cp_async_16(beside_to, at_page(beside_src, page, beside_page, 0));
        }
      }
    }
    cp_async_commit();
  };
  if constexpr (kInt4) {
    for (int i = 0; i < kStages - 1; ++i)
      copy4(i, i);
  } else {
    for (int i = 0; i < min(kStages, count); ++i)
      copy(i);
  }

  uint32_t qf[kNT][KS][2];
  int limit[kNT][2];
  float to_log2[kNT][2];                           // a row's factor from its products to scores in log2
#pragma unroll
  for (int t = 0; t < kNT; ++t) {
    const int r = r0 + t * 8 + g;
    // The four elements of each product step that this lane holds of a K row.
    const __nv_bfloat16 *src = a.q + (begin + r / group) * a.q_row + (kvh * group + r % group) * a.q_head;
    if constexpr (kInt4) {                         // pairs four apart, as a word's codes come
#pragma unroll
      for (int s = 0; s < KS; s += 2) {
        const uint4 w = r < r1 ? __ldg(reinterpret_cast<const uint4 *>(src + q4 * (D / 4) + s * 4)) : make_uint4(0, 0, 0, 0);
        qf[t][s][0] = __byte_perm(w.x, w.z, 0x5410), qf[t][s][1] = __byte_perm(w.x, w.z, 0x7632);
        qf[t][s + 1][0] = __byte_perm(w.y, w.w, 0x5410), qf[t][s + 1][1] = __byte_perm(w.y, w.w, 0x7632);
      }
    }
#pragma unroll
    for (int s = 0; s < (kInt4 ? 0 : KS); ++s) {
      const int at = kBf16 ? (s / 2 * 4 + q4) * 8 + s % 2 * 4 : (s / 4 * 4 + q4) * 16 + s % 4 * 4;
      const uint2 w = r < r1 ? __ldg(reinterpret_cast<const uint2 *>(src + at)) : make_uint2(0, 0);
      qf[t][s][0] = w.x;
      qf[t][s][1] = w.y;
    }
    float undo = 1.f;
    if constexpr (!kBf16) {
      // fp16 holds a bf16 row exactly (to 2^-35 of its largest value) once a
      // power of two has brought that value to 2^10.
      uint32_t most = 0;
#pragma unroll
      for (int s = 0; s < KS; ++s)
        most = __vmaxu2(most, __vmaxu2(qf[t][s][0] & 0x7fff7fffu, qf[t][s][1] & 0x7fff7fffu));
      most = max(most & 0xffffu, most >> 16);
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const int up = most == 0 ? 127 : min(264 - int(most >> 7), 253);   // exponent field of the power
      const float factor = __int_as_float(up << 23);
      undo = __int_as_float((254 - up) << 23) * (kInt4 ? 4.f : 1.f);   // its K is a quarter of what it is
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 x = bf16_pair(qf[t][s][e]);
          qf[t][s][e] = pack_half2(x.x * factor, x.y * factor);
        }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int rr = r0 + t * 8 + 2 * q4 + e;
      limit[t][e] = rr < r1 ? first_new + rr / group : -1;
      to_log2[t][e] = __shfl_sync(0xffffffffu, undo, (2 * q4 + e) * 4) * a.scale_log2;
    }
  }

  uint4 *query = reinterpret_cast<uint4 *>(few_sm + Shape::kRing + Shape::kScales) + warp * kNT * (KS / 2) * 32 + lane;
  if constexpr (kInt4) {
#pragma unroll
    for (int t = 0; t < kNT; ++t)
#pragma unroll
      for (int s = 0; s < KS; s += 2)
        query[(t * KS + s) / 2 * 32] = make_uint4(qf[t][s][0], qf[t][s][1], qf[t][s + 1][0], qf[t][s + 1][1]);
    __syncwarp();
  }
  float o[kNT][KS][4] = {};
  float l[kNT][2] = {}, mu[kNT][2] = {};           // mu: the maximum subtracted (0 while none)
  float top[kNT][2];                               // the running maximum
#pragma unroll
  for (int t = 0; t < kNT; ++t) {
    top[t][0] = top[t][1] = -INFINITY;
  }

  // M row g of a step is its key `mine` (and g + 8 is 8 after it); K index 2 q4
  // is key 2 q4 and 2 q4 + 1 is key `odd` of its first eight.
  const int mine = g ^ ((g & 1) << 2), odd = (2 * q4 + 1) ^ 4;
  // Their first pieces in a tile; the row 8 after has the same swizzle, the
  // next four pieces of K lie 64 bytes across, those after 128 in the next box.
  constexpr int kEight = kRowBytes >= 128 ? 1024 : 8 * kRowBytes;
  constexpr int kPart = VW < 4 ? 4 / VW : 1;       // lanes that share a piece of a V row
  const int k_off = KW == 2 ? offset_of<kRowBytes>(mine, q4 >> 1) + (q4 & 1) * 8 : offset_of<kRowBytes>(mine, q4);
  const int v_even = offset_of<kRowBytes>(2 * q4, g / kPart) + g % kPart * (VW * 4);
  const int v_odd = offset_of<kRowBytes>(odd, g / kPart) + g % kPart * (VW * 4);
  int done = 0;
  if constexpr (kInt4) {
    constexpr int kGroups = D / kFactorGroup;
    int stage = 0, next = kStages - 1;
    for (; done < count; ++done, stage = stage == kStages - 1 ? 0 : stage + 1, next = next == kStages - 1 ? 0 : next + 1) {
      const int key0 = (step0 + done * kFewWarps) << 5;
      cp_async_wait_group<kStages - 2>();
      __syncwarp();                                 // all lanes' copies of this stage; all have read the last one
      copy4(done + kStages - 1, next);
      const uint8_t *k_tile = ring + stage * 4 * kTile, *v_tile = k_tile + 2 * kTile;
      const uint8_t *side = beside + stage * 2 * Shape::kBeside;
      auto work = [&](auto some_hidden) {
        constexpr bool kMasked = some_hidden.value;
        float sc[2][kNT][4] = {};
        uint4 qs[kNT][KS / 2];
#pragma unroll
        for (int t = 0; t < kNT; ++t)
#pragma unroll
          for (int s = 0; s < KS / 2; ++s)
            qs[t][s] = query[(t * (KS / 2) + s) * 32];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t kr[2][KW];                         // K rows mine, mine + 8
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint8_t *at = k_tile + h * kTile + k_off + x * kEight;
            if constexpr (KW == 4)
              load_words<4>(kr[x], at);
            else
              load_words<2>(kr[x], at);
          }
          const uint8_t *f = side + h * Shape::kBeside + q4 * (D / 4) / kFactorGroup;
          uint32_t two;
          asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(two) : "h"(uint16_t(f[mine * kGroups] | (f[(mine + 8) * kGroups] << 8))));
          const Int4Factors lo = int4_factors(__byte_perm(two, two, 0x1010)), hi = int4_factors(__byte_perm(two, two, 0x3232));
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            uint32_t af[4];
            if (s & 1) {
              int4_to_half<1>(kr[0][s / 2], lo, masks, af[0], af[2]);
              int4_to_half<1>(kr[1][s / 2], hi, masks, af[1], af[3]);
            } else {
              int4_to_half<0>(kr[0][s / 2], lo, masks, af[0], af[2]);
              int4_to_half<0>(kr[1][s / 2], hi, masks, af[1], af[3]);
            }
#pragma unroll
            for (int t = 0; t < kNT; ++t)
              mma_half_16816(sc[h][t], af, s & 1 ? qs[t][s / 2].z : qs[t][s / 2].x, s & 1 ? qs[t][s / 2].w : qs[t][s / 2].y);
          }
          const float *k_scale = reinterpret_cast<const float *>(side + h * Shape::kBeside + 128) + mine;
          const float k_lo = k_scale[0], k_hi = k_scale[8];
#pragma unroll
          for (int t = 0; t < kNT; ++t) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              // The factors first: a large key's scale alone could overflow the product.
              float v = sc[h][t][e] * ((e < 2 ? k_lo : k_hi) * to_log2[t][e & 1]);
              if (kMasked && key0 + h * 16 + mine + (e & 2) * 4 > limit[t][e & 1])
                v = -INFINITY;
              sc[h][t][e] = v;
            }
          }
        }
        bool raise = false;
#pragma unroll
        for (int t = 0; t < kNT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            raise |= fmaxf(fmaxf(sc[0][t][e], sc[0][t][e + 2]), fmaxf(sc[1][t][e], sc[1][t][e + 2])) > top[t][e] + 8.f;
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
          for (int t = 0; t < kNT; ++t) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float m = fmaxf(fmaxf(top[t][e], fmaxf(sc[0][t][e], sc[0][t][e + 2])), fmaxf(sc[1][t][e], sc[1][t][e + 2]));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
              const float keep = top[t][e] == -INFINITY ? 1.f : exp2_fast(top[t][e] - m);   // nothing summed yet: keep it
              top[t][e] = m;
              mu[t][e] = m == -INFINITY ? 0.f : m;
              l[t][e] *= keep;
#pragma unroll
              for (int s = 0; s < KS; ++s) {
                o[t][s][e] *= keep;
                o[t][s][e + 2] *= keep;
              }
            }
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t vr[4][VW];                         // V rows 2 q4, odd, and 8 after them
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint8_t *at = v_tile + h * kTile + (x & 1 ? v_odd : v_even) + (x >> 1) * kEight;
            if constexpr (VW == 2)
              load_words<2>(vr[x], at);
            else
              vr[x][0] = *reinterpret_cast<const uint32_t *>(at);
          }
          const uint8_t *f = side + h * Shape::kBeside + 64 + g * (D / 8) / kFactorGroup;
          uint32_t vf[2], minus_24vf[2];              // of keys 2 q4 and odd, and 8 after them
#pragma unroll
          for (int x = 0; x < 2; ++x)
            vf[x] = factor_pair_bf16(f[(2 * q4 + 8 * x) * kGroups], f[(odd + 8 * x) * kGroups], minus_24vf[x]);
          const float *v_scale = reinterpret_cast<const float *>(side + h * Shape::kBeside + 192) + mine;
          const float vsc[2] = {v_scale[0], v_scale[8]};
          uint32_t pf[kNT][2];
#pragma unroll
          for (int t = 0; t < kNT; ++t) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = exp2_fast(sc[h][t][e] - mu[t][e & 1]);
              l[t][e & 1] += x;
              // A hidden key's scale may be anything.
              w[e] = kMasked && sc[h][t][e] == -INFINITY ? 0.f : x * vsc[e >> 1];
            }
            pf[t][0] = transpose_8x8(pack_bf16x2(w[0], w[1]));
            pf[t][1] = transpose_8x8(pack_bf16x2(w[2], w[3]));
          }
#pragma unroll
          for (int j = 0; j < VW; ++j) {
            // Channels 0-3 of the two keys in one word, 4-7 in the next.
            uint32_t af[4][4];
#pragma unroll
            for (int x = 0; x < 2; ++x)      // keys 2 q4 .. and 2 q4 + 8 ..
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const uint32_t y = __byte_perm(vr[2 * x][j], vr[2 * x + 1][j], c ? 0x7632 : 0x5410);
                af[2 * c][2 * x] = int4_to_bf16<0>(y, vf[x], minus_24vf[x], masks);
                af[2 * c][2 * x + 1] = int4_to_bf16<1>(y, vf[x], minus_24vf[x], masks);
                af[2 * c + 1][2 * x] = int4_to_bf16<2>(y, vf[x], minus_24vf[x], masks);
                af[2 * c + 1][2 * x + 1] = int4_to_bf16<3>(y, vf[x], minus_24vf[x], masks);
              }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int t = 0; t < kNT; ++t)
                mma_bf16_16816(o[t][4 * j + i], af[i], pf[t][0], pf[t][1]);
          }
        }
      };
      // Few steps have positions that some row does not see.
      if (key0 + 32 > all_see)
        work(std::true_type{});
      else
        work(std::false_type{});
    }
  }
  if constexpr (!kInt4) {
    for (; done < count; ++done) {
      const int step = step0 + done * kFewWarps, stage = done % kStages;
      if (!__all_sync(0xffffffffu, mbar_wait(&full[stage], uint32_t((done / kStages) & 1), kStatusTimeoutProducer)))
        break;
      const uint8_t *k_tile = ring + stage * 2 * kTile, *v_tile = k_tile + kTile;
      uint32_t kr[2][KW], vr[4][VW];                  // K rows mine, mine + 8; V rows 2 q4, odd, and 8 after them
#pragma unroll
      for (int i = 0; i < KW / 4; ++i) {
        const uint8_t *at = k_tile + (i >> 1) * 2048 + (i & 1 ? k_off ^ 64 : k_off);
        *reinterpret_cast<uint4 *>(&kr[0][i * 4]) = *reinterpret_cast<const uint4 *>(at);
        *reinterpret_cast<uint4 *>(&kr[1][i * 4]) = *reinterpret_cast<const uint4 *>(at + kEight);
      }
      float ksc[2] = {1.f, 1.f}, vsc[2] = {1.f, 1.f};
      if constexpr (!kBf16) {
        const float *s = scales + stage * 32 + mine;
        ksc[0] = s[0], ksc[1] = s[8], vsc[0] = s[16], vsc[1] = s[24];
      }
      float sc[kNT][4] = {};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        uint32_t af[4];
        if constexpr (kBf16) {
          af[0] = kr[0][2 * s], af[1] = kr[1][2 * s], af[2] = kr[0][2 * s + 1], af[3] = kr[1][2 * s + 1];
        } else {
          codes_to_half<kFormat>(kr[0][s], af[0], af[2]);
          codes_to_half<kFormat>(kr[1][s], af[1], af[3]);
        }
#pragma unroll
        for (int t = 0; t < kNT; ++t) {
          if constexpr (kBf16)
            mma_bf16_16816(sc[t], af, qf[t][s][0], qf[t][s][1]);
          else
            mma_half_16816(sc[t], af, qf[t][s][0], qf[t][s][1]);
        }
      }
      const float k_lo = ksc[0], k_hi = ksc[1];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint8_t *at = v_tile + (x & 1 ? v_odd : v_even) + (x >> 1) * kEight;
        if constexpr (VW == 2) {
          load_words<2>(vr[x], at);
        } else {
#pragma unroll
          for (int i = 0; i < VW / 4; ++i)
            *reinterpret_cast<uint4 *>(&vr[x][i * 4]) = *reinterpret_cast<const uint4 *>(at + i * 2048);
        }
      }
      __syncwarp();
      if (done + kStages < count)
        copy(done + kStages);
      const int key0 = step << 4;
      const bool masked = key0 + 16 > all_see;
      bool raise = false;
#pragma unroll
      for (int t = 0; t < kNT; ++t) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // The factors first: a large key's scale alone could overflow the product.
          float v = sc[t][e] * (kBf16 ? a.scale_log2 : (e < 2 ? k_lo : k_hi) * to_log2[t][e & 1]);
          if (masked && key0 + mine + (e & 2) * 4 > limit[t][e & 1])
            v = -INFINITY;
          sc[t][e] = v;
          raise |= v > top[t][e & 1] + 8.f;
        }
      }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int t = 0; t < kNT; ++t) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float m = fmaxf(top[t][e], fmaxf(sc[t][e], sc[t][e + 2]));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
            const float keep = top[t][e] == -INFINITY ? 1.f : exp2_fast(top[t][e] - m);   // nothing summed yet: keep it
            top[t][e] = m;
            mu[t][e] = m == -INFINITY ? 0.f : m;
            l[t][e] *= keep;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
              o[t][s][e] *= keep;
              o[t][s][e + 2] *= keep;
            }
          }
        }
      }
      uint32_t pf[kNT][2];
#pragma unroll
      for (int t = 0; t < kNT; ++t) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float w = exp2_fast(sc[t][e] - mu[t][e & 1]);
          l[t][e & 1] += w;
          // A hidden key's scale may be anything.
          sc[t][e] = kBf16 ? w : masked && sc[t][e] == -INFINITY ? 0.f : w * vsc[e >> 1];
        }
        pf[t][0] = transpose_8x8(pack_bf16x2(sc[t][0], sc[t][1]));
        pf[t][1] = transpose_8x8(pack_bf16x2(sc[t][2], sc[t][3]));
      }
      // Pairs (key, key + 1) of a column for the two halves of an M tile pair.
      auto product = [&](const uint32_t (&pp)[kNT][2]) {
#pragma unroll
        for (int j = 0; j < VW; ++j) {
          if constexpr (kBf16) {
            const uint32_t af[4] = {__byte_perm(vr[0][j], vr[1][j], 0x5410), __byte_perm(vr[0][j], vr[1][j], 0x7632),
                                    __byte_perm(vr[2][j], vr[3][j], 0x5410), __byte_perm(vr[2][j], vr[3][j], 0x7632)};
#pragma unroll
            for (int t = 0; t < kNT; ++t)
              mma_bf16_16816(o[t][j], af, pp[t][0], pp[t][1]);
          } else {
            uint32_t af[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {   // keys 2 q4 .. and 2 q4 + 8 ..
              const uint32_t x = __byte_perm(vr[2 * h][j], vr[2 * h + 1][j], 0x5140);
              const uint32_t y = __byte_perm(vr[2 * h][j], vr[2 * h + 1][j], 0x7362);
              codes_to_bf16<kFormat>(x, af[0][2 * h], af[0][2 * h + 1]);
              codes_to_bf16<kFormat>(y, af[1][2 * h], af[1][2 * h + 1]);
            }
#pragma unroll
            for (int t = 0; t < kNT; ++t) {
              mma_bf16_16816(o[t][2 * j], af[0], pp[t][0], pp[t][1]);
              mma_bf16_16816(o[t][2 * j + 1], af[1], pp[t][0], pp[t][1]);
            }
          }
        }
      };
      if constexpr (kBf16) {
        if (masked) {
          // Hidden values must not enter a product, not even times 0: positions
          // no row sees become 0 here, and where a position hidden from some
          // rows holds a value that is not finite the rows go one at a time.
          bool spoiled = false;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int key = key0 + (x & 1 ? odd : 2 * q4) + (x & 2) * 4;
#pragma unroll
            for (int j = 0; j < VW; ++j) {
              if (key >= keys)
                vr[x][j] = 0;
              else if (key >= all_see)
                spoiled |= pair_not_finite(vr[x][j]);
            }
          }
          if (__any_sync(0xffffffffu, spoiled)) {
            uint32_t kept[4][VW];
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
              for (int j = 0; j < VW; ++j)
                kept[x][j] = vr[x][j];
#pragma unroll 1
            for (int r = 0; r < kRows; ++r) {
              const int last = r0 + r < r1 ? first_new + (r0 + r) / group : -1;
              uint32_t one[kNT][2];
#pragma unroll
              for (int t = 0; t < kNT; ++t) {
                one[t][0] = t * 8 + g == r ? pf[t][0] : 0;
                one[t][1] = t * 8 + g == r ? pf[t][1] : 0;
              }
              // The product runs on columns of zeros for the other rows, so a
              // value that this row sees must not reach them either: it is
              // added to this row alone, below.
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const int key = key0 + (x & 1 ? odd : 2 * q4) + (x & 2) * 4;
#pragma unroll
                for (int j = 0; j < VW; ++j)
                  vr[x][j] = key > last ? 0 : kept[x][j];
              }
              float saved[kNT][KS][4];
#pragma unroll
              for (int t = 0; t < kNT; ++t)
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    saved[t][s][e] = o[t][s][e];
              product(one);
              // Columns of O^T are rows: keep the new sums of row r only.
#pragma unroll
              for (int t = 0; t < kNT; ++t)
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    if (t * 8 + 2 * q4 + (e & 1) != r)
                      o[t][s][e] = saved[t][s][e];
            }
            continue;
          }
        }
      }
      product(pf);
    }
  }

  // No copy is in flight past this point (at once, unless a wait gave up).
  if constexpr (kInt4) {
    cp_async_wait_group<0>();
  } else {
    for (int i = done; i < min(done + kStages, count); ++i)
      mbar_wait(&full[i % kStages], uint32_t((i / kStages) & 1), kStatusTimeoutProducer);
  }
  __syncthreads();
  // The warps' partial sums, added in warp order.
  float *so = reinterpret_cast<float *>(few_sm);                // [warps][rows][D + 4]
  float *sm = so + kFewWarps * kRows * (D + 4), *sl = sm + kFewWarps * kRows;
  float *joined = sl + kFewWarps * kRows;                       // [rows][D values, maximum, sum, -, -]
#pragma unroll
  for (int t = 0; t < kNT; ++t) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = l[t][e];
      x += __shfl_xor_sync(0xffffffffu, x, 4);
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      const int r = t * 8 + 2 * q4 + e;
      if (g == 0) {
        sm[warp * kRows + r] = top[t][e];
        sl[warp * kRows + r] = x;
      }
#pragma unroll
      for (int s = 0; s < KS; ++s) {                           // the two columns of tile s
        const int d = kBf16 ? (s / 4 * 8 + g) * 8 + s % 4 * 2 : g * (D / 8) + 2 * s;
        const float2 pair = make_float2(o[t][s][e], o[t][s][e + 2]);
        *reinterpret_cast<float2 *>(so + (warp * kRows + r) * (D + 4) + d) = pair;
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kRows * (D / 4); i += kFewWarps * 32) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    if (r0 + r >= r1)
      continue;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w)
      m = fmaxf(m, sm[w * kRows + r]);
    float total = 0.f;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
      const float mw = sm[w * kRows + r];
      const float f = mw == m ? 1.f : exp2_fast(mw - m);       // equal, -inf too: the sums as they are
      const float4 x = *reinterpret_cast<const float4 *>(so + (w * kRows + r) * (D + 4) + d);
      total += f * sl[w * kRows + r];
      sum.x += f * x.x, sum.y += f * x.y, sum.z += f * x.z, sum.w += f * x.w;
    }
    const int64_t row = begin + (r0 + r) / group;
    const int h = kvh * group + (r0 + r) % group;
    if (piece.count == 1) {
      const float inv = total == 0.f ? 0.f : 1.f / total;
      *reinterpret_cast<uint2 *>(a.out + row * a.ldo + h * D + d) =
          make_uint2(pack_bf16x2(sum.x * inv, sum.y * inv), pack_bf16x2(sum.z * inv, sum.w * inv));
    } else if (a.cluster > 0) {
      *reinterpret_cast<float4 *>(joined + r * (D + 4) + d) = sum;
      if (d == 0)
        joined[r * (D + 4) + D] = m, joined[r * (D + 4) + D + 1] = total;
    } else {
      const int64_t at = int64_t(blockIdx.x) * kRows + r;
      *reinterpret_cast<float4 *>(a.part_o + at * D + d) = sum;
      if (d == 0)
        a.part_ml[at] = make_float2(m, total);
    }
  }
  if (a.cluster > 1) {
    // The cluster's CTAs each join a share of the unit's values, reading the
    // others' shared memory, in rank order.
    cluster_sync();
    const uint32_t mine_sm = smem_u32(joined);
    for (int i = piece.index * kFewWarps * 32 + threadIdx.x; i < kRows * (D / 4); i += a.cluster * kFewWarps * 32) {
      const int r = i / (D / 4), d = i % (D / 4) * 4;
      if (r0 + r >= r1)
        continue;
      float m[8], l[8], top_of_all = -INFINITY;
      int4 x[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        if (c >= a.cluster)
          break;
        const uint32_t row = map_peer(mine_sm + r * (D + 4) * 4, c);
        m[c] = __int_as_float(ld_cluster_s32(row + D * 4));
        l[c] = __int_as_float(ld_cluster_s32(row + D * 4 + 4));
        x[c] = ld_cluster_v4(row + d * 4);
        top_of_all = fmaxf(top_of_all, m[c]);
      }
      float total = 0.f;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        if (c >= a.cluster)
          break;
        const float f = m[c] == top_of_all ? 1.f : exp2_fast(m[c] - top_of_all);
        total += f * l[c];
        sum.x += f * __int_as_float(x[c].x), sum.y += f * __int_as_float(x[c].y);
        sum.z += f * __int_as_float(x[c].z), sum.w += f * __int_as_float(x[c].w);
      }
      const float inv = total == 0.f ? 0.f : 1.f / total;
      *reinterpret_cast<uint2 *>(a.out + (begin + (r0 + r) / group) * a.ldo + (kvh * group + (r0 + r) % group) * D + d) =
          make_uint2(pack_bf16x2(sum.x * inv, sum.y * inv), pack_bf16x2(sum.z * inv, sum.w * inv));
    }
    cluster_sync();                                 // no CTA ends while others read it
  }
  if (a.cluster > 0)
    return;
  // Where the unit's pieces are, for the join: its slot counts units as the
  // sequences' first rows allow without a search.
  if (piece.index == 0 && threadIdx.x == 0) {
    const int64_t slot = ((begin * group) >> kRowsLog2) + b + tile;
    a.part_units[slot * a.hk + kvh] = make_int2(int(blockIdx.x), piece.count);
  }
}

// Joins the pieces of each (row, head): a CTA of eight warps for each, which
// take the pieces in turn and are added in warp order (one warp for all pieces:
// 170 us for one token over 30000 of one kv head, of which the join took nearly
// all).
template <int D, int kNT>
__global__ void __launch_bounds__(256) attention_join_pieces_kernel(const RaggedArgs a) {
  constexpr int E = D / 32, kRowsLog2 = kNT == 1 ? 3 : 4;
  __shared__ float so[8][D], sl[8], sm[8];
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = blockIdx.x / a.hq;
  const int h = int(blockIdx.x % a.hq), group = a.hq / a.hk, kvh = h / group;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = sequence_of_warp(a.starts, a.batch, row);
  if (b < 0)
    return;
  const int64_t begin = max(__ldg(a.starts + b), 0), r = (row - begin) * group + h % group;
  const int64_t slot = ((begin * group) >> kRowsLog2) + b + (r >> kRowsLog2);
  const int2 unit = a.part_units[slot * a.hk + kvh];
  if (unit.y < 2 || unit.x < 0 || unit.y > a.parts - unit.x)   // one piece (or starts that decrease)
    return;
  const int64_t first = (int64_t(unit.x) << kRowsLog2) + (r & ((1 << kRowsLog2) - 1));
  float top = -INFINITY;
  for (int s = threadIdx.x; s < unit.y; s += 256)
    top = fmaxf(top, a.part_ml[first + (int64_t(s) << kRowsLog2)].x);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1)
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
  if (lane == 0)
    sm[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w)
    top = fmaxf(top, sm[w]);
  float total = 0.f, sum[E] = {};
#pragma unroll 8
  for (int s = warp; s < unit.y; s += 8) {
    const int64_t at = first + (int64_t(s) << kRowsLog2);
    const float2 ml = a.part_ml[at];
    const float f = ml.x == top ? 1.f : exp2_fast(ml.x - top);   // equal, -inf too: the sums as they are
    total += f * ml.y;
    const float *p = a.part_o + at * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e)
      sum[e] += f * p[e];
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    so[warp][lane * E + e] = sum[e];
  if (lane == 0)
    sl[warp] = total;
  __syncthreads();
  if (threadIdx.x < D) {
    total = sum[0] = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      total += sl[w];
      sum[0] += so[w][threadIdx.x];
    }
    a.out[row * a.ldo + h * D + threadIdx.x] = __float2bfloat16(total == 0.f ? 0.f : sum[0] / total);
  }
}

// Joins the splits of each (row, head), in split order: a warp per row and
// head, D / 32 values per lane.
template <int D>
__global__ void __launch_bounds__(256) attention_join_kernel(const RaggedArgs a) {
  constexpr int E = D / 32;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t item = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int64_t row = item / a.hq;
  const int h = int(item % a.hq);
  if (row >= a.rows || sequence_of(a.starts, a.batch, row) < 0)
    return;
  const int64_t apart = a.rows * a.hq;
  // At most 32 splits: a lane per split holds its maximum and sum.
  const float2 ml = lane < a.splits ? a.part_ml[lane * apart + item] : make_float2(-INFINITY, 0.f);
  float m = ml.x;
#pragma unroll
  for (int x = 16; x > 0; x >>= 1)
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
  // A split that saw nothing has a sum of 0 and may have written no values.
  const float f = ml.y == 0.f ? 0.f : ml.x == m ? 1.f : exp2_fast(ml.x - m);
  float total = f * ml.y;
#pragma unroll
  for (int x = 16; x > 0; x >>= 1)
    total += __shfl_xor_sync(0xffffffffu, total, x);
  float sum[E] = {};
#pragma unroll 8
  for (int s = 0; s < a.splits; ++s) {
    const float fs = __shfl_sync(0xffffffffu, f, s);
    const float *p = a.part_o + (s * apart + item) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float x = p[e];
      sum[e] += fs == 0.f ? 0.f : fs * x;
    }
  }
  store_row<E>(a.out + row * a.ldo + h * D + lane * E, sum, total);
}

} // namespace pir2b
