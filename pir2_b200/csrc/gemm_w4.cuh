// Products of a few bf16 rows with weights held in 4 bits:
//   out[m, n] = bf16(sum_k x[m, k] code[n, k] scale[n, k / G] + bias[n]),
// codes of -8..7 in two's complement, two to a byte with the even k in the low
// bits, G = 32, 64 or 128 consecutive weights of a channel per bf16 scale.
//
// Few rows cannot fill a tcgen05 tile and the work is reading the weights, so
// the products run on warp-level MMAs (m16n8k16, fp32 sums) with channels as the
// M rows.  A CTA owns 16 channels; its warps split K in chunks of 128.  Codes
// become bf16 in registers, exactly: a nibble moved to bits 3-6 of 16 makes 16 +
// u, u = code + 8, from which 24 is taken.  (Sums that start at -24 times a group's
// x in place of that subtraction were no faster past eight rows and 4% faster below,
// and lose small values beside large ones.)  The four lanes of a channel take pieces
// of one group each, so a product step stays in a group, whose sums are scaled in
// fp32.  The only other rounding is that of the output.
//
// Sums are kept at 2^-10 of themselves, which the same instruction gives the codes:
// a group's are not scaled yet and may be 8 * 128 times the largest row value, which
// must not overflow where the scale brings it back.  Powers of two change no bits of
// ordinary sums; an addition below 2^-116 may lose half of 2^-139 (fp32's smallest
// step, 2^10 times), a 64th of bf16's smallest number.
//
// What bounds it: the start of a launch and the latency of the loads where weights
// are few (2048 -> 4096, one row: 3.2 us, the weights' bytes alone 0.7); where they are
// many, the pipes that bring codes into bf16 (2048 -> 151936, 4 rows: 35.5 us, bytes
// 25, 4.6 TB/s; the schedulers issue in 63 % of the cycles, and of a warp's time 27 %
// goes to a busy math pipe or its dispatch, 24 % to other warps' turns, 12 % to the
// result before, 9 % to loads); with more rows shared memory as well, from which every
// 16 channels read all rows (32 rows of 2048 -> 151936: 101 us, of them 50 of shared
// memory, 34 of MMAs at 8 cycles of a quarter SM each), and the start and the meetings
// (of 2048 -> 12288 in groups of 32: 14.1, bytes 2.3; 38 % of the cycles issue, 22 % of
// a warp's time is at barriers, 20 % at loads).
#pragma once
#include "attention_few.cuh"

namespace pir2b {

struct W4Args {
  const __nv_bfloat16 *x;        // [m, k], row stride ldx
  int64_t ldx;
  const uint8_t *w;              // [n, k / 2]
  const __nv_bfloat16 *scales;   // [n, k / G]
  const __nv_bfloat16 *bias;     // [n] or null
  __nv_bfloat16 *out;            // [m, n], row stride ldo
  int64_t ldo;
  int m, n, k;
  int slab;                      // wide: k whose rows are in shared memory at once
  int wk;                        // staged and wide: warps that split K
  int pairs;                     // output channels may be stored two at a time
};

// What brings a sum back.
constexpr float kW4Up = 1024.f;

// Code kAt of each half of a word as a bf16 pair, times 2^-10: (16 + u) 2^-10 - 24 2^-10.
template <int kAt>
__device__ __forceinline__ uint32_t w4_pair(uint32_t w, const Int4Masks &m) {
  const uint32_t t = kAt == 0 ? w << 3 : w >> (kAt == 0 ? 0 : 4 * kAt - 3);
  return bf162_fma(masked_xor<0x41c041c0u>(t, m.mantissa), 0x3a803a80u, 0xbcc0bcc0u);
}

// Eight values of x in the order in which w4_pair brings the codes.
__device__ __forceinline__ uint4 w4_order(uint4 x) {
  return make_uint4(__byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632), __byte_perm(x.y, x.w, 0x5410),
                    __byte_perm(x.y, x.w, 0x7632));
}

// kPieces pieces of 4 / kPieces words.
template <int kPieces>
__device__ __forceinline__ void w4_load(uint32_t (&w)[4], const uint8_t *row, int left) {
#pragma unroll
  for (int p = 0; p < kPieces; ++p) {
    const bool in = p < left;                       // pieces of the chunk before the end of K
    const uint8_t *at = row + p * (64 / kPieces);
    if constexpr (kPieces == 1) {
      const uint4 v = in ? __ldg(reinterpret_cast<const uint4 *>(at)) : make_uint4(0, 0, 0, 0);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (kPieces == 2) {
      const uint2 v = in ? __ldg(reinterpret_cast<const uint2 *>(at)) : make_uint2(0, 0);
      w[2 * p] = v.x, w[2 * p + 1] = v.y;
    } else {
      w[p] = in ? __ldg(reinterpret_cast<const uint32_t *>(at)) : 0;
    }
  }
}

// What a lane holds of a chunk of 128 k: codes and scales of two channels, and x
// of one token where that is all.
template <int kGroup, int kTiles>
struct W4Chunk {
  uint32_t w[2][4];
  __nv_bfloat16 s[2][128 / kGroup];
  uint4 x[kTiles == 1 ? 4 : 1];
};

// Few channels: every CTA loads what its products take straight into registers, one
// chunk ahead, so that nothing waits for shared memory or for other warps before the
// sums meet (2048 -> 2048 in groups of 128, one row: 2.2 us, without the chunk ahead
// 2.6).
template <int kGroup, int kTiles, int kWarps>
__global__ void __launch_bounds__(kWarps * 32) gemm_w4_kernel(const W4Args a) {
  constexpr int kPieces = 128 / kGroup, kWords = 4 / kPieces;   // of a lane and chunk; words of a piece
  constexpr int kCols = 8 * kTiles, kRow = 20;                  // words of a token's 16 sums, apart by banks
  extern __shared__ __align__(1024) uint8_t tile_raw[];
  float *red = reinterpret_cast<float *>(tile_raw);             // [warp][token][channel]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  const int groups = a.k / kGroup, chunks = (a.k + 127) >> 7, blocks = (a.n + 15) >> 4;
  const int begin = warp * chunks / kWarps, end = (warp + 1) * chunks / kWarps;
  const Int4Masks masks = int4_masks();
  auto row_of = [&](int block, int h) { return int64_t(min(block * 16 + g + h * 8, a.n - 1)); };   // past the last: not stored
  auto codes_of = [&](int block, int h) { return a.w + row_of(block, h) * (a.k >> 1) + q4 * (16 / kPieces); };
  auto load = [&](W4Chunk<kGroup, kTiles> &c, int block, int ch) {
    const int left = groups - ch * kPieces;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      w4_load<kPieces>(c.w[h], codes_of(block, h) + ch * 64, left);
      const __nv_bfloat16 *s = a.scales + row_of(block, h) * groups + ch * kPieces;
#pragma unroll
      for (int p = 0; p < kPieces; ++p)
        c.s[h][p] = p < left ? s[p] : __float2bfloat16(0.f);
    }
    if constexpr (kTiles == 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = i / kWords;
        c.x[i] = make_uint4(0, 0, 0, 0);
        if (g < a.m && p < left)
          c.x[i] = *reinterpret_cast<const uint4 *>(a.x + g * a.ldx + ch * 128 + p * kGroup + q4 * (kGroup / 4) + i % kWords * 8);
      }
    }
  };
  // The first weights start for L2 while the launch before this one ends; nothing
  // is read of them yet.
  if (begin < end) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(codes_of(blockIdx.x, h) + begin * 64));
  }
  pdl_wait();
  pdl_launch_dependents();
  W4Chunk<kGroup, kTiles> one, two;
  if (begin < end)
    load(one, blockIdx.x, begin);
  for (int block = blockIdx.x; block < blocks; block += gridDim.x) {
    float acc[kTiles][4] = {};
    auto multiply = [&](const W4Chunk<kGroup, kTiles> &c, int ch) {
      const int left = groups - ch * kPieces;
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
        float part[kTiles][4] = {};
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          const uint32_t u = c.w[0][p * kWords + i], v = c.w[1][p * kWords + i];
          const uint32_t even[4] = {w4_pair<0>(u, masks), w4_pair<0>(v, masks), w4_pair<1>(u, masks), w4_pair<1>(v, masks)};
          const uint32_t odd[4] = {w4_pair<2>(u, masks), w4_pair<2>(v, masks), w4_pair<3>(u, masks), w4_pair<3>(v, masks)};
          const int k = ch * 128 + p * kGroup + q4 * (kGroup / 4) + i * 8;
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            uint4 x = make_uint4(0, 0, 0, 0);
            if constexpr (kTiles == 1) {
              x = c.x[p * kWords + i];
            } else {
              const int token = t * 8 + g;
              if (token < a.m && p < left)
                x = *reinterpret_cast<const uint4 *>(a.x + token * a.ldx + k);
            }
            mma_bf16_16816(part[t], even, __byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632));
            mma_bf16_16816(part[t], odd, __byte_perm(x.y, x.w, 0x5410), __byte_perm(x.y, x.w, 0x7632));
          }
        }
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[t][e] = fmaf(part[t][e], __bfloat162float(c.s[e >> 1][p]), acc[t][e]);
      }
    };
#pragma unroll 1
    for (int ch = begin; ch < end; ch += 2) {
      if (ch + 1 < end)
        load(two, block, ch + 1);
      multiply(one, ch);
      if (ch + 2 < end)
        load(one, block, ch + 2);
      if (ch + 1 < end)
        multiply(two, ch + 1);
    }
    if (begin < end && block + gridDim.x < blocks)
      load(one, block + gridDim.x, begin);
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        red[(warp * kCols + t * 8 + 2 * q4 + (e & 1)) * kRow + g + (e >> 1) * 8] = acc[t][e];
    __syncthreads();
    for (int i = threadIdx.x; i < kCols * 16; i += kWarps * 32) {
      const int token = i / 16, c = i % 16, channel = block * 16 + c;
      if (token >= a.m || channel >= a.n)
        continue;
      float sum = 0.f;
#pragma unroll
      for (int x = 0; x < kWarps; ++x)              // in order of K
        sum += red[(x * kCols + token) * kRow + c];
      const float bias = a.bias != nullptr ? __bfloat162float(a.bias[channel]) : 0.f;
      a.out[token * a.ldo + channel] = __float2bfloat16_rn(fmaf(sum, kW4Up, bias));
    }
    if (block + gridDim.x < blocks)
      __syncthreads();
  }
}

// Up to eight rows and many channels: a persistent CTA keeps the rows in shared
// memory, as the lanes take them, and streams the weights of its blocks of 16
// channels through a ring per warp; `wk` warps split K, and their sums meet in
// shared memory.  One of a warp's two stages of two chunks is on its way while the
// other is read: with as many warps as fit up to 55 KB on an SM (2048 -> 151936, 4
// rows: 16 warps 4 us longer, four stages of one chunk 3).
struct W4Staged {
  static constexpr int kWarps = 24;
  static constexpr int kCols = 8;
  static constexpr int kStage = 2 * (1024 + 128);        // of two chunks: codes of 16 channels, 16 bytes for each one's scales
  static constexpr int kRedRow = 20;                     // words of a token's 16 sums, apart by banks
  static constexpr int kRed = kWarps * kCols * kRedRow * 4;
  static constexpr int kRing = kWarps * 2 * kStage;
  static constexpr int64_t bytes(int64_t k) { return k * kCols * 2 + kRing + kRed; }
};

// Place of 16-byte piece c of row r: pieces of eight rows read in any width lie
// in different banks.
__device__ __forceinline__ int w4_place(int r, int c) { return r * 64 + ((c ^ ((r & 2) | ((r >> 2) & 1))) << 4); }

template <int kBytes>
__device__ __forceinline__ void cp_async_ca(uint32_t dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(kBytes) : "memory");
}

// Codes of a block's units `from` to `to` on their way to L2 while the launch before
// this one ends; nothing is read of them yet.
__device__ __forceinline__ void w4_prefetch(const W4Args &a, int block, int from, int to) {
  const int row = block * 16 + (threadIdx.x & 15);
  if (row < a.n)
    for (int unit = from + ((threadIdx.x >> 4) & 1); unit < to; unit += 2)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(a.w + int64_t(row) * (a.k >> 1) + unit * 128));
}

template <int kGroup>
__global__ void __launch_bounds__(W4Staged::kWarps * 32, 1) gemm_w4_staged_kernel(const W4Args a) {
  using Shape = W4Staged;
  constexpr int kPieces = 128 / kGroup, kWords = 4 / kPieces, kCols = Shape::kCols, kWarps = Shape::kWarps;
  extern __shared__ __align__(1024) uint8_t tile_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  const int units = a.k >> 8, groups = a.k / kGroup;      // units of two chunks
  uint4 *xs = reinterpret_cast<uint4 *>(tile_raw);                           // [chunk][word][lane]
  uint8_t *rings = tile_raw + int64_t(a.k) * kCols * 2, *ring = rings + warp * 2 * Shape::kStage;
  float *red = reinterpret_cast<float *>(rings + Shape::kRing);              // [warp][token][channel]
  const int wk = a.wk, wc = kWarps / wk, part = warp % wk, which = warp / wk;
  const int begin = part * units / wk, end = (part + 1) * units / wk;
  // Block blockIdx + gridDim i of 16 channels is the CTA's i-th.
  const int blocks = (a.n + 15) >> 4, stride = gridDim.x * wc;
  const Int4Masks masks = int4_masks();
  w4_prefetch(a, int(blockIdx.x + gridDim.x * which), begin, min(begin + 2, end));
  pdl_wait();
  pdl_launch_dependents();

  // The next two chunks to copy: a row for every two lanes, which have alternate
  // 16-byte pieces of it.  Rows past the last are left as they are.
  int next_block = int(blockIdx.x + gridDim.x * which), next = begin;
  bool mine = false;
  const uint8_t *src = nullptr;
  const __nv_bfloat16 *scale_src = nullptr;
  const uint32_t ring_at = smem_u32(ring);
  int turn = Shape::kStage;
  uint32_t to = ring_at + w4_place(lane >> 1, lane & 1), scale_to = ring_at + 2048 + (lane >> 1) * 16;
  auto at_block = [&]() {
    const int row = next_block * 16 + (lane >> 1);
    mine = row < a.n;
    src = a.w + int64_t(row) * (a.k >> 1) + begin * 128 + (lane & 1) * 16;
    scale_src = a.scales + int64_t(row) * groups + begin * 2 * kPieces;
  };
  auto copy = [&]() {
    if (next_block < blocks && begin < end) {
      if (mine) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          cp_async_16_at((i & 1 ? to ^ 32 : to) + (i >> 1) * 1024, src + i * 32);
        if ((lane & 1) == 0) {
          if constexpr (kPieces == 4)
            cp_async_16_at(scale_to, scale_src);
          else
            cp_async_ca<4 * kPieces>(scale_to, scale_src);
        }
      }
      src += 128;
      scale_src += 2 * kPieces;
      if (++next == end) {
        next = begin;
        next_block += stride;
        at_block();
      }
    }
    to += turn, scale_to += turn, turn = -turn;     // the other stage
    cp_async_commit();
  };
  at_block();
  copy();

  // The rows as the lanes take them.
  for (int i = warp; i < groups * kWords; i += kWarps) {
    uint4 x = make_uint4(0, 0, 0, 0);
    if (g < a.m)
      x = *reinterpret_cast<const uint4 *>(a.x + g * a.ldx + i / kWords * kGroup + q4 * (kGroup / 4) + i % kWords * 8);
    xs[i * 32 + lane] = w4_order(x);
  }
  __syncthreads();

  int stage = 0;
  for (int base = int(blockIdx.x); base < blocks; base += stride) {
    const int block = base + int(gridDim.x) * which, c0 = block * 16;
    float acc[4] = {};
    auto chunk = [&](int unit, auto second) {
      constexpr int kSecond = second.value;
      const int ch = 2 * unit + kSecond;
      const uint8_t *at = ring + stage * Shape::kStage + kSecond * 1024;
      uint32_t w[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
          const uint8_t *row = at + h * 512;
          if constexpr (kPieces == 1)
            load_words<4>(w[h], row + w4_place(g, q4));
          else if constexpr (kPieces == 2)
            load_words<2>(w[h] + 2 * p, row + w4_place(g, 2 * p + (q4 >> 1)) + (q4 & 1) * 8);
          else
            w[h][p] = *reinterpret_cast<const uint32_t *>(row + w4_place(g, p) + q4 * 4);
        }
      }
      float s[2][kPieces];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t *words = reinterpret_cast<const uint32_t *>(ring + stage * Shape::kStage + 2048 + (g + h * 8) * 16);
        if constexpr (kPieces == 1) {
          s[h][0] = __uint_as_float(kSecond ? words[0] & 0xffff0000u : words[0] << 16);
        } else {
#pragma unroll
          for (int p = 0; p < kPieces; p += 2) {
            const float2 two = bf16_pair(words[kSecond * kPieces / 2 + p / 2]);
            s[h][p] = two.x, s[h][p + 1] = two.y;
          }
        }
      }
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
        float sums[4] = {};
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          const uint32_t u = w[0][p * kWords + i], v = w[1][p * kWords + i];
          const uint4 x = xs[(ch * 4 + p * kWords + i) * 32 + lane];
          const uint32_t first[4] = {w4_pair<0>(u, masks), w4_pair<0>(v, masks), w4_pair<1>(u, masks), w4_pair<1>(v, masks)};
          const uint32_t last[4] = {w4_pair<2>(u, masks), w4_pair<2>(v, masks), w4_pair<3>(u, masks), w4_pair<3>(v, masks)};
          mma_bf16_16816(sums, first, x.x, x.y);
          mma_bf16_16816(sums, last, x.z, x.w);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[e] = fmaf(sums[e], s[e >> 1][p], acc[e]);
      }
    };
    if (block < blocks) {
#pragma unroll 1
      for (int unit = begin; unit < end; ++unit) {
        cp_async_wait_group<0>();
        __syncwarp();                               // all lanes' copies of this stage; all have read the last one
        copy();
        chunk(unit, std::integral_constant<int, 0>{});
        chunk(unit, std::integral_constant<int, 1>{});
        stage ^= 1;
      }
    }
    if (wk == 1) {
      if (block < blocks) {
        const float b0 = a.bias && c0 + g < a.n ? __bfloat162float(a.bias[c0 + g]) : 0.f;
        const float b1 = a.bias && c0 + g + 8 < a.n ? __bfloat162float(a.bias[c0 + g + 8]) : 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float b = h ? b1 : b0;              // token g, channels 2 q4 and 2 q4 + 1 of the half
          const uint32_t y = transpose_8x8(pack_bf16x2(fmaf(acc[2 * h], kW4Up, b), fmaf(acc[2 * h + 1], kW4Up, b)));
          const int c = c0 + h * 8 + 2 * q4;
          uint16_t *out = reinterpret_cast<uint16_t *>(a.out + g * a.ldo + c);
          const bool one = g < a.m && c < a.n, two = g < a.m && c + 1 < a.n;
          if (two && a.pairs) {
            *reinterpret_cast<uint32_t *>(out) = y;
          } else {
            if (one)
              out[0] = uint16_t(y);
            if (two)
              out[1] = uint16_t(y >> 16);
          }
        }
      }
      continue;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      red[(warp * kCols + 2 * q4 + (e & 1)) * Shape::kRedRow + g + (e >> 1) * 8] = acc[e];
    __syncthreads();
    for (int i = threadIdx.x; i < wc * kCols * 16; i += kWarps * 32) {
      const int c = i % 16, token = i / 16 % kCols, of = i / (16 * kCols), channel = (base + int(gridDim.x) * of) * 16 + c;
      if (token >= a.m || channel >= a.n)
        continue;
      float sum = 0.f;
      for (int x = 0; x < wk; ++x)                  // in order of K
        sum += red[((of * wk + x) * kCols + token) * Shape::kRedRow + c];
      const float bias = a.bias != nullptr ? __bfloat162float(a.bias[channel]) : 0.f;
      a.out[token * a.ldo + channel] = __float2bfloat16_rn(fmaf(sum, kW4Up, bias));
    }
    __syncthreads();
  }
  cp_async_wait_group<0>();
}

// More than eight rows: they are brought into the lanes' order once for all CTAs, by
// a launch of its own, [K / 8 words of a lane][tile][lane].
template <int kGroup, int kTiles>
__global__ void __launch_bounds__(128) w4_rows_kernel(const W4Args a, uint4 *rows) {
  constexpr int kWords = kGroup / 32;
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  const int item = blockIdx.x * 4 + (threadIdx.x >> 5), i = item / kTiles, token = item % kTiles * 8 + g;
  if (i >= a.k >> 5)
    return;
  uint4 x = make_uint4(0, 0, 0, 0);
  if (token < a.m)
    x = *reinterpret_cast<const uint4 *>(a.x + token * a.ldx + i / kWords * kGroup + q4 * (kGroup / 4) + i % kWords * 8);
  rows[int64_t(item) * 32 + lane] = w4_order(x);
}

// A persistent CTA keeps those of a slab of K (all of it, where it fits) in shared
// memory and streams weights past them, 16 channels to a warp; `wk` warps split the
// slab.  The sums of a round meet where the rings were.  A weight's codes are brought
// into bf16 once for all rows of the launch.  Eight tiles take 64 registers of sums:
// eight warps, with 255 each, do 64 rows of 1024 -> 6144 in 12 us, 16 warps in 15.
template <int kTiles>
struct W4Wide {
  static constexpr int kWarps = kTiles == 8 ? 8 : 16, kCols = 8 * kTiles;
  static constexpr int kStage = 16 * (128 + 16);                 // of 256 k: codes of 16 channels, their scales
  static constexpr int kRedRow = 20;                             // words of a token's 16 sums, apart by banks
  static constexpr int kRing = kWarps * 2 * kStage, kRed = kWarps * kCols * kRedRow * 4;
  static constexpr int kMeet = kRing > kRed ? kRing : kRed;
  static constexpr int bytes(int slab) { return slab * kCols * 2 + kMeet + 16; }
};

template <int kGroup, int kTiles>
__global__ void __launch_bounds__(W4Wide<kTiles>::kWarps * 32, 1) gemm_w4_wide_kernel(const W4Args a, const uint4 *rows_of_x) {
  using Shape = W4Wide<kTiles>;
  constexpr int kPieces = 128 / kGroup, kWords = 4 / kPieces, kCols = Shape::kCols, kWarps = Shape::kWarps;
  extern __shared__ __align__(1024) uint8_t tile_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  const int groups = a.k / kGroup;
  uint4 *xs = reinterpret_cast<uint4 *>(tile_raw);                                    // [chunk][word][tile][lane]
  uint8_t *meet = tile_raw + int64_t(a.slab) * kCols * 2;
  uint8_t *ring = meet + warp * 2 * Shape::kStage;
  float *red = reinterpret_cast<float *>(meet);                                       // [warp][token][channel]
  uint64_t *full = reinterpret_cast<uint64_t *>(meet + Shape::kMeet);
  const int wk = a.wk, wc = kWarps / wk, part = warp % wk, which = warp / wk;
  const int blocks = (a.n + 15) >> 4, slabs = (a.k + a.slab - 1) / a.slab;
  const Int4Masks masks = int4_masks();
  if (threadIdx.x == 0) {
    mbar_init(full, 1);
    fence_barrier_init();
  }
  __syncthreads();
  const int units0 = min(a.slab, a.k) >> 8, block0 = int(blockIdx.x + gridDim.x * which);
  w4_prefetch(a, block0, part * units0 / wk, (part + 1) * units0 / wk);
  pdl_wait();
  pdl_launch_dependents();

  // A row for every two lanes, which have alternate 16-byte pieces of it.
  const uint32_t ring_at = smem_u32(ring);
  int loaded = 0;                                   // slabs so far
  bool ok = true;
  for (int base = int(blockIdx.x); base < blocks && ok; base += int(gridDim.x) * wc) {
    const int block = base + int(gridDim.x) * which;
    const int row = block * 16 + (lane >> 1);
    const bool live = block < blocks, mine = row < a.n;
    const uint8_t *src = a.w + int64_t(row) * (a.k >> 1) + (lane & 1) * 16;
    const __nv_bfloat16 *scale_src = a.scales + int64_t(row) * groups;
    float acc[kTiles][4] = {};
    for (int slab = 0; slab < slabs && ok; ++slab) {
      const int first = slab * a.slab, units = min(a.slab, a.k - first) >> 8;
      const int begin = part * units / wk, end = (part + 1) * units / wk;
      auto copy = [&](int unit) {
        if (live && mine && unit < end) {
          const uint32_t at = ring_at + (unit & 1) * Shape::kStage;
          const int k = first + unit * 256;
#pragma unroll
          for (int i = 0; i < 4; ++i)               // chunk i / 2, piece 2 (i % 2) + (lane & 1)
            cp_async_16_at(at + (i >> 1) * 1024 + w4_place(lane >> 1, 2 * (i & 1) + (lane & 1)), src + (k >> 1) + i * 32);
          if ((lane & 1) == 0) {
            const __nv_bfloat16 *s = scale_src + k / kGroup;
            if constexpr (kPieces == 4)
              cp_async_16_at(at + 2048 + lane * 8, s);
            else
              cp_async_ca<4 * kPieces>(at + 2048 + lane * 8, s);
          }
        }
        cp_async_commit();
      };
      copy(begin);
      if (loaded == 0 || slabs > 1) {
        if (loaded > 0)
          __syncthreads();                          // all have read the slab before
        if (threadIdx.x == 0) {
          const int bytes = units * 256 * kCols * 2;
          fence_proxy_async_smem();
          mbar_arrive_expect_tx(full, bytes);
          bulk_load(tile_raw, rows_of_x + int64_t(first >> 5) * kTiles * 32, bytes, full);
        }
        ok = __syncthreads_and(mbar_wait(full, uint32_t(loaded & 1), kStatusTimeoutProducer));
        ++loaded;
      }
      auto chunk = [&](int unit, int second) {
        const int ch = 2 * unit + second;          // of the slab
        const uint8_t *at = ring + (unit & 1) * Shape::kStage;
        uint32_t w[2][4];
        float s[2][kPieces];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint8_t *rows = at + second * 1024 + h * 512;
#pragma unroll
          for (int p = 0; p < kPieces; ++p) {
            if constexpr (kPieces == 1)
              load_words<4>(w[h], rows + w4_place(g, q4));
            else if constexpr (kPieces == 2)
              load_words<2>(w[h] + 2 * p, rows + w4_place(g, 2 * p + (q4 >> 1)) + (q4 & 1) * 8);
            else
              w[h][p] = *reinterpret_cast<const uint32_t *>(rows + w4_place(g, p) + q4 * 4);
          }
          const uint32_t *words = reinterpret_cast<const uint32_t *>(at + 2048 + (g + h * 8) * 16);
          if constexpr (kPieces == 1) {
            s[h][0] = __uint_as_float(second ? words[0] & 0xffff0000u : words[0] << 16);
          } else {
#pragma unroll
            for (int p = 0; p < kPieces; p += 2) {
              const float2 two = bf16_pair(words[second * kPieces / 2 + p / 2]);
              s[h][p] = two.x, s[h][p + 1] = two.y;
            }
          }
        }
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
          float sums[kTiles][4] = {};
#pragma unroll
          for (int i = 0; i < kWords; ++i) {
            const uint32_t u = w[0][p * kWords + i], v = w[1][p * kWords + i];
            const uint32_t first[4] = {w4_pair<0>(u, masks), w4_pair<0>(v, masks), w4_pair<1>(u, masks), w4_pair<1>(v, masks)};
            const uint32_t last[4] = {w4_pair<2>(u, masks), w4_pair<2>(v, masks), w4_pair<3>(u, masks), w4_pair<3>(v, masks)};
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
              const uint4 x = xs[((ch * 4 + p * kWords + i) * kTiles + t) * 32 + lane];
              mma_bf16_16816(sums[t], first, x.x, x.y);
              mma_bf16_16816(sums[t], last, x.z, x.w);
            }
          }
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              acc[t][e] = fmaf(sums[t][e], s[e >> 1][p], acc[t][e]);
        }
      };
#pragma unroll 1
      for (int unit = begin; unit < end && live; ++unit) {
        cp_async_wait_group<0>();
        __syncwarp();                               // all lanes' copies of this unit; all have read the last one
        copy(unit + 1);
#pragma unroll 1
        for (int second = 0; second < 2; ++second)
          chunk(unit, second);
      }
      __syncwarp();
    }
    cp_async_wait_group<0>();
    __syncthreads();                                // the rings are read
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        red[(warp * kCols + t * 8 + 2 * q4 + (e & 1)) * Shape::kRedRow + g + (e >> 1) * 8] = acc[t][e];
    __syncthreads();
    for (int i = threadIdx.x >> 4; i < wc * a.m && ok; i += kWarps * 2) {
      const int of = i / a.m, token = i % a.m, c = lane & 15, channel = (base + int(gridDim.x) * of) * 16 + c;
      if (channel >= a.n)
        continue;
      float sum = 0.f;
      for (int x = 0; x < wk; ++x)                  // in order of K
        sum += red[((of * wk + x) * kCols + token) * Shape::kRedRow + c];
      const float bias = a.bias != nullptr ? __bfloat162float(a.bias[channel]) : 0.f;
      a.out[token * a.ldo + channel] = __float2bfloat16_rn(fmaf(sum, kW4Up, bias));
    }
    __syncthreads();
  }
  if (!ok && threadIdx.x == 0)                      // a copy may still be on its way
    mbar_wait(full, uint32_t((loaded - 1) & 1), kStatusTimeoutProducer);
}

} // namespace pir2b
