// Products of a few bf16 rows with weights held in 4 bits:
//   out[m, n] = bf16(sum_k x[m, k] code[n, k] scale[n, k / G] + bias[n]),
// codes of -8..7 in two's complement, two to a byte with the even k in the low
// bits, G = 32, 64 or 128 consecutive weights of a channel per bf16 scale.
//
// Few rows cannot fill a tcgen05 tile and the work is reading the weights, so
// the products run on warp-level MMAs (m16n8k16, fp32 sums) with channels as the
// M rows.  A CTA owns 16 channels; its warps split K in chunks of 128.  Codes
// become bf16 in registers, exactly: a nibble moved to bits 3-6 of 16 makes 16 +
// u, u = code + 8, from which 24 is taken.  The four lanes of a channel take
// pieces of one group each, so a product step stays in a group, whose sums are
// scaled in fp32.
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
  int wk, stages;                // staged: warps that split K, of their rings
  int pairs;                     // output channels may be stored two at a time
};

// Code kAt of each half of a word as a bf16 pair.
template <int kAt>
__device__ __forceinline__ uint32_t w4_pair(uint32_t w, const Int4Masks &m) {
  const uint32_t t = kAt == 0 ? w << 3 : w >> (kAt == 0 ? 0 : 4 * kAt - 3);
  return bf162_fma(masked_xor<0x41c041c0u>(t, m.mantissa), 0x3f803f80u, 0xc1c0c1c0u);
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
      if (a.bias != nullptr)
        sum += __bfloat162float(a.bias[channel]);
      a.out[token * a.ldo + channel] = __float2bfloat16_rn(sum);
    }
    if (block + gridDim.x < blocks)
      __syncthreads();
  }
}

// Many channels: a persistent CTA keeps all rows in shared memory, as the lanes
// take them, and streams the weights of its blocks of 16 channels through a ring
// per warp; `wk` warps split K, and their sums meet in shared memory.
//
// x enters as fp16: a power of two brings a row's largest value to 2^10, below
// which fp16 holds the row to 2^-35 of that value.  fp16 has room for a code in
// two places: with u = code + 8, bits 2-5 make 64 + u / 4 (even k) and bits 6-9 4 +
// u / 4 (odd k), so a word of eight needs two shifts, and none of the eight a
// subtraction: a group's sums start at -66 (-6) times the sum of its even (odd) x,
// which is made once per CTA.  The fp32 sums then pass through values some 100
// times a typical result, which costs 2^-14 of it.  Where a row holds a value that
// is not finite the codes themselves are taken instead.
template <int kTiles>
struct W4Shape {
  static constexpr int kWarps = kTiles == 1 ? 24 : 16;
  static constexpr int kMostStages = 2;
  static constexpr int kCols = 8 * kTiles;
  static constexpr int kStage = 2 * (1024 + 128);        // of two chunks: codes of 16 channels, 16 bytes for each one's scales
  static constexpr int kRedRow = 20;                     // words of a token's 16 sums, apart by banks
  static constexpr int kRed = kWarps * kCols * kRedRow * 4;
  static constexpr int bytes(int64_t k, int group, int stages) {
    return int(k * kCols * 2 + k / group * kCols * 4) + kWarps * stages * kStage + kRed + kCols * 4;
  }
};

// Place of 16-byte piece c of row r: pieces of eight rows read in any width lie
// in different banks.
__device__ __forceinline__ int w4_place(int r, int c) { return r * 64 + ((c ^ ((r & 2) | ((r >> 2) & 1))) << 4); }

template <int kBytes>
__device__ __forceinline__ void cp_async_ca(uint32_t dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(kBytes) : "memory");
}

template <int kGroup, int kTiles>
__global__ void __launch_bounds__(W4Shape<kTiles>::kWarps * 32, 1) gemm_w4_staged_kernel(const W4Args a) {
  using Shape = W4Shape<kTiles>;
  constexpr int kPieces = 128 / kGroup, kWords = 4 / kPieces, kCols = Shape::kCols, kWarps = Shape::kWarps;
  extern __shared__ __align__(1024) uint8_t tile_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  const int units = a.k >> 8, groups = a.k / kGroup;      // units of two chunks
  uint4 *xs = reinterpret_cast<uint4 *>(tile_raw);                           // [chunk][word][tile][lane]
  float *offsets = reinterpret_cast<float *>(tile_raw + int64_t(a.k) * kCols * 2);   // [group][token]
  uint8_t *ring = reinterpret_cast<uint8_t *>(offsets + groups * kCols) + warp * a.stages * Shape::kStage;
  float *red = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(offsets + groups * kCols) + kWarps * a.stages * Shape::kStage);
  uint32_t *most = reinterpret_cast<uint32_t *>(red + Shape::kRed / 4);      // [token] largest magnitude
  const int wk = a.wk, wc = kWarps / wk, part = warp % wk, which = warp / wk;
  const int begin = part * units / wk, end = (part + 1) * units / wk;
  // Block blockIdx + gridDim i of 16 channels is the CTA's i-th.
  const int blocks = (a.n + 15) >> 4, stride = gridDim.x * wc;
  const Int4Masks masks = int4_masks();
  pdl_wait();
  pdl_launch_dependents();

  // The next two chunks to copy: a row for every two lanes, which have alternate
  // 16-byte pieces of it.  Rows past the last are left as they are.
  int next_block = int(blockIdx.x + gridDim.x * which), next = begin;
  bool mine = false;
  const uint8_t *src = nullptr;
  const __nv_bfloat16 *scale_src = nullptr;
  const uint32_t ring_at = smem_u32(ring);
  int stage_in = 0;
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
    const int step = ++stage_in == a.stages ? Shape::kStage - a.stages * Shape::kStage : Shape::kStage;
    stage_in = stage_in == a.stages ? 0 : stage_in;
    to += step, scale_to += step;
    cp_async_commit();
  };
  at_block();
  for (int i = 0; i < a.stages - 1; ++i)
    copy();

  // The rows' largest finite magnitudes, 256 values of a row at a time.
  for (int i = threadIdx.x; i < kCols; i += kWarps * 32)
    most[i] = 0;
  __syncthreads();
  bool odd_values = false;
  const int segments = units;
  for (int i = warp; i < a.m * segments; i += kWarps) {
    const int token = i / segments, at = (i % segments) * 256 + lane * 8;
    const uint4 x = *reinterpret_cast<const uint4 *>(a.x + token * a.ldx + at);
    uint32_t m = magnitude8(x);
    if (m >= 0x7f80u) {
      odd_values = true;
      m = magnitude8_finite(x);
      m = m > 0x7f80u ? 0 : m;                      // a NaN
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0)
      atomicMax(&most[token], m);
  }
  const bool alone = __syncthreads_or(odd_values);
  // Exponent field of a row's power of two.
  auto power_of = [&](int token) { return most[token] == 0 ? 127 : min(264 - int(most[token] >> 7), 253); };
  // The rows as the lanes take them: a warp makes a group at a time.
  for (int i = warp; i < groups * kTiles; i += kWarps) {
    const int group = i / kTiles, t = i % kTiles, token = t * 8 + g;
    const float factor = __int_as_float(power_of(token) << 23);
    float even = 0.f, odd = 0.f;
#pragma unroll
    for (int j = 0; j < kWords; ++j) {
      uint4 x = make_uint4(0, 0, 0, 0);
      if (token < a.m)
        x = *reinterpret_cast<const uint4 *>(a.x + token * a.ldx + group * kGroup + q4 * (kGroup / 4) + j * 8);
      uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float2 v = bf16_pair(y[c]);
        y[c] = pack_half2(v.x * factor, v.y * factor);
        const float2 r = __half22float2(*reinterpret_cast<const __half2 *>(&y[c]));
        even += r.x, odd += r.y;
      }
      xs[((group * kWords + j) * kTiles + t) * 32 + lane] =
          make_uint4(__byte_perm(y[0], y[2], 0x5410), __byte_perm(y[0], y[2], 0x7632), __byte_perm(y[1], y[3], 0x5410),
                     __byte_perm(y[1], y[3], 0x7632));
    }
    float sum = -66.f * even - 6.f * odd;
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    if (q4 == 0)
      offsets[group * kCols + token] = alone ? 0.f : sum;
  }
  __syncthreads();

  auto undo = [&](int token) { return 4.f * __int_as_float((254 - power_of(token)) << 23); };
  int stage = 0;
  for (int base = int(blockIdx.x); base < blocks; base += stride) {
    const int block = base + int(gridDim.x) * which, c0 = block * 16;
    float acc[kTiles][4] = {};
    auto chunk = [&](int unit, auto second, auto codes_alone) {
      constexpr bool kAlone = codes_alone.value;
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
            *reinterpret_cast<uint4 *>(w[h]) = *reinterpret_cast<const uint4 *>(row + w4_place(g, q4));
          else if constexpr (kPieces == 2)
            *reinterpret_cast<uint2 *>(w[h] + 2 * p) = *reinterpret_cast<const uint2 *>(row + w4_place(g, 2 * p + (q4 >> 1)) + (q4 & 1) * 8);
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
        float sums[kTiles][4];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          const float2 o = *reinterpret_cast<const float2 *>(offsets + (ch * kPieces + p) * kCols + t * 8 + 2 * q4);
          sums[t][0] = sums[t][2] = o.x, sums[t][1] = sums[t][3] = o.y;
        }
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          const uint32_t u = w[0][p * kWords + i], v = w[1][p * kWords + i];
          auto low = [&](uint32_t x) {              // places 0 and 4 of a word, or 2 and 6
            const uint32_t y = masked_xor<0x54205420u>(x, masks.low);
            return kAlone ? half2_fma(y, 0x3c003c00u, 0xd420d420u) : y;
          };
          auto high = [&](uint32_t x) {             // 1 and 5, or 3 and 7
            const uint32_t y = masked_xor<0x46004600u>(x, masks.high);
            return kAlone ? half2_fma(y, 0x3c003c00u, 0xc600c600u) : y;
          };
          const uint32_t first[4] = {low(u << 2), low(v << 2), high(u << 2), high(v << 2)};
          const uint32_t last[4] = {low(u >> 6), low(v >> 6), high(u >> 6), high(v >> 6)};
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            const uint4 x = xs[((ch * 4 + p * kWords + i) * kTiles + t) * 32 + lane];
            mma_half_16816(sums[t], first, x.x, x.y);
            mma_half_16816(sums[t], last, x.z, x.w);
          }
        }
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[t][e] = fmaf(sums[t][e], s[e >> 1][p], acc[t][e]);
      }
    };
    if (block < blocks) {
#pragma unroll 1
      for (int unit = begin; unit < end; ++unit) {
        if (a.stages == 2)
          cp_async_wait_group<0>();
        else if (a.stages == 3)
          cp_async_wait_group<1>();
        else
          cp_async_wait_group<2>();
        __syncwarp();                               // all lanes' copies of this stage; all have read the last one
        copy();
        if (!alone) {
          chunk(unit, std::integral_constant<int, 0>{}, std::false_type{});
          chunk(unit, std::integral_constant<int, 1>{}, std::false_type{});
        } else {
          chunk(unit, std::integral_constant<int, 0>{}, std::true_type{});
          chunk(unit, std::integral_constant<int, 1>{}, std::true_type{});
        }
        stage = stage == a.stages - 1 ? 0 : stage + 1;
      }
    }
    if (wk == 1) {
      if (block < blocks) {
        const float b0 = a.bias && c0 + g < a.n ? __bfloat162float(a.bias[c0 + g]) : 0.f;
        const float b1 = a.bias && c0 + g + 8 < a.n ? __bfloat162float(a.bias[c0 + g + 8]) : 0.f;
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float b = h ? b1 : b0;            // token g, channels 2 q4 and 2 q4 + 1 of the half
            const uint32_t y = transpose_8x8(pack_bf16x2(fmaf(acc[t][2 * h], undo(t * 8 + 2 * q4), b),
                                                         fmaf(acc[t][2 * h + 1], undo(t * 8 + 2 * q4 + 1), b)));
            const int token = t * 8 + g, c = c0 + h * 8 + 2 * q4;
            uint16_t *out = reinterpret_cast<uint16_t *>(a.out + token * a.ldo + c);
            const bool first = token < a.m && c < a.n, second = token < a.m && c + 1 < a.n;
            if (second && a.pairs) {
              *reinterpret_cast<uint32_t *>(out) = y;
            } else {
              if (first)
                out[0] = uint16_t(y);
              if (second)
                out[1] = uint16_t(y >> 16);
            }
          }
      }
      continue;
    }
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        red[(warp * kCols + t * 8 + 2 * q4 + (e & 1)) * Shape::kRedRow + g + (e >> 1) * 8] = acc[t][e];
    __syncthreads();
    for (int i = threadIdx.x; i < wc * kCols * 16; i += kWarps * 32) {
      const int c = i % 16, token = i / 16 % kCols, of = i / (16 * kCols), channel = (base + int(gridDim.x) * of) * 16 + c;
      if (token >= a.m || channel >= a.n)
        continue;
      float sum = 0.f;
      for (int x = 0; x < wk; ++x)                  // in order of K
        sum += red[((of * wk + x) * kCols + token) * Shape::kRedRow + c];
      const float b = a.bias != nullptr ? __bfloat162float(a.bias[channel]) : 0.f;
      a.out[token * a.ldo + channel] = __float2bfloat16_rn(fmaf(sum, undo(token), b));
    }
    __syncthreads();
  }
  cp_async_wait_group<0>();
}

// More than eight rows.  What a product takes of x is then made once for all CTAs,
// by a launch of its own: the rows as the lanes take them, [K / 8 words of a lane][tile]
// [lane], and -24 times each group's sum (24 + code needs no subtraction, as above),
// with a word that says whether a value of the group is past 2^100 or not finite.
struct W4Rows {
  uint4 *x;            // [4 chunks][tiles][32]
  float *offsets;      // [groups][8 tiles]
  uint32_t *odd;       // [groups][tiles]
};

template <int kGroup, int kTiles>
__global__ void __launch_bounds__(128) w4_rows_kernel(const W4Args a, const W4Rows r) {
  constexpr int kWords = kGroup / 32;
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  const int item = blockIdx.x * 4 + (threadIdx.x >> 5), group = item / kTiles, t = item % kTiles, token = t * 8 + g;
  if (group >= a.k / kGroup)
    return;
  float sum = 0.f;
  bool odd = false;
  uint4 x[kWords];
#pragma unroll
  for (int j = 0; j < kWords; ++j) {
    x[j] = make_uint4(0, 0, 0, 0);
    if (token < a.m)
      x[j] = *reinterpret_cast<const uint4 *>(a.x + token * a.ldx + group * kGroup + q4 * (kGroup / 4) + j * 8);
  }
#pragma unroll
  for (int j = 0; j < kWords; ++j) {
    odd |= magnitude8(x[j]) >= (227u << 7);
    const float2 p = bf16_pair(x[j].x), q = bf16_pair(x[j].y), u = bf16_pair(x[j].z), v = bf16_pair(x[j].w);
    sum += ((p.x + p.y) + (q.x + q.y)) + ((u.x + u.y) + (v.x + v.y));
    r.x[(int64_t(group * kWords + j) * kTiles + t) * 32 + lane] =
        make_uint4(__byte_perm(x[j].x, x[j].z, 0x5410), __byte_perm(x[j].x, x[j].z, 0x7632),
                   __byte_perm(x[j].y, x[j].w, 0x5410), __byte_perm(x[j].y, x[j].w, 0x7632));
  }
  sum += __shfl_xor_sync(0xffffffffu, sum, 1);
  sum += __shfl_xor_sync(0xffffffffu, sum, 2);
  odd = __any_sync(0xffffffffu, odd);
  if (q4 == 0)
    r.offsets[group * 8 * kTiles + token] = -24.f * sum;
  if (lane == 0)
    r.odd[group * kTiles + t] = odd;
}

// A persistent CTA keeps those of a slab of K (all of it, where it fits) in shared
// memory and streams weights past them, 16 channels to a warp; `wk` warps split the
// slab.  The sums of a round meet where the rings were.
template <int kTiles>
struct W4Wide {
  static constexpr int kWarps = 16, kCols = 8 * kTiles;
  static constexpr int kStage = 16 * (128 + 16);                 // of 256 k: codes of 16 channels, their scales
  static constexpr int kRedRow = 20;                             // words of a token's 16 sums, apart by banks
  static constexpr int kRing = kWarps * 2 * kStage, kRed = kWarps * kCols * kRedRow * 4;
  static constexpr int kMeet = kRing > kRed ? kRing : kRed;
  static constexpr int bytes(int slab, int group) { return slab * kCols * 2 + slab / group * kCols * 4 + kMeet + 16; }
};

template <int kGroup, int kTiles>
__global__ void __launch_bounds__(W4Wide<kTiles>::kWarps * 32, 1) gemm_w4_wide_kernel(const W4Args a, const W4Rows r) {
  using Shape = W4Wide<kTiles>;
  constexpr int kPieces = 128 / kGroup, kWords = 4 / kPieces, kCols = Shape::kCols, kWarps = Shape::kWarps;
  extern __shared__ __align__(1024) uint8_t tile_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  const int groups = a.k / kGroup, slab_groups = a.slab / kGroup;
  uint4 *xs = reinterpret_cast<uint4 *>(tile_raw);                                    // [chunk][word][tile][lane]
  float *offsets = reinterpret_cast<float *>(tile_raw + int64_t(a.slab) * kCols * 2);  // [group][token]
  uint8_t *meet = reinterpret_cast<uint8_t *>(offsets + slab_groups * kCols);
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
  pdl_wait();
  pdl_launch_dependents();
  bool odd = false;
  for (int i = threadIdx.x; i < groups * kTiles; i += kWarps * 32)
    odd |= r.odd[i] != 0;
  const bool alone = __syncthreads_or(odd);

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
          const int g0 = first / kGroup, bytes_x = units * 256 * kCols * 2, bytes_o = units * 256 / kGroup * kCols * 4;
          fence_proxy_async_smem();
          mbar_arrive_expect_tx(full, bytes_x + bytes_o);
          bulk_load(xs, r.x + int64_t(first >> 5) * kTiles * 32, bytes_x, full);
          bulk_load(offsets, r.offsets + g0 * kCols, bytes_o, full);
        }
        ok = __syncthreads_and(mbar_wait(full, uint32_t(loaded & 1), kStatusTimeoutProducer));
        ++loaded;
      }
      auto chunk = [&](int unit, auto second, auto codes_alone) {
        constexpr bool kAlone = codes_alone.value;
        constexpr int kSecond = second.value;
        const int ch = 2 * unit + kSecond;          // of the slab
        const uint8_t *at = ring + (unit & 1) * Shape::kStage;
        uint32_t w[2][4];
        float s[2][kPieces];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint8_t *rows = at + kSecond * 1024 + h * 512;
#pragma unroll
          for (int p = 0; p < kPieces; ++p) {
            if constexpr (kPieces == 1)
              *reinterpret_cast<uint4 *>(w[h]) = *reinterpret_cast<const uint4 *>(rows + w4_place(g, q4));
            else if constexpr (kPieces == 2)
              *reinterpret_cast<uint2 *>(w[h] + 2 * p) = *reinterpret_cast<const uint2 *>(rows + w4_place(g, 2 * p + (q4 >> 1)) + (q4 & 1) * 8);
            else
              w[h][p] = *reinterpret_cast<const uint32_t *>(rows + w4_place(g, p) + q4 * 4);
          }
          const uint32_t *words = reinterpret_cast<const uint32_t *>(at + 2048 + (g + h * 8) * 16);
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
          float sums[kTiles][4];
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            const float2 o = kAlone ? make_float2(0.f, 0.f)
                                    : *reinterpret_cast<const float2 *>(offsets + (ch * kPieces + p) * kCols + t * 8 + 2 * q4);
            sums[t][0] = sums[t][2] = o.x, sums[t][1] = sums[t][3] = o.y;
          }
#pragma unroll
          for (int i = 0; i < kWords; ++i) {
            uint32_t even[4], last[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t u = w[h][p * kWords + i];
              auto pair = [&](uint32_t t) {
                const uint32_t y = masked_xor<0x41c041c0u>(t, masks.mantissa);
                return kAlone ? bf162_fma(y, 0x3f803f80u, 0xc1c0c1c0u) : y;
              };
              even[h] = pair(u << 3), even[h + 2] = pair(u >> 1);
              last[h] = pair(u >> 5), last[h + 2] = pair(u >> 9);
            }
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
              const uint4 x = xs[((ch * 4 + p * kWords + i) * kTiles + t) * 32 + lane];
              mma_bf16_16816(sums[t], even, x.x, x.y);
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
        if (alone) {
          chunk(unit, std::integral_constant<int, 0>{}, std::true_type{});
          chunk(unit, std::integral_constant<int, 1>{}, std::true_type{});
        } else {
          chunk(unit, std::integral_constant<int, 0>{}, std::false_type{});
          chunk(unit, std::integral_constant<int, 1>{}, std::false_type{});
        }
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
      if (a.bias != nullptr)
        sum += __bfloat162float(a.bias[channel]);
      a.out[token * a.ldo + channel] = __float2bfloat16_rn(sum);
    }
    __syncthreads();
  }
}

} // namespace pir2b
