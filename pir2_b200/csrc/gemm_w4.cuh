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

constexpr int kW4Channels = 16, kW4Warps = 8;

struct W4Args {
  const __nv_bfloat16 *x;        // [m, k], row stride ldx
  int64_t ldx;
  const uint8_t *w;              // [n, k / 2]
  const __nv_bfloat16 *scales;   // [n, k / G]
  const __nv_bfloat16 *bias;     // [n] or null
  __nv_bfloat16 *out;            // [m, n], row stride ldo
  int64_t ldo;
  int m, n, k;
};

// Code kAt of each half of a word as a bf16 pair.
template <int kAt>
__device__ __forceinline__ uint32_t w4_pair(uint32_t w) {
  const uint32_t t = kAt == 0 ? w << 3 : w >> (kAt == 0 ? 0 : 4 * kAt - 3);
  return bf162_fma((t & 0x00780078u) ^ 0x41c041c0u, 0x3f803f80u, 0xc1c0c1c0u);
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

template <int kGroup, int kTiles>
__global__ void __launch_bounds__(kW4Warps * 32) gemm_w4_kernel(const W4Args a) {
  constexpr int kPieces = 128 / kGroup, kWords = 4 / kPieces;   // of a lane and chunk; words of a piece
  constexpr int kCols = 8 * kTiles;
  __shared__ float red[kW4Warps][kCols][kW4Channels];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  const int c0 = blockIdx.x * kW4Channels, groups = a.k / kGroup;
  const int chunks = (a.k + 127) >> 7;
  const int begin = warp * chunks / kW4Warps, end = (warp + 1) * chunks / kW4Warps;
  const int row[2] = {min(c0 + g, a.n - 1), min(c0 + g + 8, a.n - 1)};   // rows past the last are not stored
  float acc[kTiles][4] = {};
  pdl_wait();
  pdl_launch_dependents();
#pragma unroll 1
  for (int ch = begin; ch < end; ++ch) {
    const int left = groups - ch * kPieces;
    uint32_t w[2][4];
    float s[2][kPieces];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      w4_load<kPieces>(w[h], a.w + int64_t(row[h]) * (a.k >> 1) + ch * 64 + q4 * (16 / kPieces), left);
#pragma unroll
      for (int p = 0; p < kPieces; ++p)
        s[h][p] = p < left ? __bfloat162float(a.scales[int64_t(row[h]) * groups + ch * kPieces + p]) : 0.f;
    }
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      float part[kTiles][4] = {};
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        const uint32_t u = w[0][p * kWords + i], v = w[1][p * kWords + i];
        const uint32_t even[4] = {w4_pair<0>(u), w4_pair<0>(v), w4_pair<1>(u), w4_pair<1>(v)};
        const uint32_t odd[4] = {w4_pair<2>(u), w4_pair<2>(v), w4_pair<3>(u), w4_pair<3>(v)};
        const int k = ch * 128 + p * kGroup + q4 * (kGroup / 4) + i * 8;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          const int token = t * 8 + g;
          uint4 x = make_uint4(0, 0, 0, 0);
          if (token < a.m && p < left)
            x = *reinterpret_cast<const uint4 *>(a.x + token * a.ldx + k);
          mma_bf16_16816(part[t], even, __byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632));
          mma_bf16_16816(part[t], odd, __byte_perm(x.y, x.w, 0x5410), __byte_perm(x.y, x.w, 0x7632));
        }
      }
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[t][e] = fmaf(part[t][e], s[e >> 1][p], acc[t][e]);
    }
  }
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      red[warp][t * 8 + 2 * q4 + (e & 1)][g + (e >> 1) * 8] = acc[t][e];
  __syncthreads();
  for (int i = threadIdx.x; i < kCols * kW4Channels; i += kW4Warps * 32) {
    const int token = i / kW4Channels, c = i % kW4Channels;
    if (token >= a.m || c0 + c >= a.n)
      continue;
    float sum = 0.f;
#pragma unroll
    for (int x = 0; x < kW4Warps; ++x)
      sum += red[x][token][c];
    if (a.bias != nullptr)
      sum += __bfloat162float(a.bias[c0 + c]);
    a.out[token * a.ldo + c0 + c] = __float2bfloat16_rn(sum);
  }
}

} // namespace pir2b
