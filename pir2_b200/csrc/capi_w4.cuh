// C ABI of the products with 4-bit weights: argument checks and launches.
#pragma once
#include "capi_cache.cuh"
#include "gemm_w4.cuh"

namespace pir2b {

constexpr int kW4Rows = 64;   // rows of a launch

// How many warps split K in the staged kernel: the fewest rounds of chunks of
// 128, a round's meeting counted as one more.
static int w4_split(const W4Args &a, int warps, int ctas) {
  const int64_t blocks = (a.n + 15) / 16, units = a.k / 256;
  int best = 1;
  int64_t least = INT64_MAX;
  for (int wk = 1; wk <= warps && warps % wk == 0; wk *= 2) {
    const int64_t wc = warps / wk, rounds = ((blocks + ctas - 1) / ctas + wc - 1) / wc;
    const int64_t cost = rounds * (2 * ((units + wk - 1) / wk) + (wk > 1));
    if (cost < least)
      least = cost, best = wk;
  }
  return best;
}

static std::atomic<int> g_w4_mode{0};   // probe

template <int kGroup, int kTiles>
static int launch_w4(W4Args a, const DeviceInfo *dev, void *stream) {
  using Shape = W4Shape<kTiles>;
  const int limit = 227 * 1024;
  a.stages = Shape::kMostStages;
  while (a.stages > 2 && Shape::bytes(a.k, kGroup, a.stages) > limit)
    --a.stages;
  const int smem = Shape::bytes(a.k, kGroup, a.stages);
  const int mode = g_w4_mode.load();
  const bool fits = a.k % 256 == 0 && smem <= limit && aligned(a.scales, 16);
  if (fits && (mode == 2 || (mode == 0 && a.n >= 8192))) {
    const int64_t ctas = dev->sms;
    a.wk = w4_split(a, Shape::kWarps, int(ctas));
    const int64_t grid = std::min<int64_t>(ctas, (a.n + 15) / 16);
    cudaFuncSetAttribute(gemm_w4_staged_kernel<kGroup, kTiles>, cudaFuncAttributeMaxDynamicSharedMemorySize, limit);
    return launch_cache("gemm_w4a16 launch", gemm_w4_staged_kernel<kGroup, kTiles>, grid, 1, 1, Shape::kWarps * 32, smem, stream, a);
  }
  if constexpr (kTiles > 1) {
    if (mode == 3 && a.k % 256 == 0) {
      static uint8_t *ws = nullptr;
      if (!ws) cudaMalloc(&ws, 64 << 20);
      W4Rows r;
      r.x = reinterpret_cast<uint4 *>(ws);
      r.offsets = reinterpret_cast<float *>(ws + (32 << 20));
      r.odd = reinterpret_cast<uint32_t *>(ws + (48 << 20));
      const int64_t items = a.k / kGroup * kTiles;
      if (int x = launch_cache("w4 rows launch", w4_rows_kernel<kGroup, kTiles>, (items + 3) / 4, 1, 1, 128, 0, stream, a, r))
        return x;
      using Wide = W4Wide<kTiles>;
      a.slab = a.k;
      while (Wide::bytes(a.slab, kGroup) > limit)
        a.slab = (a.slab / 2 + 255) / 256 * 256;
      cudaFuncSetAttribute(gemm_w4_wide_kernel<kGroup, kTiles>, cudaFuncAttributeMaxDynamicSharedMemorySize, limit);
      const int64_t blocks = (a.n + 15) / 16, grid = std::min<int64_t>(blocks, dev->sms);
      int64_t least = INT64_MAX;
      const int slabs = (a.k + a.slab - 1) / a.slab;
      for (int wk = 1; wk <= Wide::kWarps; wk *= 2) {
        const int64_t wc = Wide::kWarps / wk, rounds = ((blocks + grid - 1) / grid + wc - 1) / wc;
        const int64_t cost = rounds * (slabs * 2 * ((a.slab / 256 + wk - 1) / wk) + 2);
        if (cost < least)
          least = cost, a.wk = wk;
      }
      return launch_cache("gemm_w4a16 launch", gemm_w4_wide_kernel<kGroup, kTiles>, grid, 1, 1, Wide::kWarps * 32,
                          Wide::bytes(a.slab, kGroup), stream, a, r);
    }
  }
  // Long K is split over twice the warps; a CTA takes several blocks of channels
  // only where more CTAs would not fit at once, and reads its rows through L1.
  const int warps = a.k >= 4096 ? 16 : 8, smem2 = warps * 8 * kTiles * 20 * 4;
  const int64_t grid = std::min<int64_t>((a.n + 15) / 16, int64_t(dev->sms) * (kTiles == 1 ? 5 * 8 : 2 * 8) / warps);
  if (warps == 16) {
    cudaFuncSetAttribute(gemm_w4_kernel<kGroup, kTiles, 16>, cudaFuncAttributeMaxDynamicSharedMemorySize, limit);
    return launch_cache("gemm_w4a16 launch", gemm_w4_kernel<kGroup, kTiles, 16>, grid, 1, 1, warps * 32, smem2, stream, a);
  }
  cudaFuncSetAttribute(gemm_w4_kernel<kGroup, kTiles, 8>, cudaFuncAttributeMaxDynamicSharedMemorySize, limit);
  return launch_cache("gemm_w4a16 launch", gemm_w4_kernel<kGroup, kTiles, 8>, grid, 1, 1, warps * 32, smem2, stream, a);
}

template <int kGroup>
static int launch_w4(const W4Args &a, const DeviceInfo *dev, void *stream) {
  if (a.m <= 8)
    return launch_w4<kGroup, 1>(a, dev, stream);
  if (a.m <= 16)
    return launch_w4<kGroup, 2>(a, dev, stream);
  if (a.m <= 32)
    return launch_w4<kGroup, 4>(a, dev, stream);
  return launch_w4<kGroup, 8>(a, dev, stream);
}

} // namespace pir2b

using namespace pir2b;

extern "C" {

int pir2b_set_w4_mode(int mode) { return g_w4_mode.exchange(mode); }

int pir2b_gemm_w4a16(const void *x, int64_t ldx, const void *packed, const void *scales, int group,
                     const void *bias, int64_t m, int64_t n, int64_t k, void *out, int64_t ldo,
                     void *stream) {
  if (group != 32 && group != 64 && group != 128)
    return fail(PIR2B_EINVAL, "gemm_w4a16: a group is 32, 64 or 128 weights");
  if (m < 0 || m > 0x7fffffff || n < 1 || n > 0x7ffffff0 || k < group || k > (1 << 20) || k % group != 0)
    return fail(PIR2B_EINVAL, "gemm_w4a16: needs rows >= 0, n >= 1 and k a multiple of the group, at most 2^20");
  if (m == 0)
    return PIR2B_OK;
  if (x == nullptr || packed == nullptr || scales == nullptr || out == nullptr)
    return fail(PIR2B_EINVAL, "gemm_w4a16: x, packed, scales and out must be non-null");
  if (ldx < k || ldo < n)
    return fail(PIR2B_EINVAL, "gemm_w4a16: a row stride is below its row's width");
  if (!aligned(x, 16) || ldx % 8 != 0 || !aligned(packed, 16) || !aligned(scales, 2) || !aligned(bias, 2) || !aligned(out, 2))
    return fail(PIR2B_EALIGN, "gemm_w4a16: x and packed must be 16-byte aligned, x with a row stride that is a multiple of 8");
  DeviceInfo *dev = nullptr;
  if (int r = device_info(&dev))
    return r;
  W4Args a = {};
  a.w = static_cast<const uint8_t *>(packed);
  a.scales = static_cast<const __nv_bfloat16 *>(scales);
  a.bias = static_cast<const __nv_bfloat16 *>(bias);
  a.ldx = ldx;
  a.ldo = ldo;
  a.n = int(n);
  a.k = int(k);
  a.pairs = ldo % 2 == 0 && aligned(out, 4);
  for (int64_t first = 0; first < m; first += kW4Rows) {   // more rows read the weights again
    a.x = static_cast<const __nv_bfloat16 *>(x) + first * ldx;
    a.out = static_cast<__nv_bfloat16 *>(out) + first * ldo;
    a.m = int(std::min<int64_t>(kW4Rows, m - first));
    if (int r = group == 32 ? launch_w4<32>(a, dev, stream) : group == 64 ? launch_w4<64>(a, dev, stream) : launch_w4<128>(a, dev, stream))
      return r;
  }
  return PIR2B_OK;
}

} // extern "C"
