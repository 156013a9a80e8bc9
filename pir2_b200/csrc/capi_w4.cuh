// C ABI of the products with 4-bit weights: argument checks, plans and launches.
#pragma once
#include "capi_cache.cuh"
#include "gemm_w4.cuh"

namespace pir2b {

constexpr int kW4Rows = 64;   // rows of a launch: more read the weights again
constexpr int kW4Smem = 227 * 1024;

// Plan override for tests and measurement (pir2b_set_w4_mode): 0 lets the rules
// below choose, 1 never keeps rows in shared memory, 2 does wherever they fit.
static std::atomic<int> g_w4_mode{0};

// Whether the rows are kept in shared memory (the staged kernel up to eight, the
// wide one above) while weights stream past them.  That costs a start, which many
// channels pay back; more than eight rows pay a launch more as well.  Graph replays,
// us, the direct kernel against the one that keeps rows, in groups of 128 (32), channels
// x K:
//    1 row   6144 x 1024 3.6 (4.0) 3.4 (3.7)   6144 x 2048 4.5 (7.3) 4.7 (5.2)
//            4096 x 2048 3.2 (4.3) 4.0 (4.3)   12288 x 2048 7.1 (10.8) 7.0 (7.7)
//            4096 x 4096 5.9 (8.1) 5.6 (6.2)   4096 x 6144 7.4 (11.3) 6.9 (7.4)
//            2048 x 6144 4.1 (6.1) 5.1 (5.4)   8192 x 4096 10.2 (14.4) 8.0 (8.7)
//    8 rows  4096 x 2048 3.7 (4.8) 4.2 (4.6)   2048 x 6144 4.8 (6.6) 6.7 (6.4)
//            6144 x 1536 5.1 (5.9) 4.5 (4.8)   12288 x 2048 8.4 (12.0) 7.3 (8.0)
//            4096 x 4096 6.7 (8.9) 6.4 (6.5)   4096 x 6144 8.8 (12.6) 8.6 (8.5)
//            151936 x 2048 69 (121) 36 (40)
//   16       4096 x 1024 3.6 4.7               4096 x 2048 6.2 (6.0) 5.5 (5.8)
//   32       2048 x 6144 10.2 (13.1) 12.8 (13.3)   4096 x 1024 4.7 5.8
//            4096 x 2048 7.5 (11.7) 7.1 (7.8)  6144 x 1024 7.8 6.5
//            12288 x 2048 19.8 (24.1) 12.9 (14.1)   151936 x 2048 198 (222) 99 (106)
static bool w4_keeps_rows(int64_t m, int64_t n, int64_t k) {
  const int mode = g_w4_mode.load();
  if (mode == 1 || k % 256 != 0)
    return false;
  if (m <= 8)
    return W4Staged::bytes(k) <= kW4Smem && (mode == 2 || n >= 6144 || (n >= 4096 && k >= 4096));
  return mode == 2 || (n >= 4096 && n * k >= (int64_t(6) << 20));
}

// Warps that split K: the fewest rounds of chunks of 128, a round's meeting counted
// as `meeting` more (wide, 32 rows of 4096 -> 20000: 33-36 us with 4 to 16, 36-39 with
// 2, 43-45 with 1).
static int w4_split(int64_t blocks, int64_t ctas, int warps, int slabs, int units, int meeting) {
  int best = 1;
  int64_t least = INT64_MAX;
  for (int wk = 1; wk <= warps && warps % wk == 0; wk *= 2) {
    const int64_t wc = warps / wk, rounds = ((blocks + ctas - 1) / ctas + wc - 1) / wc;
    const int64_t cost = rounds * (slabs * 2 * ((units + wk - 1) / wk) + meeting);
    if (cost < least)
      least = cost, best = wk;
  }
  return best;
}

// Eight-row tiles of a launch.
static int w4_tiles(int64_t m) { return m <= 8 ? 1 : m <= 16 ? 2 : m <= 32 ? 4 : 8; }

// Workspace of a launch's rows, in bytes.
static int64_t w4_workspace(int64_t m, int64_t n, int64_t k) {
  return m > 8 && w4_keeps_rows(m, n, k) ? k * 8 * w4_tiles(m) * 2 : 0;
}

template <int kGroup>
static int launch_w4_staged(W4Args a, const DeviceInfo *dev, void *stream) {
  const int64_t blocks = (a.n + 15) / 16, grid = std::min<int64_t>(dev->sms, blocks);
  a.wk = w4_split(blocks, grid, W4Staged::kWarps, 1, a.k / 256, 1);
  return launch_cache("gemm_w4a16 launch", gemm_w4_staged_kernel<kGroup>, grid, 1, 1, W4Staged::kWarps * 32,
                      size_t(W4Staged::bytes(a.k)), stream, a);
}

template <int kGroup, int kTiles>
static int launch_w4_wide(W4Args a, void *workspace, const DeviceInfo *dev, void *stream) {
  using Shape = W4Wide<kTiles>;
  uint4 *rows = static_cast<uint4 *>(workspace);
  const int64_t items = int64_t(a.k) / 32 * kTiles;
  if (int r = launch_cache("gemm_w4a16 rows launch", w4_rows_kernel<kGroup, kTiles>, (items + 3) / 4, 1, 1, 128, 0, stream, a, rows))
    return r;
  a.slab = a.k;
  while (Shape::bytes(a.slab) > kW4Smem)
    a.slab = (a.slab / 2 + 255) / 256 * 256;
  const int64_t blocks = (a.n + 15) / 16, grid = std::min<int64_t>(dev->sms, blocks);
  a.wk = w4_split(blocks, grid, Shape::kWarps, (a.k + a.slab - 1) / a.slab, a.slab / 256, 4);
  return launch_cache("gemm_w4a16 launch", gemm_w4_wide_kernel<kGroup, kTiles>, grid, 1, 1, Shape::kWarps * 32,
                      size_t(Shape::bytes(a.slab)), stream, a, static_cast<const uint4 *>(rows));
}

template <int kGroup, int kTiles, int kWarps>
static int launch_w4_direct(const W4Args &a, const DeviceInfo *dev, void *stream) {
  // A CTA takes several blocks of channels only where more CTAs would not fit at once.
  const int64_t grid = std::min<int64_t>((a.n + 15) / 16, int64_t(dev->sms) * (kTiles == 1 ? 40 : 16) / kWarps);
  return launch_cache("gemm_w4a16 launch", gemm_w4_kernel<kGroup, kTiles, kWarps>, grid, 1, 1, kWarps * 32,
                      kWarps * 8 * kTiles * 20 * 4, stream, a);
}

// Long K is split over twice the warps (8 rows of 6144 -> 2048: 4.9 us, with eight
// 7.4); not for eight tiles, whose sums do not fit the registers of so many (64 rows of
// 8192 -> 600: 22.0, with 16 warps 26.3).
template <int kGroup, int kTiles>
static int launch_w4(const W4Args &a, void *workspace, const DeviceInfo *dev, void *stream) {
  if (w4_keeps_rows(a.m, a.n, a.k)) {
    if constexpr (kTiles == 1)
      return launch_w4_staged<kGroup>(a, dev, stream);
    else
      return launch_w4_wide<kGroup, kTiles>(a, workspace, dev, stream);
  }
  if constexpr (kTiles < 8) {
    if (a.k >= 4096)
      return launch_w4_direct<kGroup, kTiles, 16>(a, dev, stream);
  }
  return launch_w4_direct<kGroup, kTiles, 8>(a, dev, stream);
}

template <int kGroup>
static int launch_w4(const W4Args &a, void *workspace, const DeviceInfo *dev, void *stream) {
  switch (w4_tiles(a.m)) {
  case 1: return launch_w4<kGroup, 1>(a, workspace, dev, stream);
  case 2: return launch_w4<kGroup, 2>(a, workspace, dev, stream);
  case 4: return launch_w4<kGroup, 4>(a, workspace, dev, stream);
  default: return launch_w4<kGroup, 8>(a, workspace, dev, stream);
  }
}

template <typename Kernel>
static int w4_attribute(Kernel kernel) {
  return cuda_status(cudaFuncSetAttribute(reinterpret_cast<const void *>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, kW4Smem),
                     "cudaFuncSetAttribute");
}

template <int kGroup, int kTiles>
static int w4_attributes() {
  if (int r = w4_attribute(gemm_w4_kernel<kGroup, kTiles, 8>))
    return r;
  if constexpr (kTiles < 8) {
    if (int r = w4_attribute(gemm_w4_kernel<kGroup, kTiles, 16>))
      return r;
  }
  if constexpr (kTiles == 1)
    return w4_attribute(gemm_w4_staged_kernel<kGroup>);
  else
    return w4_attribute(gemm_w4_wide_kernel<kGroup, kTiles>);
}

template <int kGroup>
static int w4_attributes_of_group() {
  if (int r = w4_attributes<kGroup, 1>())
    return r;
  if (int r = w4_attributes<kGroup, 2>())
    return r;
  if (int r = w4_attributes<kGroup, 4>())
    return r;
  return w4_attributes<kGroup, 8>();
}

// Dynamic shared memory above the default limit, once per device.
static int w4_kernel_attributes(DeviceInfo *dev) {
  std::lock_guard<std::mutex> lock(g_mutex);
  if (dev->w4_attrs_set)
    return PIR2B_OK;
  if (int r = w4_attributes_of_group<32>())
    return r;
  if (int r = w4_attributes_of_group<64>())
    return r;
  if (int r = w4_attributes_of_group<128>())
    return r;
  dev->w4_attrs_set = true;
  return PIR2B_OK;
}

} // namespace pir2b

using namespace pir2b;

extern "C" {

int pir2b_set_w4_mode(int mode) {
  if (mode < 0 || mode > 2)
    return -fail(PIR2B_EINVAL, "w4 mode must be 0, 1 or 2");   // not a mode
  return g_w4_mode.exchange(mode);
}

int64_t pir2b_gemm_w4a16_workspace(int64_t m, int64_t n, int64_t k, int group) {
  if ((group != 32 && group != 64 && group != 128) || m < 1 || n < 1 || k < group || k > (1 << 20) || k % group != 0)
    return 0;                                       // the call itself reports what is wrong
  // The largest of its launches of up to 64 rows.
  return std::max(w4_workspace(std::min<int64_t>(m, kW4Rows), n, k), w4_workspace(m % kW4Rows, n, k));
}

int pir2b_gemm_w4a16(const void *x, int64_t ldx, const void *packed, const void *scales, int group,
                     const void *bias, int64_t m, int64_t n, int64_t k, void *out, int64_t ldo,
                     void *workspace, void *stream) {
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
  if (!aligned(x, 16) || ldx % 8 != 0 || !aligned(packed, 16) || !aligned(scales, 16) || !aligned(bias, 2) || !aligned(out, 2))
    return fail(PIR2B_EALIGN, "gemm_w4a16: x, packed and scales must be 16-byte aligned, x with a row stride that is a multiple of 8");
  if (pir2b_gemm_w4a16_workspace(m, n, k, group) > 0 && (workspace == nullptr || !aligned(workspace, 16)))
    return fail(PIR2B_EALIGN, "gemm_w4a16: this shape needs a 16-byte aligned workspace");
  DeviceInfo *dev = nullptr;
  if (int r = device_info(&dev))
    return r;
  if (int r = w4_kernel_attributes(dev))
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
  for (int64_t first = 0; first < m; first += kW4Rows) {
    a.x = static_cast<const __nv_bfloat16 *>(x) + first * ldx;
    a.out = static_cast<__nv_bfloat16 *>(out) + first * ldo;
    a.m = int(std::min<int64_t>(kW4Rows, m - first));
    if (int r = group == 32   ? launch_w4<32>(a, workspace, dev, stream)
                : group == 64 ? launch_w4<64>(a, workspace, dev, stream)
                              : launch_w4<128>(a, workspace, dev, stream))
      return r;
  }
  return PIR2B_OK;
}

} // extern "C"
