// Causal attention of many rows: 128-row tiles on the tensor cores
// (tcgen05.mma), for packed prompts and for chunks over the paged cache.
//
// A CTA takes 128 kTiles rows (token x head of one kv head's group, token
// major, so the heads that share a kv head share its K and V tiles) of one
// sequence as M = 128 tiles, and walks the keys in blocks of 128:
//   S = Q K^T  (Q, K in shared memory, 128-byte swizzle; S fp32 in TMEM),
//   P = exp2(scale S - m), rounded to bf16, written over half of S in TMEM,
//   O += P V   (P from TMEM, V in shared memory as it lies: keys x D, the
//               transposed B operand; O fp32 in TMEM).
// Eight warps per tile are its softmax, two threads per row with half of a
// block's columns each (one thread per row: 64 prompts of 280-816 tokens 192 us,
// two: 179); then one warp issues the MMAs, one loads K and V by TMA into a
// ring, and one clears what a page holds past the keys.  While one tile's
// softmax runs, the tensor core works on the other's products.  Weights are
// relative to a reference near the running maximum that moves in few blocks: O
// is rescaled in TMEM by the softmax warps only then (scores of deviation 6, 10
// and 30, which move it often: the 8192 tokens below 266, 277-293 and 299 us).
// References, sums and O are fp32; weights are rounded to bf16, the type of the
// values they multiply, and a row's sum is that of the weights before that
// rounding.
//
// What bounds it, at 16 query and 8 kv heads of 128 (replayed from a graph; called
// in a loop in brackets).  One prompt of 8192 tokens: 236 us (271, at the board's
// power limit), 1165 TFLOP/s of the causal half; the tensor pipe is busy 55 % of
// the time and the exponentials' unit as long, and neither hides the other in
// full.  The 64 prompts: 179 us (197) against 67 for their bytes; a tile has three
// blocks on average, and its start, end and each block's chain of scores, softmax
// and product are overlapped only with those of the one other CTA on the SM that
// TMEM has room for.  Chunks of 250-288 tokens over 16 E4M3 histories of 544-2100:
// 120 us (121); reading each key's scales from shared memory and turning codes
// into bf16 come on top.  Over int4 histories the same, 120 us (120): half the bytes,
// and a longer conversion beside them (49 % of the cycles issue; of a warp's time 26 %
// is at the barriers between roles, 23 % at loads, TMEM's among them).
//
// TMEM columns: S/P of each tile (128 each), then O of each.
// Every wait is bounded; on expiry all roles leave their loops, the loader
// waits for its copies in flight and TMEM is freed.  The two softmax warps of 32
// rows meet at a hardware barrier, to which one that leaves still comes
// (PairMeeting; that costs 1 to 2 % against a plain barrier, and half of what an
// mbarrier with its time limit does).
#pragma once
#include <cuda.h>
#include "attention_few.cuh"

namespace pir2b {

constexpr int kSourceRows = 0;   // K and V source: packed rows, else a cache format
constexpr int kTileKeys = 128;

// kTiles = 1 fits two CTAs on an SM: one's softmax, prologue and epilogue run
// beside the other's products.
template <int kSource, int D, int kTiles>
struct TileShape {
  static constexpr bool kScaled = kSource == kCacheInt8 || kSource == kCacheE4m3 || kSource == kCacheInt4;
  static constexpr int kThreads = kTiles * 256 + 96 + (kScaled ? 128 : 0);
  static constexpr int kBytes = 128 * D * 2;            // a Q, K or V tile
  static constexpr int kStages = kTiles == 2 ? (D == 128 ? (kScaled ? 3 : 5) : (kScaled ? 6 : 8)) : (D == 128 ? 2 : 5);
  // Quantised caches: tiles of codes (int4: and their factors) on their way to the
  // converting warps, and blocks whose scales are kept.  The loader writes block j's scales when
  // item 2 j - kRaw has been converted, so item 2 j - kRaw - kStages has been
  // used; V item 2 (j - kDepth) + 1 must not come after that.
  static constexpr int kRowCodes = code_bytes(kSource, D), kRowFactors = kSource == kCacheInt4 ? D / kFactorGroup : 0;
  static constexpr int kRaw = kScaled ? 3 : 0, kRawBytes = 128 * (kRowCodes + kRowFactors);
  static constexpr int kDepth = (kStages + kRaw + 2) / 2;
  static constexpr int kScaleBytes = kScaled ? kDepth * 2 * kTileKeys * 4 : 0;
  static constexpr int kSumBytes = kTiles * 2 * 128 * 4;
  static constexpr int kSmem = (kTiles + kStages) * kBytes + kRaw * kRawBytes + kScaleBytes + kSumBytes + 512 /* barriers */;
};

// bf16 x bf16 -> fp32, A and B in shared memory.
__device__ __forceinline__ void mma_bf16_ss(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// The same with A in TMEM (two bf16 per 32-bit column).
__device__ __forceinline__ void mma_bf16_ts(uint32_t d, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// kind::f16: bf16 operands, fp32 accumulator; `b_rows`: B is stored [K][N].
__host__ __device__ constexpr uint32_t idesc_bf16(uint32_t m, uint32_t n, bool b_rows) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(b_rows) << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

// Shared-memory descriptors of operands in 128-byte swizzled rows (1024 bytes
// per 8 rows).  One thread issues every product, so a descriptor is its low word,
// made once per tile and moved by additions, and a constant high word.
//   tile_lo: rows of M or N, 64 K elements each (K-major);
//   rows_lo: rows of K, 64 columns of N each, further columns 16 KB apart.
__device__ __forceinline__ uint32_t tile_lo(uint32_t saddr) { return (saddr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t rows_lo(uint32_t saddr) { return (saddr >> 4) | ((16384u >> 4) << 16); }
__device__ __forceinline__ uint64_t tile_desc(uint32_t lo) {
  constexpr uint32_t kHi = (1024u >> 4) | (1u << 14) | (2u << 29);   // stride, descriptor version, swizzle
  return (uint64_t(kHi) << 32) | lo;
}

__device__ __forceinline__ void tmem_st_16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_ld_8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}

__device__ __forceinline__ void tmem_st_8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float m;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}

__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 3-D tiled load into this CTA's shared memory.
__device__ __forceinline__ void tma_load_3d(void *dst, const void *tmap, uint64_t *bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(tmap), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

__device__ __forceinline__ void tma_store_3d(const void *tmap, const void *src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(tmap),
               "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z)
               : "memory");
}

// What a CTA works on.  Positions count from `base`, the first of its split.
struct TileWork {
  int b;              // sequence
  int r0, r1;         // its rows [r0, min(r0 + 256, r1)) of the sequence's token x head rows
  int64_t begin;      // packed row of its first token
  int base;           // multiple of 128
  int first;          // position of the sequence's first row's token
  int keys;           // positions any row sees
  int all_see;        // positions below this are seen by every row
  int keys0, keys1;   // positions any row of each tile sees

  __device__ __forceinline__ int blocks(int u) const { return ((u ? keys1 : keys0) + kTileKeys - 1) / kTileKeys; }
  // Keys of the tile in block j, in steps of 16 (the products' granularity).
  __device__ __forceinline__ int steps(int u, int j) const {
    return (min(kTileKeys, (u ? keys1 : keys0) - j * kTileKeys) + 15) >> 4;
  }
};

struct TileBarriers {
  uint64_t full[8], empty[8], raw_full[3], raw_empty[3], q_full[2], s_full[2], p_full[2], o_full[2], to_mend, mended;
  TileWork work;
  uint32_t tmem;
};
static_assert(sizeof(TileBarriers) <= 512);

// 32 columns of a row's output from its scores, if its hidden positions (those
// of its last block past `limit`) hold values there that are not finite.
template <int kSource, int D>
__device__ __noinline__ void sum_again(const RaggedArgs &a, TileWork w, int kvh, int token, int head, int limit,
                                       float mu, float inv, int column, float (&f)[32]) {
  auto row_of = [&](const __nv_bfloat16 *rows, int64_t row, int64_t hd, const void *pages, int64_t page_stride, int key) {
    if constexpr (kSource == kSourceRows) {
      return rows + (w.begin + w.base + key) * row + kvh * hd;
    } else {
      const int64_t page = max(0, page_of(a.c, w.b, w.base + key));
      const int64_t slot = (int64_t(kvh) << a.c.shift) + (key & ((1 << a.c.shift) - 1));
      return static_cast<const __nv_bfloat16 *>(pages) + page * page_stride + slot * D;
    }
  };
  auto v_of = [&](int key) { return row_of(a.v, a.v_row, a.v_head, a.c.v, a.c.v_page, key) + column; };
  // Hidden positions that the products read: to the end of their 16 keys (of
  // the rows there are, or the keys of the pages).
  int end = (w.keys + 15) & ~15;
  if constexpr (kSource == kSourceRows)
    end = int(min(int64_t(end), a.rows - w.begin - w.base));
  else
    end = w.keys;
  bool spoiled = false;
  // A row that sees nothing here has a limit below 0: no position lies there.
  for (int key = max(0, limit + 1); key < end && !spoiled; ++key)
    for (int c = 0; c < 32; ++c)
      spoiled |= !(fabsf(__bfloat162float(v_of(key)[c])) < INFINITY);
  if (!spoiled)
    return;
  const __nv_bfloat16 *q = a.q + (w.begin + token) * a.q_row + head * a.q_head;
  for (int c = 0; c < 32; ++c)
    f[c] = 0.f;
  for (int key = 0; key <= min(limit, w.keys - 1); ++key) {
    const __nv_bfloat16 *k = row_of(a.k, a.k_row, a.k_head, a.c.k, a.c.k_page, key);
    float s = 0.f;
    for (int d = 0; d < D; ++d)
      s += __bfloat162float(q[d]) * __bfloat162float(k[d]);
    const float p = __bfloat162float(__float2bfloat16(exp2_fast(s * a.scale_log2 - mu)));
    for (int c = 0; c < 32; ++c)
      f[c] += p * inv * __bfloat162float(v_of(key)[c]);
  }
}

template <int kSource, int D, int kTiles>
__global__ void __launch_bounds__(TileShape<kSource, D, kTiles>::kThreads, kTiles == 2 ? 1 : 2)
    attention_tile_kernel(const __grid_constant__ RaggedArgs a, const __grid_constant__ CUtensorMap tm_q,
                          const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                          const __grid_constant__ CUtensorMap tm_o) {
  using Shape = TileShape<kSource, D, kTiles>;
  constexpr bool kScaled = Shape::kScaled, kPaged = kSource != kSourceRows;
  constexpr int kMmaWarp = kTiles * 8, kRows = kTiles * 128;
  constexpr uint32_t kOCols = kTiles * 128;       // TMEM: S/P of the tiles, then O
  constexpr int kStages = Shape::kStages, kBytes = Shape::kBytes;
  constexpr int kHalves = D / 64;                 // 64-column blocks of a tile, 16 KB each
  extern __shared__ __align__(1024) uint8_t tile_raw[];   // swizzled tiles need the alignment; nothing lies before
  uint8_t *q_sm = tile_raw, *ring = q_sm + kTiles * kBytes;
  uint8_t *raw = ring + kStages * kBytes;                               // [kRaw]: [128][D] codes, [128][D / 32] factors
  float *scales = reinterpret_cast<float *>(raw + Shape::kRaw * Shape::kRawBytes);   // [kDepth][K, V][128]
  float *sums = scales + Shape::kScaleBytes / 4;                        // [tile][half][row], between a row's two threads
  TileBarriers &bar = *reinterpret_cast<TileBarriers *>(sums + Shape::kSumBytes / 4);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (warp == kMmaWarp) {
    tmem_alloc(&bar.tmem, kTiles * 256);
    tmem_relinquish();
  }
  if (warp == kMmaWarp + 1) {
    if (lane == 0) {
      for (int i = 0; i < kStages; ++i) {
        mbar_init(&bar.full[i], kScaled ? 4 : 1);
        mbar_init(&bar.empty[i], 1);
      }
      for (int u = 0; u < kTiles; ++u) {
        mbar_init(&bar.q_full[u], a.q_by_tma ? 1 : 256);
        mbar_init(&bar.s_full[u], 1);
        mbar_init(&bar.p_full[u], 8);
        mbar_init(&bar.o_full[u], 1);
      }
      mbar_init(&bar.to_mend, 1);
      mbar_init(&bar.mended, 1);
      for (int i = 0; i < Shape::kRaw; ++i) {
        mbar_init(&bar.raw_full[i], 1);
        mbar_init(&bar.raw_empty[i], 4);
      }
      fence_barrier_init();
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
    __syncwarp();
  }
  pdl_wait();
  pdl_launch_dependents();
  const int group = a.group;
  const bool ordered = kPaged && a.ordered;
  // Of a prompt, later rows see more keys: they start first.
  const int unit = int((ordered ? blockIdx.x : gridDim.x - 1 - blockIdx.x) / uint32_t(a.splits));
  const int split = int(blockIdx.x % uint32_t(a.splits));
  const int kvh = int(uint32_t(unit) % uint32_t(a.hk)), slot = int(uint32_t(unit) / uint32_t(a.hk));
  // The loader warp finds out what the CTA works on; the others read it once
  // the CTA is set up.
  TileWork w = {};
  w.b = -1;
  int tile = 0, s0 = 0, s1 = 0;
  if (warp == kMmaWarp + 1)
    w.b = ordered ? unit_by_length(a, kTiles == 2 ? 8 : 7, slot, tile, s0, s1)
                  : unit_of(a, kTiles == 2 ? 8 : 7, slot, tile, s0, s1);
  if (w.b >= 0) {
    w.begin = s0;
    const int n = s1 - s0;
    w.r0 = tile * kRows;
    w.r1 = n * group;
    int length = n;
    if constexpr (kPaged) {
      length = cache_length(a.c, a.lengths, w.b);
      w.first = first_new_position(a.lengths, w.b, n);
    }
    w.all_see = max(0, min(length, w.first + over_group(a, w.r0) + 1));
#pragma unroll
    for (int u = 0; u < kTiles; ++u) {
      const int last = min(w.r0 + 128 * (u + 1), w.r1) - 1;   // last row of the tile
      const int keys = last < w.r0 + 128 * u ? 0 : max(0, min(length, w.first + over_group(a, last) + 1));
      (u ? w.keys1 : w.keys0) = keys;
      w.keys = max(w.keys, keys);
    }
    const int all = (w.keys + kTileKeys - 1) / kTileKeys;
    const int per = (a.splits == 1 ? all : (all + a.splits - 1) / a.splits) * kTileKeys;   // of a split
    w.base = split * per;
    w.keys0 = max(0, min(w.keys0 - w.base, per));
    w.keys1 = max(0, min(w.keys1 - w.base, per));
    w.keys = max(w.keys0, w.keys1);
    w.all_see = max(0, w.all_see - w.base);
  }
  int blocks = max(w.blocks(0), w.blocks(1));
  // Products read keys in steps of 16: what a page holds past the keys in the
  // last step is made 0 first.  (Past the rows of a prompt lie those of the
  // next, or zeros.)
  bool mend = kPaged && !kScaled && w.keys % 16 != 0;
  // Item 2 j is block j's K, item 2 j + 1 its V.  From pages, a lane per page
  // copies it (a bad page reads page 0: any values do).  8-bit codes go to the
  // converting warps' ring, with the block's scales.
  constexpr int kRing = kScaled ? Shape::kRaw : kStages;
  uint64_t *full = kScaled ? bar.raw_full : bar.full, *empty = kScaled ? bar.raw_empty : bar.empty;
  int copied = 0, page = 0;     // the loader warp's
  bool mine = lane == 0;
  auto copy = [&](int item) {
    const int stage = item % kRing, j = item >> 1;
    if constexpr (kPaged) {
      if (!(item & 1)) {
        const int at = j * kTileKeys + (lane << a.c.shift);
        mine = (lane << a.c.shift) < kTileKeys && at < w.keys;
        if (mine)
          page = max(0, page_of(a.c, w.b, w.base + at));
      }
    }
    const int copies = __popc(__ballot_sync(0xffffffffu, mine));
    bool free_stage = true;
    if (item >= kRing)
      free_stage = mbar_wait(&empty[stage], uint32_t((item / kRing - 1) & 1), kStatusTimeoutProducer);
    if (!__all_sync(0xffffffffu, free_stage))
      return false;
    if (lane == 0) {
      const int row_bytes = kScaled ? Shape::kRowCodes + Shape::kRowFactors + (item & 1 ? 0 : 8) : D * 2;
      mbar_arrive_expect_tx(&full[stage], kPaged ? (copies << a.c.shift) * row_bytes : kBytes);
    }
    __syncwarp();
    if (mine) {
      const void *map = (item & 1) ? &tm_v : &tm_k;
      if constexpr (kScaled) {
        const int row = lane << a.c.shift;
        tma_load_4d(raw + stage * Shape::kRawBytes + row * Shape::kRowCodes, map, &full[stage], 0, 0, kvh, page);
        if constexpr (kSource == kCacheInt4) {
          const uint8_t *factors = (item & 1) ? a.c.vf + page * a.c.vf_page : a.c.kf + page * a.c.kf_page;
          bulk_load(raw + stage * Shape::kRawBytes + 128 * Shape::kRowCodes + row * Shape::kRowFactors,
                    factors + (int64_t(kvh) << a.c.shift) * Shape::kRowFactors, uint32_t(Shape::kRowFactors) << a.c.shift,
                    &full[stage]);
        }
        if (!(item & 1)) {
          float *block_scales = scales + (j % Shape::kDepth) * 2 * kTileKeys + row;
          const int64_t slot = int64_t(kvh) << a.c.shift;
          bulk_load(block_scales, a.c.ks + page * a.c.ks_page + slot, 4u << a.c.shift, &full[stage]);
          bulk_load(block_scales + kTileKeys, a.c.vs + page * a.c.vs_page + slot, 4u << a.c.shift, &full[stage]);
        }
      } else {
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          uint8_t *dst = ring + stage * kBytes + h * 16384;
          if constexpr (kPaged)
            tma_load_4d(dst + (lane << a.c.shift) * 128, map, &full[stage], h * 64, 0, kvh, page);
          else
            tma_load_3d(dst, map, &full[stage], h * 64, kvh, int(w.begin) + w.base + j * kTileKeys);
        }
      }
    }
    if (mend && lane == 0 && item == 2 * blocks - 1)
      mbar_arrive(&bar.to_mend);
    return true;
  };
  if (warp == kMmaWarp + 1) {
    if (lane == 0)
      bar.work = w;
    // What needs no free stage is on its way before the CTA is set up.
    if (a.q_by_tma && lane < kTiles && w.blocks(lane) > 0) {
      mbar_arrive_expect_tx(&bar.q_full[lane], kBytes);
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
        tma_load_3d(q_sm + lane * kBytes + h * 16384, &tm_q, &bar.q_full[lane], h * 64, kvh * group,
                    int(w.begin) + over_group(a, w.r0 + lane * 128));
    }
    while (copied < min(kRing, 2 * blocks) && copy(copied))
      ++copied;
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar.tmem;
  if (warp != kMmaWarp + 1) {
    w = bar.work;
    blocks = max(w.blocks(0), w.blocks(1));
    mend = kPaged && !kScaled && w.keys % 16 != 0;
  }

  if (warp < kMmaWarp) {
    // Two warps per 32 rows of a tile, each with half of a block's columns (and
    // of O's): a row's two threads keep the same reference and sum.
    const int u = warp >> 3, half = (warp >> 2) & 1, t = (warp & 3) * 32 + lane;
    constexpr int kOwn = D / 2;                               // columns of O
    const uint32_t lanes = uint32_t(warp & 3) << 21;          // this warp's TMEM lanes
    const uint32_t s_tm = tmem + lanes + u * 128 + half * 64, o_tm = tmem + lanes + kOCols + u * 128 + half * kOwn;
    const bool valid = w.b >= 0 && w.r0 + u * 128 + t < w.r1;
    // Token and head of the CTA's i-th row.
    auto token_of = [&](int i, int &head) {
      const int token = over_group(a, w.r0 + i);
      head = kvh * group + w.r0 + i - token * group;
      return token;
    };
    int my_head;
    const int my_token = token_of(u * 128 + t, my_head);
    const int limit = valid ? w.first + my_token - w.base : -1;   // it sees positions 0 .. limit
    float *my_sum = sums + (u * 2 + half) * 128 + t, *other_sum = sums + (u * 2 + 1 - half) * 128 + t;
    PairMeeting pair{uint32_t(1 + u * 4 + (warp & 3))};   // the two warps of these rows
    if (w.blocks(u) > 0 && !a.q_by_tma) {
      for (int i = half * 128 + t; i < 128 * (D / 8); i += 256) {
        const int qr = i / (D / 8), c = i % (D / 8);
        uint8_t *dst = q_sm + u * kBytes + (c >> 3) * 16384 + qr * 128 + (((c & 7) ^ (qr & 7)) << 4);
        int head;
        const int token = token_of(u * 128 + qr, head);
        if (w.r0 + u * 128 + qr < w.r1)
          cp_async_16(dst, a.q + (w.begin + token) * a.q_row + head * a.q_head + c * 8);
        else
          *reinterpret_cast<uint4 *>(dst) = make_uint4(0, 0, 0, 0);
      }
      cp_async_wait_all();
      fence_proxy_async_smem();
      mbar_arrive(&bar.q_full[u]);
    }
    float mu = 0.f, sum = 0.f;    // weights are exp2(score - mu); their sum over the row
    bool none = true;             // no score seen yet
    constexpr float kAgain = kScaled ? 0x1p16f : 0x1p64f;
    for (int j = 0; j < w.blocks(u); ++j) {
      if (!__all_sync(0xffffffffu, mbar_wait(&bar.s_full[u], j & 1, kStatusTimeoutEpilogue))) {
        pair.leave();
        break;
      }
      tc_fence_after();
      // Columns above `seen` are hidden.  Only blocks past all_see have any,
      // and a warp's rows differ in few positions: a chunk of 32 columns is
      // mostly all seen or all hidden.
      const int seen = limit - j * kTileKeys - half * 64;
      int seen_by_all = kTileKeys, seen_by_any = kTileKeys;
      if ((j + 1) * kTileKeys > w.all_see) {
        seen_by_all = __reduce_min_sync(0xffffffffu, seen);
        seen_by_any = __reduce_max_sync(0xffffffffu, seen);
      }
      // Only a row's first block is searched for its maximum: the weights are
      // taken relative to mu, and their sum tells when that has become too
      // small.  A block whose weights sum to more than 2^12 raises mu by the
      // power of two in that sum and scales its weights, exactly, before they
      // meet V: products and O then overflow only where the plain sum would.
      // One whose weights pass kAgain is done again under its own maximum: 2^64,
      // or 2^16 where the weights are rounded to bf16 with V's scale in them.
      const float *block_scales = scales + (j % Shape::kDepth) * 2 * kTileKeys + half * 64;
      uint32_t s[32], p[2][16];
      auto load = [&](int i) {
        tmem_ld_32(s_tm + i * 32, s);
        tmem_ld_wait();
        if constexpr (kScaled) {
          const float4 *k_scale = reinterpret_cast<const float4 *>(block_scales + i * 32);
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const float4 x = k_scale[c / 4];
            const float2 y = __fmul2_rn(make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), make_float2(x.x, x.y));
            const float2 z = __fmul2_rn(make_float2(__uint_as_float(s[c + 2]), __uint_as_float(s[c + 3])), make_float2(x.z, x.w));
            s[c] = __float_as_uint(y.x), s[c + 1] = __float_as_uint(y.y);
            s[c + 2] = __float_as_uint(z.x), s[c + 3] = __float_as_uint(z.y);
          }
        }
        if (seen_by_all < i * 32 + 31) {
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (i * 32 + c > seen)
              s[c] = 0xff800000u;
        }
      };
      // The maximum of the row's block, by both of its threads.
      auto maximum = [&]() {
        float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
          if (seen_by_any < i * 32)
            break;
          load(i);
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            m0 = max3(m0, __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
            m1 = max3(m1, __uint_as_float(s[c + 2]), __uint_as_float(s[c + 3]));
          }
        }
        *my_sum = fmaxf(m0, m1);
        if (!pair.meet())
          return -INFINITY;
        const float m = fmaxf(*my_sum, *other_sum) * a.scale_log2;
        pair.meet();
        return m;
      };
      auto scale_o = [&](float keep) {
#pragma unroll 1
        for (int i = 0; i < kOwn / 8; ++i) {
          uint32_t o[8];
          tmem_ld_8(o_tm + i * 8, o);
          tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 8; ++c)
            o[c] = __float_as_uint(__uint_as_float(o[c]) * keep);
          tmem_st_8(o_tm + i * 8, o);
        }
      };
      // The weights of this thread's columns into p; returns the row's sum.
      auto weights = [&]() {
        const float2 scale2 = make_float2(a.scale_log2, a.scale_log2), minus = make_float2(-mu, -mu);
        float2 total = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (seen_by_any < i * 32) {
#pragma unroll
            for (int c = 0; c < 16; ++c)
              p[i][c] = 0;
            continue;
          }
          load(i);
          const float4 *v_scale = reinterpret_cast<const float4 *>(block_scales + kTileKeys + i * 32);
          float4 v4;
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const float2 x =
                __ffma2_rn(make_float2(__uint_as_float(s[2 * c]), __uint_as_float(s[2 * c + 1])), scale2, minus);
            float2 e = make_float2(exp2_fast(x.x), exp2_fast(x.y));
            total = __fadd2_rn(total, e);
            if constexpr (kScaled) {
              if (!(c & 1))
                v4 = v_scale[c / 2];
              const float2 v = (c & 1) ? make_float2(v4.z, v4.w) : make_float2(v4.x, v4.y);
              if (seen_by_all < i * 32 + 31)   // a hidden row's scale may be anything
                e = make_float2(e.x == 0.f ? 0.f : e.x * v.x, e.y == 0.f ? 0.f : e.y * v.y);
              else
                e = __fmul2_rn(e, v);
            }
            p[i][c] = pack_bf16x2(e.x, e.y);
          }
        }
        *my_sum = total.x + total.y;
        pair.meet();
        return *my_sum + *other_sum;
      };
      if (__any_sync(0xffffffffu, none && limit >= j * kTileKeys)) {
        const float m = maximum();
        if (!pair.ok)             // the other warp has left
          break;
        if (none && m > -INFINITY) {
          mu = m;
          none = false;
        }
      }
      float total = weights();
      // Of rows past the sequence nothing is kept.
      if (__any_sync(0xffffffffu, !pair.ok || (valid && !(total <= 4096.f)))) {
        if (!pair.ok)
          break;
        float keep;
        if (__any_sync(0xffffffffu, valid && !(total < kAgain))) {
          if (!pair.meet())       // both have read the sums
            break;
          const float m = fmaxf(mu, maximum());
          if (!pair.ok)
            break;
          keep = exp2_fast(mu - m);
          mu = m;
          total = weights();
          if (!pair.ok)
            break;
        } else {
          const int up = valid && total > 4096.f ? (__float_as_int(total) >> 23) - 127 : 0;
          keep = __int_as_float((127 - up) << 23);
          mu += up;
          total *= keep;
          const __nv_bfloat162 keep2 = __float2bfloat162_rn(keep);
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              const __nv_bfloat162 x = __hmul2(*reinterpret_cast<const __nv_bfloat162 *>(&p[i][c]), keep2);
              p[i][c] = *reinterpret_cast<const uint32_t *>(&x);
            }
        }
        sum *= keep;
        scale_o(keep);
      }
      sum += total;
      // P goes over the scores it came from.
      tmem_st_16(s_tm, p[0]);
      tmem_st_16(s_tm + 16, p[1]);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&bar.p_full[u]);
    }
    // 32 rows that leave by TMA; the two halves of heads of 64 in one box.
    const int first_row = w.r0 + u * 128 + (warp & 3) * 32;
    const bool whole = a.splits == 1 && a.out_by_tma && w.b >= 0 && first_row + 32 <= w.r1;
    bool done = pair.ok;
    if (done && w.blocks(u) > 0)
      done = __all_sync(0xffffffffu, mbar_wait(&bar.o_full[u], 0, kStatusTimeoutEpilogue));
    if (D == 64 && whole && pair.ok && !done)
      pair.leave();
    tc_fence_after();
    if (done && w.b >= 0 && w.r0 + u * 128 < w.r1) {
      const float inv = sum == 0.f ? 0.f : a.splits > 1 ? 1.f : 1.f / sum;   // splits are divided when joined
      const int64_t part = (int64_t(split) * a.rows + w.begin + my_token) * a.hq + my_head;
      if (a.splits > 1 && valid && half == 0)
        a.part_ml[part] = make_float2(none ? -INFINITY : mu, sum);
      // Into the tile that held Q (its products are done), in the same layout.
      constexpr int kPieces = kOwn / 8;                       // 16-byte pieces of a row
      uint8_t *own_sm = q_sm + u * kBytes + (D == 128 ? half * 16384 : 0);
      const int piece0 = D == 128 ? 0 : half * kPieces;
#pragma unroll
      for (int i = 0; i < kOwn / 32; ++i) {
        const int column = half * kOwn + i * 32;
        uint32_t o[32] = {};
        if (w.blocks(u) > 0) {
          tmem_ld_32(o_tm + i * 32, o);
          tmem_ld_wait();
        }
        float f[32];
#pragma unroll
        for (int c = 0; c < 32; ++c)
          f[c] = __uint_as_float(o[c]) * inv;
        // A weight of 0 times a value that is not finite is NaN: where a row's
        // hidden positions hold one, its values are summed again without them.
        float2 check = make_float2(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < 32; c += 2)
          check = __ffma2_rn(make_float2(f[c], f[c + 1]), make_float2(0.f, 0.f), check);
        if (!kScaled && !(check.x + check.y == 0.f) && valid && w.blocks(u) > 0) {
          float again[32];            // a copy: f stays in registers
#pragma unroll
          for (int c = 0; c < 32; ++c)
            again[c] = f[c];
          sum_again<kSource, D>(a, w, kvh, my_token, my_head, limit, mu, inv, column, again);
#pragma unroll
          for (int c = 0; c < 32; ++c)
            f[c] = again[c];
        }
        if (a.splits > 1) {
          if (valid && w.blocks(u) > 0) {
#pragma unroll
            for (int c = 0; c < 32; c += 4)
              *reinterpret_cast<float4 *>(a.part_o + part * D + column + c) = make_float4(f[c], f[c + 1], f[c + 2], f[c + 3]);
          }
          continue;
        }
#pragma unroll
        for (int c = 0; c < 32; c += 8)
          *reinterpret_cast<uint4 *>(own_sm + t * 128 + (((piece0 + i * 4 + c / 8) ^ (t & 7)) << 4)) =
              make_uint4(pack_bf16x2(f[c], f[c + 1]), pack_bf16x2(f[c + 2], f[c + 3]), pack_bf16x2(f[c + 4], f[c + 5]),
                         pack_bf16x2(f[c + 6], f[c + 7]));
      }
      // 32 rows to memory: by TMA, or the last of a sequence row by row.
      if (whole) {
        fence_proxy_async_smem();
        __syncwarp();
        if (D == 64)
          pair.meet();            // both halves are in one box
        if (pair.ok && lane == 0 && (D == 128 || half == 0)) {
          tma_store_3d(&tm_o, own_sm + (warp & 3) * 4096, D == 128 ? half * 64 : 0, kvh * group,
                       int(w.begin) + over_group(a, first_row));
          tma_store_commit_and_wait();
        }
      } else if (a.splits == 1) {
        __syncwarp();
        constexpr int kAtOnce = 32 / kPieces;
#pragma unroll 4
        for (int i = 0; i < 32; i += kAtOnce) {
          const int rr = (warp & 3) * 32 + i + lane / kPieces, piece = lane % kPieces;
          int head;
          const int token = token_of(u * 128 + rr, head);
          const uint4 x = *reinterpret_cast<const uint4 *>(own_sm + rr * 128 + (((piece0 + piece) ^ (rr & 7)) << 4));
          if (w.r0 + u * 128 + rr < w.r1)
            *reinterpret_cast<uint4 *>(a.out + (w.begin + token) * a.ldo + head * D + half * kOwn + piece * 8) = x;
        }
      }
    }
  } else {
    if (warp == kMmaWarp) {
      if (elect_one_sync()) {
        constexpr uint32_t kIdescO = idesc_bf16(128, D, true);
        const uint32_t q_addr = smem_u32(q_sm), ring_addr = smem_u32(ring);
        auto wait = [&](uint64_t *b, int parity) { return mbar_wait(b, uint32_t(parity & 1), kStatusTimeoutMma); };
        auto scores = [&](int u, int item) {
          const uint32_t k_lo = tile_lo(ring_addr + (item % kStages) * kBytes), q_lo = tile_lo(q_addr + u * kBytes);
          const uint32_t idesc = idesc_bf16(128, w.steps(u, item / 2) * 16, false);
#pragma unroll
          for (int s = 0; s < D / 16; ++s) {
            const uint32_t at = ((s >> 2) * 16384 + (s & 3) * 32) >> 4;
            mma_bf16_ss(tmem + u * 128, tile_desc(q_lo + at), tile_desc(k_lo + at), idesc, s > 0);
          }
          mma_commit(&bar.s_full[u]);
        };
        bool ok = blocks > 0 && wait(&bar.full[0], 0);
        for (int u = 0; u < kTiles && ok; ++u)
          if (w.blocks(u) > 0) {
            ok = wait(&bar.q_full[u], 0);
            if (ok)
              scores(u, 0);
          }
        if (ok)
          mma_commit(&bar.empty[0]);
        for (int j = 0; j < blocks && ok; ++j) {
          const int v_item = 2 * j + 1, k_item = 2 * j + 2;
          bool v_ready = false, k_ready = false;
          for (int u = 0; u < kTiles && ok; ++u) {
            if (j >= w.blocks(u))
              continue;
            if (!v_ready) {
              if (mend && j == blocks - 1)
                ok = wait(&bar.mended, 0);
              else
                ok = wait(&bar.full[v_item % kStages], v_item / kStages);
              v_ready = true;
            }
            const uint32_t v_lo = rows_lo(ring_addr + (v_item % kStages) * kBytes);
            auto product = [&](int s) {
              mma_bf16_ts(tmem + kOCols + u * 128, tmem + u * 128 + (s >> 2) * 64 + (s & 3) * 8, tile_desc(v_lo + s * 128),
                          kIdescO, j > 0 || s > 0);
            };
            const int steps = w.steps(u, j);
            ok = ok && wait(&bar.p_full[u], j);
            if (!ok)
              break;
            tc_fence_after();
            if (steps == 8) {
#pragma unroll
              for (int s = 0; s < 8; ++s)
                product(s);
            } else {
#pragma unroll 1
              for (int s = 0; s < steps; ++s)
                product(s);
            }
            if (j + 1 < w.blocks(u)) {
              if (!k_ready) {
                ok = wait(&bar.full[k_item % kStages], k_item / kStages);
                k_ready = true;
              }
              if (ok)
                scores(u, k_item);
            } else {
              mma_commit(&bar.o_full[u]);
            }
          }
          if (ok) {
            mma_commit(&bar.empty[v_item % kStages]);
            if (k_ready)
              mma_commit(&bar.empty[k_item % kStages]);
          }
        }
      }
    } else if (warp == kMmaWarp + 1) {
      while (copied < 2 * blocks && copy(copied))
        ++copied;
      // No copy is in flight when the CTA ends (at once, unless a wait gave up).
      if (lane == 0) {
        for (int i = max(0, copied - kRing); i < copied; ++i)
          mbar_wait(&full[i % kRing], uint32_t((i / kRing) & 1), kStatusTimeoutProducer);
        for (int u = 0; u < kTiles && a.q_by_tma; ++u)
          if (w.blocks(u) > 0)
            mbar_wait(&bar.q_full[u], 0, kStatusTimeoutProducer);
      }
    } else if (kScaled) {
      if constexpr (kScaled) {
        // Four warps turn tiles of codes into bf16 tiles, 16 bytes of a row at
        // a time (of int4 the channels of one factor).  Rows past the keys hold
        // old codes, which are numbers.
        constexpr int kRuns = Shape::kRowCodes / 16, kRowStep = 128 / kRuns;
        const Int4Masks masks = int4_masks();
        const int t = tid - (kMmaWarp + 3) * 32, run = t % kRuns, row0 = t / kRuns;
        for (int item = 0; t >= 0 && item < 2 * blocks; ++item) {
          const int from = item % Shape::kRaw, stage = item % kStages;
          bool go = mbar_wait(&bar.raw_full[from], uint32_t((item / Shape::kRaw) & 1), kStatusTimeoutConvert);
          if (go && item >= kStages)
            go = mbar_wait(&bar.empty[stage], uint32_t((item / kStages - 1) & 1), kStatusTimeoutConvert);
          if (!__all_sync(0xffffffffu, go))
            break;
          const uint8_t *src = raw + from * Shape::kRawBytes + row0 * Shape::kRowCodes + run * 16;
          constexpr int kPieces = 2 * D / kRuns / 16;         // 16-byte pieces of bf16 that a run becomes
          uint8_t *dst = ring + stage * kBytes + run * kPieces / 8 * 16384;
          const int piece = run * kPieces % 8;
#pragma unroll
          for (int i = 0; i < kTileKeys / kRowStep; ++i) {
            const int row = row0 + i * kRowStep;
            const uint4 x = *reinterpret_cast<const uint4 *>(src + i * kRowStep * Shape::kRowCodes);
            if constexpr (kSource == kCacheInt4) {
              const uint32_t byte = raw[from * Shape::kRawBytes + 128 * Shape::kRowCodes + row * Shape::kRowFactors + run];
              uint32_t minus_24f;
              const uint32_t f = factor_pair_bf16(byte, byte, minus_24f), w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const uint32_t p0 = int4_to_bf16<0>(w[c], f, minus_24f, masks), p1 = int4_to_bf16<1>(w[c], f, minus_24f, masks);
                const uint32_t p2 = int4_to_bf16<2>(w[c], f, minus_24f, masks), p3 = int4_to_bf16<3>(w[c], f, minus_24f, masks);
                *reinterpret_cast<uint4 *>(dst + row * 128 + (((piece + c) ^ (row & 7)) << 4)) =
                    make_uint4(__byte_perm(p0, p1, 0x5410), __byte_perm(p2, p3, 0x5410), __byte_perm(p0, p1, 0x7632),
                               __byte_perm(p2, p3, 0x7632));
              }
              continue;
            }
            uint4 lo, hi;
            codes_to_bf16<kSource>(x.x, lo.x, lo.y);
            codes_to_bf16<kSource>(x.y, lo.z, lo.w);
            codes_to_bf16<kSource>(x.z, hi.x, hi.y);
            codes_to_bf16<kSource>(x.w, hi.z, hi.w);
            *reinterpret_cast<uint4 *>(dst + row * 128 + ((piece ^ (row & 7)) << 4)) = lo;
            *reinterpret_cast<uint4 *>(dst + row * 128 + (((piece + 1) ^ (row & 7)) << 4)) = hi;
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&bar.full[stage]);
            mbar_arrive(&bar.raw_empty[from]);
          }
        }
      }
    } else {
      // The loader says when the last V block is on its way: only then is its
      // stage's barrier in the phase that is waited for.
      const int item = 2 * blocks - 1, stage = item % kStages;
      if (mend && mbar_wait(&bar.to_mend, 0, kStatusTimeoutConvert) &&
          mbar_wait(&bar.full[stage], uint32_t((item / kStages) & 1), kStatusTimeoutConvert)) {
        uint8_t *v = ring + stage * kBytes;
        const int end = w.keys - (blocks - 1) * kTileKeys;
        for (int i = lane; i < (16 - end % 16) * (D / 8); i += 32) {
          const int key = end + i / (D / 8), c = i % (D / 8);
          *reinterpret_cast<uint4 *>(v + (c >> 3) * 16384 + key * 128 + (((c & 7) ^ (key & 7)) << 4)) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&bar.mended);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp)
    tmem_dealloc(tmem, kTiles * 256);
}

} // namespace pir2b
