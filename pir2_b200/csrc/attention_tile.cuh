// Causal attention of many rows: 128-row tiles on the tensor cores
// (tcgen05.mma), for packed prompts and for chunks over the paged cache.
//
// A CTA takes 256 rows (token x head of one kv head's group, token major, so
// the heads that share a kv head share its K and V tiles) of one sequence as
// two M = 128 tiles, and walks the keys in blocks of 128:
//   S = Q K^T  (Q, K in shared memory, 128-byte swizzle; S fp32 in TMEM),
//   P = exp2(scale S - m), rounded to bf16, written over S in TMEM,
//   O += P V   (P from TMEM, V in shared memory as it lies: keys x D, the
//               transposed B operand; O fp32 in TMEM).
// Warps 0-3 and 4-7 are the softmax of the two tiles, one thread per row, so
// row maxima and sums need no shuffles; warp 8 issues the MMAs; warp 9 loads
// K and V by TMA into a ring; warps 10-11 mend V blocks that hold positions
// some row must not see.  While one tile's softmax runs, the tensor core
// works on the other's products.  The running maximum moves only when a score
// passes it by more than 8 (in log2): P stays below 2^8 and O is rescaled in
// TMEM by the softmax warps only then.  Maxima, sums and O are fp32.
//
// TMEM columns: S/P of the tiles at 0 and 128, O at 256 and 384.
// Every wait is bounded; on expiry all roles leave their loops, the loader
// waits for its copies in flight and TMEM is freed.
#pragma once
#include <cuda.h>
#include "attention_few.cuh"

namespace pir2b {

constexpr int kTileThreads = 384;
constexpr int kSourceRows = 0;   // K and V source: packed rows, else a cache format
constexpr int kTileKeys = 128;

template <int D>
struct TileShape {
  static constexpr int kBytes = 128 * D * 2;            // a Q, K or V tile
  static constexpr int kStages = D == 128 ? 5 : 8;
  static constexpr int kSmem = (2 + kStages) * kBytes + 1024 /* alignment */ + 256 /* barriers */;
};

struct TileBarriers {
  uint64_t full[8], empty[8], q_full[2], s_full[2], p_full[2], o_full[2], to_mend[3], mended[3];
  uint32_t tmem;
  int spoiled;   // a V block held a value that is not finite at a position hidden from some row
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

// Descriptor of a B operand stored [K rows][64 columns] in 128-byte swizzled
// rows, further 64-column blocks `block` bytes apart: 8 rows of K are 1024
// bytes.
__device__ __forceinline__ uint64_t smem_desc_rows(uint32_t saddr, uint32_t block) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>((block >> 4) & 0x3FFFu) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

__device__ __forceinline__ void tmem_st_32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, "
      "%25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 3-D and 4-D tiled loads into this CTA's shared memory.
__device__ __forceinline__ void tma_load_3d(void *dst, const void *tmap, uint64_t *bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(tmap), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

template <int kRegisters>
__device__ __forceinline__ void registers_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegisters));
}
template <int kRegisters>
__device__ __forceinline__ void registers_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegisters));
}

// What a CTA works on.
struct TileWork {
  int b;              // sequence
  int r0, r1;         // its rows [r0, min(r0 + 256, r1)) of the sequence's token x head rows
  int64_t begin;      // packed row of its first token
  int first;          // position of its first token (prompts: 0)
  int keys;           // positions any row sees
  int all_see;        // positions below this are seen by every row
  int blocks0, blocks1;   // 128-key blocks of each tile

  __device__ __forceinline__ int blocks(int u) const { return u ? blocks1 : blocks0; }
};

template <int kSource, int D>
__global__ void __launch_bounds__(kTileThreads, 1)
    attention_tile_kernel(const RaggedArgs a, const __grid_constant__ CUtensorMap tm_k,
                          const __grid_constant__ CUtensorMap tm_v) {
  using Shape = TileShape<D>;
  constexpr int kStages = Shape::kStages, kBytes = Shape::kBytes;
  constexpr int kHalves = D / 64;                 // 64-column blocks of a tile, 16 KB each
  extern __shared__ uint8_t tile_raw[];
  uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(tile_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *q_sm = sm, *ring = sm + 2 * kBytes;
  TileBarriers &bar = *reinterpret_cast<TileBarriers *>(ring + kStages * kBytes);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (warp == 8) {
    if (lane == 0) {
      for (int i = 0; i < kStages; ++i) {
        mbar_init(&bar.full[i], 1);
        mbar_init(&bar.empty[i], 1);
      }
      for (int u = 0; u < 2; ++u) {
        mbar_init(&bar.q_full[u], 128);
        mbar_init(&bar.s_full[u], 1);
        mbar_init(&bar.p_full[u], 4);
        mbar_init(&bar.o_full[u], 1);
      }
      for (int i = 0; i < 3; ++i) {
        mbar_init(&bar.to_mend[i], 1);
        mbar_init(&bar.mended[i], 2);
      }
      bar.spoiled = 0;
      fence_barrier_init();
    }
    __syncwarp();
    tmem_alloc(&bar.tmem, 512);
    tmem_relinquish();
  }
  if (warp == 9 && lane == 0) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  pdl_wait();
  pdl_launch_dependents();
  const int group = a.hq / a.hk;
  // Later rows see more keys: they start first.
  const int kvh = int(blockIdx.x % a.hk), slot = int((gridDim.x - 1 - blockIdx.x) / a.hk);
  TileWork w = {};
  int tile;
  w.b = unit_of(a, group, 8, slot, tile);
  if (w.b >= 0) {
    w.begin = max(__ldg(a.starts + w.b), 0);
    const int n = int(min(int64_t(__ldg(a.starts + w.b + 1)), a.rows) - w.begin);
    w.r0 = tile << 8;
    w.r1 = n * group;
    int length = n;
    if constexpr (kSource != kSourceRows) {
      length = cache_length(a.c, a.lengths, w.b);
      w.first = first_new_position(a.lengths, w.b, n);
    }
    w.all_see = max(0, min(length, w.first + w.r0 / group + 1));
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int last = min(w.r0 + 128 * (u + 1), w.r1) - 1;   // last row of the tile
      const int keys = last < w.r0 + 128 * u ? 0 : max(0, min(length, w.first + last / group + 1));
      (u ? w.blocks1 : w.blocks0) = (keys + kTileKeys - 1) / kTileKeys;
      w.keys = max(w.keys, keys);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar.tmem;
  const int blocks = max(w.blocks0, w.blocks1);
  // The rows' limits span at most 256 positions, so at most three blocks hold
  // positions hidden from some row; each has its barriers.
  const int first_mend = w.all_see / kTileKeys;

  if (warp < 8) {
    registers_up<208>();
    const int u = warp >> 2, t = tid & 127;
    const uint32_t lanes = uint32_t(warp & 3) << 21;          // this warp's TMEM lanes
    const uint32_t s_tm = tmem + lanes + u * 128, o_tm = tmem + lanes + 256 + u * 128;
    const int r = w.r0 + u * 128 + t;                         // this thread's row
    const bool valid = w.b >= 0 && r < w.r1;
    const int limit = valid ? w.first + r / group : -1;       // it sees positions 0 .. limit
    bool ok = true;
    if (w.blocks(u) > 0) {
      for (int i = t; i < 128 * (D / 8); i += 128) {
        const int qr = i / (D / 8), c = i % (D / 8);
        uint8_t *dst = q_sm + u * kBytes + (c >> 3) * 16384 + qr * 128 + (((c & 7) ^ (qr & 7)) << 4);
        const int rr = w.r0 + u * 128 + qr;
        if (rr < w.r1)
          cp_async_16(dst, a.q + (w.begin + rr / group) * a.q_row + (kvh * group + rr % group) * a.q_head + c * 8);
        else
          *reinterpret_cast<uint4 *>(dst) = make_uint4(0, 0, 0, 0);
      }
      cp_async_wait_all();
      fence_proxy_async_smem();
      mbar_arrive(&bar.q_full[u]);
    }
    float top = -INFINITY, mu = 0.f, l = 0.f;
    for (int j = 0; j < w.blocks(u); ++j) {
      if (!mbar_wait(&bar.s_full[u], j & 1, kStatusTimeoutEpilogue)) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        tmem_ld_32(s_tm + i * 32, s[i]);
      tmem_ld_wait();
      const int seen = limit - j * kTileKeys;                 // columns above this are hidden
      if (__any_sync(0xffffffffu, seen < kTileKeys - 1)) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (i * 32 + c > seen)
              s[i][c] = 0xff800000u;
      }
      float most = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 32; ++c)
          most = fmaxf(most, __uint_as_float(s[i][c]));
      most *= a.scale_log2;
      if (__any_sync(0xffffffffu, most > top + 8.f)) {
        const float m = fmaxf(top, most);
        const float keep = top == -INFINITY ? 1.f : exp2_fast(top - m);   // nothing summed yet: keep it
        top = m;
        mu = m == -INFINITY ? 0.f : m;
        l *= keep;
        if (j > 0) {
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            uint32_t o[32];
            tmem_ld_32(o_tm + i * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < 32; ++c)
              o[c] = __float_as_uint(__uint_as_float(o[c]) * keep);
            tmem_st_32(o_tm + i * 32, o);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t p[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const float x = exp2_fast(__uint_as_float(s[2 * i + c / 16][c * 2 % 32]) * a.scale_log2 - mu);
          const float y = exp2_fast(__uint_as_float(s[2 * i + c / 16][c * 2 % 32 + 1]) * a.scale_log2 - mu);
          l += x + y;
          p[c] = pack_bf16x2(x, y);
        }
        tmem_st_32(s_tm + i * 32, p);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&bar.p_full[u]);
    }
    if (ok && w.blocks(u) > 0)
      ok = mbar_wait(&bar.o_full[u], 0, kStatusTimeoutEpilogue);
    tc_fence_after();
    if (ok && w.b >= 0 && w.r0 + u * 128 < w.r1) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const bool spoiled = *reinterpret_cast<volatile int *>(&bar.spoiled) != 0;
      __nv_bfloat16 *out = a.out + (w.begin + r / group) * a.ldo + (kvh * group + r % group) * D;
#pragma unroll 1
      for (int i = 0; i < D / 32; ++i) {
        uint32_t o[32] = {};
        if (w.blocks(u) > 0) {
          tmem_ld_32(o_tm + i * 32, o);
          tmem_ld_wait();
        }
        float f[32];
#pragma unroll
        for (int c = 0; c < 32; ++c)
          f[c] = __uint_as_float(o[c]) * inv;
        if (spoiled) {
          // Values that are not finite were left out of the products from
          // position all_see on: they go to the rows that see them.
          for (int key = w.all_see; key <= limit; ++key) {
            const __nv_bfloat16 *v = a.v + (w.begin + key) * a.v_row + kvh * a.v_head + i * 32;
            for (int c = 0; c < 32; ++c) {
              const float x = __bfloat162float(v[c]);
              if (!(fabsf(x) < INFINITY))
                f[c] += x;
            }
          }
        }
        if (valid) {
#pragma unroll
          for (int c = 0; c < 32; c += 8)
            *reinterpret_cast<uint4 *>(out + i * 32 + c) =
                make_uint4(pack_bf16x2(f[c], f[c + 1]), pack_bf16x2(f[c + 2], f[c + 3]), pack_bf16x2(f[c + 4], f[c + 5]),
                           pack_bf16x2(f[c + 6], f[c + 7]));
        }
      }
    }
  } else {
    registers_down<80>();
    if (warp == 8) {
      if (elect_one_sync()) {
        constexpr uint32_t kIdescS = idesc_bf16(128, kTileKeys, false), kIdescO = idesc_bf16(128, D, true);
        const uint32_t q_addr = smem_u32(q_sm), ring_addr = smem_u32(ring);
        auto wait = [&](uint64_t *b, int parity) { return mbar_wait(b, uint32_t(parity & 1), kStatusTimeoutMma); };
        auto scores = [&](int u, int item) {
          const uint32_t k_addr = ring_addr + (item % kStages) * kBytes;
#pragma unroll
          for (int s = 0; s < D / 16; ++s) {
            const uint32_t at = (s >> 2) * 16384 + (s & 3) * 32;
            mma_bf16_ss(tmem + u * 128, smem_desc_sw128(q_addr + u * kBytes + at), smem_desc_sw128(k_addr + at), kIdescS,
                        s > 0);
          }
          mma_commit(&bar.s_full[u]);
        };
        bool ok = blocks > 0 && wait(&bar.full[0], 0);
        for (int u = 0; u < 2 && ok; ++u)
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
          for (int u = 0; u < 2 && ok; ++u) {
            if (j >= w.blocks(u))
              continue;
            if (!v_ready) {
              if ((j + 1) * kTileKeys > w.all_see)
                ok = wait(&bar.mended[j - first_mend], 0);
              else
                ok = wait(&bar.full[v_item % kStages], v_item / kStages);
              v_ready = true;
            }
            ok = ok && wait(&bar.p_full[u], j);
            if (!ok)
              break;
            tc_fence_after();
            const uint32_t v_addr = ring_addr + (v_item % kStages) * kBytes;
#pragma unroll
            for (int s = 0; s < kTileKeys / 16; ++s)
              mma_bf16_ts(tmem + 256 + u * 128, tmem + u * 128 + s * 8, smem_desc_rows(v_addr + s * 2048, 16384), kIdescO,
                          j > 0 || s > 0);
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
    } else if (warp == 9) {
      if (elect_one_sync()) {
        int item = 0;
        for (; item < 2 * blocks; ++item) {
          const int stage = item % kStages;
          if (item >= kStages && !mbar_wait(&bar.empty[stage], uint32_t((item / kStages - 1) & 1), kStatusTimeoutProducer))
            break;
          mbar_arrive_expect_tx(&bar.full[stage], kBytes);
          const void *map = (item & 1) ? &tm_v : &tm_k;
#pragma unroll
          for (int h = 0; h < kHalves; ++h)
            tma_load_3d(ring + stage * kBytes + h * 16384, map, &bar.full[stage], h * 64, kvh,
                        int(w.begin) + (item >> 1) * kTileKeys);
          if ((item & 1) && ((item >> 1) + 1) * kTileKeys > w.all_see)
            mbar_arrive(&bar.to_mend[(item >> 1) - first_mend]);
        }
        // No copy is in flight when the CTA ends (at once, unless a wait gave up).
        for (int i = max(0, item - kStages); i < item; ++i)
          mbar_wait(&bar.full[i % kStages], uint32_t((i / kStages) & 1), kStatusTimeoutProducer);
      }
    } else {
      // Positions some row of the tiles must not see: those past the keys
      // become 0, and a value that is not finite is left out (0 times it
      // would be NaN in the rows that do not see it).
      // The loader says when such a block is on its way: only then is its
      // stage's barrier in the phase that is waited for.
      for (int j = first_mend; j < blocks; ++j) {
        const int item = 2 * j + 1;
        if (!mbar_wait(&bar.to_mend[j - first_mend], 0, kStatusTimeoutConvert) ||
            !mbar_wait(&bar.full[item % kStages], uint32_t((item / kStages) & 1), kStatusTimeoutConvert))
          break;
        uint8_t *v = ring + (item % kStages) * kBytes;
        const int from = max(0, w.all_see - j * kTileKeys), end = w.keys - j * kTileKeys;
        bool found = false;
        for (int i = (warp - 10) * 32 + lane; i < (kTileKeys - from) * (D / 8); i += 64) {
          const int key = from + i / (D / 8), c = i % (D / 8);
          uint4 *at = reinterpret_cast<uint4 *>(v + (c >> 3) * 16384 + key * 128 + (((c & 7) ^ (key & 7)) << 4));
          if (key >= end) {
            *at = make_uint4(0, 0, 0, 0);
          } else {
            uint4 x = *at;
            uint32_t *word = reinterpret_cast<uint32_t *>(&x);
            bool bad = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if ((word[e] & 0x7f80u) == 0x7f80u)
                word[e] &= 0xffff0000u, bad = true;
              if ((word[e] & 0x7f800000u) == 0x7f800000u)
                word[e] &= 0xffffu, bad = true;
            }
            if (bad)
              *at = x, found = true;
          }
        }
        if (found)
          *reinterpret_cast<volatile int *>(&bar.spoiled) = 1;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0)
          mbar_arrive(&bar.mended[j - first_mend]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8)
    tmem_dealloc(tmem, 512);
}

} // namespace pir2b
