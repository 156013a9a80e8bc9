// C ABI of the ragged-batch operators (packed prompts, paged K/V cache):
// argument checks and launches.
#pragma once
#include <type_traits>
#include <utility>
#include "attention_few.cuh"
#include "attention_ragged.cuh"
#include "attention_tile.cuh"
#include "capi.cuh"
#include "kv_cache.cuh"

namespace pir2b {

// Rows view [rows, heads, d] of bf16: strides in elements.
static int check_view(const char *what, const void *p, int64_t row, int64_t head) {
  if (p == nullptr)
    return fail(PIR2B_EINVAL, "%s must be non-null", what);
  if (!aligned(p, 16) || row % 8 != 0 || head % 8 != 0 || row < 0 || head < 0)
    return fail(PIR2B_EALIGN, "%s must be 16-byte aligned with row and head strides that are multiples of 8", what);
  return PIR2B_OK;
}

static int check_heads(const char *what, int hq, int hk, int d) {
  if (hk < 1 || hq < 1 || hq % hk != 0 || hq > 1024 || (d != 64 && d != 128))
    return fail(PIR2B_EINVAL, "%s: hq must be a multiple of hk (at most 1024 heads), head_dim 64 or 128", what);
  return PIR2B_OK;
}

static void set_heads(RaggedArgs *a, int hq, int hk) {
  a->hq = hq;
  a->hk = hk;
  a->group = hq / hk;
  a->inverse = a->group == 1 ? 0xffffffffu : uint32_t((uint64_t(1) << 32) / a->group);
}

static int check_out(const char *what, const void *out, int64_t ldo, int64_t width) {
  if (out == nullptr || ldo < width)
    return fail(PIR2B_EINVAL, "%s: output missing or its row stride below its width", what);
  if (!aligned(out, 16) || ldo % 8 != 0)
    return fail(PIR2B_EALIGN, "%s: output must be 16-byte aligned with a row stride that is a multiple of 8", what);
  return PIR2B_OK;
}

static int check_sequences(const char *what, const pir2b_sequences *s, int64_t rows, bool lengths) {
  if (s == nullptr || s->starts == nullptr || s->batch < 1 || s->table_width < 0 || s->table_stride < s->table_width ||
      (lengths && s->lengths == nullptr) || (s->table_width > 0 && s->table == nullptr))
    return fail(PIR2B_EINVAL, "%s: sequences need starts, lengths, a table and batch >= 1", what);
  if (rows < 0 || rows > 0x7fffffff)
    return fail(PIR2B_EINVAL, "%s: rows out of range", what);
  return PIR2B_OK;
}

static int make_pages(const char *what, const pir2b_kv_pages *p, const pir2b_sequences *s, CachePages *out) {
  if (p == nullptr || p->k == nullptr || p->v == nullptr || p->pages < 1 || p->kv_heads < 1 || p->kv_heads > 1024)
    return fail(PIR2B_EINVAL, "%s: a pool needs k, v, pages >= 1 and 1 to 1024 kv heads", what);
  if (p->page_size != 16 && p->page_size != 32 && p->page_size != 64 && p->page_size != 128)
    return fail(PIR2B_EINVAL, "%s: page_size must be 16, 32, 64 or 128", what);
  if (p->head_dim != 64 && p->head_dim != 128)
    return fail(PIR2B_EINVAL, "%s: head_dim must be 64 or 128", what);
  if (p->format != PIR2B_CACHE_BF16 && p->format != PIR2B_CACHE_INT8 && p->format != PIR2B_CACHE_E4M3)
    return fail(PIR2B_EINVAL, "%s: unknown cache format %d", what, p->format);
  const int64_t tokens = int64_t(p->kv_heads) * p->page_size;
  if (p->k_page_stride < tokens * p->head_dim || p->v_page_stride < tokens * p->head_dim)
    return fail(PIR2B_EINVAL, "%s: page strides below a page's size", what);
  if (!aligned(p->k, 16) || !aligned(p->v, 16) || p->k_page_stride % 16 != 0 || p->v_page_stride % 16 != 0)
    return fail(PIR2B_EALIGN, "%s: pages must be 16-byte aligned", what);
  if (p->format != PIR2B_CACHE_BF16 &&
      (p->k_scale == nullptr || p->v_scale == nullptr || !aligned(p->k_scale, 16) || !aligned(p->v_scale, 16) ||
       p->k_scale_page_stride < tokens || p->v_scale_page_stride < tokens || p->k_scale_page_stride % 4 != 0 ||
       p->v_scale_page_stride % 4 != 0))
    return fail(PIR2B_EINVAL, "%s: 8-bit pages need 16-byte aligned fp32 scales", what);
  out->k = p->k;
  out->v = p->v;
  out->ks = p->k_scale;
  out->vs = p->v_scale;
  out->k_page = p->k_page_stride;
  out->v_page = p->v_page_stride;
  out->ks_page = p->k_scale_page_stride;
  out->vs_page = p->v_scale_page_stride;
  out->table = s->table;
  out->ldt = s->table_stride;
  out->width = s->table_width;
  out->pages = p->pages;
  out->shift = p->page_size == 16 ? 4 : p->page_size == 32 ? 5 : p->page_size == 64 ? 6 : 7;
  out->hk = p->kv_heads;
  return PIR2B_OK;
}

// A launch that may start while its predecessor drains (every kernel here
// begins with griddepcontrol.wait).
// `cluster` consecutive CTAs form a thread-block cluster.
template <typename... Args>
static int launch_cache(const char *what, void (*kernel)(Args...), int64_t grid, int grid_y, int cluster, int threads,
                        size_t smem, void *stream, const std::remove_reference_t<Args> &...args) {
  if (grid > 0x7fffffff)
    return fail(PIR2B_EINVAL, "%s: too many rows", what);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(grid), unsigned(grid_y), 1);
  cfg.blockDim = dim3(unsigned(threads), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(cluster);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, args...), what);
}

// Few tokens are spread over more warps, one row load each (8 tokens of 8 kv
// heads: 2.1 us against 3.2, 862 tokens of 4: 2.3 against 3.2); many keep four
// in flight and share the search for their sequence.
template <int kFormat, int D>
static int launch_rows(bool write, const CacheRowsArgs &a, void *stream) {
  constexpr int kRows = 32 / (D / 16);                      // rows of a warp's load
  const int64_t grid = (a.rows + kCacheWarps - 1) / kCacheWarps;
  const int loads = (2 * a.c.hk + kRows - 1) / kRows;
  if (!write)
    return launch_cache("cache_read launch", cache_read_kernel<kFormat, D>, grid, 1, 1, kCacheWarps * 32, 0, stream, a);
  if (a.rows * loads <= 4096)
    return launch_cache("cache_write launch", cache_write_kernel<kFormat, D, 1>, grid, loads, 1, kCacheWarps * 32, 0, stream, a);
  return launch_cache("cache_write launch", cache_write_kernel<kFormat, D, 4>, grid, (loads + 3) / 4, 1, kCacheWarps * 32, 0,
                      stream, a);
}

template <int kFormat>
static int launch_rows(bool write, int d, const CacheRowsArgs &a, void *stream) {
  return d == 64 ? launch_rows<kFormat, 64>(write, a, stream) : launch_rows<kFormat, 128>(write, a, stream);
}

static int launch_rows(bool write, int format, int d, const CacheRowsArgs &a, void *stream) {
  switch (format) {
  case kCacheInt8: return launch_rows<kCacheInt8>(write, d, a, stream);
  case kCacheE4m3: return launch_rows<kCacheE4m3>(write, d, a, stream);
  default: return launch_rows<kCacheBf16>(write, d, a, stream);
  }
}

// Rows a sequence has in a kv head up to which the few-row kernel takes it; it
// reads the keys once per 16 rows, the tile kernel once per 128 or 256.  Over
// 1000 tokens of 64 sequences: 16 rows 50 us against 55 (bf16) and 50 against
// 110 (int8, whose tiles are converted first), 24 rows 80 against 56 and 84
// against 111, 34 rows 115 against 55 and 125 against 110.
constexpr int kFewRowsBf16 = 16, kFewRows8Bit = 32;

// How the few-row kernel covers a call: a cluster of CTAs per unit of rows,
// which joins its sums in shared memory, or, where units are few and long, a
// list of pieces that a second launch joins.
struct FewPlan {
  int nt;            // 8 nt rows per unit
  int cluster;       // CTAs of a unit, 0: pieces
  int64_t slots;     // of units
  int64_t pieces;    // CTAs wanted
  int64_t grid;
  int64_t bytes(int hk, int d) const { return cluster ? 0 : grid * 8 * nt * (d * 4 + 8) + slots * hk * 8; }
};

static FewPlan plan_few(int64_t rows, int hq, int hk, int batch, int64_t positions, int format, int d, int sms) {
  FewPlan p = {};
  const int group = hq / hk;
  const int64_t per_sequence = (rows + batch - 1) / batch * group;
  p.nt = per_sequence <= 8 ? 1 : 2;
  p.slots = rows * group / (8 * p.nt) + batch;
  const int resident = few_ctas(format, d, p.nt);
  const int64_t units = batch * ((per_sequence + 8 * p.nt - 1) / (8 * p.nt)) * hk;
  const int64_t longest = (positions + 16 * kFewWarps - 1) / (16 * kFewWarps);    // CTAs a unit can use
  const int64_t places = int64_t(resident) * sms;
  // Pieces of equal length, in one round of CTAs, where a unit has four places
  // or more on the SMs; but up to 2560 keys a cluster, which needs no second
  // launch, and up to 6144 where clusters of four fill the SMs.  8 kv heads,
  // cluster against pieces, one token: one int8 sequence of 2000 8.8 us against
  // 10.2, of 8000 17.7 against 13.9, of 30000 50 against 22; two tokens in a group
  // of four, eight bf16 sequences: of 2000-4000 20.5 against 22.9, of 3000-6000
  // 32.3 against 34.9.
  if (4 * units >= places || longest <= (8 * units > places ? 96 : 40)) {
    // One round of CTAs; a second only where each has 1280 keys or more (eight
    // bf16 sequences of 1000-2000 12.1 us with four to a unit, 18.2 with eight;
    // 64 int8 ones of 500-4000 62 with two, 74 with four; 64 of 2000-4000, group
    // of four, 80 with two, 102 with one).
    p.cluster = 1;
    while (p.cluster < 8 && 2 * p.cluster <= longest && p.cluster * units < places &&
           (2 * p.cluster * units <= places || positions >= 1280 * 2 * p.cluster))
      p.cluster *= 2;
    p.grid = p.slots * hk * p.cluster;
  } else {
    p.pieces = places;
    p.grid = p.pieces + p.slots * hk;              // each unit may have a piece more
  }
  return p;
}

// 4-D map over pages [pages, hk, page, d], box of `rows` rows of one head: 64
// columns of bf16 or whole rows of codes, swizzled over the row's 128 or 64
// bytes or as they lie.
static int make_pages_map(CUtensorMap *map, const void *base, const CachePages &c, int d, int64_t page_stride, int bytes,
                          int rows, bool swizzled) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr)
    return fail(PIR2B_ECUDA, "cuTensorMapEncodeTiled entry point unavailable");
  const cuuint64_t page = cuuint64_t(1) << c.shift;
  const cuuint64_t dims[4] = {cuuint64_t(d), page, cuuint64_t(c.hk), cuuint64_t(c.pages)};
  const cuuint64_t strides[3] = {cuuint64_t(d) * bytes, page * d * bytes, cuuint64_t(page_stride) * bytes};
  const cuuint32_t box[4] = {bytes == 2 ? 64u : cuuint32_t(d), cuuint32_t(rows), 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = fn(map, bytes == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 4,
                  const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  !swizzled ? CU_TENSOR_MAP_SWIZZLE_NONE
                            : box[0] * bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? PIR2B_OK : fail(PIR2B_ECUDA, "cuTensorMapEncodeTiled (pages) failed (%d)", int(r));
}

// Whether CTAs start in the order of their sequences' lengths, longest first:
// where there are more than run at once and a CTA may have 1024 keys or more
// (64 sequences of 500-4000 tokens, one new token each: 62 us against 72; chunks
// of 250-288 over 16 of 544-2100: 121 against 133).  Shorter ones lose more by
// looking up the order (28 sequences of 660-1320 in eighths: 17.8 us against
// 15.6), and so do the many short CTAs of prompts (64 prompts: 196 against 179).
static bool by_length(const RaggedArgs &a, int64_t grid, int resident, int parts) {
  return a.lengths != nullptr && a.batch > 1 && a.batch <= kOrdered && grid > int64_t(resident) * a.sms &&
         (int64_t(a.c.width) << a.c.shift) >= int64_t(1024) * parts;
}

template <int kFormat, int D, int kNT>
static int launch_attention_few(const FewPlan &p, RaggedArgs a, void *stream) {
  a.ordered = by_length(a, p.grid, FewShape<kFormat, D, kNT>::kCtas, std::max(p.cluster, 1));
  constexpr int kBytes = kFormat == kCacheBf16 ? 2 : 1;
  CUtensorMap tm_k, tm_v;
  if (int r = make_pages_map(&tm_k, a.c.k, a.c, D, a.c.k_page, kBytes, 16, true))
    return r;
  if (int r = make_pages_map(&tm_v, a.c.v, a.c, D, a.c.v_page, kBytes, 16, true))
    return r;
  return launch_cache("cache_attention launch", attention_few_kernel<kFormat, D, kNT>, p.grid, 1, std::max(p.cluster, 1), kFewWarps * 32,
                      FewShape<kFormat, D, kNT>::kSmem, stream, a, tm_k, tm_v);
}

template <int kFormat>
static int launch_attention_few(const FewPlan &p, int d, const RaggedArgs &a, void *stream) {
  if (d == 64)
    return p.nt == 1 ? launch_attention_few<kFormat, 64, 1>(p, a, stream) : launch_attention_few<kFormat, 64, 2>(p, a, stream);
  return p.nt == 1 ? launch_attention_few<kFormat, 128, 1>(p, a, stream) : launch_attention_few<kFormat, 128, 2>(p, a, stream);
}

// 3-D map over packed bf16 rows [rows, heads, d], box of 64 columns in
// 128-byte swizzled rows.
static int make_rows_map(CUtensorMap *map, const void *base, int64_t rows, int heads, int d, int64_t row, int64_t head,
                         int box_heads, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr)
    return fail(PIR2B_ECUDA, "cuTensorMapEncodeTiled entry point unavailable");
  const cuuint64_t dims[3] = {cuuint64_t(d), cuuint64_t(heads), cuuint64_t(rows)};
  const cuuint64_t strides[2] = {cuuint64_t(head) * 2, cuuint64_t(row) * 2};
  const cuuint32_t box[3] = {64, cuuint32_t(box_heads), cuuint32_t(box_rows)};
  const cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? PIR2B_OK : fail(PIR2B_ECUDA, "cuTensorMapEncodeTiled (rows) failed (%d)", int(r));
}

// A query tile is one box (its heads, then its tokens) when the group divides
// 128; otherwise its rows are gathered.
static int make_q_map(CUtensorMap *map, RaggedArgs *a, int d) {
  const int group = a->hq / a->hk;
  a->q_by_tma = 128 % group == 0;
  a->out_by_tma = 32 % group == 0;
  return make_rows_map(map, a->q, a->rows, a->hq, d, a->q_row, a->q_head, a->q_by_tma ? group : 1,
                       a->q_by_tma ? 128 / group : 128);
}

// Output rows leave 32 at a time (a warp's) where the group divides 32.
static int make_o_map(CUtensorMap *map, const RaggedArgs &a, int d) {
  return make_rows_map(map, a.out, a.rows, a.hq, d, a.ldo, d, a.out_by_tma ? a.group : 1, a.out_by_tma ? 32 / a.group : 32);
}

template <int kSource, int D, int kTiles>
static int launch_tile(const char *what, RaggedArgs a, const CUtensorMap &tm_q, const CUtensorMap &tm_k,
                       const CUtensorMap &tm_v, void *stream) {
  CUtensorMap tm_o;
  if (int r = make_o_map(&tm_o, a, D))
    return r;
  using Shape = TileShape<kSource, D, kTiles>;
  const int64_t grid = (a.rows * (a.hq / a.hk) / (128 * kTiles) + a.batch) * a.hk * a.splits;
  a.ordered = by_length(a, grid, 3 - kTiles, a.splits);
  return launch_cache(what, attention_tile_kernel<kSource, D, kTiles>, grid, 1, 1, Shape::kThreads, Shape::kSmem, stream, a,
                      tm_q, tm_k, tm_v, tm_o);
}

// Tiles per CTA of the tile kernel over prompts.  One tile and two CTAs on an SM
// cover the latencies of a CTA's start and end with another's products (64 prompts
// of 280-816 tokens: 178 us against 203, one of 544: 12.5 against 13.9, one of
// 2048: 35.1 against 36.8); two tiles read K and V half as often, which carries
// long prompts of heads of 128 (16 and 8 heads, one of 8192: 235 against 236, two:
// 460 against 472, one of 16384: 880 against 912) but not of 64 (12 and 4 heads,
// one of 8192: 180 against 165, of 16384: 640 against 605).
static int tiles_per_cta(int64_t rows, int batch, int d) { return d == 128 && rows / batch >= 8192 ? 2 : 1; }

// How a call of cache_attention runs: the few-row kernel (tiles = 0) or
// 128-row tiles, and its splits along the keys.
struct CachePlan {
  int tiles;
  FewPlan few;
  int splits;
  bool joined() const { return tiles == 0 ? few.cluster == 0 : splits > 1; }
};

static CachePlan plan_cache(int64_t rows, int hq, int hk, int d, int batch, int64_t positions, int format, int sms) {
  CachePlan p = {};
  const int64_t per_sequence = (rows + batch - 1) / batch * (hq / hk);
  if (per_sequence <= (format == kCacheBf16 ? kFewRowsBf16 : kFewRows8Bit)) {
    p.few = plan_few(rows, hq, hk, batch, positions, format, d, sms);
    return p;
  }
  p.tiles = format != kCacheBf16 || per_sequence > 128 ? 2 : 1;
  const int64_t ctas = batch * ((per_sequence + 128 * p.tiles - 1) / (128 * p.tiles)) * hk;
  // Splits of two blocks or more fill the SMs, from six blocks on (one sequence
  // of 40 rows, 8 kv heads, bf16: over 1000 tokens 14.4 us against 17.0 with four
  // blocks or more, over 4000 16.2 against 16.7; 270 rows over 300: 20.8 against
  // 16.7 in one).
  p.splits = positions < 6 * kTileKeys ? 1
             : int(std::max<int64_t>(1, std::min<int64_t>({sms * (3 - p.tiles) / ctas, positions / (2 * kTileKeys), 32})));
  return p;
}

template <int kSource, int D>
static int launch_cache_tile(const CachePlan &p, RaggedArgs a, void *stream) {
  constexpr int kBytes = kSource == kCacheBf16 ? 2 : 1;
  CUtensorMap tm_q, tm_k, tm_v;
  if (int r = make_q_map(&tm_q, &a, D))
    return r;
  if (int r = make_pages_map(&tm_k, a.c.k, a.c, D, a.c.k_page, kBytes, 1 << a.c.shift, kBytes == 2))
    return r;
  if (int r = make_pages_map(&tm_v, a.c.v, a.c, D, a.c.v_page, kBytes, 1 << a.c.shift, kBytes == 2))
    return r;
  if constexpr (kSource == kCacheBf16) {
    if (p.tiles == 1)
      return launch_tile<kSource, D, 1>("cache_attention launch", a, tm_q, tm_k, tm_v, stream);
  }
  return launch_tile<kSource, D, 2>("cache_attention launch", a, tm_q, tm_k, tm_v, stream);
}

template <int kFormat>
static int launch_cache_attention(const CachePlan &p, int d, const RaggedArgs &a, void *stream) {
  if (p.tiles == 0)
    return launch_attention_few<kFormat>(p.few, d, a, stream);
  return d == 64 ? launch_cache_tile<kFormat, 64>(p, a, stream) : launch_cache_tile<kFormat, 128>(p, a, stream);
}

static int launch_join(const CachePlan &p, int d, const RaggedArgs &a, void *stream) {
  if (p.tiles == 0)
    return launch_cache("cache_attention join launch",
                        d == 64 ? (p.few.nt == 1 ? attention_join_pieces_kernel<64, 1> : attention_join_pieces_kernel<64, 2>)
                                : (p.few.nt == 1 ? attention_join_pieces_kernel<128, 1> : attention_join_pieces_kernel<128, 2>),
                        a.rows * a.hq, 1, 1, 256, 0, stream, a);
  return launch_cache("cache_attention join launch", d == 64 ? attention_join_kernel<64> : attention_join_kernel<128>,
                      (a.rows * a.hq + 7) / 8, 1, 1, 256, 0, stream, a);
}

// Dynamic shared memory above the default limit, once per device.
static int cache_kernel_attributes(DeviceInfo *dev) {
  std::lock_guard<std::mutex> lock(g_mutex);
  if (dev->cache_attrs_set)
    return PIR2B_OK;
  const std::pair<const void *, int> kernels[] = {
      {reinterpret_cast<const void *>(attention_few_kernel<kCacheBf16, 64, 1>), FewShape<kCacheBf16, 64, 1>::kSmem},
      {reinterpret_cast<const void *>(attention_few_kernel<kCacheBf16, 64, 2>), FewShape<kCacheBf16, 64, 2>::kSmem},
      {reinterpret_cast<const void *>(attention_few_kernel<kCacheBf16, 128, 1>), FewShape<kCacheBf16, 128, 1>::kSmem},
      {reinterpret_cast<const void *>(attention_few_kernel<kCacheBf16, 128, 2>), FewShape<kCacheBf16, 128, 2>::kSmem},
      {reinterpret_cast<const void *>(attention_few_kernel<kCacheInt8, 64, 1>), FewShape<kCacheInt8, 64, 1>::kSmem},
      {reinterpret_cast<const void *>(attention_few_kernel<kCacheInt8, 64, 2>), FewShape<kCacheInt8, 64, 2>::kSmem},
      {reinterpret_cast<const void *>(attention_few_kernel<kCacheInt8, 128, 1>), FewShape<kCacheInt8, 128, 1>::kSmem},
      {reinterpret_cast<const void *>(attention_few_kernel<kCacheInt8, 128, 2>), FewShape<kCacheInt8, 128, 2>::kSmem},
      {reinterpret_cast<const void *>(attention_few_kernel<kCacheE4m3, 64, 1>), FewShape<kCacheE4m3, 64, 1>::kSmem},
      {reinterpret_cast<const void *>(attention_few_kernel<kCacheE4m3, 64, 2>), FewShape<kCacheE4m3, 64, 2>::kSmem},
      {reinterpret_cast<const void *>(attention_few_kernel<kCacheE4m3, 128, 1>), FewShape<kCacheE4m3, 128, 1>::kSmem},
      {reinterpret_cast<const void *>(attention_few_kernel<kCacheE4m3, 128, 2>), FewShape<kCacheE4m3, 128, 2>::kSmem},
      {reinterpret_cast<const void *>(attention_tile_kernel<kSourceRows, 64, 1>), TileShape<kSourceRows, 64, 1>::kSmem},
      {reinterpret_cast<const void *>(attention_tile_kernel<kSourceRows, 128, 1>), TileShape<kSourceRows, 128, 1>::kSmem},
      {reinterpret_cast<const void *>(attention_tile_kernel<kSourceRows, 128, 2>), TileShape<kSourceRows, 128, 2>::kSmem},
      {reinterpret_cast<const void *>(attention_tile_kernel<kCacheBf16, 64, 1>), TileShape<kCacheBf16, 64, 1>::kSmem},
      {reinterpret_cast<const void *>(attention_tile_kernel<kCacheBf16, 64, 2>), TileShape<kCacheBf16, 64, 2>::kSmem},
      {reinterpret_cast<const void *>(attention_tile_kernel<kCacheBf16, 128, 1>), TileShape<kCacheBf16, 128, 1>::kSmem},
      {reinterpret_cast<const void *>(attention_tile_kernel<kCacheBf16, 128, 2>), TileShape<kCacheBf16, 128, 2>::kSmem},
      {reinterpret_cast<const void *>(attention_tile_kernel<kCacheInt8, 64, 2>), TileShape<kCacheInt8, 64, 2>::kSmem},
      {reinterpret_cast<const void *>(attention_tile_kernel<kCacheInt8, 128, 2>), TileShape<kCacheInt8, 128, 2>::kSmem},
      {reinterpret_cast<const void *>(attention_tile_kernel<kCacheE4m3, 64, 2>), TileShape<kCacheE4m3, 64, 2>::kSmem},
      {reinterpret_cast<const void *>(attention_tile_kernel<kCacheE4m3, 128, 2>), TileShape<kCacheE4m3, 128, 2>::kSmem},
  };
  for (const auto &k : kernels)
    if (int r = cuda_status(cudaFuncSetAttribute(k.first, cudaFuncAttributeMaxDynamicSharedMemorySize, k.second),
                            "cudaFuncSetAttribute"))
      return r;
  dev->cache_attrs_set = true;
  return PIR2B_OK;
}

} // namespace pir2b

using namespace pir2b;

extern "C" {

int pir2b_prompt_attention(const void *q, int64_t q_row, int64_t q_head, const void *k,
                           int64_t k_row, int64_t k_head, const void *v, int64_t v_row,
                           int64_t v_head, const int32_t *starts, int64_t batch, int64_t rows,
                           int hq, int hk, int head_dim, float scale, void *out, int64_t ldo,
                           void *stream) {
  const char *what = "prompt_attention";
  if (int r = check_heads(what, hq, hk, head_dim))
    return r;
  if (rows < 0 || rows > 0x7fffffff || batch < 1 || batch > 0x7fffffff || starts == nullptr)
    return fail(PIR2B_EINVAL, "prompt_attention: need starts, batch >= 1 and rows >= 0");
  if (!(scale > 0.f) || !(scale < 3.0e38f))
    return fail(PIR2B_EINVAL, "prompt_attention: scale must be positive and finite");
  if (rows == 0)
    return PIR2B_OK;
  if (int r = check_view("prompt_attention q", q, q_row, q_head))
    return r;
  if (int r = check_view("prompt_attention k", k, k_row, k_head))
    return r;
  if (int r = check_view("prompt_attention v", v, v_row, v_head))
    return r;
  if (int r = check_out(what, out, ldo, int64_t(hq) * head_dim))
    return r;
  DeviceInfo *dev = nullptr;
  if (int r = device_info(&dev))
    return r;
  RaggedArgs a = {};
  a.q = static_cast<const __nv_bfloat16 *>(q);
  a.q_row = q_row;
  a.q_head = q_head;
  a.k = static_cast<const __nv_bfloat16 *>(k);
  a.k_row = k_row;
  a.k_head = k_head;
  a.v = static_cast<const __nv_bfloat16 *>(v);
  a.v_row = v_row;
  a.v_head = v_head;
  a.starts = starts;
  a.out = static_cast<__nv_bfloat16 *>(out);
  a.ldo = ldo;
  a.rows = rows;
  a.batch = int(batch);
  set_heads(&a, hq, hk);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.sms = dev->sms;
  a.splits = 1;
  if (int r = cache_kernel_attributes(dev))
    return r;
  CUtensorMap tm_q, tm_k, tm_v;
  if (int r = make_rows_map(&tm_k, k, rows, hk, head_dim, k_row, k_head, 1, kTileKeys))
    return r;
  if (int r = make_rows_map(&tm_v, v, rows, hk, head_dim, v_row, v_head, 1, kTileKeys))
    return r;
  if (int r = make_q_map(&tm_q, &a, head_dim))
    return r;
  const bool two = tiles_per_cta(rows, int(batch), head_dim) == 2;
  return (head_dim == 64 ? launch_tile<kSourceRows, 64, 1> : two ? launch_tile<kSourceRows, 128, 2> : launch_tile<kSourceRows, 128, 1>)(
      what, a, tm_q, tm_k, tm_v, stream);
}

int pir2b_cache_write(const void *k, int64_t k_row, int64_t k_head, const void *v, int64_t v_row,
                      int64_t v_head, int64_t rows, const pir2b_kv_pages *pages,
                      const pir2b_sequences *sequences, void *stream) {
  const char *what = "cache_write";
  CacheRowsArgs a = {};
  if (int r = check_sequences(what, sequences, rows, true))
    return r;
  if (int r = make_pages(what, pages, sequences, &a.c))
    return r;
  if (rows == 0)
    return PIR2B_OK;
  if (int r = check_view("cache_write k", k, k_row, k_head))
    return r;
  if (int r = check_view("cache_write v", v, v_row, v_head))
    return r;
  DeviceInfo *dev = nullptr;
  if (int r = device_info(&dev))
    return r;
  a.k = static_cast<const __nv_bfloat16 *>(k);
  a.v = static_cast<const __nv_bfloat16 *>(v);
  a.k_row = k_row;
  a.k_head = k_head;
  a.v_row = v_row;
  a.v_head = v_head;
  a.starts = sequences->starts;
  a.lengths = sequences->lengths;
  a.batch = sequences->batch;
  a.rows = rows;
  return launch_rows(true, pages->format, pages->head_dim, a, stream);
}

int pir2b_cache_read(const pir2b_kv_pages *pages, const pir2b_sequences *sequences, int64_t rows,
                     void *k_out, void *v_out, void *stream) {
  const char *what = "cache_read";
  CacheRowsArgs a = {};
  if (int r = check_sequences(what, sequences, rows, false))
    return r;
  if (int r = make_pages(what, pages, sequences, &a.c))
    return r;
  if (rows == 0)
    return PIR2B_OK;
  if (k_out == nullptr || v_out == nullptr)
    return fail(PIR2B_EINVAL, "cache_read outputs must be non-null");
  if (!aligned(k_out, 16) || !aligned(v_out, 16))
    return fail(PIR2B_EALIGN, "cache_read outputs must be 16-byte aligned");
  DeviceInfo *dev = nullptr;
  if (int r = device_info(&dev))
    return r;
  a.k_out = static_cast<__nv_bfloat16 *>(k_out);
  a.v_out = static_cast<__nv_bfloat16 *>(v_out);
  a.starts = sequences->starts;
  a.batch = sequences->batch;
  a.rows = rows;
  return launch_rows(false, pages->format, pages->head_dim, a, stream);
}

int pir2b_cache_attention(const void *q, int64_t q_row, int64_t q_head, int64_t rows, int hq,
                          const pir2b_kv_pages *pages, const pir2b_sequences *sequences,
                          float scale, void *out, int64_t ldo, void *workspace, void *stream) {
  const char *what = "cache_attention";
  RaggedArgs a = {};
  if (int r = check_sequences(what, sequences, rows, true))
    return r;
  if (int r = make_pages(what, pages, sequences, &a.c))
    return r;
  if (int r = check_heads(what, hq, pages->kv_heads, pages->head_dim))
    return r;
  if (!(scale > 0.f) || !(scale < 3.0e38f))
    return fail(PIR2B_EINVAL, "cache_attention: scale must be positive and finite");
  if (rows == 0)
    return PIR2B_OK;
  if (int r = check_view("cache_attention q", q, q_row, q_head))
    return r;
  if (int r = check_out(what, out, ldo, int64_t(hq) * pages->head_dim))
    return r;
  DeviceInfo *dev = nullptr;
  if (int r = device_info(&dev))
    return r;
  a.q = static_cast<const __nv_bfloat16 *>(q);
  a.q_row = q_row;
  a.q_head = q_head;
  a.starts = sequences->starts;
  a.lengths = sequences->lengths;
  a.out = static_cast<__nv_bfloat16 *>(out);
  a.ldo = ldo;
  a.rows = rows;
  a.batch = sequences->batch;
  set_heads(&a, hq, pages->kv_heads);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.sms = dev->sms;
  const int d = pages->head_dim;
  if (int r = cache_kernel_attributes(dev))
    return r;
  const CachePlan plan =
      plan_cache(rows, hq, a.hk, d, a.batch, int64_t(a.c.width) << a.c.shift, pages->format, dev->sms);
  a.splits = plan.splits;
  a.cluster = plan.few.cluster;
  if (plan.joined()) {
    if (workspace == nullptr || !aligned(workspace, 16))
      return fail(PIR2B_EALIGN, "cache_attention: this shape needs a 16-byte aligned workspace");
    const int64_t parts = plan.tiles == 0 ? plan.few.grid * 8 * plan.few.nt : plan.splits * rows * hq;
    a.part_o = static_cast<float *>(workspace);
    a.part_ml = reinterpret_cast<float2 *>(a.part_o + parts * d);
    a.part_units = reinterpret_cast<int2 *>(a.part_ml + parts);
    a.pieces = int(plan.few.pieces);
    a.parts = int(plan.few.grid);
  }
  int status = PIR2B_OK;
  switch (pages->format) {
  case kCacheInt8: status = launch_cache_attention<kCacheInt8>(plan, d, a, stream); break;
  case kCacheE4m3: status = launch_cache_attention<kCacheE4m3>(plan, d, a, stream); break;
  default: status = launch_cache_attention<kCacheBf16>(plan, d, a, stream); break;
  }
  return status != PIR2B_OK || !plan.joined() ? status : launch_join(plan, d, a, stream);
}

int64_t pir2b_cache_attention_workspace(int64_t rows, int hq, const pir2b_kv_pages *pages,
                                        const pir2b_sequences *sequences) {
  DeviceInfo *dev = nullptr;
  if (pages == nullptr || sequences == nullptr || rows < 1 || pages->kv_heads < 1 || hq < pages->kv_heads ||
      sequences->batch < 1 || device_info(&dev) != PIR2B_OK)
    return 0;                                     // the call itself reports what is wrong
  const CachePlan plan = plan_cache(rows, hq, pages->kv_heads, pages->head_dim, sequences->batch,
                                    int64_t(sequences->table_width) * pages->page_size, pages->format, dev->sms);
  if (!plan.joined())
    return 0;
  return plan.tiles == 0 ? plan.few.bytes(pages->kv_heads, pages->head_dim)
                         : int64_t(plan.splits) * rows * hq * (pages->head_dim * 4 + 8);
}

} // extern "C"
