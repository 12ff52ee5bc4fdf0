// Attention entry points: checks, the choice of the split over the keys, and
// dispatch by element type (kernels: attention.h).
#include <algorithm>
#include <cmath>

#include "attention.h"

namespace nhip {
namespace {

// Checks the sizes and fills them in, chooses the kernel (vec: rows that the
// one for many rows takes; cache: over the 8-bit cache) and the number of parts
// of the keys.
int attn_args(const nhip_attention_desc* d, bool vec, bool cache, AttnArgs* a) {
  if (!d) return fail(NHIP_STATUS_NULL_POINTER, "attention: null descriptor");
  if (!elem_size(d->dtype)) return fail(NHIP_STATUS_UNSUPPORTED, "attention: dtype has to be F32, F16 or BF16");
  if (d->batch < 0 || d->queries < 0 || d->keys < 0) return fail(NHIP_STATUS_INVALID_SHAPE, "attention: negative extent");
  if (d->heads <= 0 || d->kv_heads <= 0 || d->heads % d->kv_heads)
    return fail(NHIP_STATUS_INVALID_SHAPE, "attention: kv_heads has to divide heads");
  if (d->head_dim <= 0 || d->head_dim > 256) return fail(NHIP_STATUS_INVALID_SHAPE, "attention: head_dim has to be 1 to 256");
  if (!std::isfinite(d->scale)) return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "attention: scale has to be finite");
  a->batch = d->batch;
  a->queries = d->queries;
  a->keys = d->keys;
  a->heads = d->heads;
  a->kv_heads = d->kv_heads;
  a->group = d->heads / d->kv_heads;
  a->d = d->head_dim;
  a->scale_log2 = d->scale * 1.4426950408889634f;
  // 2^30 leaves room for the last tile's keys and rows past the end
  const int64_t most = int64_t(1) << 30;
  if (d->keys > most || (int64_t)d->queries * a->group > most)
    return fail(NHIP_STATUS_SHAPE_ARITHMETIC_OVERFLOW, "attention: at most 2^30 keys, and rows of a key/value head");
  a->rows = d->queries * a->group;
  // The kernel of few rows reads all keys and values for every 16 of them, some
  // 8 TB/s from the L2s; the one of many reads them once for 128, and its parts
  // are joined in a launch of their own (5 us).  So the second where the first
  // would read longer than the second computes, unless its workgroups leave most
  // CUs idle; and where the first would have several workgroups a CU, each with
  // its own start.  The bounds are the best over 336 shapes (bf16 and fp32, heads
  // of 64 and 128; 8, 32, 80, 197, 784, 3136 keys; batch, heads, key/value heads 4,
  // 12, 12, 16, 16, 4, 1, 16, 16, 10, 8, 4; 4 to 784 rows), and 192 over the cache (256,
  // 1024, 4096 keys; 4, 12, 12, 16, 16, 4, 1, 32, 8; 4 to 256 rows), each timed with
  // both kernels (NHIP_ATTN_TILES): slower than the better one by 0.5 and 0.8% in
  // the mean.
  // us, few / many: 64 heads of 3136 keys of 128 bf16, 32 rows 38.1 / 30.9; 16 heads
  // of 784 keys of 64 fp32, 256 rows 20.5 / 31.8, of 3136 of 128 102.6 / 64.8; 64
  // heads of 197 keys, 256 rows of 64 bf16 13.4 / 9.9, of 128 24.3 / 13.6; 40 of 32
  // keys, 198 rows of 128 fp32 28.7 / 15.3; over the cache 8 heads of 1024 of 128,
  // 512 rows bf16 22.8 / 39.7, fp32 39.6 / 32.9.
  const int64_t kv_heads = (int64_t)d->batch * d->kv_heads, tiles16 = ceil_div(std::max(a->rows, 1), attn::kRowTile);
  const bool f32 = d->dtype == NHIP_DTYPE_F32;
  const double bytes = (double)kv_heads * d->keys * d->head_dim * 2 * (cache ? 1 : elem_size(d->dtype));
  const int force = setting_int("NHIP_ATTN_TILES", -1);
  const double few = (double)kv_heads * tiles16 / cu_count();  // workgroups of the first to a CU
  const bool full = cache ? few >= (f32 ? 3 : 4) : d->head_dim > 64 ? few >= 1.5 : f32 ? few > 2 : few >= 3;
  const double again = cache ? (f32 ? 28e6 : 90e6) : f32 ? 215e6 : 64e6;  // bytes
  a->tiles = vec && force != 0 && (force == 1 || full || (few >= 0.25 && (tiles16 - 1) * bytes > again));
  const int tile = a->tiles ? attn::kTilesRows : attn::kRowTile;
  a->row_tiles = (int)ceil_div(std::max(a->rows, 1), tile);
  const int64_t heads = (int64_t)d->batch * d->kv_heads;
  if (heads > 0x7fffff00 / attn::kTilesRows / a->row_tiles)
    return fail(NHIP_STATUS_SHAPE_ARITHMETIC_OVERFLOW, "attention: too many rows");
  const int64_t wgs = std::max<int64_t>(1, heads * a->row_tiles);
  a->splits = 1;
  if (!a->tiles) {
    // Few workgroups: the keys are split until there is one for every CU (three
    // over the cache), each part with at least 512 keys.  us at 1 / 2 / 4 a CU:
    // cross attention of 256 heads, 3136 keys 67.7 / 72.3 / 74.6; 2 / 3 / 4 over
    // the cache, 128 heads, 12544 keys 77.4 / 72.8 / 81.5.  Parts of 128 / 512 /
    // 1024 keys: 8 heads of 12544 keys 24.9 / 21.2 / 23.0, 4 of 500 13.1 / 9.1.
    const int64_t want = ((cache ? 3 : 1) * cu_count() + wgs / 2) / wgs;
    a->splits = (int)std::max<int64_t>(1, std::min<int64_t>({want, ceil_div(d->keys, 512), 64}));
    return ok();
  }
  // One row tile to a worker, or as many workers as there are places on the
  // CUs, the work dealt to them in equal runs of at least 256 keys, if that
  // saves more than it costs: the parts' way through memory and the launch that
  // joins them, and of each worker's pace a seventh (two row tiles' queries, all
  // CUs busy).  us, one each / dealt: 4 x 784 rows of 12 heads of 64 bf16 (336
  // row tiles) to 784 / 1500 / 3136 keys 23.5 / 33.5, 37.2 / 41.4, 68.3 / 63.7, of
  // 128 35.3 / 48.4, 55.7 / 64.3, 100 / 101, of 64 fp32 76.6 / 75.9, 132 / 116, 257 /
  // 215; 128, 256, 640 row tiles of 1024 keys of 64 bf16 20.7 / 23.3, 21.8 / 28.0,
  // 37.6 / 47.9, fp32 63.6 / 43.9, 67.9 / 67.4, 151 / 144; 784 of 12544 of 128 bf16 780 / 703.
  const int keys = a->d > (d->dtype == NHIP_DTYPE_F32 ? 64 : 128) ? 32 : 64;  // of a tile
  int64_t places = (int64_t)cu_count() * (a->d <= (d->dtype == NHIP_DTYPE_F32 ? 64 : 128) ? 2 : 1);
  a->workers = (int)wgs;
  a->units = std::max(1, (int)ceil_div(d->keys, keys));
  // Over the cache, where loads and codes are waited for, heads of 64 have room
  // for a third workgroup on a CU: us at 2 / 3, 16 heads on 4 of 509 rows to
  // 6272 keys 69.2 / 65; not in runs below 512 keys, 4 x 256 rows to 2048 keys 30.6 /
  // 32.2; nor without codes, 1024 rows and keys, 128 heads 52.0 / 70.
  if (cache && a->d <= 64 && d->dtype != NHIP_DTYPE_F32 && wgs * a->units * keys >= 512 * 3 * (int64_t)cu_count())
    places = 3 * (int64_t)cu_count();
  // TFLOP/s of a CU, measured; a workgroup alone on a CU with room for two has
  // 3/4 of what both have together (fp32: 5/8)
  const bool two = places > cu_count();
  const double rate = f32 ? (a->d <= 64 ? 0.84 : 0.55) : a->d <= 64 ? (cache ? 2.2 : 3.3) : a->d <= 128 ? 4.3 : 2.0;
  const double unit = 4e-6 * attn::kTilesRows * keys * a->d / rate;  // us
  const int64_t rounds = ceil_div(wgs, cu_count());
  const double each = rounds + (two && rounds % 2 ? (f32 ? 0.6 : 0.33) : 0.0), dealt = 1.15 * wgs / cu_count();
  const double join = 5 + 2.6 * places * attn::kTilesRows * a->d * sizeof(float) / 5e6;
  if (a->units * unit * (each - dealt) > join && wgs * a->units < 0x7fffffff) {
    const int64_t workers = std::min(places, wgs * a->units * keys / 256);
    if (workers > wgs || workers == places) a->workers = (int)std::max<int64_t>(1, workers);
  }
  const int dealt_to = setting_int("NHIP_ATTN_WORKERS", 0);
  if (dealt_to > 0 && wgs * a->units < 0x7fffffff) a->workers = (int)std::min<int64_t>(dealt_to, wgs * a->units);
  return ok();
}

// Parts' (maximum, sum) pairs, an even number; their sums follow, 16-byte aligned.
uint64_t parts_of(const AttnArgs& a) {
  if (a.tiles) return a.workers == a.batch * a.kv_heads * a.row_tiles ? 0 : (uint64_t)a.workers * 2 * attn::kTilesRows;
  return a.splits == 1 ? 0 : (uint64_t)round_up((int64_t)a.batch * a.kv_heads * a.rows * a.splits, 2);
}

uint64_t workspace_of(const AttnArgs& a) { return parts_of(a) * (a.d * sizeof(float) + sizeof(float2)); }

// The most that a call with this descriptor needs, whatever its strides.
int attn_workspace(const nhip_attention_desc* d, bool cache, uint64_t* bytes) {
  *bytes = 0;
  for (bool vec : {false, true}) {
    AttnArgs a{};
    NHIP_TRY(attn_args(d, vec, cache, &a));
    *bytes = std::max(*bytes, workspace_of(a));
  }
  return ok();
}

int attn_forward(AttnArgs& a, const nhip_attention_desc* d, int src, const void* query, const int64_t* qs, void* out,
                 void* workspace, uint64_t workspace_bytes, void* stream) {
  const int es = elem_size(d->dtype);
  if (!aligned_to(query, es) || !aligned_to(out, es))
    return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "attention: a tensor is not aligned to its type");
  a.q = query;
  a.o = out;
  for (int i = 0; i < 3; ++i) {
    if (qs[i] < 0) return fail(NHIP_STATUS_INVALID_SHAPE, "attention: negative stride");
    a.qs[i] = qs[i];
  }
  const uint64_t need = workspace_of(a);
  if (need) {
    if (!workspace) return fail(NHIP_STATUS_NULL_POINTER, "attention: null workspace");
    if (workspace_bytes < need || !aligned_to(workspace, 16))
      return fail(NHIP_STATUS_OUTPUT_CAPACITY_INSUFFICIENT, "attention: workspace too small or not 16-byte aligned");
    a.part_ml = (float2*)workspace;
    a.part_o = (float*)(a.part_ml + parts_of(a));
  }
  switch (d->dtype) {
    case NHIP_DTYPE_F32: return attn_run_f32(a, src, as_stream(stream));
    case NHIP_DTYPE_F16: return attn_run_f16(a, src, as_stream(stream));
    default: return attn_run_bf16(a, src, as_stream(stream));
  }
}

// 16-byte aligned rows, near enough for a tile's to be reached with 31 bits.
bool vec_rows(const void* p, const int64_t* strides, int es) {
  const int v = 16 / es;
  return aligned_to(p, 16) && strides[0] % v == 0 && strides[1] % v == 0 && strides[2] % v == 0 &&
         strides[1] <= (int64_t(1) << 24) / es;
}

}  // namespace
}  // namespace nhip

using namespace nhip;

extern "C" {

int nhip_cross_attention_workspace_size(const nhip_attention_desc* desc, uint64_t* bytes) {
  if (!bytes) return fail(NHIP_STATUS_NULL_POINTER, "attention: null pointer");
  return attn_workspace(desc, false, bytes);
}

int nhip_cross_attention_forward(const nhip_attention_desc* desc, const void* query, const int64_t* query_strides,
                                 const void* key, const int64_t* key_strides, const void* value,
                                 const int64_t* value_strides, const int32_t* key_lengths, const uint8_t* key_mask,
                                 int64_t mask_stride, void* out, void* workspace, uint64_t workspace_bytes,
                                 void* stream) {
  AttnArgs a{};
  NHIP_TRY(attn_args(desc, false, false, &a));
  if (desc->batch == 0 || desc->queries == 0) return ok();
  if (!query || !query_strides || !out || !key_strides || !value_strides || (desc->keys && (!key || !value)))
    return fail(NHIP_STATUS_NULL_POINTER, "attention: null pointer");
  const int es = elem_size(desc->dtype);
  if (!aligned_to(key, es) || !aligned_to(value, es) || !aligned_to(key_lengths, 4))
    return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "attention: a tensor is not aligned to its type");
  a.k = key;
  a.v = value;
  for (int i = 0; i < 3; ++i) {
    if (key_strides[i] < 0 || value_strides[i] < 0) return fail(NHIP_STATUS_INVALID_SHAPE, "attention: negative stride");
    a.ks[i] = key_strides[i];
    a.vs[i] = value_strides[i];
  }
  a.lengths = key_lengths;
  a.mask = key_mask;
  if (mask_stride < 0) return fail(NHIP_STATUS_INVALID_SHAPE, "attention: negative stride");
  a.mask_stride = mask_stride;
  const bool vec = desc->head_dim % (16 / es) == 0 && aligned_to(out, 16) && vec_rows(query, query_strides, es) &&
                   vec_rows(key, key_strides, es) && vec_rows(value, value_strides, es);
  NHIP_TRY(attn_args(desc, vec, false, &a));
  return attn_forward(a, desc, vec ? kSrcVec : kSrcAny, query, query_strides, out, workspace, workspace_bytes, stream);
}

int nhip_kv8_attention_workspace_size(const nhip_attention_desc* desc, const nhip_kv8_cache* cache, uint64_t* bytes) {
  if (!bytes || !cache) return fail(NHIP_STATUS_NULL_POINTER, "attention: null pointer");
  return attn_workspace(desc, true, bytes);
}

int nhip_kv8_attention_forward(const nhip_attention_desc* desc, const nhip_kv8_cache* cache, const void* query,
                               const int64_t* query_strides, const int32_t* block_table, int64_t table_pages,
                               const int32_t* lengths, int32_t causal, void* out, void* workspace,
                               uint64_t workspace_bytes, void* stream) {
  AttnArgs a{};
  NHIP_TRY(attn_args(desc, true, true, &a));
  NHIP_TRY(kv8_args(cache, block_table, table_pages, &a.cache));
  if (cache->kv_heads != desc->kv_heads || cache->head_dim != desc->head_dim)
    return fail(NHIP_STATUS_INVALID_SHAPE, "attention: the cache has other heads");
  if (desc->batch == 0 || desc->queries == 0) return ok();
  if (!query || !query_strides || !out || !lengths) return fail(NHIP_STATUS_NULL_POINTER, "attention: null pointer");
  if (!aligned_to(lengths, 4)) return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "attention: a tensor is not aligned to its type");
  a.lengths = lengths;
  a.causal = causal != 0;
  const int v = 16 / elem_size(desc->dtype);
  if (!aligned_to(query, 16) || !aligned_to(out, 16) || query_strides[0] % v || query_strides[1] % v || query_strides[2] % v)
    return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "attention: queries and results over the cache have to be 16-byte aligned");
  return attn_forward(a, desc, kSrcInt8, query, query_strides, out, workspace, workspace_bytes, stream);
}

}  // extern "C"
