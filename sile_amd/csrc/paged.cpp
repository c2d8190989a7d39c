// Entry points of the paged key-value cache: storing tokens, bookkeeping of the
// pages, and the attention of one new token a row.  Arguments are checked here;
// what stands in device memory (page numbers, lengths, positions) is checked by the
// kernels, which leave out what lies outside the pool or the table.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <cstring>

#include "kernels/chunk_plan.h"
#include "paged_checks.h"

using namespace sile_rt;

namespace {

// Kernel argument blocks; layouts match the structs in kernels/*.hip.
struct AppendArgs {
  const void *k, *v;
  const int32_t *rows, *positions, *tables;
  void *k_pages, *v_pages;
  int64_t tokens, ldk, ldv, page_stride, ld_table, capacity;
  int32_t heads, d, num_pages, page_shift, n_rows, per_group;
  float k_scale, v_scale, k_rcp, v_rcp;
};
constexpr int kMaxPools = 128;
constexpr int64_t kSegB = 16384;
struct Pools {
  void* base[kMaxPools];
  int64_t page_bytes, page_stride;
  int32_t count, segs;
};
struct ReserveArgs {
  const int32_t *lengths, *need, *tables_in;
  int32_t* tables_out;
  const int32_t* refs_in;
  int32_t *refs_out, *granted, *demand, *kept, *fresh;
  int64_t ld_table;
  int32_t n_rows, num_pages, page_shift;
};
struct PagedArgs {
  const void *q, *k, *v;
  void* o;
  const int32_t *tables, *lengths;
  int32_t* plan;
  float *part_ml, *part_o;
  int64_t ldq, ldo, page_stride, ld_table, capacity, window, sinks;
  int32_t batch, kv_heads, group, head_groups, d, num_pages, page_shift, groups, direct, e4m3;
  float scale_log2, v_scale;
};

struct ChunkArgs {
  const void *q, *k, *v;
  void* o;
  const int32_t *starts, *tables, *lengths;
  sile::ChunkRec* plan;
  float* parts;
  int64_t ldq, ldo, page_stride, ld_table;
  sile::ChunkShape shape;
  int32_t kv_heads, d, num_pages, page_shift, tiles, groups, direct;
  uint32_t q_and, q_xor;
  float scale_log2, v_scale;
};

int check_pools(void* const* pools, int64_t n_pools, int64_t page_bytes, int64_t page_stride,
                int64_t num_pages, Pools* out) {
  memset(out, 0, sizeof *out);
  if (n_pools < 0 || n_pools > kMaxPools)
    return fail(SILE_ERR_SHAPE, "%lld pools (0 to %d)", (long long)n_pools, kMaxPools);
  if (n_pools == 0) return SILE_OK;
  if (!pools) return fail(SILE_ERR_SHAPE, "NULL pools");
  if (page_bytes <= 0 || page_bytes % 16 != 0 || page_stride % 16 != 0 || page_stride < page_bytes ||
      page_bytes > (1ll << 32) || page_stride > (1ll << 48) / std::max<int64_t>(num_pages, 1))
    return fail(SILE_ERR_SHAPE, "pages of %lld bytes every %lld: multiples of 16, apart, at most 4 GiB each",
                (long long)page_bytes, (long long)page_stride);
  for (int64_t i = 0; i < n_pools; ++i) {
    if (!pools[i]) return fail(SILE_ERR_SHAPE, "pool %lld is NULL", (long long)i);
    if (!aligned16(pools[i])) return fail(SILE_ERR_SHAPE, "pool %lld not 16-byte aligned", (long long)i);
    out->base[i] = pools[i];
  }
  out->page_bytes = page_bytes;
  out->page_stride = page_stride;
  out->count = (int32_t)n_pools;
  out->segs = (int32_t)((page_bytes + kSegB - 1) / kSegB);
  return SILE_OK;
}

// Workgroups for `units` 16 KiB pieces of copying: at most 16 a CU, the rest in turn
// (a copy at 4096 workgroups runs at the rate of a large contiguous one).
int copy_groups(int64_t units, int64_t* out) {
  int cus = 0;
  const int rc = device_cus(&cus);
  if (rc != SILE_OK) return rc;
  *out = std::min<int64_t>(units, 16ll * cus);
  return SILE_OK;
}

int64_t kv_ints(int64_t n_rows, int64_t num_pages) {
  // reserve: demand, kept, fresh, snapshot of the counts; compact: moves, map, holes, movers
  return std::max(2 * ints16(n_rows) + 2 * ints16(num_pages), 4 + 3 * ints16(num_pages));
}

int copy_ints(const int32_t* from, int32_t* to, int64_t n, hipStream_t s) {
  if (from == to || n == 0) return SILE_OK;
  const unsigned groups = (unsigned)std::min<int64_t>((n + 255) / 256, 1024);
  void* params[] = {(void*)&from, &to, &n};
  return launch(Module::kKvCache, "sile_kv_copy_ints", dim3(groups), dim3(256), params, s);
}

// Instances of the one-token attention: width of the padded head dimension, tiles of
// 16 query heads (two where a key head has more than 16), workgroups a CU holds.
struct PagedPlan {
  int dp, q_tiles, per_cu, cus;
  int64_t head_groups, groups, plan_ints, slots, bytes;
};
void paged_shape(int64_t q_heads, int64_t kv_heads, int64_t head_dim, PagedPlan* p) {
  const int64_t group = q_heads / kv_heads;
  p->dp = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
  p->q_tiles = group > 16 && p->dp < 256 ? 2 : 1;
  p->head_groups = (group + 16 * p->q_tiles - 1) / (16 * p->q_tiles);
}
int paged_plan(bool fp8, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim, PagedPlan* p) {
  paged_shape(q_heads, kv_heads, head_dim, p);
  p->per_cu = p->dp == 64 ? (p->q_tiles == 1 ? 4 : 2) : p->dp == 128 && p->q_tiles == 1 ? (fp8 ? 3 : 2) : 1;
  const int rc = device_cus(&p->cus);
  if (rc != SILE_OK) return rc;
  p->groups = (int64_t)p->per_cu * p->cus;
  p->plan_ints = ints16(batch + 1);
  p->slots = 2 * p->groups * 16 * p->q_tiles;   // two a workgroup
  p->bytes = 4 * (p->plan_ints + p->slots * (2 + head_dim));
  return SILE_OK;
}

// The attention of pieces of prompts: width of the padded head dimension, keys of a block, the
// workgroups of a dealt list (a multiple of 8) and its workspace.
struct ChunkPlan {
  int dp, block;
  int64_t tiles, groups, plan_ints, bytes;
};
int check_chunk(int64_t n_rows, int64_t n_tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim) {
  const int rc = check_heads(n_rows, q_heads, kv_heads, head_dim);
  if (rc != SILE_OK) return rc;
  if (n_rows > kMaxRows || n_tokens < 0 || n_tokens > kIntMax / 2 / (q_heads / kv_heads))
    return fail(SILE_ERR_SHAPE, "%lld tokens of %lld rows: negative or too many", (long long)n_tokens, (long long)n_rows);
  return SILE_OK;
}
int chunk_plan(int64_t n_rows, int64_t n_tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim, ChunkPlan* p) {
  p->dp = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
  p->block = p->dp == 64 ? 64 : 32;
  p->tiles = sile::chunk_tiles(n_tokens, n_rows, q_heads / kv_heads);
  int cus = 0;
  const int rc = device_cus(&cus);
  if (rc != SILE_OK) return rc;
  p->groups = std::max<int64_t>(8, (int64_t)(p->dp == 256 ? 1 : 2) * cus / 8 * 8);
  p->plan_ints = ints16(4 * (p->tiles + 1));   // a ChunkRec each
  // O and (m, l) of a tile's 128 rows, two parts a workgroup
  p->bytes = 4 * (p->plan_ints + 2 * p->groups * 4 * (p->dp / 8 + 1) * 256);
  return SILE_OK;
}

}  // namespace

extern "C" {

int sile_hip_kv_append(sile_dtype dtype, sile_dtype cache_type, int64_t n_tokens, int64_t kv_heads,
                       int64_t head_dim, const void* k, int64_t ldk, const void* v, int64_t ldv,
                       const int32_t* rows, const int32_t* positions, void* k_pages, void* v_pages,
                       int64_t num_pages, int64_t page_size, int64_t page_stride,
                       const int32_t* tables, int64_t n_rows, int64_t ld_table, float k_scale,
                       float v_scale, sile_hip_stream stream) {
  int64_t es = 0;
  int rc = check_cache(dtype, cache_type, kv_heads, head_dim, num_pages, page_size, page_stride, &es);
  if (rc != SILE_OK) return rc;
  if ((rc = check_table(n_rows, ld_table)) != SILE_OK) return rc;
  if (n_tokens < 0 || n_tokens > kIntMax)
    return fail(SILE_ERR_SHAPE, "%lld tokens: negative or too many", (long long)n_tokens);
  if (n_tokens == 0 || n_rows == 0 || ld_table == 0 || num_pages == 0) return ok();
  if (!k || !v || !positions || !k_pages || !v_pages || !tables) return fail(SILE_ERR_SHAPE, "NULL operand");
  if (ldk < kv_heads * head_dim || ldv < kv_heads * head_dim)
    return fail(SILE_ERR_SHAPE, "leading dimension smaller than a token's heads");
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_pages) || !aligned16(v_pages) || ldk % 8 || ldv % 8)
    return fail(SILE_ERR_SHAPE, "tokens and pages have to be 16-byte aligned");
  const bool fp8 = cache_type == SILE_F8E4M3;
  const int64_t each = 2 * kv_heads * head_dim / (fp8 ? 16 : 8);   // chunks of a token
  AppendArgs a{k, v, rows, positions, tables, k_pages, v_pages, n_tokens, ldk, ldv, page_stride,
               ld_table, ld_table * page_size, (int32_t)kv_heads, (int32_t)head_dim, (int32_t)num_pages,
               page_shift_of(page_size), (int32_t)n_rows, 1, k_scale, v_scale, reciprocal(k_scale),
               reciprocal(v_scale)};
  // two chunks a thread where a token has few; at most 2^22 workgroups
  a.per_group = (int32_t)std::max<int64_t>({1, 512 / each, (n_tokens >> 22) + 1});
  const int64_t blocks = (n_tokens + a.per_group - 1) / a.per_group;
  void* params[] = {&a};
  rc = launch(Module::kKvCache, !fp8 ? "sile_kv_append" : dtype == SILE_F16 ? "sile_kv_append_f16_fp8"
                                                                            : "sile_kv_append_bf16_fp8",
              dim3((unsigned)blocks), dim3(256), params, static_cast<hipStream_t>(stream));
  return rc == SILE_OK ? ok() : rc;
}

int sile_hip_kv_copy_pages(void* const* pools, int64_t n_pools, int64_t page_bytes,
                           int64_t page_stride_bytes, int64_t num_pages, int64_t n,
                           const int32_t* src, const int32_t* dst, sile_hip_stream stream) {
  if (n < 0 || num_pages < 0 || n > kIntMax || num_pages > kIntMax)
    return fail(SILE_ERR_SHAPE, "%lld copies in a pool of %lld pages", (long long)n, (long long)num_pages);
  Pools p;
  int rc = check_pools(pools, n_pools, page_bytes, page_stride_bytes, num_pages, &p);
  if (rc != SILE_OK) return rc;
  if (n == 0 || n_pools == 0 || num_pages == 0) return ok();
  if (!src || !dst) return fail(SILE_ERR_SHAPE, "NULL operand");
  int64_t groups = 0;
  if ((rc = copy_groups(n * p.count * p.segs, &groups)) != SILE_OK) return rc;
  int32_t pages = (int32_t)num_pages;
  void* params[] = {&p, (void*)&src, (void*)&dst, &n, &pages};
  rc = launch(Module::kKvCache, "sile_kv_copy_pages", dim3((unsigned)groups), dim3(256), params,
              static_cast<hipStream_t>(stream));
  return rc == SILE_OK ? ok() : rc;
}

int sile_hip_kv_free(int64_t n_rows, int64_t ld_table, const int32_t* drop, const int32_t* tables_in,
                     int32_t* tables_out, const int32_t* lengths_in, int32_t* lengths_out,
                     int64_t num_pages, const int32_t* refs_in, int32_t* refs_out,
                     sile_hip_stream stream) {
  int rc = check_table(n_rows, ld_table);
  if (rc != SILE_OK) return rc;
  if (num_pages < 0 || num_pages > kIntMax) return fail(SILE_ERR_SHAPE, "invalid page count");
  if (num_pages > 0 && (!refs_in || !refs_out)) return fail(SILE_ERR_SHAPE, "NULL operand");
  if (n_rows > 0 && (!drop || !lengths_in || !lengths_out || (ld_table > 0 && (!tables_in || !tables_out))))
    return fail(SILE_ERR_SHAPE, "NULL operand");
  if ((rc = check_in_out(tables_in, tables_out, n_rows * ld_table, "tables")) != SILE_OK ||
      (rc = check_in_out(lengths_in, lengths_out, n_rows, "lengths")) != SILE_OK ||
      (rc = check_in_out(refs_in, refs_out, num_pages, "counts")) != SILE_OK)
    return rc;
  if (overlap(drop, n_rows, lengths_out, n_rows) || overlap(drop, n_rows, tables_out, n_rows * ld_table))
    return fail(SILE_ERR_SHAPE, "drop overlaps what is written");
  const int64_t entries = n_rows * ld_table;
  if ((rc = check_apart({{"drop", drop, n_rows, false}, {"tables", tables_in, entries, false},
                         {"tables", tables_out, entries, true}, {"lengths", lengths_in, n_rows, false},
                         {"lengths", lengths_out, n_rows, true}, {"counts", refs_in, num_pages, false},
                         {"counts", refs_out, num_pages, true}})) != SILE_OK)
    return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if ((rc = copy_ints(refs_in, refs_out, num_pages, s)) != SILE_OK) return rc;
  if (n_rows == 0) return ok();
  int32_t pages = (int32_t)num_pages;
  void* params[] = {&ld_table, (void*)&drop, (void*)&tables_in, &tables_out, (void*)&lengths_in,
                    &lengths_out, &pages, &refs_out};
  rc = launch(Module::kKvCache, "sile_kv_free", dim3((unsigned)n_rows), dim3(256), params, s);
  return rc == SILE_OK ? ok() : rc;
}

int sile_hip_kv_fork(int64_t n_in, int64_t n_out, int64_t ld_table, const int32_t* src,
                     const int32_t* tables_in, int32_t* tables_out, const int32_t* lengths_in,
                     int32_t* lengths_out, int64_t num_pages, const int32_t* refs_in,
                     int32_t* refs_out, sile_hip_stream stream) {
  int rc = check_table(n_in, ld_table);
  if (rc == SILE_OK) rc = check_table(n_out, ld_table);
  if (rc != SILE_OK) return rc;
  if (num_pages < 0 || num_pages > kIntMax) return fail(SILE_ERR_SHAPE, "invalid page count");
  if (num_pages > 0 && (!refs_in || !refs_out)) return fail(SILE_ERR_SHAPE, "NULL operand");
  if ((n_out > 0 && (!src || !lengths_out || (ld_table > 0 && !tables_out))) ||
      (n_in > 0 && (!lengths_in || (ld_table > 0 && !tables_in))))
    return fail(SILE_ERR_SHAPE, "NULL operand");
  if (overlap(tables_in, n_in * ld_table, tables_out, n_out * ld_table) ||
      overlap(lengths_in, n_in, lengths_out, n_out) || overlap(src, n_out, lengths_out, n_out) ||
      overlap(src, n_out, tables_out, n_out * ld_table))
    return fail(SILE_ERR_SHAPE, "a fork's src, old and new tables and lengths must not overlap");
  if ((rc = check_in_out(refs_in, refs_out, num_pages, "counts")) != SILE_OK) return rc;
  if ((rc = check_apart({{"src", src, n_out, false}, {"tables", tables_in, n_in * ld_table, false},
                         {"tables", tables_out, n_out * ld_table, true}, {"lengths", lengths_in, n_in, false},
                         {"lengths", lengths_out, n_out, true}, {"counts", refs_in, num_pages, false},
                         {"counts", refs_out, num_pages, true}})) != SILE_OK)
    return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if ((rc = copy_ints(refs_in, refs_out, num_pages, s)) != SILE_OK) return rc;
  if (n_in + n_out == 0) return ok();
  int32_t in = (int32_t)n_in, out = (int32_t)n_out, pages = (int32_t)num_pages;
  void* params[] = {&in, &out, &ld_table, (void*)&src, (void*)&tables_in, &tables_out,
                    (void*)&lengths_in, &lengths_out, &pages, &refs_out};
  rc = launch(Module::kKvCache, "sile_kv_fork", dim3((unsigned)(n_in + n_out)), dim3(256), params, s);
  return rc == SILE_OK ? ok() : rc;
}

int sile_hip_kv_workspace(int64_t n_rows, int64_t num_pages, size_t* bytes) {
  if (!bytes) return fail(SILE_ERR_SHAPE, "bytes is NULL");
  *bytes = 0;
  if (n_rows < 0 || num_pages < 0 || n_rows > kMaxRows || num_pages > kIntMax)
    return fail(SILE_ERR_SHAPE, "%lld rows over %lld pages", (long long)n_rows, (long long)num_pages);
  *bytes = (size_t)(4 * kv_ints(n_rows, num_pages));
  return ok();
}

int sile_hip_kv_reserve(int64_t n_rows, int64_t ld_table, int64_t page_size, const int32_t* lengths,
                        const int32_t* need, const int32_t* tables_in, int32_t* tables_out,
                        int64_t num_pages, const int32_t* refs_in, int32_t* refs_out,
                        int32_t* granted, void* const* pools, int64_t n_pools, int64_t page_bytes,
                        int64_t page_stride_bytes, void* workspace, size_t workspace_bytes,
                        sile_hip_stream stream) {
  int rc = check_table(n_rows, ld_table);
  if (rc != SILE_OK) return rc;
  const int shift = page_shift_of(page_size);
  if (shift < 0)
    return fail(SILE_ERR_SHAPE, "page_size %lld is no power of two up to 65536", (long long)page_size);
  if (num_pages < 0 || num_pages > kIntMax) return fail(SILE_ERR_SHAPE, "invalid page count");
  Pools p;
  if ((rc = check_pools(pools, n_pools, page_bytes, page_stride_bytes, num_pages, &p)) != SILE_OK) return rc;
  if (num_pages > 0 && (!refs_in || !refs_out)) return fail(SILE_ERR_SHAPE, "NULL operand");
  if (n_rows > 0 && (!lengths || !need || !granted || (ld_table > 0 && (!tables_in || !tables_out))))
    return fail(SILE_ERR_SHAPE, "NULL operand");
  if ((rc = check_in_out(tables_in, tables_out, n_rows * ld_table, "tables")) != SILE_OK ||
      (rc = check_in_out(refs_in, refs_out, num_pages, "counts")) != SILE_OK)
    return rc;
  if ((rc = check_workspace(workspace, workspace_bytes, 4 * kv_ints(n_rows, num_pages))) != SILE_OK) return rc;
  if (overlap(granted, n_rows, need, n_rows) || overlap(granted, n_rows, lengths, n_rows))
    return fail(SILE_ERR_SHAPE, "granted overlaps need or lengths");
  if ((rc = check_apart({{"lengths", lengths, n_rows, false}, {"need", need, n_rows, false},
                         {"tables", tables_in, n_rows * ld_table, false}, {"tables", tables_out, n_rows * ld_table, true},
                         {"counts", refs_in, num_pages, false}, {"counts", refs_out, num_pages, true},
                         {"granted", granted, n_rows, true},
                         {"workspace", static_cast<int32_t*>(workspace), kv_ints(n_rows, num_pages), true}})) != SILE_OK)
    return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (n_rows == 0) {
    rc = copy_ints(refs_in, refs_out, num_pages, s);
    return rc == SILE_OK ? ok() : rc;
  }
  int32_t* demand = static_cast<int32_t*>(workspace);
  int32_t* kept = demand + ints16(n_rows);
  int32_t* fresh = kept + ints16(n_rows);
  int32_t* copy = fresh + ints16(num_pages);
  const bool in_place = refs_in == refs_out;
  // in place the counts as they were go to the workspace, else they are copied on
  int32_t* snapshot = in_place ? copy : refs_out;
  ReserveArgs a{lengths, need, tables_in, tables_out, refs_in, refs_out, granted, demand, kept, fresh,
                ld_table, (int32_t)n_rows, (int32_t)num_pages, shift};
  const int64_t row_groups = (n_rows + 3) / 4;
  const int64_t ints = std::max(num_pages, tables_in != tables_out ? n_rows * ld_table : 0);
  const int64_t copies = std::max<int64_t>(1, std::min<int64_t>((ints + 1023) / 1024, 512));
  void* p1[] = {&a, (void*)&refs_in, &snapshot};
  rc = launch(Module::kKvCache, "sile_kv_reserve_need", dim3((unsigned)(row_groups + copies)), dim3(256), p1, s);
  if (rc != SILE_OK) return rc;
  if (in_place) a.refs_in = copy;
  void* p2[] = {&a};
  rc = launch(Module::kKvCache, "sile_kv_reserve_deal", dim3(1), dim3(1024), p2, s);
  if (rc != SILE_OK) return rc;
  int64_t groups = 0;
  if ((rc = copy_groups(n_rows * p.count * p.segs, &groups)) != SILE_OK) return rc;
  void* p3[] = {&a, &p};
  rc = launch(Module::kKvCache, "sile_kv_reserve_take", dim3((unsigned)(row_groups + groups)), dim3(256), p3, s);
  return rc == SILE_OK ? ok() : rc;
}

int sile_hip_kv_compact(int64_t n_rows, int64_t ld_table, const int32_t* tables_in, int32_t* tables_out,
                        int64_t num_pages, const int32_t* refs_in, int32_t* refs_out, int32_t* used,
                        void* const* pools, int64_t n_pools, int64_t page_bytes,
                        int64_t page_stride_bytes, void* workspace, size_t workspace_bytes,
                        sile_hip_stream stream) {
  int rc = check_table(n_rows, ld_table);
  if (rc != SILE_OK) return rc;
  if (num_pages < 0 || num_pages > kIntMax) return fail(SILE_ERR_SHAPE, "invalid page count");
  Pools p;
  if ((rc = check_pools(pools, n_pools, page_bytes, page_stride_bytes, num_pages, &p)) != SILE_OK) return rc;
  if (!used || (num_pages > 0 && (!refs_in || !refs_out)) ||
      (n_rows * ld_table > 0 && (!tables_in || !tables_out)))
    return fail(SILE_ERR_SHAPE, "NULL operand");
  if ((rc = check_in_out(tables_in, tables_out, n_rows * ld_table, "tables")) != SILE_OK ||
      (rc = check_in_out(refs_in, refs_out, num_pages, "counts")) != SILE_OK)
    return rc;
  if ((rc = check_workspace(workspace, workspace_bytes, 4 * kv_ints(n_rows, num_pages))) != SILE_OK) return rc;
  if ((rc = check_apart({{"tables", tables_in, n_rows * ld_table, false}, {"tables", tables_out, n_rows * ld_table, true},
                         {"counts", refs_in, num_pages, false}, {"counts", refs_out, num_pages, true},
                         {"used", used, 1, true},
                         {"workspace", static_cast<int32_t*>(workspace), kv_ints(n_rows, num_pages), true}})) != SILE_OK)
    return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  int32_t* moves = static_cast<int32_t*>(workspace);
  int32_t* map = moves + 4;
  int32_t* holes = map + ints16(num_pages);
  int32_t* movers = holes + ints16(num_pages);
  int32_t pages = (int32_t)num_pages;
  void* p1[] = {&pages, (void*)&refs_in, &used, &moves, &map, &holes, &movers};
  rc = launch(Module::kKvCache, "sile_kv_compact_plan", dim3(1), dim3(1024), p1, s);
  if (rc != SILE_OK) return rc;
  int64_t groups = 0, entries = n_rows * ld_table;
  if ((rc = copy_groups(num_pages / 2 * p.count * p.segs, &groups)) != SILE_OK) return rc;
  int32_t meta = (int32_t)std::max<int64_t>(1, std::min<int64_t>((std::max(entries, num_pages) + 255) / 256, 512));
  void* p2[] = {&meta, &entries, (void*)&tables_in, &tables_out, &pages, (void*)&refs_in, &refs_out,
                &used, &moves, &map, &holes, &movers, &p};
  rc = launch(Module::kKvCache, "sile_kv_compact_move", dim3((unsigned)(meta + groups)), dim3(256), p2, s);
  return rc == SILE_OK ? ok() : rc;
}

int sile_hip_paged_attn_workspace(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                  size_t* bytes) {
  if (!bytes) return fail(SILE_ERR_SHAPE, "bytes is NULL");
  *bytes = 0;
  int rc = check_heads(batch, q_heads, kv_heads, head_dim);
  if (rc != SILE_OK) return rc;
  PagedPlan plan;
  // (the 8-bit cache's grid is the larger one, where they differ)
  if ((rc = paged_plan(true, batch, q_heads, kv_heads, head_dim, &plan)) != SILE_OK) return rc;
  *bytes = (size_t)plan.bytes;
  return ok();
}

int sile_hip_paged_attn_decode(sile_dtype dtype, sile_dtype cache_type, int64_t batch, int64_t q_heads,
                               int64_t kv_heads, int64_t head_dim, const void* q, int64_t ldq,
                               const void* k_pages, const void* v_pages, int64_t num_pages,
                               int64_t page_size, int64_t page_stride, const int32_t* tables,
                               int64_t ld_table, const int32_t* lengths, void* o, int64_t ldo,
                               float scale, float k_scale, float v_scale, int64_t window,
                               int64_t sinks, void* workspace, size_t workspace_bytes,
                               sile_hip_stream stream) {
  int64_t es = 0;
  int rc = check_heads(batch, q_heads, kv_heads, head_dim);
  if (rc != SILE_OK) return rc;
  if ((rc = check_cache(dtype, cache_type, kv_heads, head_dim, num_pages, page_size, page_stride, &es)) != SILE_OK)
    return rc;
  if ((rc = check_table(batch, ld_table)) != SILE_OK) return rc;
  if (window < 0 || sinks < 0) return fail(SILE_ERR_SHAPE, "negative window or sinks");
  if (batch == 0) return ok();
  if (!q || !o || !lengths || (num_pages > 0 && (!k_pages || !v_pages)) || (ld_table > 0 && !tables))
    return fail(SILE_ERR_SHAPE, "NULL operand");
  if (ldq < q_heads * head_dim || ldo < q_heads * head_dim)
    return fail(SILE_ERR_SHAPE, "leading dimension smaller than a token's heads");
  if (!aligned16(q) || !aligned16(o) || !aligned16(k_pages) || !aligned16(v_pages) || ldq % 8 || ldo % 8)
    return fail(SILE_ERR_SHAPE, "q, o and the pages have to be 16-byte aligned");
  if (std::max(ldq, ldo) > (1ll << 45) / batch) return fail(SILE_ERR_SHAPE, "leading dimension too large");
  const Region out{"o", o, batch, ldo * 2, q_heads * head_dim * 2}, in{"q", q, batch, ldq * 2, q_heads * head_dim * 2};
  const int64_t page = kv_heads * page_size * head_dim * es;
  const Region kp{"K's pages", k_pages, num_pages, page_stride * es, page};
  const Region vp{"V's pages", v_pages, num_pages, page_stride * es, page};
  const Region of = array_of("lengths", lengths, 4 * batch), pages = array_of("tables", tables, 4 * batch * ld_table);
  PagedPlan plan;
  paged_shape(q_heads, kv_heads, head_dim, &plan);
  // without a page every row is empty
  const int64_t capacity = num_pages > 0 ? std::min<int64_t>(ld_table * page_size, kIntMax) : 0;
  // tiles are numbered in 32 bits, over all rows and key heads
  const int64_t seen = window > 0 ? std::min<int64_t>(capacity, std::min<int64_t>(window, kIntMax) +
                                                                    std::min<int64_t>(sinks, kIntMax))
                                  : capacity;
  const int64_t row_tiles = (seen / sile::kTileKeys + 3 + sile::kUnitTiles) * kv_heads * plan.head_groups;
  if (batch > (kIntMax - (1 << 20)) / row_tiles || batch * kv_heads * plan.head_groups > kMaxRows)
    return fail(SILE_ERR_SHAPE, "%lld rows of up to %lld keys: too many for one call", (long long)batch,
                (long long)seen);
  if ((rc = check_written({out}, {in, kp, vp, of, pages})) != SILE_OK) return rc;
  if ((rc = paged_plan(es == 1, batch, q_heads, kv_heads, head_dim, &plan)) != SILE_OK) return rc;
  if ((rc = check_workspace(workspace, workspace_bytes, plan.bytes)) != SILE_OK) return rc;
  if ((rc = check_written({array_of("workspace", workspace, plan.bytes)}, {out, in, kp, vp, of, pages})) != SILE_OK) return rc;
  PagedArgs a{};
  a.q = q;
  a.k = k_pages;
  a.v = v_pages;
  a.o = o;
  a.tables = tables;
  a.lengths = lengths;
  a.plan = static_cast<int32_t*>(workspace);
  a.part_ml = reinterpret_cast<float*>(a.plan + plan.plan_ints);
  a.part_o = a.part_ml + 2 * plan.slots;
  a.ldq = ldq;
  a.ldo = ldo;
  a.page_stride = page_stride;
  a.ld_table = ld_table;
  a.capacity = capacity;
  a.window = window;
  a.sinks = sinks;
  a.batch = (int32_t)batch;
  a.kv_heads = (int32_t)kv_heads;
  a.group = (int32_t)(q_heads / kv_heads);
  a.head_groups = (int32_t)plan.head_groups;
  a.d = (int32_t)head_dim;
  a.num_pages = (int32_t)num_pages;
  a.page_shift = page_shift_of(page_size);
  a.groups = (int32_t)plan.groups;
  a.e4m3 = es == 1;
  a.scale_log2 = scale * k_scale * 1.4426950408889634f;
  a.v_scale = v_scale;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const char* dt = dtype == SILE_F16 ? "f16" : "bf16";
  char name[64];
  snprintf(name, sizeof name, "sile_paged_attn_%s%s_%c%d_q%d", dt, cache_type == dtype ? "" : "_fp8",
           page_size < 16 ? 's' : head_dim == plan.dp ? 'd' : 'p', plan.dp, plan.q_tiles);
  void* params[] = {&a};
  const int64_t units = batch * kv_heads * plan.head_groups;
  // A workgroup a unit, in one launch, where a unit is short (what the table's width or the
  // window allows, as the lengths stand on the device): up to 512 keys in any case, up to 2048
  // (1024 of 256 16-bit dims) where there is a unit for every CU.  Us a call, dealt and so, 8
  // key heads of 128: 1 x 256 keys 10.7, 6.9; 1 x 512 10.9, 9.2; 1 x 1024 10.8, 13.3; 32 x 1024
  // 30.6, 23.5; 128 x 1024 90.6, 84.2; 32 x 2048 53.3, 44.7; 8 x 2048 22.1, 22.9; 4 of 256, 64 x
  // 2000 56, 71.  (A table wider than its rows takes the first of each.)  Past that a single
  // long row among short ones would keep its workgroups alone for long.
  a.direct = (seen <= 512 || (seen <= 2048 && seen * head_dim * es <= (1 << 19) && units >= plan.cus));
  const int32_t grid = a.direct ? (int32_t)units : sile::deal_workgroups(batch * row_tiles, a.groups);
  rc = launch(Module::kPagedAttn, name, dim3((unsigned)grid), dim3(256), params, s);
  if (rc != SILE_OK || a.direct) return rc == SILE_OK ? ok() : rc;
  // Units of one length have about grid / units parts (and one or two more): up to 16 for one
  // wave, two rounds of eight, then more waves.  A long row among short ones has more than that and
  // is joined by as few waves: one row of 100000 keys, 8 key heads of 128, takes 74 us alone, 89
  // beside 63 rows of 100.
  const int64_t heads = std::min<int64_t>(a.group, 16 * plan.q_tiles);
  const int64_t parts = grid / units + 2;
  int split = parts <= 16 ? 1 : parts <= 32 ? 2 : parts <= 64 ? 4 : 8;
  const int64_t groups = (heads * split + 7) / 8;
  snprintf(name, sizeof name, "sile_paged_attn_join_%s_q%d", dt, plan.q_tiles);
  void* join[] = {&a, &split};
  rc = launch(Module::kPagedAttn, name, dim3((unsigned)units, (unsigned)groups), dim3(512), join, s);
  return rc == SILE_OK ? ok() : rc;
}

int sile_hip_paged_attn_chunk_workspace(int64_t n_rows, int64_t n_tokens, int64_t q_heads, int64_t kv_heads,
                                        int64_t head_dim, size_t* bytes) {
  if (!bytes) return fail(SILE_ERR_SHAPE, "bytes is NULL");
  *bytes = 0;
  int rc = check_chunk(n_rows, n_tokens, q_heads, kv_heads, head_dim);
  if (rc != SILE_OK) return rc;
  ChunkPlan plan;
  if ((rc = chunk_plan(n_rows, n_tokens, q_heads, kv_heads, head_dim, &plan)) != SILE_OK) return rc;
  *bytes = (size_t)plan.bytes;
  return ok();
}

int sile_hip_paged_attn_chunk(sile_dtype dtype, sile_dtype cache_type, int64_t n_rows, int64_t n_tokens,
                              int64_t q_heads, int64_t kv_heads, int64_t head_dim, const void* q, int64_t ldq,
                              const int32_t* starts, const void* k_pages, const void* v_pages, int64_t num_pages,
                              int64_t page_size, int64_t page_stride, const int32_t* tables, int64_t ld_table,
                              const int32_t* lengths, void* o, int64_t ldo, float scale, float k_scale,
                              float v_scale, int64_t window, int64_t sinks, void* workspace,
                              size_t workspace_bytes, sile_hip_stream stream) {
  int64_t es = 0;
  int rc = check_chunk(n_rows, n_tokens, q_heads, kv_heads, head_dim);
  if (rc != SILE_OK) return rc;
  if ((rc = check_cache(dtype, cache_type, kv_heads, head_dim, num_pages, page_size, page_stride, &es)) != SILE_OK)
    return rc;
  if ((rc = check_table(n_rows, ld_table)) != SILE_OK) return rc;
  if (window < 0 || sinks < 0) return fail(SILE_ERR_SHAPE, "negative window or sinks");
  const float product = scale * k_scale;
  if (!(std::fabs(product) <= 3.402823466e38f)) return fail(SILE_ERR_SHAPE, "scale * k_scale is not finite");
  if (n_rows == 0 || n_tokens == 0) return ok();
  if (!q || !o || !starts || !lengths || (num_pages > 0 && (!k_pages || !v_pages)) || (ld_table > 0 && !tables))
    return fail(SILE_ERR_SHAPE, "NULL operand");
  const int64_t width = q_heads * head_dim;
  if (ldq < width || ldo < width) return fail(SILE_ERR_SHAPE, "leading dimension smaller than a token's heads");
  if (!aligned16(q) || !aligned16(o) || !aligned16(k_pages) || !aligned16(v_pages) || ldq % 8 || ldo % 8)
    return fail(SILE_ERR_SHAPE, "q, o and the pages have to be 16-byte aligned");
  if (std::max(ldq, ldo) > (1ll << 45) / n_tokens) return fail(SILE_ERR_SHAPE, "leading dimension too large");
  if (ld_table * page_size > (1ll << 29))
    return fail(SILE_ERR_SHAPE, "a table of %lld pages of %lld keys: at most 2^29 keys a row", (long long)ld_table,
                (long long)page_size);
  ChunkPlan plan{};
  const Region out{"o", o, n_tokens, ldo * 2, width * 2}, in{"q", q, n_tokens, ldq * 2, width * 2};
  const int64_t page = kv_heads * page_size * head_dim * es;
  const Region kp{"K's pages", k_pages, num_pages, page_stride * es, page};
  const Region vp{"V's pages", v_pages, num_pages, page_stride * es, page};
  const Region list = array_of("starts", starts, 4 * (n_rows + 1)), of = array_of("lengths", lengths, 4 * n_rows);
  const Region pages = array_of("tables", tables, 4 * n_rows * ld_table);
  if ((rc = check_written({out}, {in, kp, vp, list, of, pages})) != SILE_OK) return rc;
  const int block = head_dim <= 64 ? 64 : 32;
  // without a page every row is empty
  const int64_t capacity = num_pages > 0 ? ld_table * page_size : 0;
  const int64_t tiles = sile::chunk_tiles(n_tokens, n_rows, q_heads / kv_heads);
  // blocks of a unit: what a row holds, or its tokens' windows and the sinks
  const int64_t tokens = std::min<int64_t>(n_tokens, sile::kChunkRows / (q_heads / kv_heads) + 2);
  const int64_t seen = window > 0 ? std::min<int64_t>(capacity, std::min<int64_t>(window, kIntMax) + tokens +
                                                                    std::min<int64_t>(sinks, kIntMax))
                                  : capacity;
  const int64_t unit = seen / block + 4 + sile::kChunkUnit;
  // (units: of 256 threads each, rounded up to a multiple of 8; a launch has less than 2^32)
  if (tiles > ((1 << 24) - 8) / kv_heads || tiles > (kIntMax - (1 << 20)) / (unit * kv_heads))
    return fail(SILE_ERR_SHAPE, "%lld tokens of %lld rows of up to %lld keys: too many for one call",
                (long long)n_tokens, (long long)n_rows, (long long)seen);
  if ((rc = chunk_plan(n_rows, n_tokens, q_heads, kv_heads, head_dim, &plan)) != SILE_OK) return rc;
  if ((rc = check_workspace(workspace, workspace_bytes, plan.bytes)) != SILE_OK) return rc;
  if ((rc = check_written({array_of("workspace", workspace, plan.bytes)}, {out, in, kp, vp, list, of, pages})) != SILE_OK)
    return rc;
  ChunkArgs a{};
  a.q = q;
  a.k = k_pages;
  a.v = v_pages;
  a.o = o;
  a.starts = starts;
  a.tables = tables;
  a.lengths = lengths;
  a.plan = static_cast<sile::ChunkRec*>(workspace);
  a.parts = static_cast<float*>(workspace) + plan.plan_ints;
  a.ldq = ldq;
  a.ldo = ldo;
  a.page_stride = page_stride;
  a.ld_table = ld_table;
  a.shape = {n_tokens, capacity, window, sinks, (int32_t)n_rows, (int32_t)(q_heads / kv_heads), block};
  a.kv_heads = (int32_t)kv_heads;
  a.d = (int32_t)head_dim;
  a.num_pages = (int32_t)num_pages;
  a.page_shift = page_shift_of(page_size);
  a.tiles = (int32_t)tiles;
  a.groups = (int32_t)plan.groups;
  // the kernel wants a positive scale: a negative one's sign goes into q, under 0 all of it
  a.q_and = product == 0.0f ? 0u : 0xffffffffu;
  a.q_xor = product < 0.0f ? 0x80008000u : 0u;
  a.scale_log2 = product == 0.0f ? 1.0f : std::fabs(product) * 1.4426950408889634f;
  a.v_scale = v_scale;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const char* dt = dtype == SILE_F16 ? "f16" : "bf16";
  const bool fp8 = cache_type != dtype;
  char name[64];
  // a DMA instruction covers 1 KiB of keys, which have to lie in one page
  snprintf(name, sizeof name, "sile_paged_chunk_%s%s_%c%d", dt, fp8 ? "_fp8" : "",
           !fp8 && page_size < 512 / plan.dp ? 's' : 'd', plan.dp);
  void* params[] = {&a};
  const int64_t units = tiles * kv_heads;
  a.direct = seen <= 512;
  int64_t grid = a.direct ? (units + 7) / 8 * 8 : plan.groups;
  if (!a.direct) {
    const int64_t most = (tiles * unit * kv_heads + sile::kChunkShare + sile::kChunkUnit - 1) / (sile::kChunkShare + sile::kChunkUnit);
    grid = std::min(grid, (most + 7) / 8 * 8);
  }
  rc = launch(Module::kPagedChunk, name, dim3((unsigned)grid), dim3(256), params, s);
  if (rc != SILE_OK || a.direct) return rc == SILE_OK ? ok() : rc;
  // with few units, of many parts, the dims of a row go to several workgroups (8 tokens over 131072 keys, 8 units
  // of 64 parts: 132 -> 121 us; 568 units of one to three: 145 -> 161)
  const int split = units <= 64 ? plan.dp / 32 : 1;
  snprintf(name, sizeof name, "sile_paged_chunk_join%s_%s%s_d%d", split > 1 ? "1" : "", dt, fp8 ? "_fp8" : "", plan.dp);
  rc = launch(Module::kPagedChunk, name, dim3((unsigned)units, sile::kChunkRows / 32, split), dim3(256), params, s);
  return rc == SILE_OK ? ok() : rc;
}

}  // extern "C"
