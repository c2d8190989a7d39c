// Entry points of a serving step around the paged cache: the step's token list, rotary
// positions, the row norm and the log probabilities of a row of logits.  Arguments are checked
// here; lengths, positions and page numbers in device memory by the kernels.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>

#include "paged_checks.h"

using namespace sile_rt;

namespace {

// Kernel argument blocks; layouts match the structs in kernels/*.hip.
struct SlotsArgs {
  const int32_t *lengths, *need, *granted;
  int32_t *starts, *rows, *positions, *lengths_out;
  int32_t n_rows, tokens;
};
constexpr int64_t kSlotRows = 65536, kSlotTokens = 1024;
struct RopeArgs {
  const void *q, *k, *v;
  void *q_out, *k_out, *v_out;
  const int32_t *rows, *positions, *tables;
  const double* turns;
  int64_t tokens, ldq, ldk, ldv, ldqo, ldko, page_stride, ld_table, capacity;
  int32_t q_heads, kv_heads, d, rot, num_pages, page_shift, n_rows, per_group, rot_items, head_items, items,
      value_items, past, head_shift, value_shift, k_exact, v_exact;
  float inv_head, inv_items, inv_value, magnitude, k_scale, v_scale, k_rcp, v_rcp;
};
constexpr int64_t kRopeItems = 1024, kRopeTokens = 16, kRopeAngles = 1024;   // of a workgroup
struct NormArgs {
  const void *x, *residual, *weight;
  void *sum, *y;
  float* scales;
  int64_t rows, ldx, ldr, lds, ldy;
  int32_t cols, group;
  float eps, inv_cols, scale, rcp;
};
struct LogprobArgs {
  const void* x;
  const int32_t* targets;
  float *logp, *entropy, *top_logp;
  int32_t* top_ids;
  float *part_sums, *part_top;
  int32_t* part_ids;
  int64_t ldx;
  int32_t rows, cols, top, parts, chunks, per_part;
  float scale, scale_log2, floor;
};
constexpr int64_t kLogitChunk = 8192;

bool aligned_to(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes == 0; }

// What sile_hip_rope and sile_hip_rope_append have in common: checks, and the kernel's vector
// width (8, 4 or 1 elements; 8 only of 16 bits).
int check_rope(sile_dtype dtype, sile_rope_layout layout, int64_t n_tokens, int64_t q_heads, int64_t kv_heads,
               int64_t head_dim, int64_t rot_dim, float magnitude) {
  if (dtype != SILE_F32 && dtype != SILE_F16 && dtype != SILE_BF16)
    return fail(SILE_ERR_UNSUPPORTED_BACKEND, "rotary positions of %s not supported", dtype_name(dtype));
  if (layout != SILE_ROPE_HALF && layout != SILE_ROPE_PAIRS)
    return fail(SILE_ERR_SHAPE, "unknown rotary layout %d", (int)layout);
  if (n_tokens < 0 || n_tokens > kIntMax)
    return fail(SILE_ERR_SHAPE, "%lld tokens: negative or too many", (long long)n_tokens);
  if (q_heads < 0 || kv_heads < 0 || q_heads + kv_heads == 0 || q_heads > (1 << 15) || kv_heads > (1 << 15))
    return fail(SILE_ERR_SHAPE, "%lld query and %lld key heads", (long long)q_heads, (long long)kv_heads);
  if (head_dim <= 0 || head_dim > 2048) return fail(SILE_ERR_UNSUPPORTED_BACKEND, "head_dim past 2048 not supported");
  if (rot_dim < 0 || rot_dim > head_dim || rot_dim % 2 != 0)
    return fail(SILE_ERR_SHAPE, "rot_dim %lld of a head_dim of %lld: an even number up to it", (long long)rot_dim,
                (long long)head_dim);
  if (!(std::fabs(magnitude) <= 3.402823466e38f)) return fail(SILE_ERR_SHAPE, "magnitude is not finite");
  return SILE_OK;
}
int64_t rope_width(int64_t es, const RopeArgs& a) {
  for (int64_t e : {8, 4}) {
    if (e * es > 16) continue;
    if (a.rot / 2 % e || a.d % e) continue;
    bool fits = true;
    for (int64_t ld : {a.q ? a.ldq : 0, a.k ? a.ldk : 0, a.v ? a.ldv : 0, a.q ? a.ldqo : 0, a.ldko}) fits &= ld % e == 0;
    for (const void* p : {a.q, a.k, a.v, (const void*)a.q_out, (const void*)a.k_out, (const void*)a.v_out})
      fits &= aligned_to(p, e * es);
    if (fits) return e;
  }
  return 1;
}
int launch_rope(sile_dtype dtype, sile_rope_layout layout, const char* cache, bool values, RopeArgs* a, hipStream_t s) {
  const int64_t e = rope_width((int64_t)dtype_bytes(dtype), *a);
  a->rot_items = (int32_t)(a->rot / (2 * e));
  a->head_items = (int32_t)(a->rot_items + (a->d - a->rot + 2 * e - 1) / (2 * e));
  a->value_items = (int32_t)((a->d + 2 * e - 1) / (2 * e));
  a->items = (a->q_heads + a->kv_heads) * a->head_items + (values ? a->kv_heads * a->value_items : 0);
  if (a->items > (1 << 23)) return fail(SILE_ERR_SHAPE, "too many heads of %d dims", a->d);
  a->inv_head = 1.0f / (float)a->head_items;
  a->inv_items = 1.0f / (float)a->items;
  a->inv_value = 1.0f / (float)a->value_items;
  auto log2_of = [](int32_t n) { return n > 0 && (n & (n - 1)) == 0 ? __builtin_ctz((unsigned)n) : -1; };
  a->head_shift = log2_of(a->head_items);
  a->value_shift = log2_of(a->value_items);
  auto power = [](float x) { int e; return std::frexp(std::fabs(x), &e) == 0.5f && std::fabs(x) >= 0x1p-60f && std::fabs(x) <= 0x1p60f; };
  a->k_exact = power(a->k_scale);
  a->v_exact = power(a->v_scale);
  // queries and keys that the caches cannot hold anyway go past them
  a->past = a->tokens * (a->q_heads + a->kv_heads) * a->d * (int64_t)dtype_bytes(dtype) > (32 << 20);
  const int64_t angles = std::max(1, a->rot / 2);
  // enough tokens for one item a thread and more where there are tokens for all CUs
  int64_t per = std::min({kRopeItems / a->items, kRopeTokens, kRopeAngles / angles});
  int cus = 0;
  const int rc = device_cus(&cus);
  if (rc != SILE_OK) return rc;
  per = std::min(per, a->tokens / (4 * cus));
  a->per_group = (int32_t)std::max<int64_t>(1, per);
  const int64_t groups = (a->tokens + a->per_group - 1) / a->per_group;
  const int64_t pieces = ((int64_t)a->per_group * a->items + kRopeItems - 1) / kRopeItems;
  char name[64];
  snprintf(name, sizeof name, "sile_rope_%s_%s%s_e%d", layout == SILE_ROPE_HALF ? "half" : "pairs",
           dtype == SILE_F32 ? "f32" : dtype == SILE_F16 ? "f16" : "bf16", cache, (int)e);
  // (a launch has less than 2^32 threads; the workgroups go on to further tokens)
  void* params[] = {a};
  return launch(Module::kRope, name, dim3((unsigned)std::min<int64_t>(groups, (1 << 24) / pieces - 1), (unsigned)pieces),
                dim3(256), params, s);
}

}  // namespace

extern "C" {

int sile_hip_kv_slots(int64_t n_rows, const int32_t* lengths, const int32_t* need, const int32_t* granted,
                      int64_t max_tokens, int32_t* starts, int32_t* rows, int32_t* positions,
                      int32_t* lengths_out, sile_hip_stream stream) {
  if (n_rows < 0 || n_rows > kSlotRows)
    return fail(SILE_ERR_SHAPE, "%lld rows (0 to %lld)", (long long)n_rows, (long long)kSlotRows);
  if (max_tokens < 0 || max_tokens > kIntMax)
    return fail(SILE_ERR_SHAPE, "%lld tokens: negative or too many", (long long)max_tokens);
  if (!starts || (n_rows > 0 && (!lengths || !need || !lengths_out)) || (max_tokens > 0 && (!rows || !positions)))
    return fail(SILE_ERR_SHAPE, "NULL operand");
  int rc = check_apart({{"lengths", lengths, n_rows, false}, {"need", need, n_rows, false},
                        {"granted", granted, n_rows, false}, {"starts", starts, n_rows + 1, true},
                        {"rows", rows, max_tokens, true}, {"positions", positions, max_tokens, true},
                        {"new lengths", lengths_out, n_rows, true}});
  if (rc != SILE_OK) return rc;
  SlotsArgs a{lengths, need, granted, starts, rows, positions, lengths_out, (int32_t)n_rows, (int32_t)max_tokens};
  void* params[] = {&a};
  const int64_t groups = std::max<int64_t>(1, (max_tokens + kSlotTokens - 1) / kSlotTokens);
  rc = launch(Module::kKvCache, "sile_kv_slots", dim3((unsigned)groups), dim3(1024), params,
              static_cast<hipStream_t>(stream));
  return rc == SILE_OK ? ok() : rc;
}

int sile_hip_rope_turns(sile_rope_scaling scaling, int64_t rot_dim, double base, double factor, double original,
                        double low, double high, double* turns) {
  if (rot_dim < 0 || rot_dim % 2 != 0 || rot_dim > 2048)
    return fail(SILE_ERR_SHAPE, "rot_dim %lld: an even number up to 2048", (long long)rot_dim);
  if (rot_dim > 0 && !turns) return fail(SILE_ERR_SHAPE, "NULL operand");
  if (!(base > 0) || !std::isfinite(base)) return fail(SILE_ERR_SHAPE, "base has to be positive");
  if (scaling < SILE_ROPE_UNSCALED || scaling > SILE_ROPE_DIMS)
    return fail(SILE_ERR_SHAPE, "unknown rotary scaling %d", (int)scaling);
  if (scaling != SILE_ROPE_UNSCALED && (!(factor > 0) || !std::isfinite(factor)))
    return fail(SILE_ERR_SHAPE, "factor has to be positive");
  const bool ramp = scaling == SILE_ROPE_TURNS || scaling == SILE_ROPE_DIMS;
  if (ramp && (!(original > 0) || !std::isfinite(original) || !(low > 0) || !(high > low) || !std::isfinite(high)))
    return fail(SILE_ERR_SHAPE, "a ramp needs an original length and 0 < low < high");
  if (scaling == SILE_ROPE_DIMS && !(base > 1)) return fail(SILE_ERR_SHAPE, "a ramp over the pairs needs a base past 1");
  const double two_pi = 6.283185307179586477, r = (double)rot_dim;
  if (scaling == SILE_ROPE_BASE && rot_dim > 2) base *= std::pow(factor, r / (r - 2.0));
  // the pair that turns n times over the original length
  auto pair_of = [&](double n) { return r * std::log(original / (n * two_pi)) / (2.0 * std::log(base)); };
  const double first = ramp ? std::max(std::floor(pair_of(high)), 0.0) : 0.0;
  double last = ramp ? std::min(std::ceil(pair_of(low)), r - 1.0) : 0.0;
  if (last <= first) last = first + 0.001;
  for (int64_t j = 0; j < rot_dim / 2; ++j) {
    double t = std::pow(base, -2.0 * (double)j / r) / two_pi;
    double kept = 1.0;   // how much of the pair keeps its turns
    if (scaling == SILE_ROPE_LINEAR) kept = 0.0;
    if (scaling == SILE_ROPE_TURNS) kept = std::min(std::max((original * t - low) / (high - low), 0.0), 1.0);
    if (scaling == SILE_ROPE_DIMS) kept = 1.0 - std::min(std::max(((double)j - first) / (last - first), 0.0), 1.0);
    if (scaling != SILE_ROPE_UNSCALED && scaling != SILE_ROPE_BASE) t *= kept + (1.0 - kept) / factor;
    turns[j] = t;
  }
  return ok();
}

int sile_hip_rope(sile_dtype dtype, sile_rope_layout layout, int64_t n_tokens, int64_t q_heads, int64_t kv_heads,
                  int64_t head_dim, int64_t rot_dim, const void* q, int64_t ldq, void* q_out, int64_t ldqo,
                  const void* k, int64_t ldk, void* k_out, int64_t ldko, const int32_t* positions,
                  const double* turns, float magnitude, sile_hip_stream stream) {
  int rc = check_rope(dtype, layout, n_tokens, q_heads, kv_heads, head_dim, rot_dim, magnitude);
  if (rc != SILE_OK) return rc;
  if (n_tokens == 0) return ok();
  if (!positions || (rot_dim > 0 && !turns) || (q_heads > 0 && (!q || !q_out)) || (kv_heads > 0 && (!k || !k_out)))
    return fail(SILE_ERR_SHAPE, "NULL operand");
  if ((q_heads > 0 && (ldq < q_heads * head_dim || ldqo < q_heads * head_dim)) ||
      (kv_heads > 0 && (ldk < kv_heads * head_dim || ldko < kv_heads * head_dim)))
    return fail(SILE_ERR_SHAPE, "leading dimension smaller than a token's heads");
  const int64_t es = (int64_t)dtype_bytes(dtype), nq = q_heads * head_dim, nk = kv_heads * head_dim;
  // (a workgroup's offsets, of up to 16 tokens, are counted in 32 bits)
  if (std::max({ldq, ldqo, ldk, ldko}) > (1 << 25)) return fail(SILE_ERR_SHAPE, "leading dimension past 2^25");
  for (const void* p : {q, (const void*)q_out, k, (const void*)k_out})
    if (!aligned_to(p, es)) return fail(SILE_ERR_SHAPE, "tokens not aligned to their type");
  const Region rq{"q", q, n_tokens, ldq * es, nq * es}, ro{"q's output", q_out, n_tokens, ldqo * es, nq * es};
  const Region rk{"k", k, n_tokens, ldk * es, nk * es}, rp{"k's output", k_out, n_tokens, ldko * es, nk * es};
  if ((q_heads > 0 && !(q == q_out && ldq == ldqo) && regions_share(rq, ro)) ||
      (kv_heads > 0 && !(k == k_out && ldk == ldko) && regions_share(rk, rp)))
    return fail(SILE_ERR_SHAPE, "an output overlaps its input without being the same");
  const Region angles = array_of("turns", turns, 4 * rot_dim), at = array_of("positions", positions, 4 * n_tokens);
  if ((rc = check_written({ro, rp}, {at, angles})) != SILE_OK || (rc = check_written({ro}, {rk})) != SILE_OK ||
      (rc = check_written({rp}, {rq})) != SILE_OK)
    return rc;
  RopeArgs a{};
  if (q_heads > 0) {
    a.q = q;
    a.q_out = q_out;
    a.ldq = ldq;
    a.ldqo = ldqo;
  }
  if (kv_heads > 0) {
    a.k = k;
    a.k_out = k_out;
    a.ldk = ldk;
    a.ldko = ldko;
  }
  a.positions = positions;
  a.turns = turns;
  a.tokens = n_tokens;
  a.q_heads = (int32_t)q_heads;
  a.kv_heads = (int32_t)kv_heads;
  a.d = (int32_t)head_dim;
  a.rot = (int32_t)rot_dim;
  a.magnitude = magnitude;
  rc = launch_rope(dtype, layout, "", false, &a, static_cast<hipStream_t>(stream));
  return rc == SILE_OK ? ok() : rc;
}

int sile_hip_rope_append(sile_dtype dtype, sile_dtype cache_type, sile_rope_layout layout, int64_t n_tokens,
                         int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t rot_dim, const void* q,
                         int64_t ldq, void* q_out, int64_t ldqo, const void* k, int64_t ldk, const void* v,
                         int64_t ldv, const int32_t* rows, const int32_t* positions, const double* turns,
                         float magnitude, void* k_pages, void* v_pages, int64_t num_pages, int64_t page_size,
                         int64_t page_stride, const int32_t* tables, int64_t n_rows, int64_t ld_table,
                         float k_scale, float v_scale, sile_hip_stream stream) {
  int64_t es = 0;
  int rc = check_cache(dtype, cache_type, kv_heads, head_dim, num_pages, page_size, page_stride, &es);
  if (rc == SILE_OK) rc = check_rope(dtype, layout, n_tokens, q_heads, kv_heads, head_dim, rot_dim, magnitude);
  if (rc == SILE_OK) rc = check_table(n_rows, ld_table);
  if (rc != SILE_OK) return rc;
  if (n_tokens == 0) return ok();
  if (!positions || !k || !v || (rot_dim > 0 && !turns) || (q_heads > 0 && (!q || !q_out)) ||
      (num_pages > 0 && (!k_pages || !v_pages)) || (n_rows * ld_table > 0 && !tables))
    return fail(SILE_ERR_SHAPE, "NULL operand");
  const int64_t nq = q_heads * head_dim, nk = kv_heads * head_dim;
  if ((q_heads > 0 && (ldq < nq || ldqo < nq)) || ldk < nk || ldv < nk)
    return fail(SILE_ERR_SHAPE, "leading dimension smaller than a token's heads");
  if (std::max({ldq, ldqo, ldk, ldv}) > (1 << 25)) return fail(SILE_ERR_SHAPE, "leading dimension past 2^25");
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_pages) || !aligned16(v_pages) || ldk % 8 || ldv % 8 ||
      (q_heads > 0 && (!aligned16(q) || !aligned16(q_out) || ldq % 8 || ldqo % 8)))
    return fail(SILE_ERR_SHAPE, "tokens and pages have to be 16-byte aligned");
  const Region rq{"q", q, n_tokens, ldq * 2, nq * 2}, ro{"q's output", q_out, n_tokens, ldqo * 2, nq * 2};
  const Region rk{"k", k, n_tokens, ldk * 2, nk * 2}, rv{"v", v, n_tokens, ldv * 2, nk * 2};
  if (q_heads > 0 && !(q == q_out && ldq == ldqo) && regions_share(rq, ro))
    return fail(SILE_ERR_SHAPE, "an output overlaps its input without being the same");
  const int64_t page = kv_heads * page_size * head_dim * es;
  const Region kp{"K's pages", k_pages, num_pages, page_stride * es, page};
  const Region vp{"V's pages", v_pages, num_pages, page_stride * es, page};
  const Region angles = array_of("turns", turns, 4 * rot_dim), at = array_of("positions", positions, 4 * n_tokens);
  const Region of = array_of("rows", rows, 4 * n_tokens), pages = array_of("tables", tables, 4 * n_rows * ld_table);
  if ((rc = check_written({ro, kp, vp}, {rk, rv, at, of, angles, pages})) != SILE_OK ||
      (rc = check_written({kp, vp}, {rq})) != SILE_OK)
    return rc;
  RopeArgs a{};
  if (q_heads > 0) {
    a.q = q;
    a.q_out = q_out;
    a.ldq = ldq;
    a.ldqo = ldqo;
  }
  a.k = k;
  a.v = v;
  a.ldk = ldk;
  a.ldv = ldv;
  a.k_out = k_pages;
  a.v_out = v_pages;
  a.rows = rows;
  a.positions = positions;
  a.tables = tables;
  a.turns = turns;
  a.tokens = n_tokens;
  a.page_stride = page_stride;
  a.ld_table = ld_table;
  a.capacity = num_pages > 0 ? ld_table * page_size : 0;
  a.q_heads = (int32_t)q_heads;
  a.kv_heads = (int32_t)kv_heads;
  a.d = (int32_t)head_dim;
  a.rot = (int32_t)rot_dim;
  a.num_pages = (int32_t)num_pages;
  a.page_shift = page_shift_of(page_size);
  a.n_rows = (int32_t)n_rows;
  a.magnitude = magnitude;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.k_rcp = reciprocal(k_scale);
  a.v_rcp = reciprocal(v_scale);
  rc = launch_rope(dtype, layout, cache_type == dtype ? "_cache" : "_fp8", true, &a, static_cast<hipStream_t>(stream));
  return rc == SILE_OK ? ok() : rc;
}

int sile_hip_rmsnorm_rows(sile_dtype in_type, sile_dtype out_type, int64_t rows, int64_t cols, const void* x,
                          int64_t ldx, const void* residual, int64_t ldr, void* sum, int64_t lds,
                          const void* weight, float eps, void* y, int64_t ldy, float scale, float* scales,
                          int64_t group, sile_hip_stream stream) {
  if (in_type != SILE_F32 && in_type != SILE_F16 && in_type != SILE_BF16)
    return fail(SILE_ERR_UNSUPPORTED_BACKEND, "row norm of %s not supported", dtype_name(in_type));
  if (out_type != in_type && out_type != SILE_F8E4M3)
    return fail(SILE_ERR_UNSUPPORTED_BACKEND, "row norm of %s into %s not supported", dtype_name(in_type),
                dtype_name(out_type));
  if (rows < 0 || cols < 0 || cols > (1 << 30)) return fail(SILE_ERR_SHAPE, "row norm of %lld x %lld", (long long)rows, (long long)cols);
  const bool fp8 = out_type == SILE_F8E4M3;
  if (group < 0 || (group > 0 && (!fp8 || cols % group != 0)))
    return fail(SILE_ERR_SHAPE, "groups of %lld columns: of an 8-bit output, a divisor of %lld", (long long)group, (long long)cols);
  if (!(eps >= 0)) return fail(SILE_ERR_SHAPE, "eps is negative");
  int rc = SILE_OK;
  if (rows == 0 || cols == 0) return ok();
  if (!x || !y || (group > 0 && !scales)) return fail(SILE_ERR_SHAPE, "NULL operand");
  const int64_t es = (int64_t)dtype_bytes(in_type), ys = (int64_t)dtype_bytes(out_type);
  if (ldx < cols || (residual && ldr < cols) || (sum && lds < cols) || ldy < cols)
    return fail(SILE_ERR_SHAPE, "leading dimension smaller than a row");
  if (std::max({ldx, ldr, lds, ldy}) > (1ll << 45) / rows) return fail(SILE_ERR_SHAPE, "matrix too large");
  for (const void* p : {x, residual, (const void*)sum, weight})
    if (!aligned_to(p, es)) return fail(SILE_ERR_SHAPE, "operand not aligned to its type");
  if (!aligned_to(y, ys) || !aligned_to(scales, 4)) return fail(SILE_ERR_SHAPE, "operand not aligned to its type");
  // a row is read before it is written, element by element where the rows coincide
  const Region in{"x", x, rows, ldx * es, cols * es}, add{"residual", residual, rows, ldr * es, cols * es};
  const Region to_sum{"sum", sum, rows, lds * es, cols * es}, out{"y", y, rows, ldy * ys, cols * ys};
  const Region by = array_of("weight", weight, cols * es);
  const Region to_scales = array_of("scales", group > 0 ? scales : nullptr, group > 0 ? 4 * rows * (cols / group) : 0);
  auto own = [&](const void* to, int64_t ld, int64_t bytes, const void* from, int64_t ld_from) {
    return bytes == es && to == from && ld == ld_from;
  };
  if ((rc = check_written({to_sum, out, to_scales}, {by})) != SILE_OK || (rc = check_written({to_scales}, {in, add})) != SILE_OK)
    return rc;
  if ((!own(y, ldy, ys, x, ldx) && regions_share(out, in)) || (!own(y, ldy, ys, residual, ldr) && regions_share(out, add)) ||
      (!own(sum, lds, es, x, ldx) && regions_share(to_sum, in)) ||
      (!own(sum, lds, es, residual, ldr) && regions_share(to_sum, add)))
    return fail(SILE_ERR_SHAPE, "an output overlaps another operand without being its rows");
  NormArgs a{x, residual, weight, sum, y, scales, rows, ldx, ldr, lds, ldy, (int32_t)cols, (int32_t)group,
             eps, 1.0f / (float)cols, scale, reciprocal(scale)};
  // a row in registers, and a group in a lane, lanes of one wave or all of the row
  const bool vectors =
      cols <= 16384 && (group == 0 || group == cols || (group <= 512 && group >= 8 && (group & (group - 1)) == 0));
  int cus = 0;
  if ((rc = device_cus(&cus)) != SILE_OK) return rc;
  int threads = 256, per = 0, wg = 256;
  char name[64], form[16];
  if (vectors) {
    threads = cols <= 512 ? 64 : cols <= 8192 ? 256 : 1024;
    per = cols <= 512 ? 1 : (int)((cols + threads * 8 - 1) / (threads * 8));
    per = per == 3 ? 4 : per;
    wg = threads == 64 ? 256 : threads;
    snprintf(form, sizeof form, "t%d_v%d%s", threads, per, cols % 8 != 0 ? "p" : "");
  } else {
    snprintf(form, sizeof form, "any");
  }
  snprintf(name, sizeof name, "sile_rmsnorm_%s%s_%s", dtype_name(in_type), fp8 ? "_fp8" : "", form);
  const int64_t groups = (rows + wg / threads - 1) / (wg / threads);
  void* params[] = {&a};
  rc = launch(Module::kNorm, name, dim3((unsigned)std::min<int64_t>(groups, 2048ll * cus / wg)), dim3((unsigned)wg),
              params, static_cast<hipStream_t>(stream));
  return rc == SILE_OK ? ok() : rc;
}

// Parts of a row: workgroups for every CU's four where the rows are fewer.
static int logprob_parts(int64_t rows, int64_t cols, int64_t* chunks, int64_t* per, int64_t* parts) {
  int cus = 0;
  const int rc = device_cus(&cus);
  if (rc != SILE_OK) return rc;
  *chunks = std::max<int64_t>(1, (cols + kLogitChunk - 1) / kLogitChunk);
  const int64_t want = rows > 0 ? std::max<int64_t>(1, (4 * cus + rows - 1) / rows) : 1;
  *per = (*chunks + std::min(want, *chunks) - 1) / std::min(want, *chunks);
  *parts = (*chunks + *per - 1) / *per;
  return SILE_OK;
}
static int check_logprobs(int64_t rows, int64_t cols, int64_t top_k) {
  if (rows < 0 || cols < 0 || rows > kMaxRows || cols > (1 << 30))
    return fail(SILE_ERR_SHAPE, "logits of %lld x %lld", (long long)rows, (long long)cols);
  if (top_k < 0 || top_k > 64) return fail(SILE_ERR_SHAPE, "top_k %lld (0 to 64)", (long long)top_k);
  return SILE_OK;
}

int sile_hip_logprobs_workspace(int64_t rows, int64_t cols, int64_t top_k, size_t* bytes) {
  if (!bytes) return fail(SILE_ERR_SHAPE, "bytes is NULL");
  *bytes = 0;
  int rc = check_logprobs(rows, cols, top_k);
  if (rc != SILE_OK) return rc;
  int64_t chunks, per, parts;
  if ((rc = logprob_parts(rows, cols, &chunks, &per, &parts)) != SILE_OK) return rc;
  *bytes = (size_t)(parts > 1 ? rows * parts * (16 + 8 * top_k) : 0);
  return ok();
}

int sile_hip_logprobs_rows(sile_dtype in_type, int64_t rows, int64_t cols, const void* x, int64_t ldx, float scale,
                           const int32_t* targets, float* logp, float* entropy, int64_t top_k, float* top_logp,
                           int32_t* top_ids, void* workspace, size_t workspace_bytes, sile_hip_stream stream) {
  if (in_type != SILE_F32 && in_type != SILE_F16 && in_type != SILE_BF16)
    return fail(SILE_ERR_UNSUPPORTED_BACKEND, "logits of %s not supported", dtype_name(in_type));
  int rc = check_logprobs(rows, cols, top_k);
  if (rc != SILE_OK) return rc;
  if (!(scale >= 0x1p-60f && scale <= 0x1p60f)) return fail(SILE_ERR_SHAPE, "scale has to be in [2^-60, 2^60]");
  if (rows == 0) return ok();
  if ((cols > 0 && !x) || (logp && !targets) || (top_k > 0 && (!top_logp || !top_ids)))
    return fail(SILE_ERR_SHAPE, "NULL operand");
  if (ldx < cols || ldx > (1ll << 45) / rows) return fail(SILE_ERR_SHAPE, "leading dimension smaller than a row, or too large");
  const int64_t es = (int64_t)dtype_bytes(in_type);
  if (!aligned_to(x, es) || !aligned_to(targets, 4) || !aligned_to(logp, 4) || !aligned_to(entropy, 4) ||
      !aligned_to(top_logp, 4) || !aligned_to(top_ids, 4))
    return fail(SILE_ERR_SHAPE, "operand not aligned to its type");
  const Region in{"x", x, rows, ldx * es, cols * es}, of = array_of("targets", logp ? targets : nullptr, 4 * rows);
  const Region one = array_of("logp", logp, 4 * rows), two = array_of("entropy", entropy, 4 * rows);
  const Region top = array_of("top_logp", top_logp, 4 * rows * top_k), ids = array_of("top_ids", top_ids, 4 * rows * top_k);
  if ((rc = check_written({one, two, top, ids}, {in, of})) != SILE_OK) return rc;
  int64_t chunks, per, parts;
  if ((rc = logprob_parts(rows, cols, &chunks, &per, &parts)) != SILE_OK) return rc;
  const int64_t need = parts > 1 ? rows * parts * (16 + 8 * top_k) : 0;
  if (need > 0 && (rc = check_workspace(workspace, workspace_bytes, need)) != SILE_OK) return rc;
  if ((rc = check_written({array_of("workspace", workspace, need)}, {in, of, one, two, top, ids})) != SILE_OK) return rc;
  LogprobArgs a{};
  a.x = x;
  a.targets = targets;
  a.logp = logp;
  a.entropy = entropy;
  a.top_logp = top_k ? top_logp : nullptr;
  a.top_ids = top_k ? top_ids : nullptr;
  a.part_sums = static_cast<float*>(workspace);
  a.part_top = a.part_sums + 4 * rows * parts;
  a.part_ids = reinterpret_cast<int32_t*>(a.part_top + rows * parts * top_k);
  a.ldx = ldx;
  a.rows = (int32_t)rows;
  a.cols = (int32_t)cols;
  a.top = (int32_t)top_k;
  a.parts = (int32_t)parts;
  a.chunks = (int32_t)chunks;
  a.per_part = (int32_t)per;
  a.scale = scale;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.floor = -512.0f / a.scale_log2;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const char* dt = dtype_name(in_type);
  char name[64];
  snprintf(name, sizeof name, "sile_logprobs_%s", dt);
  void* params[] = {&a};
  rc = launch(Module::kLogprobs, name, dim3((unsigned)(rows * parts)), dim3(256), params, s);
  if (rc != SILE_OK || parts == 1) return rc == SILE_OK ? ok() : rc;
  snprintf(name, sizeof name, "sile_logprobs_join_%s", dt);
  rc = launch(Module::kLogprobs, name, dim3((unsigned)rows), dim3(256), params, s);
  return rc == SILE_OK ? ok() : rc;
}

}  // extern "C"
