// Checks of arguments that the entry points over a paged key-value cache share.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <initializer_list>

#include "runtime_internal.h"

namespace sile_rt {

constexpr int64_t kIntMax = 0x7fffffff;
// rows of a table, and units of an attention call: a launch has less than 2^32 threads
constexpr int64_t kMaxRows = 1 << 22;

// 1 / scale, or 0 where the kernel is to divide
inline float reciprocal(float scale) {
  const float x = std::fabs(scale);
  return x >= 0x1p-60f && x <= 0x1p60f ? 1.0f / scale : 0.0f;
}

// log2 of a power of two up to 65536, or -1
inline int page_shift_of(int64_t page_size) {
  for (int s = 0; s <= 16; ++s)
    if (page_size == (1ll << s)) return s;
  return -1;
}

// the types and the shape of a cache's pages; es: bytes of an element
inline int check_cache(sile_dtype dtype, sile_dtype cache_type, int64_t kv_heads, int64_t head_dim,
                       int64_t num_pages, int64_t page_size, int64_t page_stride, int64_t* es) {
  if (dtype != SILE_F16 && dtype != SILE_BF16)
    return fail(SILE_ERR_UNSUPPORTED_BACKEND, "paged cache: tokens of %s not supported", dtype_name(dtype));
  if (cache_type != dtype && cache_type != SILE_F8E4M3)
    return fail(SILE_ERR_UNSUPPORTED_BACKEND, "paged cache of %s under %s not supported",
                dtype_name(cache_type), dtype_name(dtype));
  *es = (int64_t)dtype_bytes(cache_type);
  if (kv_heads <= 0 || head_dim <= 0 || num_pages < 0) return fail(SILE_ERR_SHAPE, "invalid cache shape");
  if (head_dim > 256) return fail(SILE_ERR_UNSUPPORTED_BACKEND, "head_dim > 256 not supported");
  if (head_dim % (16 / *es) != 0)
    return fail(SILE_ERR_UNSUPPORTED_BACKEND, "paged cache of %s: head_dim %lld is no multiple of %lld",
                dtype_name(cache_type), (long long)head_dim, (long long)(16 / *es));
  if (page_shift_of(page_size) < 0)
    return fail(SILE_ERR_SHAPE, "page_size %lld is no power of two up to 65536", (long long)page_size);
  if (kv_heads > (1 << 15) || num_pages > kIntMax) return fail(SILE_ERR_SHAPE, "cache too large");
  if (num_pages > 0 && (page_stride < kv_heads * page_size * head_dim || page_stride * *es % 16 != 0))
    return fail(SILE_ERR_SHAPE, "page_stride %lld: a page has %lld elements, in steps of 16 bytes",
                (long long)page_stride, (long long)(kv_heads * page_size * head_dim));
  if (num_pages > 0 && page_stride > (1ll << 47) / num_pages)
    return fail(SILE_ERR_SHAPE, "page_stride %lld too large for %lld pages", (long long)page_stride,
                (long long)num_pages);
  return SILE_OK;
}

inline int check_table(int64_t rows, int64_t ld_table) {
  if (rows < 0 || ld_table < 0) return fail(SILE_ERR_SHAPE, "negative table extent");
  if (rows > kMaxRows || (rows > 0 && ld_table > kIntMax / rows))
    return fail(SILE_ERR_SHAPE, "page table of %lld x %lld entries too large", (long long)rows,
                (long long)ld_table);
  return SILE_OK;
}

// whether [x, x + nx) and [y, y + ny) share an element
inline bool overlap(const int32_t* x, int64_t nx, const int32_t* y, int64_t ny) {
  return x && y && nx > 0 && ny > 0 && x < y + ny && y < x + nx;
}
// The arrays of a call: one that it writes shares nothing with another, but for the old and the
// new form of the same thing (check_in_out).
struct Span {
  const char* name;
  const int32_t* p;
  int64_t n;
  bool written;
};
inline int check_apart(std::initializer_list<Span> all) {
  for (const Span& x : all)
    for (const Span& y : all)
      if (x.written && strcmp(x.name, y.name) != 0 && overlap(x.p, x.n, y.p, y.n))
        return fail(SILE_ERR_SHAPE, "%s overlaps %s", x.name, y.name);
  return SILE_OK;
}
// a call in place or out of place, nothing in between
inline int check_in_out(const int32_t* in, const int32_t* out, int64_t n, const char* what) {
  if (in != out && overlap(in, n, out, n))
    return fail(SILE_ERR_SHAPE, "old and new %s overlap without being the same", what);
  return SILE_OK;
}

// Memory of an operand: `rows` runs of `width` bytes, `pitch` bytes apart (an array: one).
struct Region {
  const char* name;
  const void* p;
  int64_t rows, pitch, width;
};
inline Region array_of(const char* name, const void* p, int64_t bytes) { return {name, p, 1, 0, bytes}; }
// Whether two share a byte.  Rows may lie in the gaps of the other's, as a fused projection's queries and
// keys do.
inline bool regions_share(const Region& x, const Region& y) {
  if (!x.p || !y.p || x.rows <= 0 || y.rows <= 0 || x.width <= 0 || y.width <= 0) return false;
  const int64_t px = x.rows > 1 ? x.pitch : 0, py = y.rows > 1 ? y.pitch : 0;
  const int64_t x0 = 0, y0 = (int64_t)(reinterpret_cast<uintptr_t>(y.p) - reinterpret_cast<uintptr_t>(x.p));
  if (x0 + (x.rows - 1) * px + x.width <= y0 || y0 + (y.rows - 1) * py + y.width <= x0) return false;
  // apart at every row, if they are so modulo a step of both
  int64_t step = px, rest = py;
  while (rest != 0) {
    const int64_t r = step % rest;
    step = rest;
    rest = r;
  }
  if (step == 0) return true;   // two arrays
  const int64_t off = (y0 % step + step) % step;
  if (off >= x.width && off + y.width <= step) return false;
  // row by row, past those that end before the other's next
  for (int64_t i = 0, j = 0; i < x.rows && j < y.rows;) {
    const int64_t xs = i * px, ys = y0 + j * py;
    if (xs + x.width <= ys)
      i = px == 0 ? x.rows : i + (ys - xs - x.width) / px + 1;
    else if (ys + y.width <= xs)
      j = py == 0 ? y.rows : j + (xs - ys - y.width) / py + 1;
    else
      return true;
  }
  return false;
}
// what a call writes apart from each other and from what it reads
inline int check_written(std::initializer_list<Region> written, std::initializer_list<Region> read) {
  for (const Region* x = written.begin(); x != written.end(); ++x) {
    for (const Region* y = x + 1; y != written.end(); ++y)
      if (regions_share(*x, *y)) return fail(SILE_ERR_SHAPE, "%s overlaps %s", x->name, y->name);
    for (const Region& y : read)
      if (regions_share(*x, y)) return fail(SILE_ERR_SHAPE, "%s overlaps %s", x->name, y.name);
  }
  return SILE_OK;
}

inline int check_heads(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim) {
  if (batch < 0 || q_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || q_heads % kv_heads != 0)
    return fail(SILE_ERR_SHAPE, "batch %lld, %lld query heads over %lld key heads of %lld",
                (long long)batch, (long long)q_heads, (long long)kv_heads, (long long)head_dim);
  if (head_dim > 256) return fail(SILE_ERR_UNSUPPORTED_BACKEND, "head_dim > 256 not supported");
  if (batch > kIntMax || q_heads > (1 << 20)) return fail(SILE_ERR_SHAPE, "attention too large");
  return SILE_OK;
}

// int32 workspaces, each part on a 16-byte boundary
inline int64_t ints16(int64_t n) { return (n + 3) / 4 * 4; }

inline int check_workspace(const void* ws, size_t have, int64_t need) {
  if (!ws || !aligned16(ws)) return fail(SILE_ERR_SHAPE, "workspace NULL or not 16-byte aligned");
  if ((int64_t)have < need)
    return fail(SILE_ERR_SHAPE, "workspace of %zu bytes, %lld needed", have, (long long)need);
  return SILE_OK;
}

}  // namespace sile_rt
