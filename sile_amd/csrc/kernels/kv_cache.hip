// The pages of a key-value cache: storing new tokens, counting, sharing, handing
// out, closing up and copying pages.
//
// A page table holds one row a sequence, `width` page numbers of a pool each, -1
// (or anything outside the pool) where the row holds none; refs counts the entries
// that name a page, and a page with no reference is free.  Every result is a whole
// number or a copy, and none depends on the order the workgroups run in: counts
// change by integer atomics, free pages are handed out by rank (lowest number
// first), and no page is read and written by one launch.
//
// All of it is bound by memory, or, at a serving step's few rows, by the launches:
// each entry point is one to three of them, and a thread moves 16 bytes a load.  Tokens and
// pages are stored past the caches (non-temporal): 16000 tokens of 8 heads of 128 into a 16-bit
// cache take 33 us with plain stores and 24 so (5.5 TB/s), closing up a pool of 4700 pages
// 39 and 31; loads that way are slower (24 us, 32).
#include "common.h"
#include "e4m3.h"

using namespace sile;

namespace {

typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));

// ---- new tokens ----

struct AppendArgs {
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* rows;       // NULL: token t is row t's
  const int32_t* positions;
  const int32_t* tables;
  uint8_t* k_pages;
  uint8_t* v_pages;
  int64_t tokens, ldk, ldv, page_stride, ld_table, capacity;
  int32_t heads, d, num_pages, page_shift, n_rows, per_group;   // tokens a workgroup
  float k_scale, v_scale, k_rcp, v_rcp;   // rcp: 1 / scale, 0 for a scale outside [2^-60, 2^60]
};

// A workgroup takes per_group tokens (K's and V's rows of all heads: `each` chunks
// of 16 bytes of the cache), a thread one chunk at a time.  kIn: 0 the type as it
// is, 1 f16 to e4m3, 2 bf16 to e4m3.
template <int kIn>
SILE_DEV void append(const AppendArgs& a) {
  constexpr int kElems = kIn == 0 ? 8 : 16;   // elements of a 16-byte chunk of the cache
  const int per_head = a.d / kElems, half = a.heads * per_head, each = 2 * half;
  const int64_t t0 = (int64_t)blockIdx.x * a.per_group;
  const int n = (int)min((int64_t)a.per_group, a.tokens - t0) * each;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int tok = i / each, c = i - tok * each;
    const int64_t t = t0 + tok;
    const int64_t row = a.rows ? a.rows[t] : t;
    const int32_t pos = a.positions[t];
    if (row < 0 || row >= a.n_rows || pos < 0 || pos >= a.capacity) continue;
    const int32_t id = a.tables[row * a.ld_table + (pos >> a.page_shift)];
    if ((uint32_t)id >= (uint32_t)a.num_pages) continue;
    const bool is_v = c >= half;
    const int hc = is_v ? c - half : c;
    const int head = hc / per_head, cc = hc - head * per_head;
    const uint16_t* src = (is_v ? a.v + t * a.ldv : a.k + t * a.ldk) + (int64_t)head * a.d + cc * kElems;
    const int64_t slot = pos & ((1 << a.page_shift) - 1);
    const int64_t at = (int64_t)id * a.page_stride + (((int64_t)head << a.page_shift) + slot) * a.d + cc * kElems;
    u32x4_t out;
    if constexpr (kIn == 0) {
      out = *reinterpret_cast<const u32x4_t*>(src);
      __builtin_nontemporal_store(out, reinterpret_cast<u32x4_t*>((is_v ? a.v_pages : a.k_pages) + 2 * at));
    } else {
      const float scale = is_v ? a.v_scale : a.k_scale, rcp = is_v ? a.v_rcp : a.k_rcp;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(src + 8 * h);
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint16_t b = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
          f[j] = e4m3_in(kIn == 1 ? f16_to_f32(b) : bf16_to_f32(b), scale, rcp);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) out[2 * h + j] = e4m3_pack4(f + 4 * j);
      }
      __builtin_nontemporal_store(out, reinterpret_cast<u32x4_t*>((is_v ? a.v_pages : a.k_pages) + at));
    }
  }
}

// ---- a step's tokens ----

struct SlotsArgs {
  const int32_t* lengths;
  const int32_t* need;
  const int32_t* granted;   // NULL: every row
  int32_t* starts;
  int32_t* rows;
  int32_t* positions;
  int32_t* lengths_out;
  int32_t n_rows, tokens;
};
constexpr int kSlotTokens = 1024;   // of the list, a workgroup

// One launch for a list of any length: every workgroup adds up the rows' tokens (a run of rows a
// thread, a scan over the threads; rows up to 65536 are in the L2), marks where the rows of its own
// 1024 tokens begin, and a running maximum over the marks names each token's row.  Every 1024th
// run of rows (or all, where there is one workgroup) also goes to starts and lengths_out.  Bound by the
// launch and three dependent reads: 256 rows and 1800 tokens 5 us, 4000 rows and 134000 tokens
// 8.7 (14.5 with a quarter of the threads, and four times the rows in each).
SILE_DEV void slots(const SlotsArgs& a) {
  __shared__ int64_t wave_sum[kSlotTokens / 64];
  // by token: row + 1 that begins there, length - start
  __shared__ int32_t mark_row[kSlotTokens], mark_base[kSlotTokens];
  __shared__ int32_t wave_top[kSlotTokens / 64], first_row, first_base;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = (a.n_rows + kSlotTokens - 1) / kSlotTokens;
  const int r0 = min(tid * per, a.n_rows), r1 = min(r0 + per, a.n_rows);
  const int32_t t0 = blockIdx.x * kSlotTokens;
  // a row's length, and how many tokens it asks for: no position passes 2^31 - 1
  auto row = [&](int r, int32_t* length) {
    const int32_t len = max(a.lengths[r], 0), n = a.granted && a.granted[r] == 0 ? 0 : max(a.need[r], 0);
    *length = len;
    return min(n, 0x7fffffff - len);
  };
  mark_row[tid] = 0;
  int64_t mine = 0;
  int32_t length;
  for (int r = r0; r < r1; ++r) mine += row(r, &length);
  int64_t incl = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t up = __shfl_up((long long)incl, off);
    if (lane >= off) incl += up;
  }
  if (lane == 63) wave_sum[wave] = incl;
  __syncthreads();
  int64_t at = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kSlotTokens / 64; ++w) {
    if (w < wave) at += wave_sum[w];
    total += wave_sum[w];
  }
  const bool keeps = tid % gridDim.x == blockIdx.x;
  if (keeps || (at < (int64_t)t0 + kSlotTokens && at + mine > t0))
    for (int r = r0; r < r1; ++r) {
      const int32_t n = row(r, &length);
      const int32_t s = (int32_t)min(at, (int64_t)a.tokens), e = (int32_t)min(at + n, (int64_t)a.tokens);
      at += n;
      if (keeps) {
        a.starts[r] = s;
        a.lengths_out[r] = length + (e - s);
      }
      if (e <= s || e <= t0 || s - t0 >= kSlotTokens) continue;
      if (s < t0) {   // (one row at most)
        first_row = r;
        first_base = length - s;
      } else {
        mark_row[s - t0] = r + 1;
        mark_base[s - t0] = length - s;
      }
    }
  if (blockIdx.x == 0 && tid == 0) a.starts[a.n_rows] = (int32_t)min(total, (int64_t)a.tokens);
  __syncthreads();
  // the last mark at or before the thread's token
  int mark = mark_row[tid] != 0 ? tid : -1;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int up = __shfl_up(mark, off);
    if (lane >= off) mark = max(mark, up);
  }
  if (lane == 63) wave_top[wave] = mark;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSlotTokens / 64 - 1; ++w)
    if (w < wave) mark = max(mark, wave_top[w]);
  if (tid >= a.tokens - t0) return;
  const bool there = (int64_t)t0 + tid < total;
  a.rows[t0 + tid] = !there ? -1 : mark < 0 ? first_row : mark_row[mark] - 1;
  a.positions[t0 + tid] = !there ? -1 : t0 + tid + (mark < 0 ? first_base : mark_base[mark]);
}

// ---- page contents ----

constexpr int kMaxPools = 128;
constexpr int kSegB = 16384;   // bytes a workgroup of 256 copies at a time

struct Pools {
  uint8_t* base[kMaxPools];
  int64_t page_bytes, page_stride;   // bytes
  int32_t count, segs;               // pools; segments of a page
};

// segment `seg` of page src of a pool to page dst: four loads of 16 bytes a
// thread in flight
SILE_DEV void copy_segment(const Pools& p, int pool, int seg, int32_t src, int32_t dst) {
  const uint8_t* from = p.base[pool] + (int64_t)src * p.page_stride;
  uint8_t* to = p.base[pool] + (int64_t)dst * p.page_stride;
  const int64_t at = (int64_t)seg * kSegB + threadIdx.x * 16;
  u32x4_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + 4096 * i < p.page_bytes) w[i] = *reinterpret_cast<const u32x4_t*>(from + at + 4096 * i);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + 4096 * i < p.page_bytes)
      __builtin_nontemporal_store(w[i], reinterpret_cast<u32x4_t*>(to + at + 4096 * i));
}

// pairs (src[i], dst[i]), i < n, workgroup `first` of `groups`
SILE_DEV void copy_pairs(const Pools& p, const int32_t* src, const int32_t* dst, int64_t n,
                         int32_t num_pages, int64_t first, int64_t groups) {
  const int64_t units = n * p.count * p.segs;
  for (int64_t u = first; u < units; u += groups) {
    const int64_t pair = u / (p.count * p.segs);
    const int r = (int)(u - pair * (p.count * p.segs));
    const int32_t s = src[pair], d = dst[pair];
    if ((uint32_t)s >= (uint32_t)num_pages || (uint32_t)d >= (uint32_t)num_pages || s == d) continue;
    copy_segment(p, r / p.segs, r % p.segs, s, d);
  }
}

SILE_DEV void copy_ints(const int32_t* from, int32_t* to, int64_t n, int64_t first, int64_t groups) {
  for (int64_t i = first * 256 + threadIdx.x; i < n; i += groups * 256) to[i] = from[i];
}

// exclusive sum over 1024 threads; *all: the whole sum
SILE_DEV int scan_1024(int v, int* lds, int* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int incl = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int up = __shfl_up(incl, off);
    if (lane >= off) incl += up;
  }
  if (lane == 63) lds[wave] = incl;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    if (w < wave) before += lds[w];
    total += lds[w];
  }
  __syncthreads();
  *all = total;
  return before + incl - v;
}

struct ReserveArgs {
  const int32_t* lengths;
  const int32_t* need;
  const int32_t* tables_in;
  int32_t* tables_out;
  const int32_t* refs_in;   // as they were before the call (a copy where the call is in place)
  int32_t* refs_out;
  int32_t* granted;
  int32_t* demand;          // workspace: [n_rows] pages a row needs (-1: cannot fit), then the rank of its first
  int32_t* kept;            // workspace: [n_rows] page whose contents the first fresh page takes, or -1
  int32_t* fresh;           // workspace: free pages, lowest first
  int64_t ld_table;
  int32_t n_rows, num_pages, page_shift;
};

// The entries a row's next `need` tokens fall into; false: they do not fit its table.
SILE_DEV bool wanted(const ReserveArgs& a, int row, int64_t* first, int64_t* last, bool* partial) {
  const int64_t cap = a.ld_table << a.page_shift;
  const int32_t raw = a.lengths[row];
  const int64_t len = raw < 0 ? 0 : raw > cap ? cap : raw;
  const int64_t need = a.need[row];
  *first = len >> a.page_shift;
  *last = need > 0 ? (len + need - 1) >> a.page_shift : *first - 1;
  *partial = (len & ((1ll << a.page_shift) - 1)) != 0;
  return need <= 0 || len + need <= cap;
}

}  // namespace

extern "C" __global__ __launch_bounds__(1024) void sile_kv_slots(SlotsArgs a) { slots(a); }
extern "C" __global__ __launch_bounds__(256) void sile_kv_append(AppendArgs a) { append<0>(a); }
extern "C" __global__ __launch_bounds__(256) void sile_kv_append_f16_fp8(AppendArgs a) { append<1>(a); }
extern "C" __global__ __launch_bounds__(256) void sile_kv_append_bf16_fp8(AppendArgs a) { append<2>(a); }

extern "C" __global__ __launch_bounds__(256) void sile_kv_copy_pages(Pools p, const int32_t* src,
                                                                     const int32_t* dst, int64_t n,
                                                                     int32_t num_pages) {
  copy_pairs(p, src, dst, n, num_pages, blockIdx.x, gridDim.x);
}

extern "C" __global__ __launch_bounds__(256) void sile_kv_copy_ints(const int32_t* from, int32_t* to,
                                                                    int64_t n) {
  copy_ints(from, to, n, blockIdx.x, gridDim.x);
}

// Rows with drop[row] != 0 let their pages go.  A workgroup a row; refs_out holds
// refs_in's values already.
extern "C" __global__ __launch_bounds__(256) void sile_kv_free(
    int64_t ld_table, const int32_t* drop, const int32_t* tables_in, int32_t* tables_out,
    const int32_t* lengths_in, int32_t* lengths_out, int32_t num_pages, int32_t* refs_out) {
  const int64_t row = blockIdx.x;
  const bool gone = drop[row] != 0;
  for (int64_t e = threadIdx.x; e < ld_table; e += 256) {
    const int32_t id = tables_in[row * ld_table + e];
    if (gone && (uint32_t)id < (uint32_t)num_pages) atomicSub(&refs_out[id], 1);
    tables_out[row * ld_table + e] = gone ? -1 : id;
  }
  if (threadIdx.x == 0) lengths_out[row] = gone ? 0 : lengths_in[row];
}

// Row i of the new table is row src[i] of the old one (empty where src[i] names
// none), and each of its pages counts once more: workgroups 0 .. n_out - 1.  Each page of
// an old row counts once less: a workgroup an old row behind them.
extern "C" __global__ __launch_bounds__(256) void sile_kv_fork(
    int32_t n_in, int32_t n_out, int64_t ld_table, const int32_t* src, const int32_t* tables_in,
    int32_t* tables_out, const int32_t* lengths_in, int32_t* lengths_out, int32_t num_pages,
    int32_t* refs_out) {
  if ((int64_t)blockIdx.x < n_out) {
    const int64_t i = blockIdx.x;
    const int32_t s = src[i];
    const bool in = s >= 0 && s < n_in;
    for (int64_t e = threadIdx.x; e < ld_table; e += 256) {
      const int32_t id = in ? tables_in[s * ld_table + e] : -1;
      if ((uint32_t)id < (uint32_t)num_pages) atomicAdd(&refs_out[id], 1);
      tables_out[i * ld_table + e] = id;
    }
    if (threadIdx.x == 0) lengths_out[i] = in ? lengths_in[s] : 0;
    return;
  }
  const int64_t row = (int64_t)blockIdx.x - n_out;
  for (int64_t e = threadIdx.x; e < ld_table; e += 256) {
    const int32_t id = tables_in[row * ld_table + e];
    if ((uint32_t)id < (uint32_t)num_pages) atomicSub(&refs_out[id], 1);
  }
}

// ---- handing out pages: (1) what each row needs, (2) which pages are free and
// which rows get theirs, (3) the tables, counts and shared pages' contents ----

// (1) A wave a row, workgroups 0 .. ceil(n_rows / 4) - 1: an entry needs a page
// where it holds none or one that another row holds too.  The workgroups behind
// them copy the counts (and, out of place, the tables).
extern "C" __global__ __launch_bounds__(256) void sile_kv_reserve_need(ReserveArgs a, const int32_t* refs,
                                                                       int32_t* snapshot) {
  const int64_t groups = (a.n_rows + 3) / 4;
  if ((int64_t)blockIdx.x >= groups) {
    const int64_t at = blockIdx.x - groups, n = gridDim.x - groups;
    // refs -> refs_out, or in place -> the snapshot the later steps read
    copy_ints(refs, snapshot, a.num_pages, at, n);
    if (a.tables_in != a.tables_out)
      copy_ints(a.tables_in, a.tables_out, a.n_rows * a.ld_table, at, n);
    return;
  }
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= a.n_rows) return;
  int64_t first, last;
  bool partial;
  const bool fits = wanted(a, row, &first, &last, &partial);
  int32_t n = 0, kept = -1;
  if (fits)
    for (int64_t e0 = first; e0 <= last; e0 += 64) {
      const int64_t e = e0 + lane;
      const int32_t id = e <= last ? a.tables_in[row * a.ld_table + e] : -1;
      const int32_t ref = (uint32_t)id < (uint32_t)a.num_pages ? refs[id] : 0;
      n += __popcll(__builtin_amdgcn_ballot_w64(e <= last && ref != 1));
      if (e == first && partial && ref > 1) kept = id;
    }
  if (lane == 0) {
    a.demand[row] = fits ? n : -1;
    a.kept[row] = kept;   // (entry `first` is lane 0's)
  }
}

// (2) One workgroup: ranks of the rows' pages, the free pages as far as they are
// asked for, and which rows get theirs: those before the first whose demand the
// free pages do not cover.
extern "C" __global__ __launch_bounds__(1024) void sile_kv_reserve_deal(ReserveArgs a) {
  __shared__ int lds[16];
  const int tid = threadIdx.x;
  int64_t total = 0;   // (a row asks for at most ld_table pages)
  for (int32_t r0 = 0; r0 < a.n_rows; r0 += 1024) {
    const int32_t r = r0 + tid;
    int all;
    (void)scan_1024(r < a.n_rows ? max(a.demand[r], 0) : 0, lds, &all);
    total += all;
  }
  int64_t found = 0;
  for (int64_t p0 = 0; p0 < a.num_pages && found < total; p0 += 4096) {
    int32_t ref[4];
    int n = 0, all;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t p = p0 + 4 * tid + i;
      ref[i] = p < a.num_pages ? a.refs_in[p] : 1;
      n += ref[i] <= 0;
    }
    int64_t at = found + scan_1024(n, lds, &all);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (ref[i] <= 0) a.fresh[at++] = (int32_t)(p0 + 4 * tid + i);
    found += all;
  }
  int64_t before = 0;
  for (int32_t r0 = 0; r0 < a.n_rows; r0 += 1024) {
    const int32_t r = r0 + tid;
    const int32_t want = r < a.n_rows ? a.demand[r] : 0;
    int all;
    const int64_t at = before + scan_1024(max(want, 0), lds, &all);
    if (r < a.n_rows) {
      const bool ok = want >= 0 && (want == 0 || at + want <= found);
      a.granted[r] = ok;
      a.demand[r] = ok ? (int32_t)at : -1;
      if (!ok) a.kept[r] = -1;
    }
    before += all;
  }
}

// (3) A wave a row (workgroups 0 .. ceil(n_rows / 4) - 1) hands its fresh pages out
// in the order of its entries; the workgroups behind them copy the contents of the
// part-filled pages that are shared.
extern "C" __global__ __launch_bounds__(256) void sile_kv_reserve_take(ReserveArgs a, Pools p) {
  const int64_t groups = (a.n_rows + 3) / 4;
  if ((int64_t)blockIdx.x >= groups) {
    const int64_t units = (int64_t)a.n_rows * p.count * p.segs;
    for (int64_t u = blockIdx.x - groups; u < units; u += gridDim.x - groups) {
      const int row = (int)(u / (p.count * p.segs)), r = (int)(u - (int64_t)row * (p.count * p.segs));
      const int32_t s = a.kept[row];
      if (s >= 0) copy_segment(p, r / p.segs, r % p.segs, s, a.fresh[a.demand[row]]);
    }
    return;
  }
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= a.n_rows) return;
  int32_t rank = a.demand[row];
  if (rank < 0) return;
  int64_t first, last;
  bool partial;
  (void)wanted(a, row, &first, &last, &partial);
  for (int64_t e0 = first; e0 <= last; e0 += 64) {
    const int64_t e = e0 + lane;
    const int32_t id = e <= last ? a.tables_in[row * a.ld_table + e] : -1;
    const int32_t ref = (uint32_t)id < (uint32_t)a.num_pages ? a.refs_in[id] : 0;
    const bool takes = e <= last && ref != 1;
    const uint64_t who = __builtin_amdgcn_ballot_w64(takes);
    if (takes) {
      const int32_t page = a.fresh[rank + __popcll(who & ((1ull << lane) - 1))];
      if (ref > 1) atomicSub(&a.refs_out[id], 1);
      a.refs_out[page] = 1;
      a.tables_out[row * a.ld_table + e] = page;
    }
    rank += __popcll(who);
  }
}

// ---- closing up: the pages in use past their number move, in order, into the
// free ones before it ----

// map: of a hole the page that moves in, of that page the hole, of any other page past
// the number in use itself; moves: their count
extern "C" __global__ __launch_bounds__(1024) void sile_kv_compact_plan(
    int32_t num_pages, const int32_t* refs, int32_t* used, int32_t* moves, int32_t* map,
    int32_t* holes, int32_t* movers) {
  __shared__ int lds[16];
  const int tid = threadIdx.x;
  // the first kHeld blocks of 4096 pages stay in registers as a bit a page
  constexpr int kHeld = 8;
  uint32_t held = 0;
  auto live4 = [&](int64_t p0) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t p = p0 + 4 * tid + i;
      if (p < num_pages && refs[p] > 0) m |= 1u << i;
    }
    return m;
  };
  int n = 0, count;
#pragma unroll
  for (int h = 0; h < kHeld; ++h)
    if (4096 * h < num_pages) held |= live4(4096 * h) << (4 * h);
  n = __popc(held);
  for (int64_t p0 = 4096 * kHeld; p0 < num_pages; p0 += 4096) n += __popc(live4(p0));
  (void)scan_1024(n, lds, &count);
  int nh = 0, nm = 0;
  for (int64_t p0 = 0; p0 < num_pages; p0 += 4096) {
    const uint32_t live = p0 < 4096 * kHeld ? (held >> (p0 / 4096 * 4)) & 15u : live4(p0);
    uint32_t hole = 0, mover = 0;
    int all;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t p = p0 + 4 * tid + i;
      const bool in = p < num_pages, is_live = (live >> i) & 1;
      if (in && !is_live && p < count) hole |= 1u << i;
      if (is_live && p >= count) mover |= 1u << i;
      if (in && p >= count && !is_live) map[p] = (int32_t)p;
    }
    // both ranks in one scan: at most 4096 of each
    const int both = scan_1024(__popc(hole) | __popc(mover) << 16, lds, &all);
    int ah = nh + (both & 0xffff), am = nm + (both >> 16);
    nh += all & 0xffff;
    nm += all >> 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int32_t p = (int32_t)(p0 + 4 * tid + i);
      if ((hole >> i) & 1) holes[ah++] = p;
      if ((mover >> i) & 1) movers[am++] = p;
    }
  }
  __syncthreads();
  for (int k = tid; k < nm; k += 1024) {   // (as many holes as movers)
    map[movers[k]] = holes[k];
    map[holes[k]] = movers[k];
  }
  if (tid == 0) {
    *used = count;
    *moves = nm;
  }
}

// Workgroups 0 .. meta - 1: counts and tables; the others: contents.  In place no
// entry is read by one thread and written by another: a hole's thread moves its
// page's count.
extern "C" __global__ __launch_bounds__(256) void sile_kv_compact_move(
    int32_t meta, int64_t entries, const int32_t* tables_in, int32_t* tables_out, int32_t num_pages,
    const int32_t* refs_in, int32_t* refs_out, const int32_t* count, const int32_t* moves,
    const int32_t* map, const int32_t* holes, const int32_t* movers, Pools p) {
  if ((int64_t)blockIdx.x >= meta) {
    if (p.count) copy_pairs(p, movers, holes, *moves, num_pages, blockIdx.x - meta, gridDim.x - meta);
    return;
  }
  const int32_t used = *count;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < entries; i += (int64_t)meta * 256) {
    const int32_t id = tables_in[i];
    tables_out[i] = id >= used && id < num_pages ? map[id] : id;
  }
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < num_pages; i += (int64_t)meta * 256) {
    if (i < used) {
      const int32_t r = refs_in[i];
      if (r > 0) {
        refs_out[i] = r;
      } else {
        const int32_t m = map[i];
        refs_out[i] = refs_in[m];
        refs_out[m] = 0;
      }
    } else if (map[i] == i) {
      refs_out[i] = 0;
    }
  }
}
