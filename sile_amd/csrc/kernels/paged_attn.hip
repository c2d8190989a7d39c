// Attention of one new token a row over a paged key-value cache.
//
//   o[b][h] = softmax_j(q[b][h] . k_j * scale) v_j over the keys j the token at
//   position lengths[b] - 1 sees (all, or the last `window` and the first `sinks`)
//
// K and V pages are [kv_heads][page][d]; key j of row b lies in page
// tables[b][j / page], slot j % page.
//
// What bounds it: every key and value is read once (HBM), against 4 g flop for
// each of their element pairs, g query heads a key head.  So the matrix cores run far below
// their rate whatever the tile, and the layout serves the loads:
//
//  * a wave takes 32 keys at a time and a tile of 16 query heads (the query
//    heads that share a key head, padded), v_mfma_f32_16x16x32.  S^T = K . Q^T
//    takes K straight from memory to registers: lane l supplies 8 consecutive
//    dims of key l % 16, as the A operand asks.  Its accumulator holds 4 keys of
//    ONE query head (l % 16), so max and sum are in-lane folds and two exchanges.
//  * O^T = V^T . P^T needs 8 keys of one dim a lane: V goes through the wave's
//    own LDS tile and is read with ds_read_b64_tr_b16.  No wave waits for
//    another until the end of its keys.
//  * P enters the product as two 16-bit parts, value and rest (16 bits of it in
//    bf16, 22 in f16): the matrix cores have the room, and the result is then as exact
//    as an fp32 P's.  But an Inf of V times a part that is zero, or has the other sign, is not
//    what the formula says: a result that is not finite is taken again with one fp32 p.
//  * while a tile is computed the next one's loads are in flight, and the page
//    numbers of the one after.
//
// The tiles of all rows and key heads are one flat list, dealt in equal shares to
// a fixed grid of workgroups (make_deal): a long row is spread over many
// workgroups and a batch of mixed lengths has no straggler, with the lengths
// known only on the device.  A workgroup whose share covers a row's key head
// whole writes its output; the others leave (O, m, l) in fp32 in the workspace, at
// most two a workgroup, and a second launch joins them.  Where the host knows that
// every row is short, a workgroup takes one unit instead, and there is nothing to join.
//
// Measured: 32 rows of up to 8192 keys, 8 key heads of 128 in 16 bits, 97 us (5.7 TB/s of K and V;
// a copy reaches 5.3), one row of 131071 91 (5.9); 64 rows of up to 4000 in e4m3 61 (4.3); 100 rows
// under a window of 1000, 4 key heads of 80, 26 (4.8); one row of 300 keys 6.1.
//
// An 8-bit cache (e4m3) is widened in registers, exactly: K into the operand, V on
// its way into LDS; the scales go into the score's and the output's factor.
#include "common.h"
#include "paged_plan.h"

using namespace sile;

namespace {

constexpr float kLowest = -3.402823466e38f;
// V's rows are loaded whole by one instruction and non-temporal; K's by several, of 64 bytes a
// row each, which the caches have to bring together (32 rows up to 8192 keys of 128: 107 us,
// V so 97, K too 94; but 128 rows up to 1000: 30, 26, 30, and 32 rows up to 2000 of 256: 65, 58, 77).
constexpr int kNonTemporal = 2;
// The probabilities of a row carry a factor 2^kLift, its maximum's being exactly
// that: f16 has no exponent below 2^-24, and a long row has many keys far below
// its maximum.  l and O carry it too, so it drops out of O / l.
template <bool kBF16>
constexpr float kLift = kBF16 ? 0.0f : 15.0f;

struct PagedArgs {
  const uint16_t* q;
  const uint8_t* k;
  const uint8_t* v;
  uint16_t* o;
  const int32_t* tables;
  const int32_t* lengths;
  int32_t* plan;        // workspace: tiles of the rows before each row, then of all rows
  float* part_ml;       // workspace: [slots][rows][2]
  float* part_o;        // workspace: [slots][rows][d]
  int64_t ldq, ldo, page_stride, ld_table, capacity, window, sinks;
  int32_t batch, kv_heads, group, head_groups, d, num_pages, page_shift, groups;
  int32_t direct;       // 1: a workgroup a unit, no list and no parts
  int32_t e4m3;         // 1: an 8-bit cache
  float scale_log2, v_scale;
};

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_ptr;

template <bool kBF16>
SILE_DEV f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (kBF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <bool kBF16>
SILE_DEV uint32_t pack2(float lo, float hi) {
  return kBF16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
}

// what is left of lo and hi beside their 16-bit values in `pk`, packed alike
template <bool kBF16>
SILE_DEV uint32_t rest2(float lo, float hi, uint32_t pk) {
  if constexpr (kBF16) {
    return pack2<kBF16>(lo - bits_f32(pk << 16), hi - bits_f32(pk & 0xffff0000u));
  } else {
    const f16x2 h = __builtin_bit_cast(f16x2, pk);
    return pack2<kBF16>(lo - (float)h[0], hi - (float)h[1]);
  }
}

// two e4m3 codes of `w` (bytes 0, 1 or 2, 3) as two 16-bit values, exactly
template <bool kBF16, bool kHigh>
SILE_DEV uint32_t widen2(uint32_t w) {
  if constexpr (kBF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, kHigh));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, kHigh));
}
template <bool kBF16>
SILE_DEV u32x4 widen8(uint32_t a, uint32_t b) {
  return u32x4{widen2<kBF16, false>(a), widen2<kBF16, true>(a), widen2<kBF16, false>(b),
               widen2<kBF16, true>(b)};
}

// max of v over lanes l, l ^ 16, l ^ 32, l ^ 48
SILE_DEV float quad_max(float v) {
  v = __builtin_fmaxf(v, swizzle_xor16(v));
  float lo, hi;
  half_swap(v, lo, hi);
  return __builtin_fmaxf(lo, hi);
}
SILE_DEV float quad_sum(float v) { return pair32_sum(v + swizzle_xor16(v)); }

template <int kDp>
struct Shape {
  static constexpr int kRow = 2 * kDp;                        // bytes of a V row in LDS
  static constexpr int kPitch = kDp + 4;                      // floats of an O row in LDS
  static constexpr int kTileB = kTileKeys * kRow;
  static constexpr int kMergeB = 16 * kPitch * 4;
  static constexpr int kWaveB = kTileB > kMergeB ? kTileB : kMergeB;
};

// Dealing: which row holds a workgroup's first tile of the flat list.  Every thread adds
// up the unit sizes of a run of rows, a scan over the 256 threads follows, and the thread
// whose run holds the row leaves it here, with the sizes before it (a row stands in the
// list once a unit).  Workgroup 0 keeps the sums for the join.
struct DealLds {
  int32_t wave_sum[4];
  int32_t row, before;
  int32_t x, x1, first_row, base;   // the workgroup's share, for paged_again
  int32_t again;                    // 1: it has rows to be taken again
};

// Whether l is a sum of probabilities that are numbers (scores of NaN, or all -inf, make a whole
// row NaN, and it stays so).
SILE_DEV bool finite_sum(float l) { return l > 0.0f && l < __builtin_inff(); }

// A query head of a row by a workgroup of kWaves, with p as one fp32 value, for a cache of 16
// bits: where V has an Inf in a seen key, the second part of P (zero, or of a sign of its own)
// makes a NaN of it on the matrix cores.  A wave takes every kWaves-th 64 keys: a lane works
// out a key's score, then the lanes take two dims each, with 16 keys' loads in flight; the waves'
// sums are added up through LDS, kWaves * (2 + 256) floats.  (One row of 131071 keys with an Inf:
// 2.9 ms in place of 92 us, 32 rows of 2000 0.36 ms in place of 42 us.)
template <bool kBF16, int kWaves>
SILE_DEV void paged_row(const PagedArgs& a, int row, int kvh, int head, const KeySpan& span, float* lds) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), d = a.d;
  auto f32_of = [](uint32_t b) { return kBF16 ? bf16_to_f32((uint16_t)b) : f16_to_f32((uint16_t)b); };
  const uint16_t* q = a.q + (int64_t)row * a.ldq + (int64_t)head * d;
  const uint16_t* const k = reinterpret_cast<const uint16_t*>(a.k);
  const uint16_t* const v = reinterpret_cast<const uint16_t*>(a.v);
  const int32_t* table = a.tables + (int64_t)row * a.ld_table;
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, m = kLowest, l = 0.0f;   // dims 2 lane, 2 lane + 1, and 128 on
  const int64_t n = (int64_t)span.sink_end + span.len - span.first;
  for (int64_t i0 = 64 * wave; i0 < n; i0 += 64 * kWaves) {
    const int64_t i = min(i0 + lane, n - 1);
    const int key = (int)(i < span.sink_end ? i : i - span.sink_end + span.first);
    const int32_t id = table[key >> a.page_shift];
    const bool ok = i0 + lane < n && (uint32_t)id < (uint32_t)a.num_pages;
    // (a key that is not seen: page 0's row of its slot, which is there)
    const int64_t off = (int64_t)(ok ? id : 0) * a.page_stride +
                        (((int64_t)kvh << a.page_shift) + (key & ((1 << a.page_shift) - 1))) * d;
    float s = 0.0f;
#pragma unroll 4
    for (int c = 0; c < d; c += 8) {
      const u32x4 qw = *reinterpret_cast<const u32x4*>(q + c), kw = *reinterpret_cast<const u32x4*>(k + off + c);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        s += f32_of(qw[j >> 1] >> (16 * (j & 1))) * f32_of(kw[j >> 1] >> (16 * (j & 1)));
    }
    s *= a.scale_log2;
    const float m_new = __builtin_fmaxf(m, wave_max(ok && s == s ? s : kLowest));
    const float alpha = exp2_fast(m - m_new), p = ok ? exp2_fast(s - m_new) : 0.0f;
    m = m_new;
    l = l * alpha + wave_sum(p);
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[t] *= alpha;
    const uint64_t seen = __builtin_amdgcn_ballot_w64(ok);
    const int off_lo = (int)(uint32_t)off, off_hi = (int)(off >> 32);
    for (int k0 = 0; k0 < 64; k0 += 16) {
      if (((seen >> k0) & 0xffff) == 0) continue;
      uint32_t w[16][2];
#pragma unroll
      for (int u = 0; u < 16; ++u) {
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane(off_lo, k0 + u);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane(off_hi, k0 + u);
        const uint16_t* vr = v + (int64_t)((uint64_t)hi << 32 | lo) + 2 * lane;
#pragma unroll
        for (int t = 0; t < 2; ++t)
          w[u][t] = 2 * lane + 128 * t < d ? *reinterpret_cast<const uint32_t*>(vr + 128 * t) : 0;
      }
#pragma unroll
      for (int u = 0; u < 16; ++u) {
        const float pu = bits_f32((uint32_t)__builtin_amdgcn_readlane((int)f32_bits(p), k0 + u));
        if ((seen >> (k0 + u)) & 1)
#pragma unroll
          for (int t = 0; t < 4; ++t) acc[t] += pu * f32_of(w[u][t >> 1] >> (16 * (t & 1)));
      }
    }
  }
  if (lane == 0) {
    lds[2 * wave] = m;
    lds[2 * wave + 1] = l;
  }
#pragma unroll
  for (int t = 0; t < 4; ++t) lds[2 * kWaves + 256 * wave + 128 * (t >> 1) + 2 * lane + (t & 1)] = acc[t];
  __syncthreads();
  const int dim = threadIdx.x;
  if (dim < d) {
    float top = kLowest, sum = 0.0f, o = 0.0f;
    for (int w = 0; w < kWaves; ++w) top = __builtin_fmaxf(top, lds[2 * w]);
    for (int w = 0; w < kWaves; ++w) {
      const float f = exp2_fast(lds[2 * w] - top);
      sum += f * lds[2 * w + 1];
      o += f * lds[2 * kWaves + 256 * w + dim];
    }
    o *= a.v_scale / sum;
    a.o[(int64_t)row * a.ldo + (int64_t)head * d + dim] = kBF16 ? bf16_rne(o) : f16_rne(o);
  }
  __syncthreads();   // (the next head's sums go to the same place)
}

// The query heads of this workgroup's whole units whose results are not finite, again.  Behind
// the rounds and from what stands in LDS, so that they keep nothing for it (called where a unit
// ends, it took 28 scalar registers of theirs: 32 rows of 1024 keys 23.4 -> 23.8 us, group 24 40 -> 43;
// so 23.7 and 41).
template <bool kBF16, int kQT>
SILE_DEV void paged_again(const PagedArgs& a, const DealLds* deal, float* lds) {
  const int lane = threadIdx.x & 63, heads = a.kv_heads * a.head_groups;
  int32_t x = __builtin_amdgcn_readfirstlane(deal->x), row = __builtin_amdgcn_readfirstlane(deal->first_row);
  int32_t base = __builtin_amdgcn_readfirstlane(deal->base);
  const int32_t x1 = __builtin_amdgcn_readfirstlane(deal->x1);
  while (x < x1 && row < a.batch) {   // as in paged_attn
    const KeySpan span = key_span(__builtin_amdgcn_readfirstlane(a.lengths[row]), a.capacity, a.window, a.sinks);
    const int32_t size = unit_size(span);
    if (x >= base + size * heads) {
      base += size * heads;
      ++row;
      continue;
    }
    const int unit = (x - base) / size;
    const int u0 = x - base - unit * size, u1 = min(size, u0 + (x1 - x));
    x += u1 - u0;
    if (u0 > kUnitTiles || u1 < size) continue;   // in parts: the join's
    const int kvh = unit / a.head_groups, hg = unit - kvh * a.head_groups;
    const int head0 = kvh * a.group + hg * 16 * kQT, rows = min(16 * kQT, a.group - hg * 16 * kQT);
    for (int r = 0; r < rows; ++r) {   // (every wave sees the same: a head is stored anew behind a barrier)
      const uint16_t* o = a.o + (int64_t)row * a.ldo + (int64_t)(head0 + r) * a.d;
      constexpr uint16_t kExp = kBF16 ? 0x7f80 : 0x7c00;
      bool bad = false;
      for (int c = lane; c < a.d; c += 64) bad |= (o[c] & kExp) == kExp;
      if (__builtin_amdgcn_ballot_w64(bad) != 0) paged_row<kBF16, kTileWaves>(a, row, kvh, head0 + r, span, lds);
    }
  }
}

template <bool kBF16, bool kFp8, int kDp, bool kExact, bool kPage16, int kQT>
__device__ __forceinline__ void paged_attn(const PagedArgs& a, uint8_t* smem, float* ml,
                                           DealLds* deal) {
  using Sh = Shape<kDp>;
  constexpr int kKK = kDp / 32;                      // d-steps of S^T
  constexpr int kDT = kDp / 16;                      // 16-dim tiles of O^T
  constexpr int kEs = kFp8 ? 1 : 2;                  // bytes of a cache element
  constexpr int kCh = kDp * kEs / 16;                // 16-byte chunks of a cache row
  constexpr int kKL = kFp8 ? kKK / 2 : kKK;          // K loads of a lane for 16 keys
  constexpr int kVL = kTileKeys * kCh / 64;          // V loads of a lane
  constexpr int kVRows = 64 / kCh;                   // V rows one load instruction covers
  static_assert(kCh <= 64 && kKK % 2 == 0, "row width");
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, l16 = lane & 15;
  const int heads = a.kv_heads * a.head_groups;      // units of a row
  const int d = kExact ? kDp : a.d;
  const int chunks = d * kEs / 16;

  int row;
  int32_t x, x1, base;   // the list's tiles x .. x1 - 1 are this workgroup's; row `row` begins at base
  if (a.direct) {
    // ---- a unit a workgroup ----
    row = blockIdx.x / heads;
    const int unit = blockIdx.x - row * heads;
    const int32_t size = unit_size(
        key_span(__builtin_amdgcn_readfirstlane(a.lengths[row]), a.capacity, a.window, a.sinks));
    base = 0;
    x = unit * size;
    x1 = x + size;
    if (size == 0) {   // a row without keys
      const int kvh = unit / a.head_groups, h0 = (unit - kvh * a.head_groups) * 16 * kQT;
      const int n = min(16 * kQT, a.group - h0) * d;
      uint16_t* o = a.o + (int64_t)row * a.ldo + (int64_t)(kvh * a.group + h0) * d;
      for (int c = tid; c < n; c += 256) o[c] = 0;
      return;
    }
  } else {
    // ---- deal ----
    const int per = (a.batch + 255) / 256;
    int32_t mine = 0;
    for (int r = tid * per; r < min((tid + 1) * per, a.batch); ++r)
      mine += unit_size(key_span(a.lengths[r], a.capacity, a.window, a.sinks));
    int32_t incl = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int32_t up = __shfl_up(incl, off);
      if (lane >= off) incl += up;
    }
    if (lane == 63) deal->wave_sum[wave] = incl;
    __syncthreads();
    int32_t before = incl - mine, rows_total = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) before += deal->wave_sum[w];
      rows_total += deal->wave_sum[w];
    }
    const int32_t total = __builtin_amdgcn_readfirstlane(rows_total) * heads;
    const Deal shares = make_deal(total, a.groups);
    x = deal_start(shares, blockIdx.x);
    x1 = deal_start(shares, blockIdx.x + 1);
    if (blockIdx.x == 0 || x < x1) {
      int32_t at = before;
      for (int r = tid * per; r < min((tid + 1) * per, a.batch); ++r) {
        const int32_t t = unit_size(key_span(a.lengths[r], a.capacity, a.window, a.sinks));
        if (blockIdx.x == 0) a.plan[r] = at;
        if (x < x1 && x / heads >= at && x / heads < at + t) {
          deal->row = r;
          deal->before = at;
        }
        at += t;
      }
      if (blockIdx.x == 0 && tid == 0) a.plan[a.batch] = rows_total;
    }
    if (x >= x1) return;
    __syncthreads();
    row = __builtin_amdgcn_readfirstlane(deal->row);
    base = __builtin_amdgcn_readfirstlane(deal->before) * heads;
  }
  uint8_t* const vt = smem + wave * Sh::kWaveB;
  if (!kFp8 && tid == 0) {
    deal->x = x;
    deal->x1 = x1;
    deal->first_row = row;
    deal->base = base;
    deal->again = 0;
  }

  while (x < x1 && row < a.batch) {
    const KeySpan span = key_span(__builtin_amdgcn_readfirstlane(a.lengths[row]), a.capacity, a.window, a.sinks);
    const int32_t size = unit_size(span);
    if (x >= base + size * heads) {   // on to the next row
      base += size * heads;
      ++row;
      continue;
    }
    const int unit = (x - base) / size;
    const int u0 = x - base - unit * size, u1 = min(size, u0 + (x1 - x));
    x += u1 - u0;
    const int t0 = max(u0 - kUnitTiles, 0), t1 = u1 - kUnitTiles;
    if (t1 <= t0) continue;   // of this unit only what it counts extra
    const int kvh = unit / a.head_groups, hg = unit - kvh * a.head_groups;
    const int rows = min(16 * kQT, a.group - hg * 16 * kQT);   // query heads of this unit
    const int head0 = kvh * a.group + hg * 16 * kQT;
    const int32_t* table = a.tables + (int64_t)row * a.ld_table;

    int qlane = lane;
    asm volatile("" : "+v"(qlane));   // (as at the end)
    const int qg = qlane >> 4, ql = qlane & 15;
    // ---- Q^T fragments: query head l16 of tile qt, zeros past the heads and dims ----
    u32x4 qf[kQT][kKK];
#pragma unroll
    for (int qt = 0; qt < kQT; ++qt) {
      const bool in = qt * 16 + ql < rows;
      const uint16_t* qr = a.q + (int64_t)row * a.ldq + (int64_t)(head0 + (in ? qt * 16 + ql : 0)) * d;
#pragma unroll
      for (int kk = 0; kk < kKK; ++kk) {
        const int dim = kFp8 ? 64 * (kk / 2) + 16 * qg + 8 * (kk & 1) : 32 * kk + 8 * qg;
        u32x4 w = {0u, 0u, 0u, 0u};
        if (in && (kExact || dim < d)) w = *reinterpret_cast<const u32x4*>(qr + dim);
        qf[qt][kk] = w;
      }
    }
    f32x4 oacc[kQT][kDT];
    float m_run[kQT], l_run[kQT];
#pragma unroll
    for (int qt = 0; qt < kQT; ++qt) {
      m_run[qt] = -__builtin_inff();
      l_run[qt] = 0.0f;
#pragma unroll
      for (int dt = 0; dt < kDT; ++dt) oacc[qt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // ---- loads ----
    // table entry of key (lane & 31) of tile t (any entry of the row's past its
    // keys); read a round ahead and looked at by load_tile alone, which then does
    // not wait for it
    auto page_of = [&](int t) {
      const int key = span_key(span, min(t, t1 - 1)) + (lane & 31);
      return table[min(key, span.len - 1) >> a.page_shift];
    };
    // (defined by an empty asm: left undefined before a unit's first loads, they are kept
    // in registers a second time, from the unit before)
    u32x4 kr[2][kKL], vr[kVL];
#pragma unroll
    for (int i = 0; i < kKL; ++i) asm volatile("" : "=v"(kr[0][i]), "=v"(kr[1][i]));
#pragma unroll
    for (int i = 0; i < kVL; ++i) asm volatile("" : "=v"(vr[i]));
    const int64_t head_off = (int64_t)kvh * d << a.page_shift;
    const int row_b = d * kEs;
    // issues tile t's loads; returns the mask of its keys that are seen
    auto load_tile = [&](int t, int32_t id) -> uint32_t {
      if constexpr (kPage16) {
        // 16 keys lie in one page: a buffer resource over their rows, which ends at
        // the row's last key and is empty where the page does not exist, so
        // that what lies past it is never read (it loads as zeros); all of it scalar
        const int32_t ids[2] = {__builtin_amdgcn_readlane(id, 0), __builtin_amdgcn_readlane(id, 16)};
        const int key0 = span_key(span, min(t, t1 - 1));
        uint32_t seen = t < t1 ? span_bits(span, key0) : 0u;
#pragma unroll
        for (int s = 0; s < 2; ++s)
          if ((uint32_t)ids[s] >= (uint32_t)a.num_pages) seen &= s ? 0x0000ffffu : 0xffff0000u;
        if (seen == 0) return 0;
        const int slot = key0 & ((1 << a.page_shift) - 1);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const bool ok = (uint32_t)ids[s] < (uint32_t)a.num_pages;
          // (through readfirstlane: the clamp is a vector instruction, and a resource in
          // vector registers costs a loop around every load)
          const int rows_in =
              __builtin_amdgcn_readfirstlane(ok ? min(max(span.len - key0 - 16 * s, 0), 16) : 0);
          const int64_t at = (int64_t)(ok ? ids[s] : 0) * a.page_stride + head_off +
                             (int64_t)((slot + 16 * s) & ((1 << a.page_shift) - 1)) * d;
          const __amdgpu_buffer_rsrc_t kb = __builtin_amdgcn_make_buffer_rsrc(
              (void*)(a.k + at * kEs), (short)0, rows_in * row_b, 0x00020000);
          const __amdgpu_buffer_rsrc_t vb = __builtin_amdgcn_make_buffer_rsrc(
              (void*)(a.v + at * kEs), (short)0, rows_in * row_b, 0x00020000);
#pragma unroll
          for (int i = 0; i < kKL; ++i) {
            const int c = 4 * i + g;   // (a chunk past the dims: past the resource, zeros)
            const int off = kExact || c < chunks ? l16 * row_b + 16 * c : 0x7fff0000;
            kr[s][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(kb, off, 0, 0));
          }
#pragma unroll
          for (int i = 0; i < kVL / 2; ++i) {
            const int c = lane % kCh;
            const int off = kExact || c < chunks ? (kVRows * i + lane / kCh) * row_b + 16 * c : 0x7fff0000;
            vr[s * (kVL / 2) + i] =
                __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(vb, off, 0, kNonTemporal));
          }
        }
        return seen;
      } else {
        // pages of 1 to 8 keys: every lane works out its own key's row, the lanes that
        // load it ask that lane
        const int key = span_key(span, min(t, t1 - 1)) + (lane & 31);
        const bool ok = t < t1 && span_sees(span, key) && (uint32_t)id < (uint32_t)a.num_pages;
        const uint32_t seen = (uint32_t)__builtin_amdgcn_ballot_w64(ok);
        if (seen == 0) return 0;
        const int slot = key & ((1 << a.page_shift) - 1);
        // keys that are not seen take page 0's row of the same slot, which is there
        const int64_t off = ((int64_t)(ok ? id : 0) * a.page_stride + head_off + (int64_t)slot * d) * kEs;
        const int off_lo = (int)(uint32_t)off, off_hi = (int)(off >> 32);
        auto row_off = [&](int k) {
          const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * k, off_lo);
          const int32_t hi = __builtin_amdgcn_ds_bpermute(4 * k, off_hi);
          return (int64_t)(((uint64_t)(uint32_t)hi << 32) | lo);
        };
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const uint8_t* p = a.k + row_off(16 * s + l16);
#pragma unroll
          for (int i = 0; i < kKL; ++i) {
            const int c = 4 * i + g;
            u32x4 w = {0u, 0u, 0u, 0u};
            if (kExact || c < chunks) w = *reinterpret_cast<const u32x4*>(p + 16 * c);
            kr[s][i] = w;
          }
        }
#pragma unroll
        for (int i = 0; i < kVL; ++i) {
          const int c = lane % kCh;   // a chunk past the dims reads chunk 0 (its O^T rows are not kept)
          const uint8_t* p = a.v + row_off(kVRows * i + lane / kCh);
          vr[i] = __builtin_nontemporal_load(
              reinterpret_cast<const u32x4*>(p + 16 * (kExact || c < chunks ? c : 0)));
        }
        return seen;
      }
    };
    auto vswz = [](int r) { return (kDp == 64 ? 2 : 4) * (r & 3); };

    // one round of a wave: S and V of the tile that has arrived, the next tile's
    // loads into the registers they leave, softmax and P V beside those.  A tile
    // without any key (the round before the first; holes) is passed over.
    int t = t0 + wave - kTileWaves;
    int32_t id = page_of(t0 + wave);
    uint32_t seen = 0;
    while (true) {
      const uint32_t now = seen;
      f32x4 sacc[kQT][2];
      if (now != 0) {
      // S^T: keys 16 s + 4 g + i of query head l16
#pragma unroll
      for (int qt = 0; qt < kQT; ++qt)
#pragma unroll
        for (int s = 0; s < 2; ++s) sacc[qt][s] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int kk = 0; kk < kKK; ++kk)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          u32x4 kf;
          if constexpr (kFp8)
            kf = widen8<kBF16>(kr[s][kk / 2][2 * (kk & 1)], kr[s][kk / 2][2 * (kk & 1) + 1]);
          else
            kf = kr[s][kk];
#pragma unroll
          for (int qt = 0; qt < kQT; ++qt) sacc[qt][s] = mma16<kBF16>(kf, qf[qt][kk], sacc[qt][s]);
        }
      // V into the wave's LDS tile; a key that is not seen as zeros (0 times what
      // lies there could be NaN)
#pragma unroll
      for (int i = 0; i < kVL; ++i) {
        const int r = kVRows * i + lane / kCh, c = lane % kCh;
        u32x4 w = vr[i];
        if (now != 0xffffffffu && !((now >> r) & 1)) w = u32x4{0u, 0u, 0u, 0u};
        if constexpr (kFp8) {
          *reinterpret_cast<u32x4*>(vt + r * Sh::kRow + (((2 * c) ^ vswz(r)) << 4)) =
              widen8<kBF16>(w[0], w[1]);
          *reinterpret_cast<u32x4*>(vt + r * Sh::kRow + (((2 * c + 1) ^ vswz(r)) << 4)) =
              widen8<kBF16>(w[2], w[3]);
        } else {
          *reinterpret_cast<u32x4*>(vt + r * Sh::kRow + ((c ^ vswz(r)) << 4)) = w;
        }
      }
      }
      __builtin_amdgcn_sched_barrier(0);
      t += kTileWaves;
      seen = load_tile(t, id);
      id = page_of(t + kTileWaves);
      __builtin_amdgcn_sched_barrier(0);

      if (now != 0) {
      // online softmax in units of log2 e; a seen key's score counts as at least
      // the lowest float in the max, so that a row of -inf scores is told from an
      // empty one (0 / 0 against zeros)
      u32x4 pf[kQT], pr[kQT];
      const uint32_t bits = ((now >> (4 * g)) & 0xfu) | (((now >> (16 + 4 * g)) & 0xfu) << 4);
#pragma unroll
      for (int qt = 0; qt < kQT; ++qt) {
        float sc[8];
        float mx = kLowest;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          sc[i] = sacc[qt][i >> 2][i & 3] * a.scale_log2;
          if (now != 0xffffffffu) sc[i] = (bits >> i) & 1 ? sc[i] : -__builtin_inff();
          mx = __builtin_fmaxf(mx, sc[i]);
        }
        const float m_new = __builtin_fmaxf(m_run[qt], quad_max(mx));   // (> -inf: a key is seen)
        const float alpha = exp2_fast(m_run[qt] - m_new);
        m_run[qt] = m_new;
        float rs = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float p0 = exp2_fast(sc[i] - m_new + kLift<kBF16>);
          const float p1 = exp2_fast(sc[i + 1] - m_new + kLift<kBF16>);
          rs += p0 + p1;
          const uint32_t pk = pack2<kBF16>(p0, p1);
          pf[qt][i >> 1] = pk;
          pr[qt][i >> 1] = rest2<kBF16>(p0, p1, pk);
        }
        l_run[qt] = l_run[qt] * alpha + rs;
        if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
          for (int dt = 0; dt < kDT; ++dt) oacc[qt][dt] *= alpha;
        }
      }
      __builtin_amdgcn_wave_barrier();
      // O^T += V^T . P^T: slots 0-3 keys 4 g + j, slots 4-7 keys 16 + 4 g + j
#pragma unroll
      for (int dt = 0; dt < kDT; ++dt) {
        u32x4 vf;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int key = 16 * h + 4 * g + (l16 >> 2);
          const int c = 2 * dt + ((l16 & 3) >> 1);
          const s16x4 w = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_s16x4_ptr)(vt + key * Sh::kRow + ((c ^ vswz(key)) << 4) + 8 * (l16 & 1)));
          const u32x2 w2 = __builtin_bit_cast(u32x2, w);
          vf[2 * h] = w2[0];
          vf[2 * h + 1] = w2[1];
        }
#pragma unroll
        for (int qt = 0; qt < kQT; ++qt) {
          oacc[qt][dt] = mma16<kBF16>(vf, pf[qt], oacc[qt][dt]);
          oacc[qt][dt] = mma16<kBF16>(vf, pr[qt], oacc[qt][dt]);
        }
      }
      __builtin_amdgcn_wave_barrier();
      }
      if (t >= t1) break;
    }

    // ---- the four waves' (m, l, O) added up ----
    // (the thread number through an empty asm: addresses worked out here are not
    // kept in registers through the rounds)
    int et = tid;
    asm volatile("" : "+v"(et));
    const int eg = (et & 63) >> 4, el = et & 15;
    const bool whole = t0 == 0 && t1 == span.tiles;
    const int slot = 2 * blockIdx.x + (t0 == 0 ? 1 : 0);
#pragma unroll
    for (int qt = 0; qt < kQT; ++qt) {
      const float l = quad_sum(l_run[qt]);
      if (eg == 0) {
        ml[(wave * 16 + el) * 2] = m_run[qt];
        ml[(wave * 16 + el) * 2 + 1] = l;
      }
      float* ot = reinterpret_cast<float*>(vt) + el * Sh::kPitch + 4 * eg;
#pragma unroll
      for (int dt = 0; dt < kDT; ++dt) *reinterpret_cast<f32x4*>(ot + 16 * dt) = oacc[qt][dt];
      __syncthreads();
      const int r = et >> 4, head = qt * 16 + r;
      float w[4], m = -__builtin_inff(), sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) m = __builtin_fmaxf(m, ml[(i * 16 + r) * 2]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float mi = ml[(i * 16 + r) * 2];
        w[i] = mi == -__builtin_inff() ? 0.0f : exp2_fast(mi - m);
        sum += w[i] * ml[(i * 16 + r) * 2 + 1];
      }
      if (head < rows) {
        // a row without keys gives zeros; scores that are all -inf give 0 / 0
        const float f = whole ? (m == -__builtin_inff() ? 0.0f : a.v_scale / sum) : 1.0f;
        const int64_t at = (int64_t)slot * 16 * kQT + head;
        float z = 0.0f;
        for (int c = 4 * (et & 15); c < d; c += 64) {
          f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(
                reinterpret_cast<const float*>(smem + i * Sh::kWaveB) + r * Sh::kPitch + c);
            acc += v * w[i];
          }
          acc *= f;
          if constexpr (!kFp8) z = __builtin_fmaf((acc[0] + acc[1]) + (acc[2] + acc[3]), 0.0f, z);
          if (whole) {
            const u32x2 out = {pack2<kBF16>(acc[0], acc[1]), pack2<kBF16>(acc[2], acc[3])};
            *reinterpret_cast<u32x2*>(a.o + (int64_t)row * a.ldo + (int64_t)(head0 + head) * d + c) = out;
          } else {
            *reinterpret_cast<f32x4*>(a.part_o + at * d + c) = acc;
          }
        }
        // (codes of e4m3 have no Inf)
        if (!kFp8 && whole && !(z == 0.0f) && finite_sum(sum)) deal->again = 1;
        if (!whole && (et & 15) == 0) {
          a.part_ml[at * 2] = m;
          a.part_ml[at * 2 + 1] = sum;
        }
      }
      __syncthreads();
    }
  }
  if constexpr (!kFp8) {
    __syncthreads();   // (a share may have no round and so no barrier since the flag was cleared)
    if (__builtin_amdgcn_readfirstlane(deal->again) != 0) paged_again<kBF16, kQT>(a, deal, reinterpret_cast<float*>(smem));
  }
}

// Joins the parts of a unit (row, key head, head group: blockIdx.x), or writes the zeros
// of a row without keys.  A part is a few hundred bytes and there are two or three of
// it, or, where a long row is all there is, one a workgroup: `split` (1, 2, 4 or 8) of a
// workgroup's eight waves take a query head's parts in turn, each lane up to four dims, eight
// parts' loads in flight, and the waves' sums are added up through LDS in their order;
// the waves left over take the next query heads (blockIdx.y: groups of 8 / split).
constexpr int kJoinWaves = 8;
template <bool kBF16, int kQT>
__device__ __forceinline__ void paged_join(const PagedArgs& a, int split, float* lds, int32_t* again) {
  const int heads = a.kv_heads * a.head_groups;
  const int row = blockIdx.x / heads, unit = blockIdx.x - row * heads;
  const int kvh = unit / a.head_groups, hg = unit - kvh * a.head_groups;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int part0 = wave % split, r = blockIdx.y * (kJoinWaves / split) + wave / split;
  const bool in = r < min(16 * kQT, a.group - hg * 16 * kQT);
  const int32_t length = a.lengths[row], before = a.plan[row], all_rows = a.plan[a.batch];
  const KeySpan span = key_span(length, a.capacity, a.window, a.sinks);
  uint16_t* o = a.o + (int64_t)row * a.ldo + (int64_t)(kvh * a.group + hg * 16 * kQT + r) * a.d;
  if (span.tiles == 0) {
    if (in && part0 == 0)
      for (int c = lane; c < a.d; c += 64) o[c] = 0;
    return;
  }
  const Deal shares = make_deal(all_rows * heads, a.groups);
  const int32_t x0 = before * heads + unit * unit_size(span) + kUnitTiles;
  const int32_t g0 = deal_workgroup(shares, x0), g1 = deal_workgroup(shares, x0 + span.tiles - 1);
  if (g0 == g1) return;   // one workgroup had it whole
  auto at = [&](int32_t w) { return ((int64_t)(2 * w + (w == g0 ? 1 : 0)) * 16 * kQT + r); };
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sum = 0.0f, m = -__builtin_inff();
  for (int32_t w0 = g0 + part0; in && w0 <= g1; w0 += 8 * split) {
    float mi[8], li[8], v[8][4];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int32_t w = w0 + u * split;
      mi[u] = -__builtin_inff();
      li[u] = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[u][i] = 0.0f;
      if (w <= g1) {
        mi[u] = a.part_ml[at(w) * 2];
        li[u] = a.part_ml[at(w) * 2 + 1];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (lane + 64 * i < a.d) v[u][i] = a.part_o[at(w) * a.d + lane + 64 * i];
      }
    }
    float m_new = m;
#pragma unroll
    for (int u = 0; u < 8; ++u) m_new = __builtin_fmaxf(m_new, mi[u]);
    if (m_new == -__builtin_inff()) continue;   // no key seen so far
    const float alpha = exp2_fast(m - m_new);
    m = m_new;
    sum *= alpha;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= alpha;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float f = exp2_fast(mi[u] - m);   // (a part without keys: m_i = -inf, 0)
      sum += f * li[u];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] += f * v[u][i];
    }
  }
  float top = m, all = sum;
  if (split > 1) {
    if (lane == 0) {
      lds[2 * wave] = m;
      lds[2 * wave + 1] = sum;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) lds[2 * kJoinWaves + 256 * wave + 64 * i + lane] = acc[i];
    __syncthreads();
    if (part0 == 0) {
      for (int w = wave; w < wave + split; ++w) top = __builtin_fmaxf(top, lds[2 * w]);
      all = acc[0] = acc[1] = acc[2] = acc[3] = 0.0f;
      for (int w = wave; w < wave + split; ++w) {
        const float f = lds[2 * w] == -__builtin_inff() ? 0.0f : exp2_fast(lds[2 * w] - top);
        all += f * lds[2 * w + 1];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] += f * lds[2 * kJoinWaves + 256 * w + 64 * i + lane];
      }
    }
  }
  bool bad = false;   // (codes of e4m3 have no Inf)
  if (in && part0 == 0) {
    const float f = top == -__builtin_inff() ? 0.0f : a.v_scale / all;
    float z = 0.0f;   // (dims past the head's: zeros)
#pragma unroll
    for (int i = 0; i < 4; ++i) z = __builtin_fmaf(acc[i] * f, 0.0f, z);
    bad = !a.e4m3 && finite_sum(all) && __builtin_amdgcn_ballot_w64(!(z == 0.0f)) != 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (!bad && lane + 64 * i < a.d) o[lane + 64 * i] = kBF16 ? bf16_rne(acc[i] * f) : f16_rne(acc[i] * f);
  }
  if (a.e4m3) return;
  if (lane == 0) again[wave] = bad;
  __syncthreads();
  uint64_t waves = __builtin_amdgcn_ballot_w64(lane < kJoinWaves && again[lane & (kJoinWaves - 1)] != 0);
  for (; waves != 0; waves &= waves - 1) {
    const int head = blockIdx.y * (kJoinWaves / split) + __builtin_ctzll(waves) / split;
    paged_row<kBF16, kJoinWaves>(a, row, kvh, kvh * a.group + hg * 16 * kQT + head, span, lds);
  }
}

}  // namespace

#define SILE_PAGED_KERNEL(NAME, BF, F8, DP, EX, P16, QT, EU)                              \
  extern "C" __global__ __launch_bounds__(256, EU) void NAME(PagedArgs a) {               \
    __shared__ __attribute__((aligned(1024))) uint8_t smem[4 * Shape<DP>::kWaveB];        \
    __shared__ float ml[4 * 16 * 2];                                                      \
    __shared__ DealLds deal;                                                              \
    paged_attn<BF, F8, DP, EX, P16, QT>(a, smem, ml, &deal);                              \
  }
// d<D>: that head dimension; p<D>: any smaller one; s<D>: any up to it, pages below 16
// keys.  q<N>: N tiles of 16 query heads.
#define SILE_PAGED_TYPES(SUFFIX, DP, EX, P16, QT, EU)                                  \
  SILE_PAGED_KERNEL(sile_paged_attn_f16_##SUFFIX, false, false, DP, EX, P16, QT, EU)   \
  SILE_PAGED_KERNEL(sile_paged_attn_bf16_##SUFFIX, true, false, DP, EX, P16, QT, EU)   \
  SILE_PAGED_KERNEL(sile_paged_attn_f16_fp8_##SUFFIX, false, true, DP, EX, P16, QT, EU) \
  SILE_PAGED_KERNEL(sile_paged_attn_bf16_fp8_##SUFFIX, true, true, DP, EX, P16, QT, EU)
#define SILE_PAGED_DIM(DP, QT, EU)                         \
  SILE_PAGED_TYPES(d##DP##_q##QT, DP, true, true, QT, EU)  \
  SILE_PAGED_TYPES(p##DP##_q##QT, DP, false, true, QT, EU) \
  SILE_PAGED_TYPES(s##DP##_q##QT, DP, false, false, QT, EU)
SILE_PAGED_DIM(64, 1, 2)
SILE_PAGED_DIM(64, 2, 2)
SILE_PAGED_DIM(128, 1, 2)
SILE_PAGED_DIM(128, 2, 1)
SILE_PAGED_DIM(256, 1, 1)

#define SILE_PAGED_JOIN(NAME, BF, QT)                                             \
  extern "C" __global__ __launch_bounds__(64 * kJoinWaves) void NAME(PagedArgs a, int split) { \
    __shared__ float lds[(2 + 256) * kJoinWaves];                                 \
    __shared__ int32_t again[kJoinWaves];                                         \
    paged_join<BF, QT>(a, split, lds, again);                                         \
  }
SILE_PAGED_JOIN(sile_paged_attn_join_f16_q1, false, 1)
SILE_PAGED_JOIN(sile_paged_attn_join_bf16_q1, true, 1)
SILE_PAGED_JOIN(sile_paged_attn_join_f16_q2, false, 2)
SILE_PAGED_JOIN(sile_paged_attn_join_bf16_q2, true, 2)
