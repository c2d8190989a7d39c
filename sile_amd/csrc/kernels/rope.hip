// Rotary positions for the queries and keys of new tokens, the keys kept contiguous or
// stored, with the values, into a paged cache.
//
//   (a, b) -> magnitude * (a cos x - b sin x, b cos x + a sin x),   x = 2 pi frac(position * turns[j])
//
// for pair j < rot / 2 of every head: dims (j, rot / 2 + j), or (2 j, 2 j + 1); dims from rot on
// stay.  turns[j] is how often the pair turns a position, in 64 bits: the product is taken
// there, too, and only its fraction goes on, so that an angle is as good at position 2^30 (off
// by at most 2^-23 turns even there, 2^-33 at a million) as at 0, whatever scaling for long
// contexts the turns hold.  Angles and rotations are in fp32 and a result is rounded once, for
// an e4m3 cache once to the fp32 quotient and once to the code.
//
// Every element is read and written once and little is done to it, so memory bounds it, or at a
// few tokens the launch and three dependent reads (row, page table, page).  A workgroup takes
// whole tokens, or, of one token of many heads, 1024 items: its threads first issue the loads of
// up to four items (two vectors, of E pairs or of E dims and the E next), then work out each
// angle of the tokens once, for all heads, into LDS, and then rotate and store.
//
// Measured: 16382 tokens of 32 + 2 x 8 heads of 128, bf16, with append 90 us (4.5 TB/s), into e4m3 pages
// 97 (3.8 TB/s: the vector units are busy for 61 % of it); 5000 tokens of f16, 32 of 128 dims rotated, 38.5
// (4.3 TB/s); 64 tokens 5.  The loads are non-temporal: 96, 100 and 41 us without.  Rows that lie on no whole
// vectors go an element a load: 5000 tokens of 32 + 8 heads of 128, bf16, 24 us, from an odd element on, or of
// 126 dims, 71.
#include "common.h"
#include "e4m3.h"

using namespace sile;

namespace {

constexpr int kItems = 4;           // of a thread
constexpr int kMaxTokens = 16;      // of a workgroup
constexpr int kMaxAngles = 1024;    // of a workgroup: tokens * rot / 2

struct RopeArgs {
  const void *q, *k, *v;            // v: only into a cache
  void *q_out, *k_out, *v_out;      // k_out, v_out: the pages of a cache
  const int32_t *rows, *positions, *tables;   // rows NULL: token t is row t's
  const double* turns;
  int64_t tokens, ldq, ldk, ldv, ldqo, ldko, page_stride, ld_table, capacity;
  int32_t q_heads, kv_heads, d, rot, num_pages, page_shift, n_rows;
  int32_t per_group;                // tokens of a workgroup
  int32_t rot_items, head_items, items;   // of a head's rotated dims, of a head, of a token
  int32_t value_items;              // of a head of values
  int32_t past;                     // 1: the queries' stores past the caches
  int32_t head_shift, value_shift;  // log2 of head_items and value_items, -1: no powers of two
  int32_t k_exact, v_exact;         // 1: x * rcp is x / scale (the scale is a power of two)
  float inv_head, inv_items, inv_value;   // 1 / head_items, items, value_items
  float magnitude, k_scale, v_scale, k_rcp, v_rcp;
};

// cos and sin of 2 pi t, t in [0, 1): the quarter turn nearest to t and a rest of at most an
// eighth of a turn either way, whose Taylor sums leave less than 2^-29 (x = pi / 4: x^12 / 12!
// of the cosine, x^13 / 13! of the sine).
SILE_DEV void turn(double t, float* c, float* s) {
  const double quarter = __builtin_rint(4.0 * t);
  const float x = (float)((t - 0.25 * quarter) * 6.283185307179586477);
  const float z = x * x;
  const float sx = x * (1.0f + z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880 + z * (-1.0f / 39916800))))));
  const float cx = 1.0f + z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320 + z * (-1.0f / 3628800)))));
  const int k = (int)quarter & 3;
  const float a = (k & 1) ? sx : cx, b = (k & 1) ? cx : sx;
  *c = k == 1 || k == 2 ? -a : a;
  *s = k >= 2 ? -b : b;
}

template <int kType>   // sile_dtype
SILE_DEV float to_f32(const void* p, int i) {
  if constexpr (kType == 0) return reinterpret_cast<const float*>(p)[i];
  const uint16_t h = reinterpret_cast<const uint16_t*>(p)[i];
  return kType == 1 ? f16_to_f32(h) : bf16_to_f32(h);
}

// E elements as they lie in memory
template <int kBytes>
struct Raw {
  typedef uint32_t T __attribute__((ext_vector_type(kBytes / 4)));
};
template <>
struct Raw<4> {
  typedef uint32_t T;
};
template <>
struct Raw<2> {
  typedef uint16_t T;
};

// kType: f32, f16 or bf16 tokens; kCache: 0 keys as the queries, into memory, 1 into pages of
// the tokens' type, 2 into e4m3 pages; kE: elements of a vector; kPairs: pairs lie side by side.
template <int kType, int kCache, int kE, bool kPairs>
SILE_DEV void rope(const RopeArgs& a) {
  constexpr int kEs = kType == 0 ? 4 : 2;
  using V = typename Raw<kE * kEs>::T;
  __shared__ float cs[kMaxAngles], sn[kMaxAngles];
  __shared__ int64_t slot_off[kMaxTokens];   // elements to the token's slot of head 0, -1: it has none
  __shared__ uint8_t there[kMaxTokens];      // its position is one
  const int tid = threadIdx.x, h = a.rot / 2;
  for (int64_t t0 = (int64_t)blockIdx.x * a.per_group; t0 < a.tokens; t0 += (int64_t)gridDim.x * a.per_group) {
  const int tokens = (int)min((int64_t)a.per_group, a.tokens - t0);
  const int n = tokens * a.items;
  const int first = blockIdx.y * (256 * kItems);

  // n / by for n below 2^24 (inv: 1 / by, so the product's whole part is off by one at most)
  auto divide = [](int n, int by, float inv, int* rest) {
    int q = (int)((float)n * inv);
    int m = n - q * by;
    if (m < 0) {
      --q;
      m += by;
    } else if (m >= by) {
      ++q;
      m -= by;
    }
    *rest = m;
    return q;
  };
  // item i: token, head (queries', then keys', then values'), its two vectors' dims
  struct Item {
    int tok, head, o0, o1, pair;   // pair: of the first dim, -1 where nothing turns
    bool two;                      // the second vector is there
  };
  auto item = [&](int i) {
    Item m;
    int r = i, c;
    m.tok = a.per_group == 1 ? 0 : divide(i, a.items, a.inv_items, &r);
    const int turned = (a.q_heads + a.kv_heads) * a.head_items;
    m.two = true;
    if (r < turned) {
      if (a.head_shift >= 0) {
        m.head = r >> a.head_shift;
        c = r & (a.head_items - 1);
      } else {
        m.head = divide(r, a.head_items, a.inv_head, &c);
      }
    } else {   // a value's head has only dims that stay
      r -= turned;
      if (a.value_shift >= 0) {
        m.head = r >> a.value_shift;
        c = r & (a.value_items - 1);
      } else {
        m.head = divide(r, a.value_items, a.inv_value, &c);
      }
      m.head += a.q_heads + a.kv_heads;
      c += a.rot_items;
    }
    if (c < a.rot_items) {
      m.pair = c * kE;
      m.o0 = kPairs ? 2 * c * kE : c * kE;
      m.o1 = kPairs ? m.o0 + kE : h + c * kE;
    } else {
      m.pair = -1;
      m.o0 = (m.head >= a.q_heads + a.kv_heads ? 0 : a.rot) + 2 * (c - a.rot_items) * kE;
      m.o1 = m.o0 + kE;
      m.two = m.o1 < a.d;
    }
    return m;
  };
  // (offsets from the workgroup's first token fit 32 bits)
  const uint8_t* const qb = static_cast<const uint8_t*>(a.q) + t0 * a.ldq * kEs;
  const uint8_t* const kb = static_cast<const uint8_t*>(a.k) + t0 * a.ldk * kEs;
  const uint8_t* const vb = static_cast<const uint8_t*>(a.v) + t0 * a.ldv * kEs;
  uint8_t* const qo = static_cast<uint8_t*>(a.q_out) + t0 * a.ldqo * kEs;
  uint8_t* const ko = static_cast<uint8_t*>(a.k_out) + (kCache == 0 ? t0 * a.ldko * kEs : 0);
  const uint32_t ldq = (uint32_t)a.ldq, ldk = (uint32_t)a.ldk, ldv = (uint32_t)a.ldv, ldqo = (uint32_t)a.ldqo, ldko = (uint32_t)a.ldko;
  // key or value head of an item's head
  auto source = [&](const Item& m) -> const uint8_t* {
    if (m.head < a.q_heads) return qb + (m.tok * ldq + (uint32_t)m.head * a.d) * kEs;
    const int u = m.head - a.q_heads;
    if (u < a.kv_heads) return kb + (m.tok * ldk + (uint32_t)u * a.d) * kEs;
    return vb + (m.tok * ldv + (uint32_t)(u - a.kv_heads) * a.d) * kEs;
  };

  V raw[kItems][2];
#pragma unroll
  for (int u = 0; u < kItems; ++u) {
    const int i = first + u * 256 + tid;
    if (i >= n) break;
    const Item m = item(i);
    const uint8_t* p = source(m);
    raw[u][0] = __builtin_nontemporal_load(reinterpret_cast<const V*>(p + m.o0 * kEs));
    if (m.two) raw[u][1] = __builtin_nontemporal_load(reinterpret_cast<const V*>(p + m.o1 * kEs));
  }

  // ---- the tokens' angles, positions and slots ----
  for (int i = tid; i < tokens * h; i += 256) {
    const int tok = i / h, j = i - tok * h;
    const double x = (double)a.positions[t0 + tok] * a.turns[j];
    float c, s;
    turn(x - __builtin_floor(x), &c, &s);
    cs[i] = c * a.magnitude;
    sn[i] = s * a.magnitude;
  }
  if (tid < tokens) {
    const int32_t pos = a.positions[t0 + tid];
    there[tid] = pos >= 0;
    if constexpr (kCache != 0) {
      const int64_t row = a.rows ? a.rows[t0 + tid] : t0 + tid;
      int64_t off = -1;
      if (row >= 0 && row < a.n_rows && pos >= 0 && pos < a.capacity) {
        const int32_t id = a.tables[row * a.ld_table + (pos >> a.page_shift)];
        if ((uint32_t)id < (uint32_t)a.num_pages)
          off = (int64_t)id * a.page_stride + (int64_t)(pos & ((1 << a.page_shift) - 1)) * a.d;
      }
      slot_off[tid] = off;
    }
  }
  __syncthreads();

#pragma unroll
  for (int u = 0; u < kItems; ++u) {
    const int i = first + u * 256 + tid;
    if (i >= n) break;
    const Item m = item(i);
    if (!there[m.tok]) continue;
    const bool is_q = m.head < a.q_heads, is_v = m.head >= a.q_heads + a.kv_heads;
    const bool cached = kCache != 0 && !is_q;
    if (cached && slot_off[m.tok] < 0) continue;
    float x[2 * kE];   // first vector, second vector
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      x[e] = to_f32<kType>(&raw[u][0], e);
      x[kE + e] = m.two ? to_f32<kType>(&raw[u][1], e) : 0.0f;
    }
    if (m.pair >= 0) {
      const float* cp = cs + m.tok * h + m.pair;
      const float* sp = sn + m.tok * h + m.pair;
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        float& p = kPairs ? x[2 * e] : x[e];
        float& q = kPairs ? x[2 * e + 1] : x[kE + e];
        const float c = cp[e], s = sp[e], p0 = p, q0 = q;
        p = p0 * c - q0 * s;
        q = q0 * c + p0 * s;
      }
    }
    if (kCache == 2 && cached) {
      const int head = m.head - a.q_heads - (is_v ? a.kv_heads : 0);
      const float scale = is_v ? a.v_scale : a.k_scale, rcp = is_v ? a.v_rcp : a.k_rcp;
      uint8_t* to = static_cast<uint8_t*>(is_v ? a.v_out : a.k_out) + slot_off[m.tok] +
                    ((int64_t)head << a.page_shift) * a.d;
      if (is_v ? a.v_exact : a.k_exact) {
#pragma unroll
        for (int e = 0; e < 2 * kE; ++e) {
          const float y = x[e] * rcp;
          x[e] = y != y ? y : __builtin_amdgcn_fmed3f(y, -448.0f, 448.0f);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 2 * kE; ++e) x[e] = e4m3_in(x[e], scale, rcp);
      }
      if (kE == 8 && m.two && m.o1 == m.o0 + kE && (m.o0 & 15) == 0) {
        const u32x4 out = {e4m3_pack4(x), e4m3_pack4(x + 4), e4m3_pack4(x + 8), e4m3_pack4(x + 12)};
        __builtin_nontemporal_store(out, reinterpret_cast<u32x4*>(to + m.o0));
        continue;
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint8_t* w = to + (half ? m.o1 : m.o0);
        if (half && !m.two) break;
        if constexpr (kE == 8) {
          const u32x2 out = {e4m3_pack4(x + half * kE), e4m3_pack4(x + half * kE + 4)};
          __builtin_nontemporal_store(out, reinterpret_cast<u32x2*>(w));
        } else if constexpr (kE == 4) {
          __builtin_nontemporal_store(e4m3_pack4(x + half * kE), reinterpret_cast<uint32_t*>(w));
        } else {
          *w = e4m3_code(x[half]);
        }
      }
      continue;
    }
    uint8_t* to;
    if (is_q)
      to = qo + (m.tok * ldqo + (uint32_t)m.head * a.d) * kEs;
    else if (kCache == 0)
      to = ko + (m.tok * ldko + (uint32_t)(m.head - a.q_heads) * a.d) * kEs;
    else
      to = static_cast<uint8_t*>(is_v ? a.v_out : a.k_out) +
           (slot_off[m.tok] + ((int64_t)(m.head - a.q_heads - (is_v ? a.kv_heads : 0)) << a.page_shift) * a.d) * kEs;
    V out[2] = {raw[u][0], raw[u][1]};
    if (m.pair >= 0) {
#pragma unroll
      for (int e = 0; e < 2 * kE; ++e) {
        if constexpr (kType == 0)
          reinterpret_cast<float*>(&out[e / kE])[e % kE] = x[e];
        else
          reinterpret_cast<uint16_t*>(&out[e / kE])[e % kE] = kType == 1 ? f16_rne(x[e]) : bf16_rne(x[e]);
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (half && !m.two) break;
      V* w = reinterpret_cast<V*>(to + (half ? m.o1 : m.o0) * kEs);
      if (cached || a.past)
        __builtin_nontemporal_store(out[half], w);
      else
        *w = out[half];
    }
  }
  __syncthreads();   // (the next tokens' angles go to the same place)
  }
}

}  // namespace

#define SILE_ROPE(NAME, TYPE, CACHE, E)                                                        \
  extern "C" __global__ __launch_bounds__(256) void sile_rope_half_##NAME##_e##E(RopeArgs a) { \
    rope<TYPE, CACHE, E, false>(a);                                                            \
  }                                                                                            \
  extern "C" __global__ __launch_bounds__(256) void sile_rope_pairs_##NAME##_e##E(RopeArgs a) { \
    rope<TYPE, CACHE, E, true>(a);                                                             \
  }
SILE_ROPE(f32, 0, 0, 1)
SILE_ROPE(f32, 0, 0, 4)
#define SILE_ROPE16(CACHE, SUFFIX)    \
  SILE_ROPE(f16##SUFFIX, 1, CACHE, 1) \
  SILE_ROPE(f16##SUFFIX, 1, CACHE, 4) \
  SILE_ROPE(f16##SUFFIX, 1, CACHE, 8) \
  SILE_ROPE(bf16##SUFFIX, 2, CACHE, 1) \
  SILE_ROPE(bf16##SUFFIX, 2, CACHE, 4) \
  SILE_ROPE(bf16##SUFFIX, 2, CACHE, 8)
SILE_ROPE16(0, )
SILE_ROPE16(1, _cache)
SILE_ROPE16(2, _fp8)
