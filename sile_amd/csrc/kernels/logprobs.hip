// Log probabilities of given tokens, the entropy and the k most probable tokens of each row of
// logits, in one pass over them.
//
//   t_c = scale x_c     lse = log sum exp t_c     logp = t_target - lse
//   entropy = lse - sum p_c t_c                   top: the k largest x_c, ties to the lower c
//
// Memory bounds it: every logit is read once (16 bytes a load, two chunks of 8192 in flight) and
// kept in registers while a lane folds it into its own running (max m, sum l of p = 2^(c (x - m)),
// sum e of p (x - m)), c = scale log2 e.  The difference comes first, so that logits at the type's
// lowest value stay numbers; e keeps the entropy's digits where one token has nearly all the mass.  What the top ones cost beside that: one comparison of a chunk's
// largest value of a lane with the k-th best so far, and where one passes (rarely, after the
// first chunk) one of each element.  Candidates go to a list in LDS, and whoever has fewer than k
// before it stays.  The first chunk has no k-th best: the ceil(k / 4)-th largest of a wave's lanes, the
// least of the four waves', has k elements at or above it, and so has the k-th largest of any wave.
// Where more than the list holds are as good (rows of equal logits), the k best are looked for one
// at a time.
//
// Few long rows: a row's chunks go to several workgroups, and a second launch joins their parts.
#include <type_traits>

#include "common.h"

using namespace sile;

namespace {

constexpr int kThreads = 256;
constexpr int kElems = 32;                    // of a thread, a chunk
constexpr int kChunk = kThreads * kElems;
constexpr int kCap = 1024;                    // of the list
constexpr int kMaxTop = 64;

struct LogprobArgs {
  const void* x;
  const int32_t* targets;
  float *logp, *entropy, *top_logp;           // each may be NULL (top_logp with top_ids)
  int32_t* top_ids;
  float* part_sums;                           // [rows][parts][4]: m, l, e
  float* part_top;                            // [rows][parts][top]: values
  int32_t* part_ids;                          // their columns, -1: none
  int64_t ldx;
  int32_t rows, cols, top, parts, chunks, per_part;   // chunks of a row, of a part
  float scale, scale_log2;
  float floor;          // -512 / scale_log2: p is 0 there, and a factor of it finite
};

// 16 bytes at any multiple of the element's size
typedef uint32_t raw_f32 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t raw_16 __attribute__((ext_vector_type(4), aligned(2)));

struct List {
  float value[kCap + kMaxTop];
  int32_t column[kCap + kMaxTop];
  float kept_value[kMaxTop];
  int32_t kept_column[kMaxTop];
  int32_t added[3];     // entries that a chunk added, three chunks in turn
  float wave_least[4], wave_kth[4];
  float best_value[4];
  int32_t best_column[4];
  float sums[4][3];
};

template <int kType>   // sile_dtype
SILE_DEV float logit(const void* x, int64_t i) {
  if constexpr (kType == 0) return static_cast<const float*>(x)[i];
  const uint16_t h = static_cast<const uint16_t*>(x)[i];
  return kType == 1 ? f16_to_f32(h) : bf16_to_f32(h);
}

// (m, l, e) of two sets of elements, joined; m = -inf: an empty set, or one of probability 0
SILE_DEV void join_sums(const LogprobArgs& a, float& m, float& l, float& e, float m2, float l2, float e2) {
  const float top = __builtin_fmaxf(m, m2);
  if (top == -__builtin_inff()) {   // (sums of NaN stay)
    l += l2;
    e += e2;
    return;
  }
  const float d1 = m - top, d2 = m2 - top;   // <= 0, -inf of an empty set; NaN if top is +inf
  const float a1 = exp2_fast(d1 * a.scale_log2), a2 = exp2_fast(d2 * a.scale_log2);
  e = a1 * (e + l * __builtin_fmaxf(d1, a.floor)) + a2 * (e2 + l2 * __builtin_fmaxf(d2, a.floor));
  l = a1 * l + a2 * l2;
  m = top;
}

// The largest float, of 16 significant bits, that at least k of the wave's values reach; -inf
// where fewer than k are above -inf.  NaN counts as reaching nothing.
SILE_DEV float reached_by(float v, int k) {
  const uint32_t b = f32_bits(v);
  const bool is_number = v == v;
  const uint32_t key = !is_number ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;   // ordered
  uint32_t least = 0;
#pragma unroll
  for (int bit = 31; bit >= 16; --bit) {
    const uint32_t with = least | (1u << bit);
    if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(key >= with)) >= k) least = with;
  }
  // (keys of -inf: 0x007fffff, so a least of at most 0x007f0000 is below every number's)
  if (least <= 0x007f0000u) return -__builtin_inff();
  return bits_f32((least & 0x80000000u) ? least & 0x7fffffffu : ~least);
}

SILE_DEV bool before(float v, int32_t c, float w, int32_t d) { return v > w || (v == w && c < d); }

// Keeps the `top` first of the list's n entries (at most kCap + kMaxTop), in order, and returns how
// many they are; all threads.
SILE_DEV int keep_first(List* s, int n, int top) {
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const float v = s->value[i];
    const int32_t c = s->column[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += before(s->value[j], s->column[j], v, c) ? 1 : 0;
    if (rank < top) {
      s->kept_value[rank] = v;
      s->kept_column[rank] = c;
    }
  }
  __syncthreads();
  const int kept = min(n, top);
  if ((int)threadIdx.x < kept) {
    s->value[threadIdx.x] = s->kept_value[threadIdx.x];
    s->column[threadIdx.x] = s->kept_column[threadIdx.x];
  }
  __syncthreads();
  return kept;
}

// the sums of all threads, joined
SILE_DEV void all_sums(const LogprobArgs& a, List* s, float& m, float& l, float& e) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const float m2 = __shfl_xor(m, off), l2 = __shfl_xor(l, off), e2 = __shfl_xor(e, off);
    join_sums(a, m, l, e, m2, l2, e2);
  }
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    s->sums[wave][0] = m;
    s->sums[wave][1] = l;
    s->sums[wave][2] = e;
  }
  __syncthreads();
  m = s->sums[0][0];
  l = s->sums[0][1];
  e = s->sums[0][2];
#pragma unroll
  for (int w = 1; w < 4; ++w) join_sums(a, m, l, e, s->sums[w][0], s->sums[w][1], s->sums[w][2]);
}

// the workgroup's first of one (value, column) a thread; all threads have it
SILE_DEV void first_of_all(List* s, float& v, int32_t& c) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const float w = __shfl_xor(v, off);
    const int32_t d = __shfl_xor(c, off);
    if (before(w, d, v, c)) {
      v = w;
      c = d;
    }
  }
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    s->best_value[wave] = v;
    s->best_column[wave] = c;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w)
    if (before(s->best_value[w], s->best_column[w], v, c)) {
      v = s->best_value[w];
      c = s->best_column[w];
    }
  __syncthreads();
}

// the results of a row from its sums and its list
template <int kType>
SILE_DEV void finish(const LogprobArgs& a, const List* s, int row, int n, float m, float l, float e) {
  const int tid = threadIdx.x;
  const float log_l = logf(l);
  const bool none = m == -__builtin_inff() && l == 0.0f;   // every logit is -inf
  auto logp_of = [&](float x) {
    return none ? -__builtin_inff() : (x - m) * a.scale - log_l;
  };
  if (tid == 0) {
    if (a.logp) {
      const int32_t t = a.targets[row];
      a.logp[row] = t >= 0 && t < a.cols ? logp_of(logit<kType>(a.x, row * a.ldx + t)) : 0.0f;
    }
    if (a.entropy) {
      const float h = none ? 0.0f : log_l - e / l * a.scale;
      a.entropy[row] = h < 0.0f ? 0.0f : h;   // (by rounding; NaN stays)
    }
  }
  if (a.top_ids && tid < a.top) {
    a.top_logp[(int64_t)row * a.top + tid] = tid < n ? logp_of(s->value[tid]) : -__builtin_inff();
    a.top_ids[(int64_t)row * a.top + tid] = tid < n ? s->column[tid] : -1;
  }
}

template <int kType>
SILE_DEV void logprobs(const LogprobArgs& a, List* s) {
  constexpr int kPer = kType == 0 ? 4 : 8;    // elements of a load
  constexpr int kLoads = kElems / kPer;
  using raw_t = std::conditional_t<kType == 0, raw_f32, raw_16>;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
  const int c_first = part * a.per_part, c_last = min(c_first + a.per_part, a.chunks);
  const uint8_t* base = static_cast<const uint8_t*>(a.x) + (int64_t)row * a.ldx * (kType == 0 ? 4 : 2);
  if (tid == 0) s->added[0] = 0;
  const float c = a.scale_log2;

  u32x4 next[kLoads];
  // (loads need no alignment beyond the element's; a load that runs past the row's end is made
  // element by element, the rest as -inf)
  auto load = [&](int chunk) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int64_t at = (int64_t)chunk * kChunk + (i * kThreads + tid) * kPer;
      if (at + kPer <= a.cols) {
        next[i] = *reinterpret_cast<const raw_t*>(base + at * (kType == 0 ? 4 : 2));
      } else {
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = kType == 0 ? 0xff800000u : kType == 1 ? 0xfc00fc00u : 0xff80ff80u;
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          if (at + j < a.cols) {
            if constexpr (kType == 0) {
              w[j] = reinterpret_cast<const uint32_t*>(base)[at + j];
            } else {
              const uint32_t h = reinterpret_cast<const uint16_t*>(base)[at + j];
              w[j >> 1] = (j & 1) ? (w[j >> 1] & 0xffffu) | h << 16 : (w[j >> 1] & 0xffff0000u) | h;
            }
          }
        next[i] = w;
      }
    }
  };
  auto element = [](const u32x4* w, int i) {   // i: constant after unrolling
    const uint32_t u = w[i / kPer][kType == 0 ? i % kPer : (i % kPer) >> 1];
    if constexpr (kType == 0) return bits_f32(u);
    if constexpr (kType == 2) return bits_f32((i & 1) ? u & 0xffff0000u : u << 16);
    return f16_to_f32((uint16_t)(u >> (16 * (i & 1))));
  };

  float m = -__builtin_inff(), l = 0.0f, e = 0.0f;
  float kth = -__builtin_inff();   // the list's last, once it has `top` entries
  bool full = false;
  int had = 0;                     // entries of the list
  load(c_first);
  __syncthreads();
  for (int chunk = c_first; chunk < c_last; ++chunk) {
    u32x4 w[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) w[i] = next[i];
    if (chunk + 1 < c_last) load(chunk + 1);
    float most = -__builtin_inff();   // (NaN does not enter)
#pragma unroll
    for (int i = 0; i < kElems; ++i) most = __builtin_fmaxf(most, element(w, i));
    // the lane's sums
    const float m_new = __builtin_fmaxf(m, most);
    const float m_use = m_new == -__builtin_inff() ? 0.0f : m_new;
    if (m_new > m) {
      const float d = m - m_new, f = exp2_fast(d * c);
      e = f * (e + l * __builtin_fmaxf(d, a.floor));
      l *= f;
      m = m_new;
    }
#pragma unroll
    for (int i = 0; i < kElems; ++i) {
      const float d = element(w, i) - m_use;
      const float p = exp2_fast(d * c);
      l += p;
      e = __builtin_fmaf(p, __builtin_fmaxf(d, a.floor), e);
    }
    if (a.top == 0) continue;
    // ---- candidates ----
    float least = kth;
    if (!full) {
      const float quarter = reached_by(most, (a.top + 3) / 4), alone = reached_by(most, a.top);
      if (lane == 0) {
        s->wave_least[wave] = quarter;
        s->wave_kth[wave] = alone;
      }
      __syncthreads();
      float q = s->wave_least[0];
      least = s->wave_kth[0];
#pragma unroll
      for (int i = 1; i < 4; ++i) {
        q = __builtin_fminf(q, s->wave_least[i]);
        least = __builtin_fmaxf(least, s->wave_kth[i]);
      }
      least = __builtin_fmaxf(least, q);
    }
    const int32_t col0 = chunk * kChunk + tid * kPer;
    auto column = [&](int i) { return col0 + (i / kPer) * kThreads * kPer + i % kPer; };
    // (the list's entries are of lower columns: an equal one is behind them)
    auto enters = [&](float v) { return full ? v > least : v >= least && v > -__builtin_inff(); };
    const int turn = (chunk - c_first) % 3;
    if (tid == 0) s->added[turn == 2 ? 0 : turn + 1] = 0;   // (last read two chunks ago)
    if (__builtin_amdgcn_ballot_w64(enters(most)) != 0) {
#pragma unroll
      for (int i = 0; i < kElems; ++i) {
        const float v = element(w, i);
        if (enters(v)) {
          const int at = had + atomicAdd(&s->added[turn], 1);
          if (at < kCap + kMaxTop) {
            s->value[at] = v;
            s->column[at] = column(i);
          }
        }
      }
    }
    __syncthreads();
    int n = had + s->added[turn];
    if (n == had) continue;
    if (n > kCap + kMaxTop) {   // the chunk's best after (v, d), one at a time
      float v = __builtin_inff();
      int32_t d = -1;
      n = had;
      for (int k = 0; k < a.top; ++k) {
        float bv = -__builtin_inff();
        int32_t bc = 0x7fffffff;
#pragma unroll
        for (int i = 0; i < kElems; ++i) {
          const float x = element(w, i);
          if (before(v, d, x, column(i)) && before(x, column(i), bv, bc)) {
            bv = x;
            bc = column(i);
          }
        }
        first_of_all(s, bv, bc);
        if (bv == -__builtin_inff()) break;
        if (tid == 0) {
          s->value[n] = bv;
          s->column[n] = bc;
        }
        ++n;
        v = bv;
        d = bc;
      }
      __syncthreads();
    }
    had = keep_first(s, n, a.top);
    full = had == a.top;
    if (full) kth = s->value[a.top - 1];
  }
  all_sums(a, s, m, l, e);
  if (a.parts == 1) {
    finish<kType>(a, s, row, had, m, l, e);
    return;
  }
  const int64_t at = (int64_t)row * a.parts + part;
  if (tid == 0) *reinterpret_cast<f32x4*>(a.part_sums + 4 * at) = f32x4{m, l, e, 0.0f};
  if (tid < a.top) {
    a.part_top[at * a.top + tid] = tid < had ? s->value[tid] : -__builtin_inff();
    a.part_ids[at * a.top + tid] = tid < had ? s->column[tid] : -1;
  }
}

// Joins the parts of row blockIdx.x.
template <int kType>
SILE_DEV void logprobs_join(const LogprobArgs& a, List* s) {
  const int tid = threadIdx.x, row = blockIdx.x;
  const int64_t first = (int64_t)row * a.parts;
  float m = -__builtin_inff(), l = 0.0f, e = 0.0f;
  // a part that has `top` entries has that many at or above its last
  float least = -__builtin_inff();
  for (int p = tid; p < a.parts; p += kThreads) {
    const f32x4 w = *reinterpret_cast<const f32x4*>(a.part_sums + 4 * (first + p));
    join_sums(a, m, l, e, w[0], w[1], w[2]);
    if (a.top) least = __builtin_fmaxf(least, a.part_top[(first + p) * a.top + a.top - 1]);
  }
  all_sums(a, s, m, l, e);
  int had = 0;
  if (a.top) {
    int32_t none = 0;
    first_of_all(s, least, none);
    const int64_t entries = (int64_t)a.parts * a.top;
    int turn = 0;
    if (tid == 0) s->added[0] = 0;
    __syncthreads();
    for (int64_t e0 = 0; e0 < entries; e0 += kCap, turn = turn == 2 ? 0 : turn + 1) {
      if (tid == 0) s->added[turn == 2 ? 0 : turn + 1] = 0;
#pragma unroll
      for (int u = 0; u < kCap / kThreads; ++u) {
        const int64_t i = e0 + u * kThreads + tid;
        if (i >= entries) break;
        const float v = a.part_top[first * a.top + i];
        const int32_t c = a.part_ids[first * a.top + i];
        if (c >= 0 && v >= least) {
          const int at = had + atomicAdd(&s->added[turn], 1);
          s->value[at] = v;
          s->column[at] = c;
        }
      }
      __syncthreads();
      const int n = had + s->added[turn];
      if (n != had) had = keep_first(s, n, a.top);
    }
  }
  finish<kType>(a, s, row, had, m, l, e);
}

}  // namespace

#define SILE_LOGPROBS(NAME, TYPE)                                                                       \
  extern "C" __global__ __launch_bounds__(kThreads) void sile_logprobs_##NAME(LogprobArgs a) {          \
    __shared__ List s;                                                                                  \
    logprobs<TYPE>(a, &s);                                                                              \
  }                                                                                                     \
  extern "C" __global__ __launch_bounds__(kThreads) void sile_logprobs_join_##NAME(LogprobArgs a) {     \
    __shared__ List s;                                                                                  \
    logprobs_join<TYPE>(a, &s);                                                                         \
  }
SILE_LOGPROBS(f32, 0)
SILE_LOGPROBS(f16, 1)
SILE_LOGPROBS(bf16, 2)
