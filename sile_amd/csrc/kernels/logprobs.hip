// Log probabilities of given tokens, the entropy and the k most probable tokens of each row of
// logits, in one pass over them.
//
//   t_c = scale x_c     lse = log sum exp t_c     logp = t_target - lse
//   entropy = lse - sum p_c t_c                   top: the k largest x_c, ties to the lower c
//
// Memory bounds it: every logit is read once (16 bytes a load, two chunks of 8192 in flight) and
// kept in registers while a lane folds it into its own running (max m, sum l of p = 2^(c (x - m)),
// sum e of p (x - m)), c = scale log2 e.  The difference comes first, so that logits at the type's
// lowest value stay numbers.
//
// One token often has nearly all the mass, and what counts is then the rest: with u = l less the p = 1
// of one column that has the maximum, log l = log1p(u) and the entropy log1p(u) - scale e / (1 + u), of
// two terms of one sign, keep their digits however small u is (from l itself, a u of 1e-8 is gone and
// one of 1e-3 good to 1e-4).  A wave whose l is below 1.25 works its u out anew: the other lanes' l, and the
// columns of one lane that has the maximum again, a 64th of the wave's, without it; above, l - 1 has
// lost two or three bits at most.  (Of the rows of 32000 below a quarter has such a wave: without top
// ones 25.5 -> 27.5 us in bf16 and 41.2 -> 42 in f32; where every row has one 28 and 44.  In every wave
// it took 29.5 and 46, a sum of its own of what is below the maximum, in every lane, 30 and 44.)
//
// What the top ones cost beside that: every wave keeps the k best of its columns in order, an
// entry a lane, and a chunk's largest value of a lane is compared with the k-th; where one passes
// (rarely, after the first chunk) its elements are, and what passes is put in its place by a shift
// of the lanes behind it.  In the first chunk the ceil(k / 4)-th largest of the lanes' maxima, the
// least of the four waves', stands for the k-th best: k elements reach it.  After that no wave waits
// for another before its last column.  (Candidates of the workgroup in LDS, ranked by counting after
// each chunk: 77 us both below; sorted and merged by one wave: 24 and 82.)
//
// Few long rows: a row's chunks go to several workgroups, and a second launch joins their parts.
//
// The loads are non-temporal (below 54 -> 52, without top ones 45 -> 41 and 27 -> 25).
//
// Measured: 64 rows of 131072 in bf16, 20 top ones, 20 us (14 and the join 7; without top ones 9.5), one
// row 15; 2000 rows of 32001 in f32, 5 top ones, 53 - 55 (4.8 TB/s; without 42), of 32000 in bf16, 20 top
// ones, 50 (without 27).  What holds them is the latency of the list's steps, then instructions: a quarter
// of the time without top ones is exp2's.
#include <type_traits>

#include "common.h"

using namespace sile;

namespace {

constexpr int kThreads = 256;
constexpr int kElems = 32;                    // of a thread, a chunk
constexpr int kChunk = kThreads * kElems;
constexpr int kMaxTop = 64;
constexpr float kLowest = -3.402823466e38f;

struct LogprobArgs {
  const void* x;
  const int32_t* targets;
  float *logp, *entropy, *top_logp;           // each may be NULL (top_logp with top_ids)
  int32_t* top_ids;
  float* part_sums;                           // [rows][parts][4]: m, u, e
  float* part_top;                            // [rows][parts][top]: values
  int32_t* part_ids;                          // their columns
  int64_t ldx;
  int32_t rows, cols, top, parts, chunks, per_part;   // chunks of a row, of a part
  float scale, scale_log2;
  float floor;          // -512 / scale_log2: p is 0 there, and a factor of it finite
};

// 16 bytes at any multiple of the element's size
typedef uint32_t raw_f32 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t raw_16 __attribute__((ext_vector_type(4), aligned(2)));

struct List {
  float value[4][kMaxTop];      // the waves' lists; [0]: the workgroup's
  int32_t column[4][kMaxTop];
  float sums[4][3];
  float quarter[4];
};

template <int kType>   // sile_dtype
SILE_DEV float logit(const void* x, int64_t i) {
  if constexpr (kType == 0) return static_cast<const float*>(x)[i];
  const uint16_t h = static_cast<const uint16_t*>(x)[i];
  return kType == 1 ? f16_to_f32(h) : bf16_to_f32(h);
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

// ---- up to 64 entries in order, one a lane ----
struct Entry {
  float v;
  int32_t c;
};
SILE_DEV Entry no_entry() { return {-__builtin_inff(), 0x7fffffff}; }
// v of lane ^ kMask, by moves between lanes alone (through LDS each of a merge's steps, one after the
// other, waits some 100 cycles)
template <int kMask>
SILE_DEV int lane_xor(int v) {
  constexpr int kRowRor8 = 0x128, kQuadReverse = 0x1B;
  if constexpr (kMask == 1) return dpp_int<kDppXor1>(v);
  if constexpr (kMask == 2) return dpp_int<kDppXor2>(v);
  if constexpr (kMask == 4) return dpp_int<kQuadReverse>(dpp_int<kDppHalfMirror>(v));   // ^ 7 ^ 3
  if constexpr (kMask == 8) return dpp_int<kRowRor8>(v);
  const unsigned u = (unsigned)v;
  if constexpr (kMask == 16) {   // two copies trade odd and even rows: (0, 0, 2, 2) and (1, 1, 3, 3)
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned even = r[0], odd = r[1];
    return (int)((threadIdx.x & 16) ? even : odd);
  }
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const unsigned lo = r[0], hi = r[1];
  return (int)((threadIdx.x & 32) ? lo : hi);
}
template <int kMask>
SILE_DEV Entry lane_xor(const Entry& t) {
  return {bits_f32((uint32_t)lane_xor<kMask>((int)f32_bits(t.v))), lane_xor<kMask>(t.c)};
}
// the earlier of the lane's entry and that of lane ^ kMask in the lower lane, the later in the upper
template <int kMask>
SILE_DEV void exchange(Entry& t) {
  const Entry u = lane_xor<kMask>(t);
  if (before(u.v, u.c, t.v, t.c) == ((threadIdx.x & kMask) == 0)) t = u;
}
// puts (x, col), which all lanes have, in its place
SILE_DEV void insert(Entry& t, float x, int32_t col) {
  const uint64_t ahead = __builtin_amdgcn_ballot_w64(before(t.v, t.c, x, col));
  const int place = (int)__builtin_popcountll(ahead), lane = threadIdx.x & 63;
  constexpr int kWaveShr1 = 0x138;   // lane i takes lane i - 1's
  const float v = dpp<kWaveShr1>(t.v);
  const int32_t c = dpp_int<kWaveShr1>(t.c);
  t.v = lane == place ? x : lane > place ? v : t.v;
  t.c = lane == place ? col : lane > place ? c : t.c;
}
// The first 64 of two lists in order, of which the first `top` count: what of u precedes t's last of
// them is put in its place one by one, or, where that is more than a few, by a bitonic merge.
SILE_DEV void merge64(Entry& t, const Entry& u, int top) {
  const float kth = bits_f32((uint32_t)__builtin_amdgcn_readlane((int)f32_bits(t.v), top - 1));
  const int32_t kth_c = __builtin_amdgcn_readlane(t.c, top - 1);
  const int n = (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(before(u.v, u.c, kth, kth_c)));
  if (n <= 6) {
    for (int i = 0; i < n; ++i)
      insert(t, bits_f32((uint32_t)__builtin_amdgcn_readlane((int)f32_bits(u.v), i)), __builtin_amdgcn_readlane(u.c, i));
    return;
  }
  // u backwards: lane ^ 63, and a row's mirror is ^ 15
  const Entry m = {dpp<kDppMirror>(u.v), dpp_int<kDppMirror>(u.c)};
  const Entry w = lane_xor<32>(lane_xor<16>(m));
  if (before(w.v, w.c, t.v, t.c)) t = w;
  exchange<32>(t);
  exchange<16>(t);
  exchange<8>(t);
  exchange<4>(t);
  exchange<2>(t);
  exchange<1>(t);
}
// the waves' lists into one, in s->value[0]
SILE_DEV void merge_waves(List* s, Entry t, int top) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (wave > 0) {
    s->value[wave][lane] = t.v;
    s->column[wave][lane] = t.c;
  }
  __syncthreads();
  if (wave == 0) {
#pragma unroll 1
    for (int w = 1; w < 4; ++w) merge64(t, {s->value[w][lane], s->column[w][lane]}, top);
    s->value[0][lane] = t.v;
    s->column[0][lane] = t.c;
  }
  __syncthreads();
}

// the sums l and e of a maximum m as those of a maximum of `top`, which is at least m (both -inf:
// nothing to scale)
SILE_DEV void rescale(const LogprobArgs& a, float m, float& l, float& e, float top) {
  const float d = m == top ? 0.0f : m - top, f = exp2_fast(d * a.scale_log2);
  e = f * (e + l * __builtin_fmaxf(d, a.floor));
  l *= f;
}
// The same with u, l less the 1 of a maximum of its own: where m is less than `top` that one counts with
// the rest; where not, u stays as it is, and the function is 1.  (m = -inf, no column: u means nothing, and
// becomes 0 under a larger maximum.)
SILE_DEV float rescale_rest(const LogprobArgs& a, float m, float& u, float& e, float top) {
  if (m == top) return 1.0f;
  u += 1.0f;
  rescale(a, m, u, e, top);
  return 0.0f;
}
// the waves' sums (m, u, e), joined
SILE_DEV void waves_sums(const LogprobArgs& a, List* s, float& m, float& u, float& e) {
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    s->sums[wave][0] = m;
    s->sums[wave][1] = u;
    s->sums[wave][2] = e;
  }
  __syncthreads();
  m = __builtin_fmaxf(__builtin_fmaxf(s->sums[0][0], s->sums[1][0]), __builtin_fmaxf(s->sums[2][0], s->sums[3][0]));
  u = e = 0.0f;
  float largest = -1.0f;   // waves that have the maximum, but one
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    float uw = s->sums[w][1], ew = s->sums[w][2];
    largest += rescale_rest(a, s->sums[w][0], uw, ew, m);
    u += uw;
    e += ew;
  }
  u += largest;
}

// the logit of the row's target, asked for ahead of its use; thread 0
template <int kType>
SILE_DEV float target_logit(const LogprobArgs& a, int row, bool* there) {
  *there = false;
  if (threadIdx.x != 0 || !a.logp) return 0.0f;
  const int32_t t = a.targets[row];
  *there = t >= 0 && t < a.cols;
  return *there ? logit<kType>(a.x, row * a.ldx + t) : 0.0f;
}
// the results of a row from its sums and the list
SILE_DEV void finish(const LogprobArgs& a, const List* s, int row, float target, bool there, float m, float u, float e) {
  const int tid = threadIdx.x;
  const float log_l = log1pf(u);
  const bool none = m == -__builtin_inff() && u == u;   // every logit is -inf
  auto logp_of = [&](float x) { return none ? -__builtin_inff() : (x - m) * a.scale - log_l; };
  if (tid == 0) {
    if (a.logp) a.logp[row] = there ? logp_of(target) : 0.0f;
    if (a.entropy) a.entropy[row] = none ? 0.0f : log_l - e / (1.0f + u) * a.scale;
  }
  if (a.top_ids && tid < a.top) {
    const float v = s->value[0][tid];
    const bool is = v > -__builtin_inff();
    a.top_logp[(int64_t)row * a.top + tid] = is ? logp_of(v) : -__builtin_inff();
    a.top_ids[(int64_t)row * a.top + tid] = is ? s->column[0][tid] : -1;
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
  bool there = false;
  const float target = a.parts == 1 ? target_logit<kType>(a, row, &there) : 0.0f;
  const float c = a.scale_log2;

  u32x4 next[kLoads];
  // (loads need no alignment beyond the element's; what the last one of a row would read past its end
  // comes behind the chunks)
  const int whole = a.cols / kPer * kPer;
  auto load = [&](int chunk) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int64_t at = (int64_t)chunk * kChunk + (i * kThreads + tid) * kPer;
      constexpr uint32_t kNone = kType == 0 ? 0xff800000u : kType == 1 ? 0xfc00fc00u : 0xff80ff80u;   // -inf
      u32x4 w = {kNone, kNone, kNone, kNone};
      if (at < whole) w = __builtin_nontemporal_load(reinterpret_cast<const raw_t*>(base + at * (kType == 0 ? 4 : 2)));
      next[i] = w;
    }
  };
  auto element = [](const u32x4* w, int i) {   // i: constant after unrolling
    const uint32_t u = w[i / kPer][kType == 0 ? i % kPer : (i % kPer) >> 1];
    if constexpr (kType == 0) return bits_f32(u);
    if constexpr (kType == 2) return bits_f32((i & 1) ? u & 0xffff0000u : u << 16);
    return f16_to_f32((uint16_t)(u >> (16 * (i & 1))));
  };

  float m = -__builtin_inff(), l = 0.0f, e = 0.0f;
  const int few = max((a.top + 3) / 4, 1);
  Entry best = no_entry();
  float least = kLowest;           // what does not reach it, or is -inf, cannot be among the wave's best
  float kth = -__builtin_inff();   // the list's last, -inf while it has fewer than `top`
  int32_t kth_c = 0x7fffffff;
  auto grow = [&](float v) {   // the lane's maximum is at least v
    if (v > m) {
      const float d = m - v, f = exp2_fast(d * c);
      e = f * (e + l * __builtin_fmaxf(d, a.floor));
      l *= f;
      m = v;
    }
  };
  auto add = [&](float v, float m_use) {
    const float d = v - m_use, p = exp2_fast(d * c);
    l += p;
    e = __builtin_fmaf(p, __builtin_fmaxf(d, a.floor), e);
  };
  auto place = [&](float v, int32_t col) {   // the lanes' values into the list, where they belong there
    uint64_t in = __builtin_amdgcn_ballot_w64(v >= least && before(v, col, kth, kth_c));
    for (; in != 0; in &= in - 1) {
      const int from = __builtin_ctzll(in);
      insert(best, bits_f32((uint32_t)__builtin_amdgcn_readlane((int)f32_bits(v), from)),
             __builtin_amdgcn_readlane(col, from));
    }
    kth = bits_f32((uint32_t)__builtin_amdgcn_readlane((int)f32_bits(best.v), a.top - 1));
    kth_c = __builtin_amdgcn_readlane(best.c, a.top - 1);
    least = __builtin_fmaxf(least, kth);
  };
  load(c_first);
  for (int chunk = c_first; chunk < c_last; ++chunk) {
    u32x4 w[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) w[i] = next[i];
    if (chunk + 1 < c_last) load(chunk + 1);
    float most = -__builtin_inff();   // (NaN does not enter)
#pragma unroll
    for (int i = 0; i < kElems; ++i) most = __builtin_fmaxf(most, element(w, i));
    // the lane's sums
    grow(most);
    const float m_use = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < kElems; ++i) add(element(w, i), m_use);
    if (a.top == 0) continue;
    // ---- the wave's best ----
    // (what every wave has ceil(top / 4) of, the workgroup has top of; later than it was written will do)
    if (chunk == c_first) {
      const float some = reached_by(most, few);
      if (lane == 0) s->quarter[wave] = some;
      __syncthreads();
    }
    float all = __builtin_inff();
#pragma unroll
    for (int i = 0; i < 4; ++i)
      all = __builtin_fminf(all, __hip_atomic_load(&s->quarter[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
    if (chunk == c_first && all == -__builtin_inff()) all = reached_by(most, a.top);
    least = __builtin_fmaxf(least, all);
    if (__builtin_amdgcn_ballot_w64(most >= least) == 0) continue;
    // a lane's elements that reach it, as bits; they are loaded again, one of each lane at a time (with
    // the insertion behind each of the 32 its code was 10 KB, fetched anew in each launch)
    uint32_t passed = 0;
#pragma unroll
    for (int i = 0; i < kElems; ++i) passed |= element(w, i) >= least ? 1u << i : 0u;
    while (__builtin_amdgcn_ballot_w64(passed != 0) != 0) {
      const int i = __builtin_ctz(passed | 0x80000000u);
      const int32_t col = chunk * kChunk + tid * kPer + (i / kPer) * kThreads * kPer + i % kPer;
      const float v = passed != 0 ? logit<kType>(base, col) : -__builtin_inff();
      passed &= passed - 1;
      place(v, col);
    }
    const float some = bits_f32((uint32_t)__builtin_amdgcn_readlane((int)f32_bits(best.v), few - 1));
    if (lane == 0 && chunk != c_first) __hip_atomic_store(&s->quarter[wave], some, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  }
  float tail = -__builtin_inff();
  if (part == a.parts - 1 && whole < a.cols && wave == 0) {   // the row's last few: a lane one
    if (tid < a.cols - whole) tail = logit<kType>(base, whole + tid);
    grow(tail);
    add(tail, m == -__builtin_inff() ? 0.0f : m);
    if (a.top != 0) place(tail, whole + tid);
  }
  // ---- the wave's sums, its maximum's 1 apart ----
  const float top_m = wave_max(m);
  rescale(a, m, l, e, top_m);
  float u = wave_sum(l) - 1.0f;
  if (top_m > -__builtin_inff() && !(u >= 0.25f)) {
    // the columns of a lane that has the maximum again, but for the first at it (m is no NaN)
    const int owner = __builtin_ctzll(__builtin_amdgcn_ballot_w64(m == top_m));
    u = lane == owner ? 0.0f : l;
    bool found = false;
    const int n = (c_last - c_first) * kElems, first = (wave * 64 + owner) * kPer;
    for (int j0 = 0; j0 < n; j0 += 256) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = j0 + 64 * i + lane;
        const int64_t at = (int64_t)(c_first + j / kElems) * kChunk + first + j % kElems / kPer * (kThreads * kPer) + j % kPer;
        v[i] = j < n && at < whole ? logit<kType>(base, at) : -__builtin_inff();
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint64_t at_top = __builtin_amdgcn_ballot_w64(v[i] == top_m);
        const bool out = !found && at_top != 0 && lane == __builtin_ctzll(at_top);
        found |= at_top != 0;
        const float d = v[i] - top_m;   // (of a +inf NaN, also where it is left out)
        u += out ? d : exp2_fast(d * c);
      }
    }
    const float d = bits_f32((uint32_t)__builtin_amdgcn_readlane((int)f32_bits(tail), owner)) - top_m;
    if (lane == 0) u += found ? exp2_fast(d * c) : d;
    u = wave_sum(u);
  }
  e = wave_sum(e);
  m = top_m;
  if (a.top != 0) merge_waves(s, best, a.top);
  waves_sums(a, s, m, u, e);
  if (a.parts == 1) {
    finish(a, s, row, target, there, m, u, e);
    return;
  }
  const int64_t at = (int64_t)row * a.parts + part;
  if (tid == 0) *reinterpret_cast<f32x4*>(a.part_sums + 4 * at) = f32x4{m, u, e, 0.0f};
  if (tid < a.top) {
    a.part_top[at * a.top + tid] = s->value[0][tid];
    a.part_ids[at * a.top + tid] = s->column[0][tid];
  }
}

// Joins the parts of row blockIdx.x.
template <int kType>
SILE_DEV void logprobs_join(const LogprobArgs& a, List* s) {
  const int tid = threadIdx.x, row = blockIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t first = (int64_t)row * a.parts;
  bool there;
  const float target = target_logit<kType>(a, row, &there);
  float m = -__builtin_inff(), u = 0.0f, e = 0.0f;
  for (int p = tid; p < a.parts; p += kThreads) {
    const f32x4 w = *reinterpret_cast<const f32x4*>(a.part_sums + 4 * (first + p));
    const float top = __builtin_fmaxf(m, w[0]);
    float uw = w[1], ew = w[2];
    const float both = rescale_rest(a, m, u, e, top) * rescale_rest(a, w[0], uw, ew, top);
    m = top;
    u += uw + both;
    e += ew;
  }
  if (a.top) {
    // a part's list is in order; the next one is on its way
    auto list = [&](int p) {
      Entry some = no_entry();
      if (lane < a.top && p < a.parts) some = {a.part_top[(first + p) * a.top + lane], a.part_ids[(first + p) * a.top + lane]};
      return some;
    };
    Entry t = list(wave), next = list(wave + 4);
#pragma unroll 1
    for (int p = wave + 4; p < a.parts; p += 4) {
      const Entry ahead = list(p + 4);
      merge64(t, next, a.top);
      next = ahead;
    }
    merge_waves(s, t, a.top);
  }
  const float top_m = wave_max(m);
  const float own = rescale_rest(a, m, u, e, top_m);
  u = wave_sum(u) + (wave_sum(own) - 1.0f);
  e = wave_sum(e);
  m = top_m;
  waves_sums(a, s, m, u, e);
  finish(a, s, row, target, there, m, u, e);
}

}  // namespace

#define SILE_LOGPROBS(NAME, TYPE)                                                                       \
  extern "C" __global__ __launch_bounds__(kThreads, 4) void sile_logprobs_##NAME(LogprobArgs a) {          \
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
