// Row norm by the root of the mean square, with the residual's addition before it and, if
// asked, an 8-bit output with scales behind it.
//
//   s = x + residual     y = s / sqrt(mean(s^2) + eps) * weight     (codes: y / scale)
//
// fp32 throughout: s goes into the norm unrounded and is stored rounded once, y is rounded once
// (to e4m3: to the fp32 quotient and then to the code).  A scale is the given one, or max |y| of
// each `group` columns over 448 (the maximum counts as at least 2^-100).  Where the sum of squares
// leaves fp32 (a value past 1.8e19; with eps below 2^-100 also where it is below 2^-80, and squares
// lose digits or vanish), it is taken again of values scaled by a power of two.
//
// Every element is read once and written once, so memory bounds it: a row stays in the
// registers of its threads between the sum and the result.  Rows of up to 512 columns take a
// wave each, others a workgroup; the weights are read once a workgroup, which goes on to
// further rows.
//
// Measured, bf16 with residual and stored sum: 8000 rows of 8192 100 us (5.2 TB/s), into e4m3 codes in groups
// 107 (4.3 TB/s: the codes' conversion is 36 % of the vector units' cycles), 64 rows of 8192 5; rows of
// 8191, which are no whole vectors, 136.  The form for any width reads an element a load, the row twice or,
// for a scale of its own, three times: 4000 rows of 16392 280 us, of 17000 into codes in groups of 1000 455.
#include "common.h"
#include "e4m3.h"

using namespace sile;

namespace {

constexpr float kTop = 448.0f;
constexpr float kLeast = 0x1p-100f;

struct NormArgs {
  const void *x, *residual, *weight;   // residual, weight: may be NULL
  void *sum, *y;                       // sum: may be NULL
  float* scales;                       // group > 0: [rows][cols / group]
  int64_t rows, ldx, ldr, lds, ldy;
  int32_t cols, group;
  float eps, inv_cols, scale, rcp;
};

template <int kType>   // sile_dtype
SILE_DEV float load1(const void* p, int64_t i) {
  if constexpr (kType == 0) return static_cast<const float*>(p)[i];
  const uint16_t h = static_cast<const uint16_t*>(p)[i];
  return kType == 1 ? f16_to_f32(h) : bf16_to_f32(h);
}
template <int kType>
SILE_DEV void store1(void* p, int64_t i, float v) {
  if constexpr (kType == 0)
    static_cast<float*>(p)[i] = v;
  else
    static_cast<uint16_t*>(p)[i] = kType == 1 ? f16_rne(v) : bf16_rne(v);
}

// rows may begin anywhere: whole vectors all the same, which the memory takes at any element
typedef uint32_t raw_16 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t raw_8 __attribute__((ext_vector_type(2), aligned(1)));

// 8 elements as they lie in memory, of which the first n are there (the others: zeros)
template <int kType>
struct Vec {
  u32x4 w[kType == 0 ? 2 : 1];
  SILE_DEV void load(const void* p, int64_t i, int n) {
    if (n >= 8) {
      const raw_16* q = reinterpret_cast<const raw_16*>(static_cast<const uint8_t*>(p) + i * (kType == 0 ? 4 : 2));
      w[0] = q[0];
      if constexpr (kType == 0) w[1] = q[1];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (kType == 0) {
          w[j >> 2][j & 3] = j < n ? static_cast<const uint32_t*>(p)[i + j] : 0u;
        } else {
          const uint32_t h = j < n ? static_cast<const uint16_t*>(p)[i + j] : 0u;
          w[0][j >> 1] = (j & 1) ? w[0][j >> 1] | h << 16 : h;
        }
      }
    }
  }
  SILE_DEV void unpack(float* f) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (kType == 0) {
        const uint32_t u = w[j >> 2][j & 3];
        f[j] = bits_f32(u);
      } else {
        const uint32_t u = w[0][j >> 1];
        if constexpr (kType == 2)
          f[j] = bits_f32((j & 1) ? u & 0xffff0000u : u << 16);
        else
          f[j] = f16_to_f32((uint16_t)(u >> (16 * (j & 1))));
      }
    }
  }
};
template <int kType>
SILE_DEV void store8(void* p, int64_t i, int n, const float* f) {
  if (n < 8) {
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (j < n) store1<kType>(p, i + j, f[j]);
  } else if constexpr (kType == 0) {
    raw_16* q = reinterpret_cast<raw_16*>(static_cast<float*>(p) + i);
    q[0] = raw_16{f32_bits(f[0]), f32_bits(f[1]), f32_bits(f[2]), f32_bits(f[3])};
    q[1] = raw_16{f32_bits(f[4]), f32_bits(f[5]), f32_bits(f[6]), f32_bits(f[7])};
  } else {
    raw_16 w;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = kType == 1 ? pack_f16x2(f[2 * j], f[2 * j + 1]) : pack_bf16x2(f[2 * j], f[2 * j + 1]);
    *reinterpret_cast<raw_16*>(static_cast<uint16_t*>(p) + i) = w;
  }
}

// the sum or maximum over the row's kThreads threads; lds: 2 * 16 floats, used in turn
template <int kThreads, bool kMax>
SILE_DEV float row_reduce(float v, float* lds) {
  v = kMax ? wave_max(v) : wave_sum(v);
  if constexpr (kThreads == 64) return v;
  constexpr int kWaves = kThreads / 64;
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = lds[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) r = kMax ? fmax_ordered(r, lds[w]) : r + lds[w];
  return r;
}

// max over groups of `lanes` lanes (a power of two up to 64)
SILE_DEV float lanes_max(float v, int lanes) {
  if (lanes >= 2) v = fmax_ordered(v, dpp<kDppXor1>(v));
  if (lanes >= 4) v = fmax_ordered(v, dpp<kDppXor2>(v));
  if (lanes >= 8) v = fmax_ordered(v, dpp<kDppHalfMirror>(v));
  if (lanes >= 16) v = fmax_ordered(v, dpp<kDppMirror>(v));
  if (lanes >= 32) v = fmax_ordered(v, swizzle_xor16(v));
  if (lanes >= 64) v = pair32_max(v);
  return v;
}

// Whether a sum of squares is outside fp32, and the power of two whose square brings the values back: a
// finite row's squares, of up to 2^30 columns, then add up to less than 2^126, and a row's least
// sum is 2^-138; a row with Inf stays Inf.
SILE_DEV bool out_of_range(float ss, float eps) {
  return ss == __builtin_inff() || (ss < 0x1p-80f && eps < 0x1p-100f);
}
SILE_DEV float back_in_range(float ss) { return ss > 1.0f ? 0x1p-40f : 0x1p40f; }
// a value that all lanes of a wave have, in a scalar register
SILE_DEV float scalar(float v) { return bits_f32((uint32_t)__builtin_amdgcn_readfirstlane((int)f32_bits(v))); }

SILE_DEV float scale_of(float top) { return __builtin_fmaxf(top, kLeast) / kTop; }
SILE_DEV float rcp_of(float scale) { return scale >= 0x1p-60f && scale <= 0x1p60f ? 1.0f / scale : 0.0f; }

// Columns in vectors of 8, the last one (kPart) perhaps in part: a row takes kThreads threads of kV vectors.
// kF8: codes out.  kWg: threads of the workgroup.  (With the parts' code in the way, 8000 x 8192 into codes
// took 125 us, 106 without; 8000 x 8191 through the form for any width 277, 136 here.)
template <int kType, bool kF8, int kThreads, int kV, int kWg, bool kPart>
SILE_DEV void norm_rows(const NormArgs& a) {
  __shared__ float lds[3][2][16];
  const int tid = threadIdx.x % kThreads, cols = a.cols;
  float w[kV][8];
  Vec<kType> wv[kV];
#pragma unroll
  for (int v = 0; v < kV; ++v)
    if (a.weight && 8 * (v * kThreads + tid) < cols) {
      const int c = 8 * (v * kThreads + tid);
      wv[v].load(a.weight, c, kPart ? cols - c : 8);
    }
  int turn = 0;
  constexpr int kRows = kWg / kThreads;
  const int groups = a.group > 0 ? cols / a.group : 0;
  for (int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / kThreads; r < a.rows;
       r += (int64_t)gridDim.x * kRows, turn ^= 1) {
    Vec<kType> xv[kV], rv[kV];
#pragma unroll
    for (int v = 0; v < kV; ++v) {
      const int c = 8 * (v * kThreads + tid);
      if (c < cols) {
        xv[v].load(a.x, r * a.ldx + c, kPart ? cols - c : 8);
        if (a.residual) rv[v].load(a.residual, r * a.ldr + c, kPart ? cols - c : 8);
      }
    }
    float s[kV][8], ss = 0.0f;
#pragma unroll
    for (int v = 0; v < kV; ++v) {
      const int c = 8 * (v * kThreads + tid);
      if (c < cols) {
        xv[v].unpack(s[v]);
        if (a.residual) {
          float f[8];
          rv[v].unpack(f);
#pragma unroll
          for (int j = 0; j < 8; ++j) s[v][j] += f[j];
        }
        if (a.sum) store8<kType>(a.sum, r * a.lds + c, kPart ? cols - c : 8, s[v]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) s[v][j] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = __builtin_fmaf(s[v][j], s[v][j], ss);
    }
    ss = scalar(row_reduce<kThreads, false>(ss, lds[0][turn]));
    float eps = a.eps, back = 1.0f;
    if (out_of_range(ss, eps)) {   // (all of the row's threads)
      back = back_in_range(ss);
      eps = eps * back * back * back * back;
      ss = 0.0f;
#pragma unroll
      for (int v = 0; v < kV; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          s[v][j] *= back;
          const float t = s[v][j] * back;
          ss = __builtin_fmaf(t, t, ss);
        }
      ss = row_reduce<kThreads, false>(ss, lds[2][turn]);
    }
    const float inv = back / __builtin_sqrtf(__builtin_fmaf(ss, a.inv_cols, eps));
    float top = 0.0f;
#pragma unroll
    for (int v = 0; v < kV; ++v) {
      const int c = 8 * (v * kThreads + tid);
      if (a.weight && c < cols) wv[v].unpack(w[v]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s[v][j] *= inv;
        if (a.weight && c < cols) s[v][j] *= w[v][j];
        if constexpr (kF8) top = __builtin_fmaxf(top, __builtin_fabsf(s[v][j]));
      }
    }
    if constexpr (!kF8) {
#pragma unroll
      for (int v = 0; v < kV; ++v) {
        const int c = 8 * (v * kThreads + tid);
        if (c < cols) store8<kType>(a.y, r * a.ldy + c, kPart ? cols - c : 8, s[v]);
      }
    } else {
      float scale = a.scale, rcp = a.rcp;
      if (a.group == cols) {
        scale = scale_of(row_reduce<kThreads, true>(top, lds[1][turn]));
        rcp = rcp_of(scale);
        if (tid == 0) a.scales[r] = scale;
      }
#pragma unroll
      for (int v = 0; v < kV; ++v) {
        const int c = 8 * (v * kThreads + tid);
        if (a.group != 0 && a.group != cols) {   // 8 to 512 columns: lanes of one wave
          float m = 0.0f;
#pragma unroll
          for (int j = 0; j < 8; ++j) m = __builtin_fmaxf(m, __builtin_fabsf(s[v][j]));
          scale = scale_of(lanes_max(m, a.group / 8));
          rcp = rcp_of(scale);
          if (c < cols && tid % (a.group / 8) == 0) a.scales[r * groups + c / 8 * 8 / a.group] = scale;
        }
        if (c < cols) {
          float f[8];
          // a group's own scale leaves no quotient past 448 but by a rounding, which the code takes back
          // (the remainder as q scale - s, whose zero is +0, and taken off: so a -0 stays one)
          if (a.group != 0 && rcp != 0.0f) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float q = s[v][j] * rcp;
              f[j] = __builtin_fmaf(-__builtin_fmaf(q, scale, -s[v][j]), rcp, q);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = e4m3_in(s[v][j], scale, rcp);
          }
          const raw_8 out = {e4m3_pack4(f), e4m3_pack4(f + 4)};
          uint8_t* y = static_cast<uint8_t*>(a.y) + r * a.ldy + c;
          if (!kPart || cols - c >= 8) {
            __builtin_nontemporal_store(out, reinterpret_cast<raw_8*>(y));
          } else {
#pragma unroll
            for (int j = 0; j < 7; ++j)
              if (j < cols - c) y[j] = (uint8_t)(out[j >> 2] >> (8 * (j & 3)));
          }
        }
      }
    }
  }
}

// Any width and group: a workgroup of 256 a row, which reads it once for the sum and
// once more for each pass behind it.  s is kept nowhere: `sum` may be x or the residual itself,
// so it is written by the last pass, each element by the thread that reads it there.
template <int kType, bool kF8>
SILE_DEV void norm_any(const NormArgs& a) {
  __shared__ float lds[3][2][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int turn = 0;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, turn ^= 1) {
    auto at = [&](int c) {
      const float v = load1<kType>(a.x, r * a.ldx + c);
      return a.residual ? v + load1<kType>(a.residual, r * a.ldr + c) : v;
    };
    float ss = 0.0f;
    for (int c = tid; c < a.cols; c += 256) {
      const float s = at(c);
      ss = __builtin_fmaf(s, s, ss);
    }
    ss = scalar(row_reduce<256, false>(ss, lds[0][turn]));
    float eps = a.eps, back = 1.0f;
    if (out_of_range(ss, eps)) {
      back = back_in_range(ss);
      eps = eps * back * back * back * back;
      ss = 0.0f;
      for (int c = tid; c < a.cols; c += 256) {
        const float t = at(c) * back * back;
        ss = __builtin_fmaf(t, t, ss);
      }
      ss = row_reduce<256, false>(ss, lds[2][turn]);
    }
    const float inv = back / __builtin_sqrtf(__builtin_fmaf(ss, a.inv_cols, eps));
    auto norm = [&](float s, int c) {
      if (back != 1.0f) s *= back;
      s *= inv;
      return a.weight ? s * load1<kType>(a.weight, c) : s;
    };
    auto put = [&](int c, float scale, float rcp) {
      const float s = at(c), y = norm(s, c);
      if (a.sum) store1<kType>(a.sum, r * a.lds + c, s);
      if constexpr (kF8)
        static_cast<uint8_t*>(a.y)[r * a.ldy + c] = e4m3_code(e4m3_in(y, scale, rcp));
      else
        store1<kType>(a.y, r * a.ldy + c, y);
    };
    if (!kF8 || a.group == 0) {
      for (int c = tid; c < a.cols; c += 256) put(c, a.scale, a.rcp);
    } else if (a.group == a.cols) {
      float top = 0.0f;
      for (int c = tid; c < a.cols; c += 256) top = __builtin_fmaxf(top, __builtin_fabsf(norm(at(c), c)));
      const float scale = scale_of(row_reduce<256, true>(top, lds[1][turn])), rcp = rcp_of(scale);
      if (tid == 0) a.scales[r] = scale;
      for (int c = tid; c < a.cols; c += 256) put(c, scale, rcp);
    } else {   // a wave a group
      const int groups = a.cols / a.group;
      for (int g = wave; g < groups; g += 4) {
        const int c0 = g * a.group, c1 = c0 + a.group;
        float top = 0.0f;
        for (int c = c0 + lane; c < c1; c += 64) top = __builtin_fmaxf(top, __builtin_fabsf(norm(at(c), c)));
        const float scale = scale_of(wave_max(top)), rcp = rcp_of(scale);
        if (lane == 0) a.scales[r * groups + g] = scale;
        for (int c = c0 + lane; c < c1; c += 64) put(c, scale, rcp);
      }
    }
  }
}

}  // namespace

// t<threads of a row>_v<vectors of a thread>, p: columns that are no whole vectors
// (Waves a SIMD: without the second bound the parts' form of 16 bits has registers for three, and 8000 x 8191
// takes 157 us for 136; the form for any width takes 730 for 454, 4000 x 17000 into codes in groups of 1000.
// Asked for four, the parts' forms into codes and of f32 would spill.)
#define SILE_NORM(NAME, TYPE, F8, T, V, WG)                                                         \
  extern "C" __global__ __launch_bounds__(WG) void sile_rmsnorm_##NAME##_t##T##_v##V(NormArgs a) {  \
    norm_rows<TYPE, F8, T, V, WG, false>(a);                                                        \
  }                                                                                                 \
  extern "C" __global__ __launch_bounds__(WG, TYPE == 0 || F8 ? 1 : 4) void sile_rmsnorm_##NAME##_t##T##_v##V##p(NormArgs a) { \
    norm_rows<TYPE, F8, T, V, WG, true>(a);                                                         \
  }
#define SILE_NORM_TYPES(NAME, TYPE, F8)                                                        \
  SILE_NORM(NAME, TYPE, F8, 64, 1, 256)                                                        \
  SILE_NORM(NAME, TYPE, F8, 256, 1, 256)                                                       \
  SILE_NORM(NAME, TYPE, F8, 256, 2, 256)                                                       \
  SILE_NORM(NAME, TYPE, F8, 256, 4, 256)                                                       \
  SILE_NORM(NAME, TYPE, F8, 1024, 2, 1024)                                                     \
  extern "C" __global__ __launch_bounds__(256, 8) void sile_rmsnorm_##NAME##_any(NormArgs a) { \
    norm_any<TYPE, F8>(a);                                                                     \
  }
SILE_NORM_TYPES(f32, 0, false)
SILE_NORM_TYPES(f16, 1, false)
SILE_NORM_TYPES(bf16, 2, false)
SILE_NORM_TYPES(f32_fp8, 0, true)
SILE_NORM_TYPES(f16_fp8, 1, true)
SILE_NORM_TYPES(bf16_fp8, 2, true)
