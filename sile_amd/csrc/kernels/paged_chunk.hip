// Attention of the new tokens of many sequences over a paged key-value cache: pieces of prompts and
// single tokens together.
//
//   o[t][h] = softmax_j(q[t][h] . k_j * scale) v_j over the keys j <= p (the token's position),
//   j > p - window or j < sinks
//
// 4 d flop for each pair of a query row and a key: with many tokens the matrix cores' work, with few
// the keys' and values' way from HBM.  A tile is 128 query rows of one key head, its tokens times the
// query heads that share the key head (a piece of 32 tokens under 4 heads, or 25 drafts under 5), 32 a wave;
// for every row of it a key is read once.  The pipeline is that of the windowed attention
// (flash_window.hip): K and V blocks of 32 or 64 keys go to LDS, two stages of each;
// iteration j issues S_{j+1} = K_{j+1} Q^T and O^T += V_{j-1}^T P_{j-1} on the matrix cores beside
// the online softmax of S_j, whose accumulator holds one query row a lane; V^T is read with
// ds_read_b64_tr_b16.  What the pages and the list of sequences change:
//
//  * A wave's LDS-DMA covers 2 to 8 keys; the buffer resource over them is built by scalar
//    instructions from the page's number, and ends at the sequence's last key or is empty where the
//    page does not exist, so that nothing past them is read (it arrives as zeros).  The page
//    numbers are loaded two iterations ahead of it.  Pages smaller than that, and e4m3 codes, which
//    are widened, exactly, go through registers.
//  * The tiles of all sequences and key heads are one list of key blocks, dealt in equal shares to
//    a fixed grid, with the lengths known only on the device: every workgroup works the list's sums out
//    for itself.  A tile that one workgroup has whole is written by it; the others leave (m, l, O) in
//    fp32 in the workspace, at most two a workgroup, and a second launch joins them.
//  * Workgroups of one XCD take a contiguous run of the list, key head by key head, so that tiles of a
//    sequence read its keys from that XCD's L2.
//  * Rows past the tile's last and waves without any compute nothing and store nothing.
//  * A tile of at most 32 rows (single tokens, drafts) has another code: each wave takes every fourth key block
//    for all of its rows, with no barrier, and the four results are joined in LDS.
//  * A row whose result is not finite (Inf or NaN in a masked key's V makes it so: 0 times it) is
//    taken again by the workgroup over its seen keys, in fp32.
//
// The probabilities enter the product in 16 bits (half a step, 2^-8 of each in bf16, 2^-11 in f16,
// their sum is of the rounded ones); f16 ones carry a factor 2^7 beside the up to 2^8 that the lazy
// maximum allows, so that those far below the maximum keep their bits.
//
// Measured, 32 query heads of 128 over 8 key heads: 2048 tokens behind 30000 keys 1.13 to 1.2 ms by card (870 to 920
// TFLOP/s: the matrix cores are busy for 41 % of the cycles, a third of the waves' cycles waits to issue and a
// quarter for data, and their power leaves 2.0 GHz of 2.4), 8192 from none 0.71 ms; 32 pieces of 8 tokens over up
// to 8192 keys 115 us (4.8 TB/s), as e4m3 codes 86 us; 1 piece of 4 over 300 13 us.  The kernels spill 70 to 290
// scalar registers into vector ones, the e4m3 forms at 256 dims also 21 vector registers to memory.
#include <type_traits>

#include "common.h"
#include "chunk_plan.h"

using namespace sile;

namespace {

constexpr float kRescaleLog2 = 8.0f;  // lazy-rescale threshold: p <= 2^8
constexpr float kLowest = -3.402823466e38f;

template <bool kBF16>
constexpr float kLift = kBF16 ? 0.0f : 7.0f;
// fast-path limit on one lane's block sum of p: below it every p is <= 2^8 (lifted)
template <bool kBF16>
constexpr float kBlockSumLimit = kBF16 ? 256.0f : 32768.0f;

template <bool kBF16>
SILE_DEV f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (kBF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <bool kBF16>
SILE_DEV uint32_t pack2(float lo, float hi) {
  return kBF16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
}

// lo + hi of the packed 16-bit pair, added to acc
template <bool kBF16>
SILE_DEV float pair_sum(uint32_t pk, float acc) {
  if constexpr (kBF16)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pk),
                                           __builtin_bit_cast(bf16x2, 0x3f803f80u), acc, false);
  else
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pk),
                                  f16x2{(_Float16)1.0f, (_Float16)1.0f}, acc, false);
}

// four e4m3 codes as four 16-bit values, exactly
template <bool kBF16>
SILE_DEV u32x2 widen4(uint32_t w) {
  if constexpr (kBF16)
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true))};
  else
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true))};
}

struct ChunkArgs {
  const uint16_t* q;
  const uint8_t* k;
  const uint8_t* v;
  uint16_t* o;
  const int32_t* starts;
  const int32_t* tables;
  const int32_t* lengths;
  ChunkRec* plan;        // workspace: of a key head's tiles, then all of its blocks
  float* parts;          // workspace: [slots][4 waves][4 d-tiles x 4 + 1][64 lanes][4]
  int64_t ldq, ldo, page_stride, ld_table;
  ChunkShape shape;
  int32_t kv_heads, d, num_pages, page_shift;
  int32_t tiles;         // of a key head, empty ones counted
  int32_t groups;
  int32_t direct;        // 1: a workgroup a unit, no shares and no parts
  uint32_t q_and, q_xor; // the sign, or a zero, of the scale
  float scale_log2, v_scale;
};

struct ChunkLds {
  int64_t wave_sum[4];
  int32_t tile, before, rows;   // the share's first tile
  int32_t x, x1, base;   // the workgroup's share, for chunk_again
  int32_t first_tile, kvh, seq;
  int32_t again;         // rows that are not finite: 1 in a tile of its own, in the join their bits
  float ml[4][2];
  float acc[4][256];
};

// 8 elements of the cache at p, in fp32
template <bool kBF16, bool kFp8>
SILE_DEV void load8(const uint8_t* p, float* f) {
  u32x4 w;
  if constexpr (kFp8) {
    const u32x2 c = *reinterpret_cast<const u32x2*>(p);
    const u32x2 lo = widen4<kBF16>(c[0]), hi = widen4<kBF16>(c[1]);
    w = u32x4{lo[0], lo[1], hi[0], hi[1]};
  } else {
    w = *reinterpret_cast<const u32x4*>(p);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint16_t h = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
    f[j] = kBF16 ? bf16_to_f32(h) : f16_to_f32(h);
  }
}

// One query row, at position p, of sequence `seq`, by the workgroup, in fp32 and over the seen
// keys only.  A wave takes every fourth 64 keys: a lane a key's score, then 8 dims of 2 keys at a
// time; the waves' sums are joined through LDS.  Its dims dim0 .. dim1 - 1 are stored.
template <bool kBF16, bool kFp8>
SILE_DEV void chunk_row(const ChunkArgs& a, int32_t seq, int kvh, int32_t p, const uint16_t* q, uint16_t* o,
                        int dim0, int dim1, ChunkLds* lds) {
  constexpr int kEs = kFp8 ? 1 : 2;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), d = a.d;
  const KeySpan span = key_span(p + 1, a.shape.capacity, a.shape.window, a.shape.sinks);
  const int32_t* table = a.tables + (int64_t)seq * a.ld_table;
  // lanes 0 .. 31 and 32 .. 63 a key each, 8 dims a lane
  const int half = lane >> 5, dim = 8 * (lane & 31);
  float acc[8], m = kLowest, l = 0.0f;
  bool any = false;   // a key is there: its page may not be
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = 0.0f;
  const int64_t n = (int64_t)span.sink_end + span.len - span.first;
  for (int64_t i0 = 64 * wave; i0 < n; i0 += 256) {
    const int64_t i = min(i0 + lane, n - 1);
    const int key = (int)(i < span.sink_end ? i : i - span.sink_end + span.first);
    const int32_t id = table[key >> a.page_shift];
    const bool ok = i0 + lane < n && (uint32_t)id < (uint32_t)a.num_pages;
    const uint64_t seen = __builtin_amdgcn_ballot_w64(ok);
    if (seen == 0) continue;
    any = true;
    // (a key that is not seen: page 0's row of its slot, which is there)
    const int64_t off = ((int64_t)(ok ? id : 0) * a.page_stride +
                         (((int64_t)kvh << a.page_shift) + (key & ((1 << a.page_shift) - 1))) * d) * kEs;
    float s = 0.0f;
    for (int c = 0; c < d; c += 8) {
      float qf[8], kf[8];
      const u32x4 qw = *reinterpret_cast<const u32x4*>(q + c);
      load8<kBF16, kFp8>(a.k + off + c * kEs, kf);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint16_t h = (uint16_t)(((qw[j >> 1] & a.q_and) ^ a.q_xor) >> (16 * (j & 1)));
        qf[j] = kBF16 ? bf16_to_f32(h) : f16_to_f32(h);
        s += qf[j] * kf[j];
      }
    }
    s *= a.scale_log2;
    // a seen score counts as at least the lowest float in the max: scores that are all -inf
    // give 0 / 0, a row without keys zeros
    const float m_new = __builtin_fmaxf(m, wave_max(ok && s == s ? s : kLowest));
    const float alpha = exp2_fast(m - m_new), pr = ok ? exp2_fast(s - m_new) : 0.0f;
    m = m_new;
    l = l * alpha + wave_sum(pr);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] *= alpha;
    for (int k0 = 0; k0 < 64; k0 += 2) {
      const int from = k0 + half;
      const float pu = __shfl(pr, from);
      const int64_t at = __shfl((long long)off, from);
      if (dim < d && ((seen >> from) & 1)) {
        float vf[8];
        load8<kBF16, kFp8>(a.v + at + dim * kEs, vf);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += pu * vf[j];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float other = __shfl_xor(acc[j], 32);
    if (half == 0) lds->acc[wave][dim + j] = acc[j] + other;
  }
  if (lane == 0) {
    lds->ml[wave][0] = any ? m : -__builtin_inff();
    lds->ml[wave][1] = l;
  }
  __syncthreads();
  if ((int)threadIdx.x < d) {
    float top = kLowest, sum = 0.0f, r = 0.0f;
    any = false;
    for (int w = 0; w < 4; ++w) {
      top = __builtin_fmaxf(top, lds->ml[w][0]);
      any |= lds->ml[w][0] > -__builtin_inff();
    }
    for (int w = 0; w < 4; ++w) {
      const float f = exp2_fast(lds->ml[w][0] - top);
      sum += f * lds->ml[w][1];
      r += f * lds->acc[w][threadIdx.x];
    }
    r = any ? r * (a.v_scale / sum) : 0.0f;
    if ((int)threadIdx.x >= dim0 && (int)threadIdx.x < dim1) o[threadIdx.x] = kBF16 ? bf16_rne(r) : f16_rne(r);
  }
  __syncthreads();
}

// The rows of this workgroup's whole tiles whose results are not finite, again.  Behind its units and
// from what stands in LDS, so that they keep nothing for it.
template <bool kBF16, bool kFp8>
SILE_DEV void chunk_again(const ChunkArgs& a, ChunkLds* lds) {
  ChunkAt at{sgpr(lds->x), sgpr(lds->x1), sgpr(lds->base), sgpr(lds->first_tile), sgpr(lds->kvh), sgpr(lds->seq)};
  ChunkUnitAt u;
  const int lane = threadIdx.x & 63, G = a.shape.group;
  while (next_unit(a, at, u)) {
    if (u.b0 != 0 || u.b1 < u.tile.blocks) continue;   // in parts: the join's
    // (every wave sees the same: a row is stored anew behind a barrier)
    for (int r = 0; r < u.tile.rows; ++r) {
      const int64_t packed = (int64_t)(at.tile - u.first) * kChunkRows + r;
      const int32_t token = (int32_t)(packed / G), head = at.kvh * G + (int32_t)(packed - (int64_t)token * G);
      const int64_t t = u.seq.start + token;
      uint16_t* o = a.o + t * a.ldo + (int64_t)head * a.d;
      constexpr uint16_t kExp = kBF16 ? 0x7f80 : 0x7c00;
      bool bad = false;
      for (int c = lane; c < a.d; c += 64) bad |= (o[c] & kExp) == kExp;
      if (__builtin_amdgcn_ballot_w64(bad) != 0)
        chunk_row<kBF16, kFp8>(a, at.seq, at.kvh, u.seq.len - u.seq.tokens + token,
                               a.q + t * a.ldq + (int64_t)head * a.d, o, 0, a.d, lds);
    }
  }
}

typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_ptr;

enum Source { kDma = 0, kStaged = 1, kCodes = 2 };

// floats of a part: O of 128 rows and (m, l)
template <int kDh>
constexpr int kPartFloats = 4 * (4 * (kDh / 32) + 1) * 64 * 4;

// Whether units of at most 32 rows have a code of their own.  (Not staged 16-bit keys, whose loads of a wave's
// block take 64 registers: 32 pieces of 8 over up to 8192 keys, a page each, 173 us for 151.)
template <Source kSrc>
constexpr bool kOwnTiles = kSrc != kStaged;

// This workgroup's units of more than 32 rows, or (kNarrow) those of at most 32: two codes, each with the
// registers to itself.  True: it has units of the other kind.
template <bool kBF16, Source kSrc, int kNK, int kDh, int kDp, bool kNarrow>
__device__ __forceinline__ bool chunk_units(const ChunkArgs& a, const uint16_t* __restrict__ Q, const uint8_t* __restrict__ K,
                                            const uint8_t* __restrict__ V, uint16_t* __restrict__ O, uint8_t* smem,
                                            ChunkLds* deal) {
  constexpr int kWG = 4;
  constexpr int kST = kNK / 32;
  constexpr int kRow = 2 * kDp;          // bytes of a K or V row in LDS
  constexpr int kChunks = kRow / 16;
  constexpr int kKK = kDh / 16;          // d-steps of S^T
  constexpr int kDT = kDh / 32;          // 32-d tiles of O^T
  constexpr int kDmaRows = 1024 / kRow;  // rows one 1 KiB DMA instruction fills
  constexpr int kPN = 2 * kST;           // 16-key chunks of a P block
  constexpr int kTileB = kNK * kRow;
  constexpr int kStageB = 2 * kTileB;
  constexpr int kDmaPerWave = kTileB / 1024 / kWG;
  constexpr int kEs = kSrc == kCodes ? 1 : 2;
  constexpr int kLoadElems = 16 / kEs;                       // elements of a staged load
  constexpr int kLoads = kNK * kDp / kLoadElems / 256;       // staged loads of a thread
  static_assert(kDh % 32 == 0 && kDh <= kDp && (kDp == 64 || kDp == 128 || kDp == 256), "row width");
  static_assert((kNK == 32 || kNK == 64) && kDmaPerWave >= 1 && kLoads >= 1, "tiles in 1 KiB slices over the waves");
  // (the thread's number through an empty asm: what the two codes work out from it is not kept from one
  // for the other)
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 5, l32 = lane & 31;
  const int d = a.d, row_b = 2 * d, chunks_g = row_b / 16;
  const int G = a.shape.group;

  auto kswz = [](int r) { return kChunks == 8 ? ((r >> 1) & 7) : (r & 15); };
  auto vswz = [](int r) { return (kChunks == 8 ? 2 : 4) * (r & 3); };
  const float c = a.scale_log2;
  const int win = a.shape.window > 0 ? (int)min(a.shape.window, (int64_t)1 << 30) : 1 << 30;
  const int sinks = a.shape.window > 0 ? (int)min(a.shape.sinks, (int64_t)1 << 30) : 0;
  const int page_mask = (1 << a.page_shift) - 1;

  // byte offsets of a lane's chunk within a DMA instruction's keys; chunks past the row's data fall past
  // the resource, which makes them zeros
  int k_voff[kDmaPerWave], v_voff[kDmaPerWave];
  if constexpr (kSrc == kDma) {
#pragma unroll
    for (int i = 0; i < kDmaPerWave; ++i) {
      const int row = kDmaRows * (wave + kWG * i) + lane / kChunks, pos = lane % kChunks;
      const int kc = pos ^ kswz(row), vc = pos ^ vswz(row);
      k_voff[i] = kc < chunks_g ? lane / kChunks * row_b + kc * 16 : 0x7fff0000;
      v_voff[i] = vc < chunks_g ? lane / kChunks * row_b + vc * 16 : 0x7fff0000;
    }
  }
  const int kf_off = l32 * kRow, kf_swz = kswz(l32);
  const int tr_i = lane & 15, tr_s = (lane >> 4) & 1;

  ChunkAt at{sgpr(deal->x), sgpr(deal->x1), sgpr(deal->base), sgpr(deal->first_tile), sgpr(deal->kvh), sgpr(deal->seq)};
  ChunkUnitAt u;
  // A share's first unit, where it is the rest of one whose start another workgroup has, comes last: the
  // workgroups of an XCD, each with the end of one tile and the start of the next, then go over the
  // same keys at the same time.
  bool others = false;
  int32_t first_end = -1;   // where that unit ends; -1: none is left over
  bool begun = false;
  for (;;) {
    if (!next_unit(a, at, u)) {
      if (kNarrow || first_end < 0) break;
      at = {sgpr(deal->x), first_end, sgpr(deal->base), sgpr(deal->first_tile), sgpr(deal->kvh), sgpr(deal->seq)};
      first_end = -1;
      if (!next_unit(a, at, u)) break;
    } else if (kOwnTiles<kSrc> && kNarrow != (u.tile.rows <= 32)) {
      others = true;
      continue;
    } else if (!kNarrow && !begun) {
      begun = true;
      if (u.b0 > 0 && at.x < at.x1) {
        first_end = at.x;
        continue;
      }
    }
    const ChunkTile& tl = u.tile;
    const int32_t b0 = u.b0, b1 = u.b1, n_blocks = tl.blocks, len = u.seq.len, rows = tl.rows, kvh = at.kvh;
    const bool whole = b0 == 0 && b1 >= n_blocks;
    const int32_t first_row = (at.tile - u.first) * kChunkRows;
    const int32_t* table = a.tables + (int64_t)at.seq * a.ld_table;
    const int rw = kNarrow ? 0 : wave;   // the wave's 32 rows; a tile of at most 32 is all waves'
    const bool active = 32 * rw < rows;

    // the lane's query row: token t of the sequence, query head `head` of the key head's
    const int m_row = min(32 * rw + l32, rows - 1);
    const uint32_t packed = (uint32_t)(first_row + m_row);
    const int32_t token = (int32_t)(packed / (uint32_t)G), head = (int32_t)(packed - (uint32_t)token * G);
    const int32_t p = len - u.seq.tokens + token;
    const int64_t q_off = (int64_t)(u.seq.start + token) * a.ldq + (int64_t)(kvh * G + head) * d;
    // positions of the wave's first and last row
    const int32_t pw0 = __builtin_amdgcn_readlane(p, 0), pw1 = __builtin_amdgcn_readlane(p, 31);

    u32x4 qf[kKK];
    {
      const uint16_t* qrow = Q + q_off + 8 * g;
#pragma unroll
      for (int kk = 0; kk < kKK; ++kk) {
        u32x4 w = {0u, 0u, 0u, 0u};
        if (16 * kk + 8 * g < d) w = *reinterpret_cast<const u32x4*>(qrow + 16 * kk);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (w[i] & a.q_and) ^ a.q_xor;
        qf[kk] = w;
      }
    }
    int32_t whole0, whole1;
    chunk_whole(a.shape, tl, &whole0, &whole1);
    whole0 = sgpr(whole0);
    whole1 = sgpr(whole1);
    auto block_of = [&](int e) { return chunk_block(tl, e); };
    auto wave_sees = [&](int e) {   // any key of entry e for any of the wave's rows
      const int k0 = block_of(e) * kNK;
      return e >= b0 && e < b1 && k0 <= pw1 && (k0 + kNK - 1 > pw0 - win || k0 < sinks);
    };

    // ---- where an entry's keys lie, a key a lane (past the part: its last entry's) ----
    auto key_of = [&](int e) { return block_of(min(e, b1 - 1)) * kNK + (lane & (kNK - 1)); };
    auto ids_of = [&](int e) { return table[min(key_of(e), len - 1) >> a.page_shift]; };
    struct Keys {
      uint32_t lo;   // byte offset of the key's row
      int32_t hi;    // below 0: no such page
    };
    auto keys_at = [&](int e, int32_t id) {
      const uint64_t off = ((uint64_t)(uint32_t)id * (uint64_t)a.page_stride +
                            (((uint64_t)kvh << a.page_shift) + (uint32_t)(key_of(e) & page_mask)) * (uint32_t)d) * kEs;
      return Keys{(uint32_t)off, (uint32_t)id < (uint32_t)a.num_pages ? (int32_t)(off >> 32) : -1};
    };
    // of the entry's keys those whose page is there (past the last key: as the last)
    auto pages_there = [&](const Keys& k) { return __builtin_amdgcn_ballot_w64(k.hi >= 0); };

    // ---- K and V of an entry to a stage ----
    auto dma = [&](const uint8_t* from, const int (&voff)[kDmaPerWave], uint8_t* to, int e, const Keys& k) {
      const int end = len - block_of(min(e, b1 - 1)) * kNK;   // of the sequence's keys, from the entry's first
#pragma unroll
      for (int i = 0; i < kDmaPerWave; ++i) {
        const int row0 = kDmaRows * (wave + kWG * i);
        const int hi = __builtin_amdgcn_readlane(k.hi, row0);
        const uint64_t at = (uint64_t)(uint32_t)hi << 32 | (uint32_t)__builtin_amdgcn_readlane((int)k.lo, row0);
        const int rows_in = sgpr(min(max(end - row0, 0), kDmaRows));
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
            (void*)(from + at), (short)0, hi < 0 ? 0 : rows_in * row_b, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)(to + (wave + i * kWG) * 1024), 16, voff[i], 0, 0, 0);
      }
    };
    // through registers: thread t takes chunks t, t + 256, .. of the block's rows
    u32x4 stage_k[kLoads], stage_v[kLoads];
    auto fetch = [&](const uint8_t* from, u32x4 (&to)[kLoads], int e, const Keys& k) {
      const int end = len - block_of(min(e, b1 - 1)) * kNK;
      constexpr int kPer = kDp / kLoadElems;   // loads of a row
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int row = (tid + 256 * i) / kPer, ch = (tid + 256 * i) % kPer;
        const int hi = __shfl(k.hi, row);
        const uint64_t at = (uint64_t)(uint32_t)hi << 32 | (uint32_t)__shfl((int)k.lo, row);
        u32x4 w = {0u, 0u, 0u, 0u};
        if (hi >= 0 && row < end && ch * kLoadElems < d) w = *reinterpret_cast<const u32x4*>(from + at + ch * 16);
        to[i] = w;
      }
    };
    // load number ch of a row to the row's place in LDS
    auto put = [&](const u32x4& from, uint8_t* row, int ch, int swz) {
      if constexpr (kSrc == kCodes) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x2 lo = widen4<kBF16>(from[2 * h]), hi = widen4<kBF16>(from[2 * h + 1]);
          *reinterpret_cast<u32x4*>(row + (((2 * ch + h) ^ swz) << 4)) = u32x4{lo[0], lo[1], hi[0], hi[1]};
        }
      } else {
        *reinterpret_cast<u32x4*>(row + ((ch ^ swz) << 4)) = from;
      }
    };
    auto commit = [&](const u32x4 (&from)[kLoads], uint8_t* to, bool is_v) {
      constexpr int kPer = kDp / kLoadElems;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int row = (tid + 256 * i) / kPer, ch = (tid + 256 * i) % kPer;
        put(from[i], to + row * kRow, ch, is_v ? vswz(row) : kswz(row));
      }
    };
    auto k_stage = [&](int s) { return smem + s * kStageB; };
    auto v_stage = [&](int s) { return smem + s * kStageB + kTileB; };
    auto begin_k = [&](int e, int stage, const Keys& k) {
      if constexpr (kSrc == kDma) dma(K, k_voff, k_stage(stage), e, k);
      else fetch(K, stage_k, e, k);
    };
    auto begin_v = [&](int e, int stage, const Keys& k) {
      if constexpr (kSrc == kDma) dma(V, v_voff, v_stage(stage), e, k);
      else fetch(V, stage_v, e, k);
    };
    auto end_k = [&](int stage) {
      if constexpr (kSrc != kDma) commit(stage_k, k_stage(stage), false);
    };
    auto end_v = [&](int stage) {
      if constexpr (kSrc != kDma) commit(stage_v, v_stage(stage), true);
    };

    auto k_frag = [&](const uint8_t* ks, int st, int kk) {
      return *reinterpret_cast<const u32x4*>(ks + 32 * st * kRow + (((2 * kk + g) ^ kf_swz) << 4));
    };
    auto v_frag = [&](const uint8_t* vs, int dt, int cc) {
      u32x4 out;
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int key = 16 * cc + 8 * hh + 4 * g + (tr_i >> 2);
        const int chunk = (32 * dt + 16 * tr_s + 4 * (tr_i & 3)) >> 3;
        const int off = key * kRow + ((chunk ^ vswz(key)) << 4) + 8 * (tr_i & 1);
        const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(vs + off));
        const u32x2 w = __builtin_bit_cast(u32x2, v);
        out[2 * hh] = w[0];
        out[2 * hh + 1] = w[1];
      }
      return out;
    };
    auto zero_s = [](f32x16 (&s)[kST]) {
#pragma unroll
      for (int st = 0; st < kST; ++st)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[st][i] = 0.0f;
    };
    auto s_block = [&](int stage, f32x16 (&s)[kST]) {
      const uint8_t* ks = k_stage(stage) + kf_off;
      zero_s(s);
#pragma unroll
      for (int st = 0; st < kST; ++st)
#pragma unroll
        for (int kk = 0; kk < kKK; ++kk) s[st] = mma32<kBF16>(k_frag(ks, st, kk), qf[kk], s[st]);
    };
    auto pv_block = [&](int stage, const u32x4 (&pf)[kPN], f32x16 (&oa)[kDT]) {
      const uint8_t* vs = v_stage(stage);
#pragma unroll
      for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
        for (int cc = 0; cc < kPN; ++cc) oa[dt] = mma32<kBF16>(v_frag(vs, dt, cc), pf[cc], oa[dt]);
    };
    // S_{j+1} and PV_{j-1}, a step of each at a time
    auto mma_block = [&](int stage, f32x16 (&s)[kST], const u32x4 (&pf)[kPN], f32x16 (&oa)[kDT]) {
      const uint8_t* ks = k_stage(stage) + kf_off;
      const uint8_t* vs = v_stage(stage);
      zero_s(s);
#pragma unroll
      for (int step = 0; step < kKK * kST; ++step) {
        const int st = step / kKK, kk = step % kKK;
        s[st] = mma32<kBF16>(k_frag(ks, st, kk), qf[kk], s[st]);
        const int dt = step % kDT, cc = step / kDT;
        oa[dt] = mma32<kBF16>(v_frag(vs, dt, cc), pf[cc], oa[dt]);
      }
    };

    f32x16 oacc[kDT];
#pragma unroll
    for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) oacc[dt][i] = 0.0f;
    float m_run = -__builtin_inff(), l_run = 0.0f;
    u32x4 pa[kPN], pb[kPN];
#pragma unroll
    for (int cc = 0; cc < kPN; ++cc) pa[cc] = pb[cc] = u32x4{0u, 0u, 0u, 0u};

    auto softmax_block = [&](int j, auto masked, uint64_t there, f32x16 (&s)[kST], u32x4 (&pnew)[kPN]) {
      constexpr bool kMasked = decltype(masked)::value;
      if constexpr (kMasked) {
        const int e = b0 + j;
        const int kb = (e < b1 ? block_of(e) * kNK : 0x40000000) + 4 * g;
        const int hi = p - kb;             // key offsets > hi are not seen
        const int lo = p - win - kb;       // <= lo neither, unless
        const int sk = sinks - kb;         // below sk
        const uint64_t mine = there >> (4 * g);
#pragma unroll
        for (int st = 0; st < kST; ++st)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int off = 32 * st + 8 * (i >> 2) + (i & 3);
            const bool in = off <= hi && (off > lo || off < sk) && ((mine >> off) & 1);
            s[st][i] = in ? s[st][i] : -__builtin_inff();
          }
      }
      // fast path: P_j against the running max; a lane whose block sum is larger than the limit, or
      // NaN, sends the wave to the block-max update
      auto probs = [&](float mc) {
        float rs = 0.0f;
#pragma unroll
        for (int st = 0; st < kST; ++st)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            u32x4 w;
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
              const float x0 = exp2_fast(__builtin_fmaf(s[st][8 * h + 2 * jj], c, -mc));
              const float x1 = exp2_fast(__builtin_fmaf(s[st][8 * h + 2 * jj + 1], c, -mc));
              w[jj] = pack2<kBF16>(x0, x1);
              rs = pair_sum<kBF16>(w[jj], rs);
            }
            pnew[2 * st + h] = w;
          }
        return rs;
      };
      float rs = probs(m_run * c - kLift<kBF16>);
      if (__builtin_amdgcn_ballot_w64(!(rs <= kBlockSumLimit<kBF16>)) != 0) {
#pragma unroll
        for (int st = 0; st < kST; ++st) asm volatile("" : "+v"(s[st]));
        float m = s[0][0];
#pragma unroll
        for (int st = 0; st < kST; ++st)
#pragma unroll
          for (int i = 0; i < 16; ++i) m = __builtin_fmaxf(m, s[st][i]);
        const float mx = pair32_max(m);
        const bool grow = __builtin_amdgcn_ballot_w64((mx - m_run) * c > kRescaleLog2) != 0;
        const float m_new = grow ? __builtin_fmaxf(m_run, mx) : m_run;
        // a row may have masked keys only so far: then every p is 0
        const float m_use = m_new == -__builtin_inff() ? 0.0f : m_new;
        const float alpha = exp2_fast((m_run - m_use) * c);
        m_run = m_new;
        rs = probs(m_use * c - kLift<kBF16>);
        l_run *= alpha;
        if (grow) {
#pragma unroll
          for (int dt = 0; dt < kDT; ++dt) oacc[dt] *= alpha;
        }
      }
      l_run += rs;
    };

    // ---- at most 32 rows: a wave takes every fourth block, in a K and a V tile of its own, and waits for
    // no other; the waves' results are joined through LDS.  (One wave with all blocks, the others
    // loading for it, as with more rows, was held up by its products and softmax: with e4m3
    // codes 32 pieces of 8 over up to 8192 keys took 108 us, now 90; 3 pieces of up to 700 and 48 single
    // tokens 164, now 146.) ----
    if constexpr (kNarrow) {
      constexpr int kN = kTileB / 1024;                          // DMAs of a tile
      constexpr int kOwn = kNK * kDp / kLoadElems / 64;          // or loads of a lane
      constexpr int kPer = kDp / kLoadElems;                     // loads of a row
      u32x4 own_k[kSrc == kDma ? 1 : kOwn], own_v[kSrc == kDma ? 1 : kOwn];
      // past the part nothing is read; the loads are non-temporal, as no other tile of the sequence, or at most
      // the larger ones before it, reads these keys (32 pieces of 8: 129 -> 115 us, of e4m3 90 -> 86)
      constexpr int kOnce = 2;
      auto own_dma = [&](const uint8_t* from, uint8_t* to, bool is_v, int e, const Keys& k) {
        const int end = e < b1 ? len - block_of(e) * kNK : 0;
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          const int row0 = kDmaRows * i, row = row0 + lane / kChunks;
          const int ch = lane % kChunks ^ (is_v ? vswz(row) : kswz(row));
          const int off = ch < chunks_g ? lane / kChunks * row_b + ch * 16 : 0x7fff0000;
          const int hi = __builtin_amdgcn_readlane(k.hi, row0);
          const uint64_t at = (uint64_t)(uint32_t)hi << 32 | (uint32_t)__builtin_amdgcn_readlane((int)k.lo, row0);
          const int rows_in = sgpr(min(max(end - row0, 0), kDmaRows));
          const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
              (void*)(from + at), (short)0, hi < 0 ? 0 : rows_in * row_b, 0x00020000);
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)(to + i * 1024), 16, off, 0, 0, kOnce);
        }
      };
      auto own_fetch = [&](const uint8_t* from, u32x4* to, int e, const Keys& k) {
        const int end = e < b1 ? len - block_of(e) * kNK : 0;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
          const int row = (lane + 64 * i) / kPer, ch = (lane + 64 * i) % kPer;
          const int hi = __shfl(k.hi, row);
          const uint64_t at = (uint64_t)(uint32_t)hi << 32 | (uint32_t)__shfl((int)k.lo, row);
          u32x4 w = {0u, 0u, 0u, 0u};
          if (hi >= 0 && row < end && ch * kLoadElems < d) 
            w = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(from + at + ch * 16));
          to[i] = w;
        }
      };
      auto own_commit = [&](const u32x4* from, uint8_t* to, bool is_v) {
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
          const int row = (lane + 64 * i) / kPer, ch = (lane + 64 * i) % kPer;
          put(from[i], to + row * kRow, ch, is_v ? vswz(row) : kswz(row));
        }
      };
      auto load_k = [&](int e, const Keys& k) {
        if constexpr (kSrc == kDma) own_dma(K, k_stage(wave), false, e, k);
        else own_fetch(K, own_k, e, k);
      };
      auto load_v = [&](int e, const Keys& k) {
        if constexpr (kSrc == kDma) own_dma(V, v_stage(wave), true, e, k);
        else own_fetch(V, own_v, e, k);
      };
      // the tile whose loads are older than those of the last kN DMAs is there; reads before have ended
      auto arrived = [&] {
        static_assert(kN <= 63, "vmcnt");
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt((kN & 15) | (7 << 4) | (15 << 8) | ((kN >> 4) << 14));
        asm volatile("" ::: "memory");
      };
      auto reads_done = [&] {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));
        asm volatile("" ::: "memory");
      };
      if (b0 + wave < b1) {
        const int e0 = b0 + wave;
        const int32_t id0 = ids_of(e0), id1 = ids_of(e0 + 4);
        int32_t id2 = ids_of(e0 + 8);
        Keys keys0 = keys_at(e0, id0), keys1 = keys_at(e0 + 4, id1);
        load_k(e0, keys0);
        load_v(e0, keys0);
        for (int e = e0; e < b1; e += 4) {
          const uint64_t there = pages_there(keys0);
          keys0 = keys1;
          if constexpr (kSrc == kDma) arrived();
          else {
            own_commit(own_k, k_stage(wave), false);
            load_k(e + 4, keys0);
          }
          f32x16 s[kST];
          s_block(wave, s);
          if constexpr (kSrc == kDma) {
            reads_done();
            load_k(e + 4, keys0);
          }
          softmax_block(e - b0, std::true_type{}, there, s, pa);
          if constexpr (kSrc == kDma) arrived();
          else {
            own_commit(own_v, v_stage(wave), true);
            load_v(e + 4, keys0);
          }
          pv_block(wave, pa, oacc);
          if constexpr (kSrc == kDma) {
            reads_done();
            load_v(e + 4, keys0);
          }
          keys1 = keys_at(e + 8, id2);
          id2 = ids_of(e + 12);
        }
      }
      // the four waves' results: in their own tiles' place, then a wave a quarter of the dims
      static_assert(kDT * 4096 <= kStageB, "O in the place of K and V");
      asm volatile("" ::: "memory");
      // vmcnt(0) lgkmcnt(0): nothing more is written there
      __builtin_amdgcn_s_waitcnt(0 | (7 << 4) | (0 << 8));
      asm volatile("" ::: "memory");
      // (through an empty asm: addresses worked out here are not kept in registers through the blocks)
      int el = lane;
      asm volatile("" : "+v"(el));
#pragma unroll
      for (int t = 0; t < 4 * kDT; ++t) {
        const int e = 4 * (t % 4);
        *reinterpret_cast<f32x4*>(smem + wave * kStageB + 1024 * t + 16 * el) =
            f32x4{oacc[t / 4][e], oacc[t / 4][e + 1], oacc[t / 4][e + 2], oacc[t / 4][e + 3]};
      }
      deal->acc[wave][el] = m_run;
      deal->acc[wave][64 + el] = pair32_sum(l_run);
      __syncthreads();
      float m = deal->acc[0][el], l = 0.0f;
#pragma unroll
      for (int w = 1; w < 4; ++w) m = __builtin_fmaxf(m, deal->acc[w][el]);
      const float m_use = m == -__builtin_inff() ? 0.0f : m;   // no key seen
      f32x4 o[kDT];
#pragma unroll
      for (int t = 0; t < kDT; ++t) o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = exp2_fast((deal->acc[w][el] - m_use) * c);
        l += f * deal->acc[w][64 + el];
#pragma unroll
        for (int t = 0; t < kDT; ++t)
          o[t] += *reinterpret_cast<const f32x4*>(smem + w * kStageB + 1024 * (kDT * wave + t) + 16 * el) * f;
      }
      if (!whole) {
        const int32_t w = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
        float* part = a.parts + (int64_t)(2 * w + (b0 == 0 ? 1 : 0)) * kPartFloats<kDh> + 4 * el;
#pragma unroll
        for (int t = 0; t < kDT; ++t) *reinterpret_cast<f32x4*>(part + 256 * (kDT * wave + t)) = o[t];
        if (wave == 0) *reinterpret_cast<f32x4*>(part + 256 * 4 * kDT) = f32x4{m, l, 0.0f, 0.0f};
      } else if ((el & 31) < rows) {
        const bool none = p < 0;   // no key: zeros
        const float inv = none ? 0.0f : a.v_scale / l;
        float z = none ? 0.0f : l * inv * 0.0f;
        uint16_t* orow = O + (int64_t)(u.seq.start + token) * a.ldo + (int64_t)(kvh * G + head) * d;
#pragma unroll
        for (int t = 0; t < kDT; ++t) {
          const int tt = kDT * wave + t, dim = 32 * (tt / 4) + 8 * (tt % 4) + 4 * (el >> 5);
          if (dim >= d) continue;
          const f32x4 f = o[t] * inv;
#pragma unroll
          for (int i = 0; i < 4; ++i) z = __builtin_fmaf(f[i], 0.0f, z);
          *reinterpret_cast<u32x2*>(orow + dim) = u32x2{pack2<kBF16>(f[0], f[1]), pack2<kBF16>(f[2], f[3])};
        }
        if (!(z == 0.0f)) deal->again = 1;
      }
      __syncthreads();   // (the next unit's tiles go to the same place)
      continue;
    }

    int nb = b1 - b0;
    nb += nb & 1;
    if (nb > 0 && n_blocks > 0) {
      // K_0, K_1 and, for the empty PV_{-1}, a V tile in stage 1: P_{-1} = 0 meets V_0, whose NaN a
      // seen row may well hold only in a masked key; such rows are taken again in any case
      const int32_t id0 = ids_of(b0), id1 = ids_of(b0 + 1), id2 = ids_of(b0 + 2);
      int32_t id3 = ids_of(b0 + 3);
      Keys keys0 = keys_at(b0, id0), keys1 = keys_at(b0 + 1, id1), keys2 = keys_at(b0 + 2, id2);
      begin_k(b0, 0, keys0);
      begin_v(b0, 1, keys0);
      end_k(0);
      end_v(1);
      begin_k(b0 + 1, 1, keys1);
      end_k(1);
      __syncthreads();
      f32x16 sa[kST], sb[kST];
      if (active) s_block(0, sa);
      __syncthreads();

      auto loads = [&](int e, int stage) {
        begin_k(e + 2, stage, keys2);
        begin_v(e, stage, keys0);
        keys0 = keys1;
        keys1 = keys2;
        keys2 = keys_at(e + 3, id3);
        id3 = ids_of(e + 4);
      };
      if (!active) {   // a wave without rows loads its share only
        for (int j = 0; j < nb; ++j) {
          loads(b0 + j, j & 1);
          end_k(j & 1);
          end_v(j & 1);
          __syncthreads();
        }
      } else {
      auto iteration = [&](int j, auto stage_c, auto masked, f32x16 (&scur)[kST], f32x16 (&snext)[kST],
                           const u32x4 (&pprev)[kPN], u32x4 (&pnew)[kPN]) {
        constexpr int kS = decltype(stage_c)::value;
        constexpr bool kMasked = decltype(masked)::value;
        const int e = b0 + j;
        const uint64_t there = kMasked ? pages_there(keys0) : 0;
        loads(e, kS);
        // (the unmasked form without a branch: behind one the compiler waits for the loads first)
        if (!kMasked || wave_sees(e - 1) || wave_sees(e) || wave_sees(e + 1)) {
          mma_block(kS ^ 1, snext, pprev, oacc);
          softmax_block(j, masked, there, scur, pnew);
        } else {
#pragma unroll
          for (int cc = 0; cc < kPN; ++cc) pnew[cc] = u32x4{0u, 0u, 0u, 0u};
        }
        // keep P_j and l in this region, beside the MFMAs
#pragma unroll
        for (int cc = 0; cc < kPN; ++cc) asm volatile("" : "+v"(pnew[cc]));
        asm volatile("" : "+v"(l_run));
        end_k(kS);
        end_v(kS);
        __syncthreads();
      };
      using Z = std::integral_constant<int, 0>;
      using One = std::integral_constant<int, 1>;
      auto masked_pairs = [&](int j, int to) {
        for (; j < to; j += 2) {
          iteration(j, Z{}, std::true_type{}, sa, sb, pa, pb);
          iteration(j + 1, One{}, std::true_type{}, sb, sa, pb, pa);
        }
      };
      // the pairs of iterations whose entries every row sees whole, up to the first with a page that
      // does not exist (a choice of masked or not for each pair in one loop took 60 registers more)
      const int j0 = min((max(whole0 - b0, 0) + 1) / 2 * 2, nb), j1 = max((min(whole1, b1) - b0) / 2 * 2, j0);
      masked_pairs(0, j0);
      int j = j0;
      for (; j < j1 && (pages_there(keys0) & pages_there(keys1)) == ~0ull; j += 2) {
        iteration(j, Z{}, std::false_type{}, sa, sb, pa, pb);
        iteration(j + 1, One{}, std::false_type{}, sb, sa, pb, pa);
      }
      masked_pairs(j, nb);
      // PV of the last block (nb is even: P_{nb-1} is in pa, V_{nb-1} in stage 1)
      if (wave_sees(b0 + nb - 1)) pv_block(1, pa, oacc);
      }
    }

    // ---- the end of the unit ----
    // (the lane's number through an empty asm: addresses worked out here are not kept in
    // registers through the blocks)
    int el = lane;
    asm volatile("" : "+v"(el));
    const int e32 = el & 31, eg = el >> 5;
    const float l = pair32_sum(l_run);
    if (!whole) {
      if (active) {
        const int32_t w = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
        float* part = a.parts + (int64_t)(2 * w + (b0 == 0 ? 1 : 0)) * kPartFloats<kDh> + wave * (4 * kDT + 1) * 256 + 4 * el;
#pragma unroll
        for (int t = 0; t < 4 * kDT; ++t) {
          const int e = 4 * (t % 4);
          *reinterpret_cast<f32x4*>(part + 256 * t) =
              f32x4{oacc[t / 4][e], oacc[t / 4][e + 1], oacc[t / 4][e + 2], oacc[t / 4][e + 3]};
        }
        *reinterpret_cast<f32x4*>(part + 256 * 4 * kDT) = f32x4{m_run, l, 0.0f, 0.0f};
      }
    } else if (32 * wave + e32 < rows) {
      const uint32_t pk = (uint32_t)(first_row + 32 * wave + e32);
      const int32_t tk = (int32_t)(pk / (uint32_t)G), hd = kvh * G + (int32_t)(pk - (uint32_t)tk * G);
      const bool none = len - u.seq.tokens + tk < 0;   // no key: zeros
      const float inv = none ? 0.0f : a.v_scale / l;
      float z = none ? 0.0f : l * inv * 0.0f;
      uint16_t* orow = O + (int64_t)(u.seq.start + tk) * a.ldo + (int64_t)hd * d;
#pragma unroll
      for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int dim = 32 * dt + 8 * r + 4 * eg;
          if (dim >= d) continue;
          f32x4 f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f[i] = oacc[dt][4 * r + i] * inv;
            z = __builtin_fmaf(f[i], 0.0f, z);
          }
          const u32x2 w = {pack2<kBF16>(f[0], f[1]), pack2<kBF16>(f[2], f[3])};
          *reinterpret_cast<u32x2*>(orow + dim) = w;
        }
      if (!(z == 0.0f)) deal->again = 1;
    }
    __syncthreads();   // (the next unit's tiles go to the same place)
  }
  return others;
}

template <bool kBF16, Source kSrc, int kNK, int kDh, int kDp>
__device__ __forceinline__ void chunk_attn(const ChunkArgs& a, const uint16_t* __restrict__ Q, const uint8_t* __restrict__ K,
                                           const uint8_t* __restrict__ V, uint16_t* __restrict__ O, uint8_t* smem,
                                           ChunkLds* deal) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // ---- this workgroup's blocks: x .. x1 - 1 of the list, in tile `tile` of key head kvh, which
  // begins at `base` ----
  int32_t tile, kvh, seq;
  int32_t x, x1, base, first_rows;
  if (a.direct) {
    // (an XCD takes a contiguous run of units; the last tiles of a piece see the most keys: first)
    const int units = a.tiles * a.kv_heads, per_xcd = (units + 7) / 8;
    const int unit = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if (unit >= units) return;
    kvh = sgpr(unit / a.tiles);
    tile = a.tiles - 1 - (unit - kvh * a.tiles);
    seq = __builtin_amdgcn_readfirstlane(seq_of_tile(a, tile));
    const ChunkTile t = chunk_tile(a.shape, load_seq(a, seq),
                                   tile - chunk_base(a.shape, chunk_clamp(a.starts[seq], a.shape.n_tokens), seq));
    base = x = 0;
    x1 = sgpr(chunk_size(t));
    if (x1 == 0) return;
    first_rows = sgpr(t.rows);
  } else {
    const int per = (a.tiles + 255) / 256;
    const int32_t c0 = min(tid * per, a.tiles), c1 = min(c0 + per, a.tiles);
    // the sizes of a run of tiles, in order
    auto run = [&](auto visit) { chunk_run(a, c0, c1, visit); };
    int64_t mine = 0;
    run([&](int32_t, int32_t size, int32_t, int32_t, int32_t) { mine += size; });
    int64_t incl = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int64_t up = __shfl_up((long long)incl, off);
      if (lane >= off) incl += up;
    }
    if (lane == 63) deal->wave_sum[wave] = incl;
    __syncthreads();
    int64_t before = incl - mine, head_total = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) before += deal->wave_sum[w];
      head_total += deal->wave_sum[w];
    }
    // (at most 2^31 - 1 by the host's bound)
    const int32_t per_head = __builtin_amdgcn_readfirstlane((int32_t)head_total);
    const int64_t total = (int64_t)per_head * a.kv_heads;
    const int64_t share = chunk_share(total, a.groups);
    // an XCD (workgroup i runs on XCD i % 8) takes a contiguous run of shares
    const int32_t w = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    x = sgpr((int32_t)min((int64_t)w * share, total));
    x1 = sgpr((int32_t)min(x + share, total));
    if (w != 0 && x >= x1) return;
    kvh = per_head == 0 ? 0 : sgpr(x / per_head);
    const int32_t in_head = x - kvh * per_head;
    if (w == 0 || (in_head >= before && in_head < before + mine)) {
      int64_t at = before;
      run([&](int32_t t, int32_t size, int32_t r, int32_t first, int32_t rows) {
        if (w == 0) a.plan[t] = {(int32_t)at, r, first, rows};
        if (in_head >= at && in_head < at + size) {
          deal->tile = t;
          deal->before = (int32_t)at;
          deal->seq = r;
          deal->rows = rows;
        }
        at += size;
      });
    }
    if (w == 0 && tid == 0) a.plan[a.tiles].at = per_head;
    if (x >= x1) return;
    __syncthreads();
    tile = __builtin_amdgcn_readfirstlane(deal->tile);
    seq = __builtin_amdgcn_readfirstlane(deal->seq);
    first_rows = sgpr(deal->rows);
    base = kvh * per_head + sgpr(deal->before);
  }

  if (tid == 0) {
    deal->x = x;
    deal->x1 = x1;
    deal->base = base;
    deal->first_tile = tile;
    deal->kvh = kvh;
    deal->seq = seq;
    deal->again = 0;
  }
  __syncthreads();
  if constexpr (kOwnTiles<kSrc>) {
    // those like the share's first unit first: most shares have no others to look for
    bool narrow = first_rows <= 32, more = true;
    for (int i = 0; i < 2 && more; ++i, narrow = !narrow)
      more = narrow ? chunk_units<kBF16, kSrc, kNK, kDh, kDp, true>(a, Q, K, V, O, smem, deal)
                    : chunk_units<kBF16, kSrc, kNK, kDh, kDp, false>(a, Q, K, V, O, smem, deal);
  } else {
    chunk_units<kBF16, kSrc, kNK, kDh, kDp, false>(a, Q, K, V, O, smem, deal);
  }
  __syncthreads();   // (a share may have no unit and so no barrier since the flag was cleared)
  if (__builtin_amdgcn_readfirstlane(deal->again) != 0) chunk_again<kBF16, kSrc == kCodes>(a, deal);
}

// Joins the parts of unit blockIdx.x (key head, tile), 32 rows a workgroup (blockIdx.y); each wave has
// kQ 4-dim columns of every lane, all of a row's in one workgroup, or (kQ 1) over blockIdx.z.
template <bool kBF16, bool kFp8, int kDh, int kQ>
__device__ __forceinline__ void chunk_join(const ChunkArgs& a, ChunkLds* deal) {
  constexpr int kDT = kDh / 32;
  const int kvh = blockIdx.x / a.tiles, tile = blockIdx.x - kvh * a.tiles;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 5, l32 = lane & 31, rw = blockIdx.y, d = a.d, G = a.shape.group;
  const int col0 = kQ * (4 * blockIdx.z + wave);   // the wave's first column, of 8 dims
  const ChunkRec rec = a.plan[tile];
  const int32_t at = rec.at, size = a.plan[tile + 1].at - at, per_head = a.plan[a.tiles].at;
  if (size <= kChunkUnit || 32 * rw >= rec.rows) return;   // without keys, or rows
  const int64_t share = chunk_share((int64_t)per_head * a.kv_heads, a.groups);
  const int64_t x0 = (int64_t)kvh * per_head + at + kChunkUnit;
  const int32_t g0 = (int32_t)(x0 / share), g1 = (int32_t)((x0 + size - kChunkUnit - 1) / share);
  if (g0 == g1) return;   // one workgroup had it whole
  const int32_t seq = rec.seq, rows = rec.rows;
  const ChunkSeq q_seq = load_seq(a, seq);
  const int64_t packed0 = (int64_t)(tile - rec.first) * kChunkRows + 32 * rw;   // the first row's
  const int64_t packed = packed0 + min(l32, rows - 1 - 32 * rw);
  const int32_t token = (int32_t)(packed / G), head = (int32_t)(packed - (int64_t)token * G);
  const int32_t p = q_seq.len - q_seq.tokens + token;
  auto part = [&](int32_t w) {
    return a.parts + (int64_t)(2 * w + (w == g0 ? 1 : 0)) * kPartFloats<kDh> + rw * (4 * kDT + 1) * 256 + 4 * lane;
  };
  if (threadIdx.x == 0) deal->again = 0;
  __syncthreads();
  f32x4 acc[kQ];
#pragma unroll
  for (int t = 0; t < kQ; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -__builtin_inff(), l = 0.0f;
  constexpr int kTake = kQ == 1 ? 16 : 4;   // parts whose loads are in flight
  for (int32_t w0 = g0; w0 <= g1; w0 += kTake) {
    f32x4 ml[kTake], o[kTake][kQ];
#pragma unroll
    for (int u = 0; u < kTake; ++u) {
      const float* from = part(min(w0 + u, g1));
      ml[u] = *reinterpret_cast<const f32x4*>(from + 256 * 4 * kDT);
#pragma unroll
      for (int t = 0; t < kQ; ++t) o[u][t] = *reinterpret_cast<const f32x4*>(from + 256 * (col0 + t));
      if (w0 + u > g1) ml[u] = f32x4{-__builtin_inff(), 0.0f, 0.0f, 0.0f};
    }
    float m_new = m;
#pragma unroll
    for (int u = 0; u < kTake; ++u) m_new = __builtin_fmaxf(m_new, ml[u][0]);
    const float m_use = m_new == -__builtin_inff() ? 0.0f : m_new;   // no key seen so far
    const float alpha = exp2_fast((m - m_use) * a.scale_log2);
    m = m_new;
    l *= alpha;
#pragma unroll
    for (int t = 0; t < kQ; ++t) acc[t] *= alpha;
#pragma unroll
    for (int u = 0; u < kTake; ++u) {
      if (w0 + u > g1) continue;
      const float f = exp2_fast((ml[u][0] - m_use) * a.scale_log2);   // (a part without seen keys: 0)
      l += f * ml[u][1];
#pragma unroll
      for (int t = 0; t < kQ; ++t) acc[t] += o[u][t] * f;
    }
  }
  const bool none = p < 0;
  const float inv = none ? 0.0f : a.v_scale / l;
  float z = none ? 0.0f : l * 0.0f;
#pragma unroll
  for (int t = 0; t < kQ; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) z = __builtin_fmaf(acc[t][i] * inv, 0.0f, z);
  const uint64_t bad = __builtin_amdgcn_ballot_w64((!(z == 0.0f) || (!none && l == 0.0f)) && 32 * rw + l32 < rows);
  if (lane == 0 && bad != 0) atomicOr(&deal->again, (int)((uint32_t)bad | (uint32_t)(bad >> 32)));
  __syncthreads();
  const uint32_t again = (uint32_t)__builtin_amdgcn_readfirstlane(deal->again);
  if (32 * rw + l32 < rows && !((again >> l32) & 1)) {
    uint16_t* orow = a.o + (int64_t)(q_seq.start + token) * a.ldo + (int64_t)(kvh * G + head) * d;
#pragma unroll
    for (int t = 0; t < kQ; ++t) {
      const int dim = 8 * (col0 + t) + 4 * g;
      if (dim >= d) continue;
      const u32x2 w = {pack2<kBF16>(acc[t][0] * inv, acc[t][1] * inv), pack2<kBF16>(acc[t][2] * inv, acc[t][3] * inv)};
      *reinterpret_cast<u32x2*>(orow + dim) = w;
    }
  }
  for (uint32_t left = again; left != 0; left &= left - 1) {
    const int64_t r = packed0 + __builtin_ctz(left);
    const int32_t tk = (int32_t)(r / G), hd = kvh * G + (int32_t)(r - (int64_t)tk * G);
    const int64_t t = q_seq.start + tk;
    chunk_row<kBF16, kFp8>(a, seq, kvh, q_seq.len - q_seq.tokens + tk, a.q + t * a.ldq + (int64_t)hd * d,
                           a.o + t * a.ldo + (int64_t)hd * d, 32 * kQ * blockIdx.z, 32 * kQ * (blockIdx.z + 1), deal);
  }
}

}  // namespace

// One LDS array for all of it, and the operands as restrict pointers: else (two arrays have an alias scope
// each; without restrict the transposing reads have none at all) the compiler takes every read of LDS for one of
// what a DMA has just been told to write, and waits for the next blocks before the products of this one.
// d<D>: head dimensions up to D; s: pages below a DMA instruction's keys
#define SILE_CHUNK_KERNEL(NAME, BF, SRC, EU, NK, DH, DP)                                  \
  extern "C" __global__ __launch_bounds__(256, EU) void NAME(ChunkArgs a) {               \
    __shared__ __attribute__((aligned(1024))) uint8_t smem[4 * 2 * NK * 2 * DP + sizeof(ChunkLds)]; \
    chunk_attn<BF, SRC, NK, DH, DP>(a, a.q, a.k, a.v, a.o, smem, reinterpret_cast<ChunkLds*>(smem + 4 * 2 * NK * 2 * DP)); \
  }
#define SILE_CHUNK_JOIN(NAME, BF, F8, DH, Q)                                     \
  extern "C" __global__ __launch_bounds__(256) void NAME(ChunkArgs a) {       \
    __shared__ ChunkLds deal;                                                 \
    chunk_join<BF, F8, DH, Q>(a, &deal);                                         \
  }
#define SILE_CHUNK_TYPES(T, BF, EU, NK, DH, DP)                                  \
  SILE_CHUNK_KERNEL(sile_paged_chunk_##T##_d##DH, BF, kDma, EU, NK, DH, DP)      \
  SILE_CHUNK_KERNEL(sile_paged_chunk_##T##_s##DH, BF, kStaged, EU, NK, DH, DP)   \
  SILE_CHUNK_KERNEL(sile_paged_chunk_##T##_fp8_d##DH, BF, kCodes, EU, NK, DH, DP) \
  SILE_CHUNK_JOIN(sile_paged_chunk_join_##T##_d##DH, BF, false, DH, DH / 32)     \
  SILE_CHUNK_JOIN(sile_paged_chunk_join_##T##_fp8_d##DH, BF, true, DH, DH / 32)  \
  SILE_CHUNK_JOIN(sile_paged_chunk_join1_##T##_d##DH, BF, false, DH, 1)          \
  SILE_CHUNK_JOIN(sile_paged_chunk_join1_##T##_fp8_d##DH, BF, true, DH, 1)
#define SILE_CHUNK_DIM(EU, NK, DH, DP)          \
  SILE_CHUNK_TYPES(f16, false, EU, NK, DH, DP)  \
  SILE_CHUNK_TYPES(bf16, true, EU, NK, DH, DP)
SILE_CHUNK_DIM(2, 64, 64, 64)
SILE_CHUNK_DIM(2, 32, 128, 128)
SILE_CHUNK_DIM(1, 32, 256, 256)
