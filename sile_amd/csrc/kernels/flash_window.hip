// Flash-attention forward of a prompt over a sliding window, with the first tokens
// kept visible and query heads sharing key heads.
//
//   O = softmax(Q K^T * scale + mask) V    Q, O [B, Hq, Sq, D]   K, V [B, Hk, Sk, D]
//   query i, at position p = start + i, sees key j <= p with j > p - window or j < sinks
//
// Its work is the matrix cores', 4 D flop for each seen pair, and the keys of a window are
// read again for every block of queries, out of the L2; but they are not what holds it (39 % busy at
// 2.1 GHz in the first case measured below, the causal kernel's 55 % at 1.78): a block of queries
// has few rounds of keys, each with its barrier, around a start and an end of some 5 us.  The
// pipeline is that of the causal kernel (flash_attn.hip): a workgroup of 4 waves, two of them a
// CU up to D = 128, takes 32 queries a wave; K and V blocks go from memory to LDS by
// LDS-DMA, two stages of each; iteration j issues S_{j+1} = K_{j+1} Q^T and O^T += V_{j-1}^T P_{j-1} on the matrix cores beside
// the online softmax of S_j, whose accumulator holds one query a lane; V^T is read
// with ds_read_b64_tr_b16.  What the window changes:
//
//  * The key blocks of a query block are a list: the blocks of the sinks, then those
//    from the first query's window to the last query's own position.  Blocks that
//    every query of the workgroup sees whole skip the mask.
//  * A wave passes over an iteration whose three blocks none of its queries sees
//    (at both ends of the window); its P is then zero.
//  * The waves of a workgroup take up to four query heads of one key head (the K and V tiles
//    are theirs alike) before further queries: 32 queries of four heads need 34 blocks of
//    32 keys for a window of 1024, 128 queries of one 37.
//  * Workgroups that read the same keys run together: an XCD takes a contiguous run of
//    (batch x key head, query block, query heads of that key head), so that a window's keys
//    are read from its L2 by all of them.
//  * A row whose result is not finite (Inf or NaN in a masked key's V makes it so: 0 times
//    it), or that sees no key, is taken again by one wave that reads its seen keys only.
//
// Two workgroups of 4 waves a CU and not one of 8: the first loads and the stores of one run beside
// the other's products, and a block's window ends sooner (8192 queries, 32 heads of 128, window
// 1024: 201 us with one, 172 with two; of 64: 150, 107).
//
// Key groups (kG = 2, 4): few query blocks leave CUs idle, so the blocks of the list can be
// dealt to groups of the waves of a workgroup of 8, which join their (m, l, O) at the end.
//
// Measured: 8192 queries, 32 heads of 128 over 8 key heads, window 1024 and 4 sinks: 154 - 169 us by
// card (765 - 840 TFLOP/s of seen pairs; MFMA 39 %, VALU 34 % of the cycles; of the waves' 40 %
// wait to issue, 27 % for data or a barrier); window 4096 381 - 413 (1000 - 1080); heads of 64, window
// 1024, 96 - 98 (670); 4096 queries, heads of 192 and 256, window 1024, 168 (540) and 207 (580); 2 x
// 4096 queries, 32 heads of 96, window 256, 60 (415); 2 x 512 queries x 16 heads behind 7680 keys,
// window 4096, 45 - 49 (740).
//
// The head dimension is rounded up to kDh (32, 64, 96, 128, 192 or 256): the chunks of a
// row past D are loaded as zeros and its O^T rows past D are not stored.
//
// The probabilities enter the product in 16 bits (half a step, 2^-8 of each in bf16, 2^-11 in
// f16, and their sum is of the rounded ones): the matrix cores are the bound here.  In f16 they carry a factor 2^7
// beside the up to 2^8 that the lazy maximum allows, so that those far below the
// maximum keep their bits; it drops out of O / l.
#include <type_traits>

#include "common.h"

using namespace sile;

namespace {

constexpr float kRescaleLog2 = 8.0f;  // lazy-rescale threshold: p <= 2^8

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

struct WindowArgs {
  int64_t q_len, kv_len, start, window, sinks;   // each below 2^31
  int32_t items;        // batch * kv_heads * q_blocks * group / heads
  int32_t q_blocks, group, d;
  int32_t heads;        // query heads of one key head that a workgroup takes: 1, 2 or 4, a divisor of group
  float scale_log2;     // softmax scale * log2(e)
};

// Query row i of Q's head (qi, oi) over its seen keys, a wave, fp32 throughout: keys
// 0 .. sink_end - 1 and first .. last.  None: zeros.
template <bool kBF16>
SILE_DEV void window_row(const uint16_t* qi, const uint16_t* kb, const uint16_t* vb, uint16_t* oi,
                         int64_t sink_end, int64_t first, int64_t last, int d, float scale_log2) {
  const int lane = threadIdx.x & 63;
  auto ld16 = [](const uint16_t* p) { return kBF16 ? bf16_to_f32(*p) : f16_to_f32(*p); };
  float qv[4], acc[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int dd = lane + 64 * t;
    qv[t] = dd < d ? ld16(qi + dd) : 0.0f;
    acc[t] = 0.0f;
  }
  // a seen score counts as at least the lowest float in the max: scores that are all
  // -inf give 0 / 0, a row without keys zeros
  float m = -3.402823466e38f, l = 0.0f;
  const int64_t n = max(last - first + 1, (int64_t)0);
  for (int64_t t = 0; t < sink_end + n; ++t) {
    const int64_t j = t < sink_end ? t : first + t - sink_end;
    const uint16_t* kj = kb + j * d;
    float s = 0.0f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int dd = lane + 64 * u;
      if (dd < d) s += qv[u] * ld16(kj + dd);
    }
    s = wave_sum(s) * scale_log2;
    const float m_new = s != s ? m : fmax_ordered(m, s);
    const float alpha = exp2_fast(m - m_new), p = exp2_fast(s - m_new);
    l = l * alpha + p;
    const uint16_t* vj = vb + j * d;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int dd = lane + 64 * u;
      if (dd < d) acc[u] = acc[u] * alpha + p * ld16(vj + dd);
    }
    m = m_new;
  }
  const float inv = sink_end + n == 0 ? 0.0f : 1.0f / l;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int dd = lane + 64 * u;
    if (dd < d) oi[dd] = kBF16 ? bf16_rne(acc[u] * inv) : f16_rne(acc[u] * inv);
  }
}

// the keys that the query at position p sees: sink_end, first, last as above
SILE_DEV void seen_range(const WindowArgs& a, int64_t p, int64_t* sink_end, int64_t* first, int64_t* last) {
  *last = min(p, a.kv_len - 1);
  *first = max(p - a.window + 1, (int64_t)0);
  *sink_end = min(min(a.sinks, *first), a.kv_len);
}

typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_ptr;

// LDS bytes: two stages of K and V tiles of kNK keys for each key group; at least the
// (m, l, O) of the groups but one
template <int kNK, int kDh, int kDp, int kW, int kG>
constexpr int lds_bytes() {
  const int stages = kG * 2 * 2 * kNK * 2 * kDp;
  const int parts = (kG - 1) * (kW / kG) * (16 * (kDh / 32) + 4) * 64 * 4;
  return stages > parts ? stages : parts;
}

template <bool kBF16, int kW, int kNK, int kDh, int kDp, int kG>
__device__ __forceinline__ void window_fwd(const uint16_t* __restrict__ Q, const uint16_t* __restrict__ K,
                                           const uint16_t* __restrict__ V, uint16_t* __restrict__ O,
                                           const WindowArgs& a, uint8_t* smem_all) {
  constexpr int kWG = kW / kG;           // waves sharing a key group's tiles
  constexpr int kBQ = kWG * 32;
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
  static_assert(kDh % 32 == 0 && kDh <= kDp && (kDp == 64 || kDp == 128 || kDp == 256), "row width");
  static_assert(kNK % 32 == 0 && kDmaPerWave >= 1 && (kTileB / 1024) % kWG == 0,
                "tiles in 1 KiB slices, evenly over the waves");
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(kG == 1 ? tid >> 6 : (tid >> 6) % kWG);
  const int kg = kG == 1 ? 0 : __builtin_amdgcn_readfirstlane((tid >> 6) / kWG);
  const int g = lane >> 5, l32 = lane & 31;
  uint8_t* const smem = smem_all + kg * 2 * kStageB;
  const int d = a.d, row_b = 2 * d, chunks_g = row_b / 16;

  // an XCD (workgroup i runs on XCD i % 8) takes a contiguous run of items
  const int per_xcd = (a.items + 7) / 8;
  const int item = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per_xcd || item >= a.items) return;
  const int head_sets = a.group / a.heads;
  // (through readfirstlane: the divisions are vector instructions, and a buffer resource
  // in vector registers costs a loop around its loads)
  const int kvh = __builtin_amdgcn_readfirstlane(item / (a.q_blocks * head_sets));
  const int rest = item - kvh * (a.q_blocks * head_sets);
  const int qb = a.q_blocks - 1 - __builtin_amdgcn_readfirstlane(rest / head_sets);   // the longest windows first
  // wave w: query head w % heads of the set, 32 queries w / heads of the block
  const int64_t head = (int64_t)kvh * a.group +
                       __builtin_amdgcn_readfirstlane(rest % head_sets * a.heads + (wave & (a.heads - 1)));
  const int64_t S = a.q_len;
  const int64_t q_off = head * S * d, kv_off = (int64_t)kvh * a.kv_len * d;
  const int heads_log2 = __builtin_ctz(a.heads);
  const int bq = kBQ >> heads_log2;       // queries of the block
  const int q0 = qb * bq;
  const int wq0 = q0 + (wave >> heads_log2) * 32;
  auto kswz = [](int r) { return kChunks == 8 ? ((r >> 1) & 7) : (r & 15); };
  auto vswz = [](int r) { return (kChunks == 8 ? 2 : 4) * (r & 3); };

  // ---- Q^T fragments; queries past the last read it and are not stored ----
  u32x4 qf[kKK];
  {
    const uint16_t* qrow = Q + q_off + min((int64_t)(wq0 + l32), S - 1) * d + 8 * g;
#pragma unroll
    for (int kk = 0; kk < kKK; ++kk) {
      u32x4 w = {0u, 0u, 0u, 0u};
      if (16 * kk + 8 * g < d) w = *reinterpret_cast<const u32x4*>(qrow + 16 * kk);
      qf[kk] = w;
    }
  }

  // ---- the list of key blocks ----
  const int kv_last = (int)a.kv_len - 1;
  const int win = (int)a.window;
  const int p0 = (int)(a.start + q0), p1 = (int)(a.start + min((int64_t)q0 + bq, S) - 1);
  const int lo0 = max(p0 - win + 1, 0);                // first key of the first query's window
  const int end = min(p1, kv_last);                    // last key of the last query
  const int blk0 = lo0 / kNK;
  const int n_win = end >= lo0 ? end / kNK - blk0 + 1 : 0;
  // (without window blocks every sink may count)
  const int sink_keys = (int)min(min(a.sinks, (int64_t)end + 1), a.kv_len);
  const int ns = n_win > 0 ? min((sink_keys + kNK - 1) / kNK, blk0) : (sink_keys + kNK - 1) / kNK;
  const int n_list = ns + n_win;
  auto block_of = [&](int i) { return i < ns ? i : i - ns + blk0; };   // also past the list: keys not seen
  // list entries that all queries see whole
  const int full_lo = max(p1 - win + 1, 0);
  const int whole0 = ns + max((full_lo + kNK - 1) / kNK - blk0, 0);
  const int whole1 = ns + max((min(p0, kv_last) + 1) / kNK - blk0, 0);   // one past the last
  // the wave's own queries
  const int pw0 = (int)(a.start + wq0), pw1 = pw0 + 31;
  auto wave_sees = [&](int i) {   // any key of entry i for any of the wave's queries
    const int k0 = block_of(i) * kNK;
    return i >= 0 && k0 <= min(pw1, kv_last) && (k0 + kNK - 1 > pw0 - win || k0 < (int)a.sinks);
  };

  // ---- LDS-DMA: as in flash_attn.hip; chunks past the row's data as zeros ----
  const int kv_bytes = (int)(a.kv_len * row_b);
  int k_voff[kDmaPerWave], v_voff[kDmaPerWave];
#pragma unroll
  for (int i = 0; i < kDmaPerWave; ++i) {
    const int row = kDmaRows * (wave + kWG * i) + lane / kChunks, pos = lane % kChunks;
    const int kc = pos ^ kswz(row), vc = pos ^ vswz(row);
    k_voff[i] = kc < chunks_g ? row * row_b + kc * 16 : kv_bytes;
    v_voff[i] = vc < chunks_g ? row * row_b + vc * 16 : kv_bytes;
  }
  const __amdgpu_buffer_rsrc_t k_rsrc =
      __builtin_amdgcn_make_buffer_rsrc((void*)(K + kv_off), (short)0, kv_bytes, 0x00020000);
  const __amdgpu_buffer_rsrc_t v_rsrc =
      __builtin_amdgcn_make_buffer_rsrc((void*)(V + kv_off), (short)0, kv_bytes, 0x00020000);
  const int list_end = max(n_list - 1, 0);
  // (an entry past the list loads the list's last block, whose scores are then masked)
  auto byte_of = [&](int j) { return block_of(min(j * kG + kg, list_end)) * kNK * row_b; };
  auto dma_k = [&](int j, int stage) {
    uint8_t* base = smem + stage * kStageB + wave * 1024;
    const int soff = byte_of(j);
#pragma unroll
    for (int i = 0; i < kDmaPerWave; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(k_rsrc, (lds_ptr_t)(base + i * kWG * 1024), 16,
                                               k_voff[i], soff, 0, 0);
  };
  auto dma_v = [&](int j, int stage) {
    uint8_t* base = smem + stage * kStageB + kTileB + wave * 1024;
    const int soff = byte_of(j);
#pragma unroll
    for (int i = 0; i < kDmaPerWave; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(v_rsrc, (lds_ptr_t)(base + i * kWG * 1024), 16,
                                               v_voff[i], soff, 0, 0);
  };

  const int kf_off = l32 * kRow, kf_swz = kswz(l32);
  auto k_frag = [&](const uint8_t* ks, int st, int kk) {
    return *reinterpret_cast<const u32x4*>(ks + 32 * st * kRow + (((2 * kk + g) ^ kf_swz) << 4));
  };
  const int tr_i = lane & 15, tr_s = (lane >> 4) & 1;
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
    const uint8_t* ks = smem + stage * kStageB + kf_off;
    zero_s(s);
#pragma unroll
    for (int st = 0; st < kST; ++st)
#pragma unroll
      for (int kk = 0; kk < kKK; ++kk) s[st] = mma32<kBF16>(k_frag(ks, st, kk), qf[kk], s[st]);
  };
  auto pv_block = [&](int stage, const u32x4 (&pf)[kPN], f32x16 (&oa)[kDT]) {
    const uint8_t* vs = smem + stage * kStageB + kTileB;
#pragma unroll
    for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
      for (int cc = 0; cc < kPN; ++cc) oa[dt] = mma32<kBF16>(v_frag(vs, dt, cc), pf[cc], oa[dt]);
  };
  // S_{j+1} and PV_{j-1}, a step of each at a time
  auto mma_block = [&](int stage, f32x16 (&s)[kST], const u32x4 (&pf)[kPN], f32x16 (&oa)[kDT]) {
    const uint8_t* ks = smem + stage * kStageB + kf_off;
    const uint8_t* vs = smem + stage * kStageB + kTileB;
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
  const float c = a.scale_log2;

  // iterations: the entries of a key group, rounded up to even
  int nb = (n_list + kG - 1) / kG;
  nb += nb & 1;
  if (nb > 0) {
    // Prologue: K_0, K_1 and a V tile in stage 1 for the empty PV_{-1}: it has to be
    // finite times zero, so P_{-1} = 0 meets V_0, whose NaN a seen row may well hold
    // only in a masked key; such rows are taken again in any case
    dma_k(0, 0);
    dma_k(1, 1);
    dma_v(0, 1);
    __syncthreads();
    f32x16 sa[kST], sb[kST];
    s_block(0, sa);
    __syncthreads();

    // The order of a region: fragment reads some steps ahead of the products that take
    // them, and the softmax spread between the products.  Up to head_dim 96 (4096 queries x 64
    // heads of 96, window 256: 66 -> 59 us); at 128, where it frees 40 registers, the compiler's own
    // order is 3 % faster.
    auto spread = [] {
      constexpr int kMfmas = 2 * kKK * kST, kReads = 3 * kKK * kST, kAhead = 3;
      constexpr int kValu = (48 * kST + kMfmas - 1) / kMfmas;
      __builtin_amdgcn_sched_group_barrier(sched::kDsRead, kAhead, 0);
#pragma unroll
      for (int i = 0; i < kMfmas; ++i) {
        __builtin_amdgcn_sched_group_barrier(sched::kMfma, 1, 0);
        __builtin_amdgcn_sched_group_barrier(sched::kValu, kValu, 0);
        if (kAhead + 3 * i / 2 < kReads) {
          if (i & 1)
            __builtin_amdgcn_sched_group_barrier(sched::kDsRead, 2, 0);
          else
            __builtin_amdgcn_sched_group_barrier(sched::kDsRead, 1, 0);
        }
      }
    };

    auto softmax_block = [&](int j, auto masked, f32x16 (&s)[kST], u32x4 (&pnew)[kPN]) {
      constexpr bool kMasked = decltype(masked)::value;
      if constexpr (kMasked) {
        const int e = j * kG + kg;
        const int kb = (e < n_list ? block_of(e) * kNK : 0x40000000) + 4 * g;
        const int p = pw0 + l32;
        const int hi = min(p, kv_last) - kb;   // key offsets > hi are not seen
        const int lo = p - win - kb;           // <= lo neither, unless
        const int sk = (int)a.sinks - kb;      // below sk
#pragma unroll
        for (int st = 0; st < kST; ++st)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int off = 32 * st + 8 * (i >> 2) + (i & 3);
            const bool in = off <= hi && (off > lo || off < sk);
            s[st][i] = in ? s[st][i] : -__builtin_inff();
          }
      }
      // fast path: P_j against the running max; a lane whose block sum is larger than
      // the limit, or NaN, sends the wave to the block-max update
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
      if constexpr (kDh <= 96) spread();
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
        // a query may have masked keys only so far: then every p is 0
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

    auto iteration = [&](int j, auto stage_c, auto masked, f32x16 (&scur)[kST], f32x16 (&snext)[kST],
                         const u32x4 (&pprev)[kPN], u32x4 (&pnew)[kPN]) {
      constexpr int kS = decltype(stage_c)::value;
      constexpr bool kMasked = decltype(masked)::value;
      dma_k(j + 2, kS);
      dma_v(j, kS);
      const int e = j * kG + kg;
      if (!kMasked || wave_sees(e - kG) || wave_sees(e) || wave_sees(e + kG)) {
        mma_block(kS ^ 1, snext, pprev, oacc);
        softmax_block(j, masked, scur, pnew);
      } else {
#pragma unroll
        for (int cc = 0; cc < kPN; ++cc) pnew[cc] = u32x4{0u, 0u, 0u, 0u};
      }
      // keep P_j and l in this region, beside the MFMAs
#pragma unroll
      for (int cc = 0; cc < kPN; ++cc) asm volatile("" : "+v"(pnew[cc]));
      asm volatile("" : "+v"(l_run));
      __syncthreads();
    };
    using Z = std::integral_constant<int, 0>;
    using One = std::integral_constant<int, 1>;
    // the pairs of iterations whose entries every query sees whole
    const int j0 = min((whole0 + 2 * kG - 1) / (2 * kG) * 2, nb), j1 = max(whole1 / (2 * kG) * 2, j0);
    auto masked_pairs = [&](int j, int to) {
      for (; j < to; j += 2) {
        iteration(j, Z{}, std::true_type{}, sa, sb, pa, pb);
        iteration(j + 1, One{}, std::true_type{}, sb, sa, pb, pa);
      }
    };
    masked_pairs(0, j0);
    for (int j = j0; j < j1; j += 2) {
      iteration(j, Z{}, std::false_type{}, sa, sb, pa, pb);
      iteration(j + 1, One{}, std::false_type{}, sb, sa, pb, pa);
    }
    masked_pairs(j1, nb);
    // PV of the last block (nb is even: P_{nb-1} is in pa, V_{nb-1} in stage 1)
    if (wave_sees((nb - 1) * kG + kg)) pv_block(1, pa, oacc);
  }

  // ---- key groups: groups 1 .. hand (m, l, O) to group 0 through LDS ----
  if constexpr (kG > 1) {
    constexpr int kRegs = 16 * kDT;
    __syncthreads();   // every read of the K and V stages is done
    float* part = reinterpret_cast<float*>(smem_all);
    auto slot = [&](int grp, int reg4) {
      return part + (((grp - 1) * kWG + wave) * (kRegs + 4) + 4 * reg4) * 64 + 4 * lane;
    };
    if (kg > 0) {
#pragma unroll
      for (int t = 0; t < kRegs / 4; ++t) {
        const int e = 4 * (t % 4);
        *reinterpret_cast<f32x4*>(slot(kg, t)) =
            f32x4{oacc[t / 4][e], oacc[t / 4][e + 1], oacc[t / 4][e + 2], oacc[t / 4][e + 3]};
      }
      *reinterpret_cast<f32x4*>(slot(kg, kRegs / 4)) = f32x4{m_run, l_run, 0.0f, 0.0f};
    }
    __syncthreads();
    if (kg > 0) return;
    float mg[kG], lg[kG];
    mg[0] = m_run;
    lg[0] = l_run;
    float m_all = m_run;
#pragma unroll
    for (int grp = 1; grp < kG; ++grp) {
      const f32x4 w = *reinterpret_cast<const f32x4*>(slot(grp, kRegs / 4));
      mg[grp] = w[0];
      lg[grp] = w[1];
      m_all = __builtin_fmaxf(m_all, mg[grp]);
    }
    // (a group without seen keys weighs nothing; a row without any has l = 0)
    auto weight = [&](float m) { return m == -__builtin_inff() ? 0.0f : exp2_fast((m - m_all) * c); };
    const float w0 = weight(mg[0]);
    l_run = lg[0] * w0;
#pragma unroll
    for (int dt = 0; dt < kDT; ++dt) oacc[dt] *= w0;
#pragma unroll
    for (int grp = 1; grp < kG; ++grp) {
      const float w = weight(mg[grp]);
      l_run += lg[grp] * w;
#pragma unroll
      for (int t = 0; t < kRegs / 4; ++t) {
        const f32x4 o4 = *reinterpret_cast<const f32x4*>(slot(grp, t));
#pragma unroll
        for (int e = 0; e < 4; ++e) oacc[t / 4][4 * (t % 4) + e] += o4[e] * w;
      }
    }
  }

  // ---- epilogue: O[q][d] = O^T[d][q] / l; rows that are not finite again ----
  const float l = pair32_sum(l_run);
  const float inv = 1.0f / l;
  const int q = wq0 + l32;
  float z = l * 0.0f;
#pragma unroll
  for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) z = __builtin_fmaf(oacc[dt][i] * inv, 0.0f, z);
  const uint64_t bad = __builtin_amdgcn_ballot_w64(!(z == 0.0f) && q < S);
  uint32_t rows = (uint32_t)bad | (uint32_t)(bad >> 32);   // query l32: bit l32
  const bool again = (rows >> l32) & 1;
  for (; rows; rows &= rows - 1) {
    const int64_t row = wq0 + __builtin_ctz(rows);
    int64_t sink_end, first, last;
    seen_range(a, a.start + row, &sink_end, &first, &last);
    window_row<kBF16>(Q + q_off + row * d, K + kv_off, V + kv_off, O + q_off + row * d, sink_end, first, last, d, c);
  }
  if (q >= S || again) return;
  uint16_t* orow = O + q_off + (int64_t)q * d;
#pragma unroll
  for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int dim = 32 * dt + 8 * r + 4 * g;
      if (dim >= d) continue;
      const f32x16& acc = oacc[dt];
      const u32x2 w = {pack2<kBF16>(acc[4 * r] * inv, acc[4 * r + 1] * inv),
                       pack2<kBF16>(acc[4 * r + 2] * inv, acc[4 * r + 3] * inv)};
      *reinterpret_cast<u32x2*>(orow + dim) = w;
    }
}

}  // namespace

#define SILE_FW_KERNEL(NAME, BF, W, EU, NK, DH, DP, G)                                  \
  extern "C" __global__ __launch_bounds__(W * 64, EU) void NAME(                        \
      const uint16_t* Q, const uint16_t* K, const uint16_t* V, uint16_t* O, WindowArgs a) { \
    __shared__ __attribute__((aligned(1024))) uint8_t smem[lds_bytes<NK, DH, DP, W, G>()]; \
    window_fwd<BF, W, NK, DH, DP, G>(Q, K, V, O, a, smem);                              \
  }
// d<D>: head dimensions up to D; g<N>: key groups
#define SILE_FW_DTYPES(W, EU, NK, DH, DP, G)                                          \
  SILE_FW_KERNEL(sile_flash_window_f16_d##DH##_g##G, false, W, EU, NK, DH, DP, G)     \
  SILE_FW_KERNEL(sile_flash_window_bf16_d##DH##_g##G, true, W, EU, NK, DH, DP, G)
#define SILE_FW_GROUPS(NK, DH, DP) \
  SILE_FW_DTYPES(4, 2, NK, DH, DP, 1) \
  SILE_FW_DTYPES(8, 2, NK, DH, DP, 2) \
  SILE_FW_DTYPES(8, 2, NK, DH, DP, 4)
SILE_FW_GROUPS(64, 32, 64)
SILE_FW_GROUPS(64, 64, 64)
SILE_FW_GROUPS(32, 96, 128)
SILE_FW_GROUPS(32, 128, 128)
SILE_FW_DTYPES(4, 1, 32, 192, 256, 1)
SILE_FW_DTYPES(4, 1, 32, 256, 256, 1)

// Any head dimension up to 256, alignment and scale: a wave a query row, and the next past the grid.
template <bool kBF16>
SILE_DEV void window_rowwise(const uint16_t* Q, const uint16_t* K, const uint16_t* V, uint16_t* O,
                             const WindowArgs& a, int64_t rows) {
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += (int64_t)gridDim.x * 4) {
    const int64_t head = r / a.q_len, i = r - head * a.q_len, kv = head / a.group * a.kv_len * a.d;
    int64_t sink_end, first, last;
    seen_range(a, a.start + i, &sink_end, &first, &last);
    window_row<kBF16>(Q + r * a.d, K + kv, V + kv, O + r * a.d, sink_end, first, last, a.d, a.scale_log2);
  }
}
extern "C" __global__ __launch_bounds__(256) void sile_flash_window_rowwise_f16(
    const uint16_t* Q, const uint16_t* K, const uint16_t* V, uint16_t* O, WindowArgs a, int64_t rows) {
  window_rowwise<false>(Q, K, V, O, a, rows);
}
extern "C" __global__ __launch_bounds__(256) void sile_flash_window_rowwise_bf16(
    const uint16_t* Q, const uint16_t* K, const uint16_t* V, uint16_t* O, WindowArgs a, int64_t rows) {
  window_rowwise<true>(Q, K, V, O, a, rows);
}
