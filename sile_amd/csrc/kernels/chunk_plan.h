// The arithmetic of the paged attention of pieces of prompts that host and device share, with
// no memory access but the step's token list: tiles of query rows, the key blocks each sees, and
// how they are dealt to workgroups.
#pragma once

#include "paged_plan.h"

namespace sile {

// A tile is kChunkRows query rows of one key head: the tokens of a sequence times the query
// heads that share the key head, packed token by token.
constexpr int kChunkRows = 128;
// A unit (a tile of a key head) counts kChunkUnit key blocks more than it has: its start and end.
constexpr int kChunkUnit = 4;
constexpr int kChunkShare = 4;   // blocks that a workgroup has at least

struct ChunkShape {
  int64_t n_tokens, capacity, window, sinks;   // capacity at most 2^29; window 0: none
  int32_t n_rows, group, block;                // block: keys of a key block
};

// The new tokens of a sequence: `tokens` of them from `start` of the list on, the last at
// position len - 1.
struct ChunkSeq {
  int32_t start, tokens, len;
};
SILE_HD int32_t chunk_clamp(int32_t v, int64_t most) { return v < 0 ? 0 : v > most ? (int32_t)most : v; }
SILE_HD ChunkSeq chunk_seq(const ChunkShape& s, int32_t start, int32_t end, int32_t length) {
  ChunkSeq q;
  q.start = chunk_clamp(start, s.n_tokens);
  q.tokens = chunk_clamp(end, s.n_tokens) - q.start;
  if (q.tokens < 0) q.tokens = 0;
  q.len = chunk_clamp(length, s.capacity);
  return q;
}

// Numbers of the tiles: those of sequence r are chunk_base(start of r) .. , one number for each of
// its tiles and at most one more, which is empty.  (floor(b) - floor(a) + 1 >= ceil(b - a).)
SILE_HD int32_t chunk_base(const ChunkShape& s, int32_t start, int32_t r) {
  return (int32_t)((int64_t)start * s.group / kChunkRows) + r;
}
SILE_HD int64_t chunk_tiles(int64_t n_tokens, int64_t n_rows, int64_t group) {
  return n_tokens * group / kChunkRows + n_rows;
}

// Tile i of a sequence: `rows` query rows (0: none) of the tokens t0 .. t1 at positions p0 .. p1
// (below 0: a token without any key), and its key blocks: those of the sinks, then those from
// the first token's window to the last token's own key.
struct ChunkTile {
  int32_t rows, t0, p0, p1;
  int32_t sink_blocks, first_block, blocks;
};
SILE_HD ChunkTile chunk_tile(const ChunkShape& s, const ChunkSeq& q, int32_t i) {
  ChunkTile t;
  const int64_t m = (int64_t)q.tokens * s.group - (int64_t)i * kChunkRows;
  t.rows = m <= 0 || i < 0 ? 0 : m < kChunkRows ? (int32_t)m : kChunkRows;
  t.t0 = t.p0 = t.p1 = t.sink_blocks = t.first_block = t.blocks = 0;
  if (t.rows == 0) return t;
  t.t0 = (int32_t)((int64_t)i * kChunkRows / s.group);
  const int32_t t1 = (int32_t)(((int64_t)i * kChunkRows + t.rows - 1) / s.group);
  t.p0 = q.len - q.tokens + t.t0;
  t.p1 = q.len - q.tokens + t1;
  if (t.p1 < 0) return t;
  int64_t lo = s.window > 0 ? (int64_t)t.p0 - s.window + 1 : 0;
  if (lo < 0) lo = 0;
  t.first_block = (int32_t)(lo / s.block);
  const int64_t sinks = s.window <= 0 ? 0 : s.sinks < t.p1 + 1 ? s.sinks : t.p1 + 1;
  const int64_t sink_blocks = (sinks + s.block - 1) / s.block;
  t.sink_blocks = (int32_t)(sink_blocks < t.first_block ? sink_blocks : t.first_block);
  t.blocks = t.sink_blocks + t.p1 / s.block - t.first_block + 1;
  return t;
}
SILE_HD int32_t chunk_block(const ChunkTile& t, int32_t e) {
  return e < t.sink_blocks ? e : e - t.sink_blocks + t.first_block;
}
// Blocks that every one of the tile's tokens sees whole: entries whole0 .. whole1 - 1 of its list.
SILE_HD void chunk_whole(const ChunkShape& s, const ChunkTile& t, int32_t* whole0, int32_t* whole1) {
  int64_t lo = s.window > 0 ? (int64_t)t.p1 - s.window + 1 : 0;
  if (lo < 0) lo = 0;
  const int32_t first = (int32_t)((lo + s.block - 1) / s.block) - t.first_block;
  const int32_t last = (t.p0 + 1 > 0 ? (t.p0 + 1) / s.block : 0) - t.first_block;
  *whole0 = t.sink_blocks + (first > 0 ? first : 0);
  *whole1 = t.sink_blocks + (last > 0 ? last : 0);
}
// What a unit counts.
SILE_HD int32_t chunk_size(const ChunkTile& t) { return t.rows > 0 ? t.blocks + kChunkUnit : 0; }

// What the attention's launch leaves of a tile for the one that joins its parts: the blocks before
// it, its sequence, that one's first tile, and its rows.
struct ChunkRec {
  int32_t at, seq, first, rows;
};

// The shares of `total` blocks for `groups` workgroups.
SILE_HD int64_t chunk_share(int64_t total, int32_t groups) {
  const int64_t per = (total + groups - 1) / groups;
  return per < kChunkShare + kChunkUnit ? kChunkShare + kChunkUnit : per;
}

// ---- walking the list ----
// A: starts, lengths (the step's, in device memory), shape, tiles (of a key head, empty ones
// counted) and kv_heads of a call.

// A value that all lanes have, in a scalar register (loads and divisions are vector instructions,
// and what they give is kept through a workgroup's key blocks).
SILE_HD int32_t sgpr(int32_t v) {
#ifdef __HIP_DEVICE_COMPILE__
  return __builtin_amdgcn_readfirstlane(v);
#else
  return v;
#endif
}

// the last sequence whose tiles begin at or before tile t
template <class A>
SILE_HD int32_t seq_of_tile(const A& a, int32_t t) {
  int32_t lo = 0, hi = a.shape.n_rows;   // base(lo) <= t < base(hi)
  while (hi - lo > 1) {   // (in nine parts: their loads do not wait for one another)
    const int32_t step = (hi - lo + 8) / 9, from = lo;
    for (int32_t i = 1; i < 9; ++i) {
      const int32_t r = from + i * step < hi ? from + i * step : hi - 1;
      if (chunk_base(a.shape, chunk_clamp(a.starts[r], a.shape.n_tokens), r) <= t && r > lo) lo = r;
    }
    hi = lo + step < hi ? lo + step : hi;
  }
  return lo;
}
template <class A>
SILE_HD ChunkSeq load_seq(const A& a, int32_t r) {
  return chunk_seq(a.shape, a.starts[r], a.starts[r + 1], a.lengths[r]);
}

// Where a workgroup is in the list: unit (kvh, tile), a tile of sequence seq, begins at base.
struct ChunkAt {
  int32_t x, x1, base;
  int32_t tile, kvh, seq;
};
// The next unit of the share that has anything to do: its blocks b0 .. b1 - 1 are this workgroup's.
struct ChunkUnitAt {
  ChunkSeq seq;
  ChunkTile tile;
  int32_t first;    // number of the sequence's first tile
  int32_t b0, b1;
};
template <class A>
SILE_HD bool next_unit(const A& a, ChunkAt& at, ChunkUnitAt& u) {
  while (at.x < at.x1) {
    if (at.tile >= a.tiles) {   // the next key head
      ++at.kvh;
      at.tile = 0;
      at.seq = 0;
      if (at.kvh >= a.kv_heads) return false;   // (a list whose starts fall)
    }
    u.seq = load_seq(a, at.seq);
    u.seq = {sgpr(u.seq.start), sgpr(u.seq.tokens), sgpr(u.seq.len)};
    u.first = sgpr(chunk_base(a.shape, u.seq.start, at.seq));
    if (at.seq + 1 < a.shape.n_rows &&
        at.tile >= sgpr(chunk_base(a.shape, chunk_clamp(a.starts[at.seq + 1], a.shape.n_tokens), at.seq + 1))) {
      ++at.seq;
      continue;
    }
    u.tile = chunk_tile(a.shape, u.seq, at.tile - u.first);
    u.tile = {sgpr(u.tile.rows), sgpr(u.tile.t0), sgpr(u.tile.p0), sgpr(u.tile.p1),
              sgpr(u.tile.sink_blocks), sgpr(u.tile.first_block), sgpr(u.tile.blocks)};
    const int32_t size = chunk_size(u.tile);
    if (size == 0 || at.x >= at.base + size) {
      at.base += size;
      ++at.tile;
      continue;
    }
    const int32_t u0 = at.x - at.base, u1 = size < u0 + (at.x1 - at.x) ? size : u0 + (at.x1 - at.x);
    at.x += u1 - u0;
    u.b0 = u0 > kChunkUnit ? u0 - kChunkUnit : 0;
    u.b1 = u1 - kChunkUnit;
    // (else of this unit only what it counts extra; a tile without keys is its last workgroup's)
    if (u.b1 > u.b0 || (u.tile.blocks == 0 && u1 == size)) return true;
  }
  return false;
}

// visit(t, size of tile t, its sequence, that one's first tile, tile t's rows) for c0 <= t < c1, in order
template <class A, class F>
SILE_HD void chunk_run(const A& a, int32_t c0, int32_t c1, F&& visit) {
  if (c0 >= c1) return;
  int32_t r = seq_of_tile(a, c0);
  ChunkSeq q = load_seq(a, r);
  int32_t first = chunk_base(a.shape, q.start, r);
  for (int32_t t = c0; t < c1; ++t) {
    while (r + 1 < a.shape.n_rows) {
      const int32_t next = chunk_base(a.shape, chunk_clamp(a.starts[r + 1], a.shape.n_tokens), r + 1);
      if (next > t) break;
      ++r;
      q = load_seq(a, r);
      first = next;
    }
    const ChunkTile tile = chunk_tile(a.shape, q, t - first);
    visit(t, chunk_size(tile), r, first, tile.rows);
  }
}

}  // namespace sile
