// The arithmetic of the paged cache that host and device share, without any
// memory access: which keys of a cached row its newest token sees, as tiles of
// 32 keys, and how the tiles of all rows are dealt to workgroups.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define SILE_HD __host__ __device__ __forceinline__
#else
#define SILE_HD inline
#endif

namespace sile {

constexpr int kTileKeys = 32;   // keys a wave takes at a time
constexpr int kTileWaves = 4;   // waves of a workgroup, a tile each a round

// The keys j < len that the token at position len - 1 sees: j >= first (the
// window) or j < sink_end.  Its tiles are those of the sinks, then those of the
// window; a tile that holds both is counted once.
struct KeySpan {
  int32_t len, first, sink_end;
  int32_t sink_tiles;   // tiles 0 .. sink_tiles - 1 of the row
  int32_t first_tile;   // then tiles first_tile ..
  int32_t tiles;        // all of them (0: no key)
};

// length: as it stands in the cache's lengths (negative counts as 0, past the
// row's capacity as the capacity); window <= 0: every key.
SILE_HD KeySpan key_span(int32_t length, int64_t capacity, int64_t window, int64_t sinks) {
  KeySpan s;
  const int64_t len = length < 0 ? 0 : length > capacity ? capacity : length;
  const int64_t first = window > 0 && window < len ? len - window : 0;
  const int64_t sink_end = sinks < 0 ? 0 : sinks < first ? sinks : first;
  s.len = (int32_t)len;
  s.first = (int32_t)first;
  s.sink_end = (int32_t)sink_end;
  s.first_tile = (int32_t)(first / kTileKeys);
  const int32_t sink_tiles = (int32_t)((sink_end + kTileKeys - 1) / kTileKeys);
  s.sink_tiles = sink_tiles < s.first_tile ? sink_tiles : s.first_tile;
  s.tiles = s.sink_tiles + (int32_t)((len + kTileKeys - 1) / kTileKeys) - s.first_tile;
  return s;
}

// The first key of tile t of the span.
SILE_HD int32_t span_key(const KeySpan& s, int32_t t) {
  return kTileKeys * (t < s.sink_tiles ? t : t - s.sink_tiles + s.first_tile);
}

SILE_HD bool span_sees(const KeySpan& s, int32_t key) {
  return key >= 0 && key < s.len && (key >= s.first || key < s.sink_end);
}

// The seen keys among the 32 from key0 on (a tile's first, below len), bit i key0 + i.
SILE_HD uint32_t span_bits(const KeySpan& s, int32_t key0) {
  const int32_t left = s.len - key0;
  uint32_t m = left >= 32 ? 0xffffffffu : (1u << left) - 1u;
  if (key0 < s.first) {
    const int32_t w = s.first - key0, e = s.sink_end - key0;
    const uint32_t in_window = w >= 32 ? 0u : 0xffffffffu << w;
    const uint32_t in_sinks = e <= 0 ? 0u : e >= 32 ? 0xffffffffu : (1u << e) - 1u;
    m &= in_window | in_sinks;
  }
  return m;
}

// Tiles a workgroup takes: an equal share of all tiles, at least one round of
// its waves, in whole rounds.
SILE_HD int32_t deal_chunk(int32_t total, int32_t workgroups) {
  const int32_t c = (total + workgroups - 1) / workgroups;
  return (c + kTileWaves - 1) / kTileWaves * kTileWaves > kTileWaves
             ? (c + kTileWaves - 1) / kTileWaves * kTileWaves
             : kTileWaves;
}

}  // namespace sile
