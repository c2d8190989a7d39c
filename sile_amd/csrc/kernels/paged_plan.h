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

// A unit (a row's keys of one key head) counts kUnitTiles tiles more than it has: what a
// workgroup spends on its query, its first loads and its result, about a round of its waves.
// (64 rows of up to 4000 keys, 512 units of 1 to 125 tiles: without it the workgroups that had
// ten short units took 70 us, the others 28 to 55.)
constexpr int kUnitTiles = 4;
SILE_HD int32_t unit_size(const KeySpan& s) { return s.tiles > 0 ? s.tiles + kUnitTiles : 0; }

// The shares of a flat list of `total` tiles: equal ones, in whole rounds, for `groups`
// workgroups, which all run at once.  (Three quarters dealt so, and the rest in small
// shares to workgroups that start as the first end, was slower: one row of 131071 keys
// 100 -> 108 us, for the starts and the parts to join.)
struct Deal {
  int32_t share, total;
};
SILE_HD Deal make_deal(int32_t total, int32_t groups) {
  const int64_t per = ((int64_t)total + groups - 1) / groups;
  const int64_t share = (per + kTileWaves - 1) / kTileWaves * kTileWaves;
  return {(int32_t)(share < kTileWaves ? kTileWaves : share), total};
}
// Workgroups that any list of up to `total` tiles needs.
SILE_HD int32_t deal_workgroups(int64_t total, int32_t groups) {
  const int64_t n = (total + kTileWaves - 1) / kTileWaves;
  return (int32_t)(n < 1 ? 1 : n < groups ? n : groups);
}
SILE_HD int32_t deal_start(const Deal& d, int32_t w) {   // at most total
  const int64_t x = (int64_t)w * d.share;
  return (int32_t)(x < d.total ? x : d.total);
}
SILE_HD int32_t deal_workgroup(const Deal& d, int32_t x) { return x / d.share; }   // whose share holds tile x

}  // namespace sile
