"""The walk over the list of the paged attention of pieces where its starts fall, as a caller's mistake leaves
them: it ends, and every row, key block, part and page entry that it names is one of the call's."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = r"""
#include "PLAN_H"
using namespace sile;
struct Args { const int32_t *starts, *lengths; ChunkShape shape; int32_t tiles, kv_heads; };
extern "C" {
// s: n_tokens, capacity, window, sinks, n_rows, group, block, kv_heads.  -1: a walk that does not end; -2: a row,
// -3: a key block, -4: a key head, -5: a part, -6: a tile's place, -7: a sequence out of range; else how many shares were
// left before their end.  at_of: tiles + 1.
int32_t walk(const int32_t* starts, const int32_t* lengths, const int64_t* s, int32_t groups, int32_t* at_of) {
  Args a{starts, lengths, {s[0], s[1], s[2], s[3], (int32_t)s[4], (int32_t)s[5], (int32_t)s[6]}, 0, (int32_t)s[7]};
  a.tiles = (int32_t)chunk_tiles(s[0], s[4], s[5]);
  // (a thread of the kernel takes a run of tiles from a search of its own)
  const int32_t per = (a.tiles + 255) / 256;
  int64_t per_head = 0;
  int32_t bad = 0, left = 0;
  for (int32_t t0 = 0; t0 < a.tiles; t0 += per)
    chunk_run(a, t0, t0 + per < a.tiles ? t0 + per : a.tiles, [&](int32_t t, int32_t size, int32_t r, int32_t first, int32_t rows) {
      if (t < 0 || t >= a.tiles || size < 0) bad = -6;
      if (r < 0 || r >= a.shape.n_rows) bad = -7;
      const ChunkSeq q = load_seq(a, r);
      const int64_t row = (int64_t)q.start * a.shape.group + (int64_t)(t - first) * kChunkRows;
      if (rows > 0 && (row < 0 || row + rows > a.shape.n_tokens * a.shape.group)) bad = -2;
      if (!bad) at_of[t] = (int32_t)per_head;
      per_head += size;
    });
  if (bad) return bad;
  at_of[a.tiles] = (int32_t)per_head;
  const int64_t total = per_head * a.kv_heads, share = chunk_share(total, groups);
  for (int32_t w = 0; w < groups; ++w) {
    const int64_t x = w * share < total ? w * share : total, x1 = x + share < total ? x + share : total;
    if (x >= x1) continue;
    ChunkAt at{(int32_t)x, (int32_t)x1, 0, 0, (int32_t)(x / per_head), 0};
    for (int32_t t = 0; t < a.tiles; ++t)
      if (x % per_head >= at_of[t] && x % per_head < at_of[t + 1]) at.tile = t;
    at.seq = seq_of_tile(a, at.tile);
    at.base = (int32_t)(at.kvh * per_head + at_of[at.tile]);
    ChunkUnitAt u;
    int64_t guard = 0;
    while (next_unit(a, at, u)) {
      if (++guard > 4 * (total + a.tiles + 8)) return -1;
      if (at.kvh < 0 || at.kvh >= a.kv_heads) return -4;
      if (at.seq < 0 || at.seq >= a.shape.n_rows) return -7;
      if (at.tile < 0 || at.tile >= a.tiles) return -6;
      const int64_t row = (int64_t)u.seq.start * a.shape.group + (int64_t)(at.tile - u.first) * kChunkRows;
      if (u.tile.rows < 1 || u.tile.rows > kChunkRows || row < 0 || row + u.tile.rows > a.shape.n_tokens * a.shape.group) return -2;
      // (an own query row's token of the sequence)
      const int64_t packed = (int64_t)(at.tile - u.first) * kChunkRows + u.tile.rows - 1;
      if (packed / a.shape.group >= u.seq.tokens || u.tile.p1 >= u.seq.len) return -2;
      if (u.b0 < 0 || u.b1 > u.tile.blocks || u.b0 > u.b1) return -5;
      for (int32_t b = u.b0; b < u.b1; ++b) {
        const int64_t key = (int64_t)chunk_block(u.tile, b) * a.shape.block;
        if (key < 0 || key >= u.seq.len) return -3;
      }
    }
    left += at.x != at.x1;
  }
  return left;
}
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    d = tmp_path_factory.mktemp("bounds")
    src = d / "bounds.cpp"
    src.write_text(SOURCE.replace("PLAN_H", os.path.join(ROOT, "sile_amd", "csrc", "kernels", "chunk_plan.h")))
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-shared", "-fPIC", "-o",
                    str(d / "bounds.so"), str(src)], check=True)
    f = ctypes.CDLL(str(d / "bounds.so")).walk
    f.argtypes, f.restype = [ctypes.c_void_p] * 3 + [ctypes.c_int32, ctypes.c_void_p], ctypes.c_int32

    def call(starts, lengths, tokens, group, kv_heads, window, sinks, block, groups, capacity=4096):
        starts, lengths = np.array(starts, np.int32), np.array(lengths, np.int32)
        shape = np.array([tokens, capacity, window, sinks, len(lengths), group, block, kv_heads], np.int64)
        at = np.zeros(tokens * group // 128 + len(lengths) + 1, np.int32)
        return f(starts.ctypes.data, lengths.ctypes.data, shape.ctypes.data, groups, at.ctypes.data)
    return call


def test_starts_that_fall(walk):
    r = np.random.default_rng(1)
    left = 0
    for _ in range(1500):
        n = int(r.integers(1, 40))
        tokens = int(r.integers(1, 900))
        got = walk(r.integers(-50, tokens + 200, n + 1), r.integers(-5, 5000, n), tokens, int(r.choice([1, 3, 4, 24, 200])), int(r.integers(1, 4)),
                   int(r.choice([0, 0, 1, 100, 3000])), int(r.integers(0, 200)), int(r.choice([32, 64])), int(r.choice([8, 64, 512])))
        assert got >= 0, got
        left += got > 0
    assert left > 0   # (such lists do leave shares before their end)


def test_starts_that_rise(walk):
    """Every share is gone through to its end."""
    r = np.random.default_rng(2)
    for _ in range(500):
        n = int(r.integers(1, 40))
        new = r.integers(0, 60, n) * (r.random(n) < 0.7)
        starts = np.concatenate([[0], np.cumsum(new)]) + int(r.integers(0, 5))
        got = walk(starts, r.integers(-5, 5000, n), int(starts[-1]) + int(r.integers(0, 9)), int(r.choice([1, 3, 4, 24, 200])), int(r.integers(1, 4)),
                   int(r.choice([0, 0, 1, 100, 3000])), int(r.integers(0, 200)), int(r.choice([32, 64])), int(r.choice([8, 64, 512])))
        assert got == 0, got
