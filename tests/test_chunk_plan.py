"""The arithmetic of the paged attention of pieces of prompts, which host and kernels share, compiled for
the CPU and held against counting: every query row of every key head has each block of its keys in
exactly one part, parts have slots of their own, and the join finds them."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = r"""
#include <cstring>
#include "PLAN_H"
using namespace sile;
struct Args { const int32_t *starts, *lengths; ChunkShape shape; int32_t tiles, kv_heads; };
static Args args(const int32_t* starts, const int32_t* lengths, const int64_t* s) {
  Args a{starts, lengths, {s[0], s[1], s[2], s[3], (int32_t)s[4], (int32_t)s[5], (int32_t)s[6]}, 0, (int32_t)s[7]};
  a.tiles = (int32_t)chunk_tiles(s[0], s[4], s[5]);
  return a;
}
extern "C" {
// seen[(head, query row of the list)][block] counts the blocks that the parts have of each row, parts[slot]
// their uses, zeros[..] the rows of tiles without keys.  s: n_tokens, capacity, window, sinks, n_rows,
// group, block, kv_heads; returns the total, -1 on a walk that does not end.
int32_t walk(const int32_t* starts, const int32_t* lengths, const int64_t* s, int32_t groups, int32_t blocks,
             int32_t* seen, int32_t* parts, int32_t* zeros, int32_t* at_of) {
  const Args a = args(starts, lengths, s);
  int64_t per_head = 0;
  chunk_run(a, 0, a.tiles, [&](int32_t t, int32_t size, auto...) { at_of[t] = (int32_t)per_head; per_head += size; });
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
    int32_t guard = 0;
    while (next_unit(a, at, u)) {
      if (++guard > 100000) return -1;
      const bool whole = u.b0 == 0 && u.b1 >= u.tile.blocks;
      if (!whole) ++parts[2 * w + (u.b0 == 0 ? 1 : 0)];
      for (int32_t r = 0; r < u.tile.rows; ++r) {
        const int64_t row = (int64_t)u.seq.start * a.shape.group + (int64_t)(at.tile - u.first) * kChunkRows + r;
        const int64_t of = (int64_t)at.kvh * a.shape.n_tokens * a.shape.group + row;
        if (u.tile.blocks == 0) ++zeros[of];
        for (int32_t b = u.b0; b < u.b1; ++b) ++seen[of * blocks + chunk_block(u.tile, b)];
      }
    }
    if (at.x != at.x1) return -1;
  }
  return (int32_t)total;
}
// blocks of each tile that all of its tokens see whole
void whole(const int32_t* starts, const int32_t* lengths, const int64_t* s, int32_t t, int32_t* out) {
  const Args a = args(starts, lengths, s);
  const int32_t r = seq_of_tile(a, t);
  const ChunkSeq q = load_seq(a, r);
  const ChunkTile tl = chunk_tile(a.shape, q, t - chunk_base(a.shape, q.start, r));
  out[0] = tl.rows; out[1] = tl.p0; out[2] = tl.p1; out[3] = tl.blocks;
  chunk_whole(a.shape, tl, out + 4, out + 5);
  for (int32_t e = 0; e < tl.blocks && e < 1000; ++e) out[6 + e] = chunk_block(tl, e);
}
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("chunk")
    src = d / "plan.cpp"
    src.write_text(SOURCE.replace("PLAN_H", os.path.join(ROOT, "sile_amd", "csrc", "kernels", "chunk_plan.h")))
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-shared", "-fPIC",
                    "-o", str(d / "plan.so"), str(src)], check=True)
    lib = ctypes.CDLL(str(d / "plan.so"))
    p, i32 = ctypes.c_void_p, ctypes.c_int32
    lib.walk.argtypes, lib.walk.restype = [p, p, p, i32, i32, p, p, p, p], i32
    lib.whole.argtypes = [p, p, p, i32, p]
    return lib


def run(plan, new, lengths, group, kv_heads, window, sinks, block, groups, pad=0, capacity=4096, starts=None):
    n = len(new)
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32) if starts is None else np.array(starts, np.int32)
    lengths = np.array(lengths, np.int32)
    tokens = int(max(starts.max(), 0)) + pad
    shape = np.array([tokens, capacity, window, sinks, n, group, block, kv_heads], np.int64)
    blocks = capacity // block + 1
    tiles = tokens * group // 128 + n
    rows = kv_heads * tokens * group
    seen, zeros = np.zeros((rows, blocks), np.int32), np.zeros(rows, np.int32)
    parts, at = np.zeros(2 * groups, np.int32), np.zeros(tiles + 1, np.int32)
    total = plan.walk(starts.ctypes.data, lengths.ctypes.data, shape.ctypes.data, groups, blocks, seen.ctypes.data,
                      parts.ctypes.data, zeros.ctypes.data, at.ctypes.data)
    return total, seen.reshape(kv_heads, tokens, group, blocks), zeros.reshape(kv_heads, tokens, group), parts, at, shape, starts, lengths


CASES = [([1], [1], 1, 1, 0, 0), ([5], [300], 4, 2, 0, 0), ([1] * 40, list(range(0, 4000, 100)), 4, 1, 0, 0),
         ([700], [700], 3, 1, 0, 0), ([300, 1, 0, 77, 2], [900, 50, 10, 77, 4000], 5, 2, 0, 0),
         ([200, 30], [1000, 2000], 4, 1, 100, 4), ([64, 64], [4000, 3000], 2, 1, 33, 300), ([10], [4], 4, 1, 0, 0),
         ([0, 0, 3], [5, 0, 1], 8, 1, 0, 0), ([130, 1], [130, 1], 1, 3, 1, 0), ([400], [500], 1, 1, 128, 40),
         ([3, 3], [5000, -2], 24, 1, 0, 0)]


@pytest.mark.parametrize("block", [32, 64])
@pytest.mark.parametrize("groups", [8, 64, 512])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_every_block_of_every_row_once(plan, case, groups, block):
    new, lengths, group, kv_heads, window, sinks = CASES[case]
    total, seen, zeros, parts, at, shape, starts, lens = run(plan, new, lengths, group, kv_heads, window, sinks, block, groups, pad=3)
    assert total >= 0 and (parts <= 1).all()
    for r, n in enumerate(new):
        length = min(max(lengths[r], 0), 4096)
        for i in range(n):
            p = length - n + i
            t = starts[r] + i
            j = np.arange(max(p + 1, 0))
            keys = j if window <= 0 else j[(j > p - window) | (j < sinks)]
            got = seen[:, t]
            need = np.zeros(got.shape[-1], bool)
            need[np.unique(keys // block)] = True
            assert (got <= 1).all() and (got[..., need] == 1).all()
            assert ((zeros[:, t] == 1) | (got.sum(-1) > 0)).all()
    assert (seen[:, starts[-1]:] == 0).all() and (zeros[:, starts[-1]:] == 0).all()


def test_whole_blocks(plan):
    """Blocks taken without a mask are seen whole by every token of the tile."""
    r = np.random.default_rng(0)
    for _ in range(400):
        n, group, block = int(r.integers(1, 300)), int(r.integers(1, 9)), int(r.choice([32, 64]))
        length = int(r.integers(0, 4000))
        window = int(r.choice([0, 0, 1, 50, 200, 1000]))
        sinks = int(r.integers(0, 100))
        shape = np.array([n, 4096, window, sinks, 1, group, block, 1], np.int64)
        starts, lengths = np.array([0, n], np.int32), np.array([length], np.int32)
        for t in range(n * group // 128 + 1):
            out = np.zeros(1100, np.int32)
            plan.whole(starts.ctypes.data, lengths.ctypes.data, shape.ctypes.data, t, out.ctypes.data)
            rows, p0, p1, blocks, w0, w1 = out[:6]
            for e in range(max(w0, 0), min(w1, blocks)):
                k0 = out[6 + e] * block
                assert k0 + block - 1 <= p0 and (window == 0 or k0 > p1 - window), (n, group, length, window, sinks, t)


def test_starts_that_fall(plan):
    """Nonsense in the list ends: no walk past the key heads, no row out of range."""
    r = np.random.default_rng(1)
    for _ in range(200):
        n = int(r.integers(1, 12))
        starts = r.integers(-50, 300, n + 1)
        got = run(plan, [0] * n, r.integers(-5, 5000, n), int(r.integers(1, 6)), 2, 0, 0, 32, 64, starts=starts, pad=5)
        assert got[0] >= -1
