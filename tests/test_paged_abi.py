"""The paged cache's host side without a GPU: refusals come before any device work, and
the arithmetic that host and kernels share (tiles of a row, shares of the workgroups) is
compiled for the CPU and held against counting."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from sile_amd import _abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = r"""
#include "PLAN_H"
extern "C" {
void span(int32_t len, int64_t cap, int64_t window, int64_t sinks, int32_t* out) {
  const sile::KeySpan s = sile::key_span(len, cap, window, sinks);
  out[0] = s.len; out[1] = s.tiles; out[2] = s.sink_tiles; out[3] = s.first_tile;
}
// how often each key 0 .. n - 1 is covered by a tile and seen
void cover(int32_t len, int64_t cap, int64_t window, int64_t sinks, int32_t n, int32_t* out) {
  const sile::KeySpan s = sile::key_span(len, cap, window, sinks);
  for (int32_t t = 0; t < s.tiles; ++t)
    for (int32_t i = 0; i < sile::kTileKeys; ++i) {
      const int32_t key = sile::span_key(s, t) + i;
      const bool bit = (sile::span_bits(s, sile::span_key(s, t)) >> i) & 1;
      if (bit != sile::span_sees(s, key)) out[0] = -1000;
      if (bit && key < n) ++out[key];
    }
}
// the shares of a list; returns the workgroups that have one, -1 if a share's tiles do not name it
int32_t deal(int32_t total, int32_t groups) {
  const sile::Deal d = sile::make_deal(total, groups);
  const int32_t n = sile::deal_workgroups(total, groups);
  int32_t at = 0, used = 0;
  for (int32_t w = 0; w < n; ++w) {
    const int32_t x0 = sile::deal_start(d, w), x1 = sile::deal_start(d, w + 1);
    if (x0 != at || x1 < x0) return -1;
    if (x1 > x0) {
      ++used;
      if (sile::deal_workgroup(d, x0) != w || sile::deal_workgroup(d, x1 - 1) != w) return -1;
      if ((x1 - x0) % sile::kTileWaves && x1 != total) return -1;
    }
    at = x1;
  }
  return at == total ? used : -1;
}
int32_t workgroups(int64_t total, int32_t groups) { return sile::deal_workgroups(total, groups); }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    src = d / "plan.cpp"
    src.write_text(SOURCE.replace("PLAN_H", os.path.join(ROOT, "sile_amd", "csrc", "kernels", "paged_plan.h")))
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-shared", "-fPIC",
                    "-o", str(d / "plan.so"), str(src)], check=True)
    lib = ctypes.CDLL(str(d / "plan.so"))
    i32, i64 = ctypes.c_int32, ctypes.c_int64
    lib.span.argtypes = [i32, i64, i64, i64, ctypes.c_void_p]
    lib.cover.argtypes = [i32, i64, i64, i64, i32, ctypes.c_void_p]
    lib.deal.argtypes, lib.deal.restype = [i32, i32], i32
    lib.workgroups.argtypes, lib.workgroups.restype = [i64, i32], i32
    return lib


def test_tiles_cover_the_seen_keys_once(plan):
    r = np.random.default_rng(0)
    cases = [(n, w, s) for n in (0, 1, 31, 32, 33, 64, 100, 257) for w in (0, 1, 5, 32, 33, 100, 400)
             for s in (0, 1, 31, 32, 40, 300)]
    cases += [tuple(int(x) for x in r.integers(0, 700, 3)) for _ in range(300)]
    for n, w, s in cases:
        got = np.zeros(800, np.int32)
        plan.cover(n, 10 ** 9, w, s, 800, got.ctypes.data)
        want = np.zeros(800, np.int32)
        j = np.arange(n)
        want[j[(w <= 0) | (j >= n - w) | (j < s)]] = 1
        assert (got == want).all(), (n, w, s)


def test_lengths_are_held_to_the_table(plan):
    out = np.zeros(4, np.int32)
    for length, cap, want in ((-1, 64, 0), (-2 ** 31, 64, 0), (65, 64, 64), (2 ** 31 - 1, 48, 48), (5, 0, 0),
                              (2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1)):
        for w, s in ((0, 0), (7, 3), (2 ** 62, 2 ** 62), (1, 2 ** 62)):
            plan.span(length, cap, w, s, out.ctypes.data)
            assert out[0] == want and 0 <= out[1] <= want // 32 + 1


def test_shares_cover_the_tiles(plan):
    """Every tile in one share, the shares in order; never more workgroups than a larger
    list needs (the grid is sized for the largest)."""
    r = np.random.default_rng(1)
    for groups in (1, 3, 256, 512, 1024):
        totals = [0, 1, 3, 4, 5, groups * 4, groups * 4 + 1, groups * 47, groups * 48 - 1, groups * 48, groups * 48 + 1,
                  99999, 2 ** 30, 2 ** 31 - 2 ** 20] + [int(x) for x in r.integers(0, groups * 200, 50)]
        most = 0
        for total in sorted(totals):
            used = plan.deal(total, groups)
            assert 0 <= used <= plan.workgroups(total, groups) <= groups, (groups, total)
            assert plan.workgroups(total, groups) >= most
            most = plan.workgroups(total, groups)


P = 4096   # an aligned address that nothing reads
F16, BF16, F8, F32 = _abi.F16, _abi.BF16, _abi.F8E4M3, _abi.F32


def refused(name, args, code, needle):
    assert _abi.status(name, *args) == code, (_abi.last_error(), args)
    assert needle in _abi.last_error(), _abi.last_error()


APPEND = [F16, F16, 3, 2, 64, P, 128, P, 128, None, P, P, P, 10, 16, 2048, P, 4, 8, 1.0, 1.0, None]


@pytest.mark.parametrize("at,value,code,needle", [
    (0, F32, 2, "tokens of f32"), (1, BF16, 2, "under f16"), (1, F32, 2, "under f16"), (2, -1, 5, "negative"),
    (2, 2 ** 31, 5, "too many"), (3, 2 ** 15 + 1, 5, "too large"), (3, 0, 5, "cache shape"), (4, 0, 5, "cache shape"), (4, 264, 2, "head_dim > 256"), (4, 60, 2, "no multiple"),
    (5, None, 5, "NULL"), (5, P + 8, 5, "aligned"), (6, 120, 5, "leading dimension"), (6, 132, 5, "aligned"),
    (8, 127, 5, "leading dimension"), (10, None, 5, "NULL"), (11, P + 4, 5, "aligned"), (13, -1, 5, "cache shape"),
    (14, 24, 5, "power of two"), (14, 0, 5, "power of two"), (14, 131072, 5, "power of two"), (15, 2047, 5, "page_stride"),
    (15, 2052, 5, "page_stride"), (15, 2 ** 46, 5, "too large for"), (17, -1, 5, "negative"), (18, -1, 5, "negative"), (17, 2 ** 31, 5, "too large"),
    (18, 2 ** 30, 5, "too large")])
def test_append_refusals(at, value, code, needle):
    args = list(APPEND)
    args[at] = value
    refused("sile_hip_kv_append", args, code, needle)


def test_append_e4m3_needs_whole_chunks():
    args = list(APPEND)
    args[1], args[4] = F8, 72
    refused("sile_hip_kv_append", args, 2, "no multiple of 16")


def test_nothing_to_do_is_fine():
    """(no GPU is asked for)"""
    args = list(APPEND)
    args[2] = 0
    assert _abi.status("sile_hip_kv_append", *args) == 0
    assert _abi.status("sile_hip_kv_copy_pages", None, 0, 0, 0, 5, 3, P, P, None) == 0
    assert _abi.status("sile_hip_kv_free", 0, 4, None, None, None, None, None, 0, None, None, None) == 0
    assert _abi.status("sile_hip_kv_fork", 0, 0, 4, None, None, None, None, None, 0, None, None, None) == 0


DECODE = [F16, F16, 2, 4, 2, 64, P, 256, P, P, 10, 16, 2048, P, 8, P, P, 256, 0.1, 1.0, 1.0, 0, 0, P, 1 << 30, None]


@pytest.mark.parametrize("at,value,code,needle", [
    (0, F32, 2, "tokens of f32"), (1, BF16, 2, "under f16"), (2, -1, 5, "batch"), (3, 5, 5, "query heads"),
    (3, 0, 5, "query heads"), (5, 257, 2, "head_dim"), (6, None, 5, "NULL"), (6, P + 2, 5, "aligned"),
    (7, 255, 5, "leading dimension"), (7, 260, 5, "aligned"), (8, None, 5, "NULL"), (9, P + 8, 5, "aligned"),
    (11, 48, 5, "power of two"), (12, 8, 5, "page_stride"), (13, None, 5, "NULL"), (14, 2 ** 31, 5, "too large"),
    (15, None, 5, "NULL"), (16, P + 8, 5, "aligned"), (17, 100, 5, "leading dimension"), (21, -1, 5, "negative"),
    (22, -1, 5, "negative")])
def test_decode_refusals(at, value, code, needle):
    args = list(DECODE)
    args[at] = value
    refused("sile_hip_paged_attn_decode", args, code, needle)


TABLES = 1 << 20


@pytest.mark.parametrize("name,args,code,needle", [
    ("sile_hip_kv_copy_pages", [None, 1, 16, 16, 4, 1, P, P, None], 5, "NULL"),
    ("sile_hip_kv_copy_pages", [(ctypes.c_void_p * 1)(P), 129, 16, 16, 4, 1, P, P, None], 5, "pools"),
    ("sile_hip_kv_copy_pages", [(ctypes.c_void_p * 1)(P), 1, 8, 16, 4, 1, P, P, None], 5, "multiples of 16"),
    ("sile_hip_kv_copy_pages", [(ctypes.c_void_p * 1)(P), 1, 32, 16, 4, 1, P, P, None], 5, "multiples of 16"),
    ("sile_hip_kv_copy_pages", [(ctypes.c_void_p * 1)(P), 1, 16, 1 << 40, 1 << 20, 1, P, P, None], 5, "4 GiB"),
    ("sile_hip_kv_copy_pages", [(ctypes.c_void_p * 1)(P), 1, 1 << 33, 1 << 33, 4, 1, P, P, None], 5, "4 GiB"),
    ("sile_hip_kv_copy_pages", [(ctypes.c_void_p * 1)(P + 8), 1, 16, 16, 4, 1, P, P, None], 5, "aligned"),
    ("sile_hip_kv_copy_pages", [(ctypes.c_void_p * 1)(P), 1, 16, 16, 4, 1, None, P, None], 5, "NULL"),
    ("sile_hip_kv_copy_pages", [(ctypes.c_void_p * 1)(P), 1, 16, 16, 4, -1, P, P, None], 5, "copies"),
    ("sile_hip_kv_free", [4, 4, P, P, P + 4, P, P, 9, P, P, None], 5, "tables overlap"),
    ("sile_hip_kv_free", [4, 4, P, P, P, P, P + 4, 9, P, P, None], 5, "lengths overlap"),
    ("sile_hip_kv_free", [4, 4, P, P, P, P, P, 9, P, P + 4, None], 5, "counts overlap"),
    ("sile_hip_kv_free", [4, 4, None, P, P, P, P, 9, P, P, None], 5, "NULL"),
    ("sile_hip_kv_fork", [4, 4, 4, P, P, P, TABLES, 2 * TABLES, 9, P, P, None], 5, "must not overlap"),
    ("sile_hip_kv_fork", [4, 4, 4, P, TABLES, 2 * TABLES, P, P, 9, P, P, None], 5, "must not overlap"),
    ("sile_hip_kv_fork", [4, 2 ** 22 + 1, 1, P, TABLES, 2 * TABLES, P, P, 9, P, P, None], 5, "too large"),
    ("sile_hip_kv_workspace", [2 ** 22 + 1, 4, ctypes.byref(ctypes.c_size_t())], 5, "rows"),
    ("sile_hip_kv_fork", [-1, 4, 4, P, TABLES, 2 * TABLES, P, P, 9, P, P, None], 5, "negative"),
    ("sile_hip_kv_reserve", [4, 4, 3, P, P, P, P, 9, P, P, P, None, 0, 0, 0, P, 1 << 20, None], 5, "power of two"),
    ("sile_hip_kv_reserve", [4, 4, 16, P, P, P, P, 9, P, P, P, None, 0, 0, 0, None, 0, None], 5, "workspace"),
    ("sile_hip_kv_reserve", [4, 4, 16, P, P, P, P, 9, P, P, P, None, 0, 0, 0, P, 64, None], 5, "workspace"),
    ("sile_hip_kv_reserve", [4, 4, 16, P, P, P, P, 9, P, P, None, None, 0, 0, 0, P, 1 << 20, None], 5, "NULL"),
    ("sile_hip_kv_reserve", [4, 4, 16, P, P, P, P + 4, 9, P, P, P, None, 0, 0, 0, P, 1 << 20, None], 5, "tables overlap"),
    ("sile_hip_kv_compact", [4, 4, P, P, 9, P, P, None, None, 0, 0, 0, P, 1 << 20, None], 5, "NULL"),
    ("sile_hip_kv_compact", [4, 4, P, P, 9, P, P, P, None, 0, 0, 0, P + 4, 1 << 20, None], 5, "aligned"),
    ("sile_hip_kv_workspace", [-1, 4, ctypes.byref(ctypes.c_size_t())], 5, "rows"),
    ("sile_hip_kv_workspace", [4, 4, None], 5, "NULL"),
    ("sile_hip_paged_attn_workspace", [1, 5, 2, 64, ctypes.byref(ctypes.c_size_t())], 5, "query heads"),
])
def test_bookkeeping_refusals(name, args, code, needle):
    refused(name, args, code, needle)


APART = 1 << 24


@pytest.mark.parametrize("name,args,needle", [
    ("sile_hip_kv_free", [4, 4, P, APART, APART, P, P, 9, P, P, None], "drop overlaps"),
    ("sile_hip_kv_free", [4, 4, P + 60, P, P, APART, APART, 9, P, P, None], "drop overlaps"),
    ("sile_hip_kv_fork", [4, 4, 4, P, TABLES, 2 * TABLES, APART, P + 8, 9, P, P, None], "must not overlap"),
    ("sile_hip_kv_fork", [4, 4, 4, 2 * TABLES + 16, TABLES, 2 * TABLES, APART, P, 9, P, P, None],
     "must not overlap"),
    ("sile_hip_kv_reserve", [4, 4, 16, P, APART, P, P, 9, P, P, APART, None, 0, 0, 0, P, 1 << 20, None],
     "granted overlaps"),
    ("sile_hip_kv_reserve", [4, 4, 16, P, APART, P, P, 9, P, P, P + 4, None, 0, 0, 0, P, 1 << 20, None],
     "granted overlaps"),
])
def test_arrays_of_their_own_are_refused_when_they_overlap(name, args, needle):
    refused(name, args, 5, needle)


WINDOW = [F16, 2, 4, 2, 10, 20, 64, P, P, P, P, 0.125, 10, 5, 1, None]


@pytest.mark.parametrize("at,value,code,needle", [
    (0, F32, 2, "f32"), (1, -1, 5, "shape"), (3, 3, 5, "query heads"), (3, 0, 5, "query heads"), (4, -1, 5, "shape"),
    (6, 0, 5, "shape"), (6, 257, 2, "head_dim"), (7, None, 5, "NULL"), (8, None, 5, "NULL"), (10, None, 5, "NULL"),
    (12, -1, 5, "start"), (13, 0, 5, "window"), (14, -1, 5, "sinks"), (12, 2 ** 29, 5, "too long"), (5, 2 ** 24, 5, "too long"),
    (1, 2 ** 31, 5, "too large")])
def test_window_refusals(at, value, code, needle):
    args = list(WINDOW)
    args[at] = value
    refused("sile_hip_flash_attn_window_fwd", args, code, needle)


def test_window_without_queries_is_fine():
    for at in (1, 2, 4):
        args = list(WINDOW)
        args[at] = 0
        assert _abi.status("sile_hip_flash_attn_window_fwd", *args) == 0


@pytest.mark.parametrize("over,needle", [
    ({1: 1, 2: 64, 3: 1, 4: 2 ** 25 - 1}, "blocks of one key head"), ({2: 2 ** 15, 3: 2 ** 15, 4: 2 ** 16}, "too large"),
    ({4: 2 ** 29, 12: 1}, "too long"), ({5: 2 ** 29 + 1, 6: 1}, "too long")])
def test_window_limits(over, needle):
    args = list(WINDOW)
    for at, value in over.items():
        args[at] = value
    refused("sile_hip_flash_attn_window_fwd", args, 5, needle)


@pytest.mark.parametrize("over", [
    {2: 2 ** 21, 3: 8, 4: 4, 7: 512, 12: 4096, 17: 512},               # units: rows x key heads
    {2: 2 ** 21, 3: 129, 4: 1, 7: 129 * 64, 17: 129 * 64, 12: 1024},   # and groups of query heads
    {2: 2 ** 14, 14: 2 ** 16, 11: 64, 12: 8192}])                      # tiles of rows of 2^22 keys
def test_decode_limits(over):
    args = list(DECODE)
    for at, value in over.items():
        args[at] = value
    refused("sile_hip_paged_attn_decode", args, 5, "too many for one call")


def _apart():
    """(call, arguments far apart, i, j): array i moved into array j, for every pair of them that
    the call must not take: one of the two is written, and they are not the old and the new
    form of the same thing."""
    far = lambda n: n << 24  # noqa: E731
    t, n, p, ws = 16, 4, 9, 1 << 18   # elements: 4 x 4 tables, 4 rows, 9 pages, the workspace
    calls = {
        "sile_hip_kv_free": ([4, 4, far(2), far(3), far(4), far(5), far(6), 9, far(8), far(9), None],
                             {2: ("drop", n, 0), 3: ("tables", t, 0), 4: ("tables", t, 1), 5: ("lengths", n, 0),
                              6: ("lengths", n, 1), 8: ("counts", p, 0), 9: ("counts", p, 1)}),
        "sile_hip_kv_fork": ([4, 4, 4, far(3), far(4), far(5), far(6), far(7), 9, far(9), far(10), None],
                             {3: ("src", n, 0), 4: ("tables", t, 0), 5: ("tables", t, 1), 6: ("lengths", n, 0),
                              7: ("lengths", n, 1), 9: ("counts", p, 0), 10: ("counts", p, 1)}),
        "sile_hip_kv_reserve": ([4, 4, 16, far(3), far(4), far(5), far(6), 9, far(8), far(9), far(10), None, 0, 0, 0, far(15),
                                 4 * ws, None],
                                {3: ("lengths", n, 0), 4: ("need", n, 0), 5: ("tables", t, 0), 6: ("tables", t, 1),
                                 8: ("counts", p, 0), 9: ("counts", p, 1), 10: ("granted", n, 1), 15: ("workspace", 16, 1)}),
        "sile_hip_kv_compact": ([4, 4, far(2), far(3), 9, far(5), far(6), far(7), None, 0, 0, 0, far(12), 4 * ws, None],
                                {2: ("tables", t, 0), 3: ("tables", t, 1), 5: ("counts", p, 0), 6: ("counts", p, 1),
                                 7: ("used", 1, 1), 12: ("workspace", 16, 1)})}
    for name, (args, arrays) in calls.items():
        for i, (what, _, written) in arrays.items():
            for j, (other, size, written_j) in arrays.items():
                if what != "workspace" and what != other and (written or written_j):
                    for at in sorted({0, size - 1}):
                        yield pytest.param(name, args, i, args[j] + 4 * at, id=f"{name[9:]}-{what}{i}-{other}{j}-{at}")


@pytest.mark.parametrize("name,args,i,address", _apart())
def test_arrays_that_a_call_writes_lie_apart(name, args, i, address):
    args = list(args)
    args[i] = address
    refused(name, args, 5, "overlap")
