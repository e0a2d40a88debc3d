"""How a ragged batch is cut into key tiles and work items (csrc/bfa_paged.h): built for
the host and compared with enumeration, broken offsets and page ids among the inputs."""
from __future__ import annotations

import ctypes
import random
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "braidinfer_amd" / "csrc"
SOURCE = r"""
#include "bfa_paged.h"
using namespace bfa;
extern "C" {
int seq(const int* in, long long tokens, long long indices, int ps, int* out) {
  bool bad;
  PagedSeq s = paged_seq(in[0], in[1], in[2], in[3], in[4], tokens, indices, ps, bad);
  out[0] = s.q0; out[1] = s.qlen; out[2] = s.page0; out[3] = s.npages; out[4] = s.kvlen;
  return bad;
}
long long page(long long id, long long pages) { return paged_page(id, pages); }
int tiles(int first, int last, int kvlen, int window, int sinks, int tile, int* out) {
  KeyTiles k = paged_key_tiles(first, last, kvlen, paged_shape(16, 1, tile, window, sinks));
  for (int i = 0; i < k.count && i < 4096; ++i) out[i] = k.at(i);
  return k.count;
}
int split(int qlen, int kvlen, int group, int bm, int window, int sinks, int tile, int* blocks) {
  PagedSeq s{0, qlen, 0, 0, kvlen};
  PagedSplit p = paged_split(s, paged_shape(bm, group, tile, window, sinks));
  *blocks = p.blocks;
  return p.tiles;
}
int chunks(int blocks, int tiles, int per) { return PagedSplit{blocks, tiles}.chunks(per); }
int even(int tiles, int chunks) { return paged_even(tiles, chunks); }
int work(int blocks, int tiles, int shift) { return paged_work(PagedSplit{blocks, tiles}, shift); }
int items(int blocks, int tiles, int per) { return paged_items(PagedSplit{blocks, tiles}, per); }
int add(int a, int b) { return paged_add(a, b); }
int line(int item, int items, int row0, int n, int all, long long rows, int bm) {
  return paged_line_inside(item, items, row0, n, all, rows, bm);
}
int per_item(int work, int shift, int target, int least) { return paged_per_item(work, shift, target, least); }
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    d = tmp_path_factory.mktemp("paged_plan")
    (d / "plan.cpp").write_text(SOURCE)
    subprocess.run([cxx, "-O1", "-std=c++17", "-shared", "-fPIC", f"-I{CSRC}", str(d / "plan.cpp"), "-o",
                    str(d / "plan.so")], check=True)
    lib = ctypes.CDLL(str(d / "plan.so"))
    lib.page.restype = ctypes.c_longlong
    lib.page.argtypes = [ctypes.c_longlong] * 2
    lib.line.argtypes = [ctypes.c_int] * 5 + [ctypes.c_longlong, ctypes.c_int]
    lib.seq.argtypes = [ctypes.c_void_p, ctypes.c_longlong, ctypes.c_longlong, ctypes.c_int, ctypes.c_void_p]
    return lib


def seq(lib, *given, tokens=100, indices=50, ps=16):
    a, out = (ctypes.c_int * 5)(*given), (ctypes.c_int * 5)()
    bad = lib.seq(a, tokens, indices, ps, out)
    return bool(bad), list(out)


def test_requests_inside_the_arrays(lib):
    assert seq(lib, 0, 4, 0, 3, 7) == (False, [0, 4, 0, 3, 39])
    assert seq(lib, 96, 100, 49, 50, 16) == (False, [96, 4, 49, 1, 16])
    assert seq(lib, 5, 5, 7, 7, 0) == (False, [5, 0, 7, 0, 0])
    assert seq(lib, 5, 6, 7, 8, 0) == (False, [5, 1, 7, 1, 0])


@pytest.mark.parametrize("given,cut", [
    ((-1, 4, 0, 3, 7), [0, 0, 0, 3, 39]), ((5, 4, 0, 3, 7), [0, 0, 0, 3, 39]), ((0, 101, 0, 3, 7), [0, 0, 0, 3, 39]),
    ((0, 4, -1, 3, 7), [0, 4, 0, 0, 0]), ((0, 4, 3, 2, 7), [0, 4, 0, 0, 0]), ((0, 4, 0, 51, 7), [0, 4, 0, 0, 0]),
    ((0, 4, 0, 3, 17), [0, 4, 0, 3, 48]), ((0, 4, 0, 3, -2), [0, 4, 0, 3, 32]),
    ((-2 ** 31, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 2 ** 31 - 1), [0, 0, 0, 0, 0])])
def test_broken_offsets_leave_nothing_outside(lib, given, cut):
    assert seq(lib, *given) == (True, cut)


def test_page_ids(lib):
    assert [lib.page(i, 5) for i in (0, 4, -1, -5, 5, -6, 2 ** 31 - 1, -2 ** 31)] == [0, 4, 4, 0, -1, -1, -1, -1]
    assert lib.page(0, 0) == -1


def visible(p, j, window, sinks):
    return j <= p and (window == 0 or p - j < window or j < sinks)


def key_tiles(lib, *args):
    out = (ctypes.c_int * 4096)()
    n = lib.tiles(*args, out)
    return list(out[:n])


def test_key_tiles_hold_every_visible_key_once(lib):
    rng = random.Random(1)
    for _ in range(3000):
        tile = rng.choice([32, 64])
        kvlen = rng.choice([0, 1, rng.randint(1, 900)])
        last = rng.randint(-3, max(kvlen - 1, 0))
        first = last - rng.choice([0, 0, 3, rng.randint(0, 200)])
        window = rng.choice([0, 1, rng.randint(1, 300), 2 ** 31 - 1])
        sinks = rng.choice([0, 1, 4, rng.randint(0, 200), 2 ** 31 - 1])
        got = key_tiles(lib, first, last, kvlen, window, sinks, tile)
        assert got == sorted(set(got)) and all(0 <= t * tile < max(kvlen, 1) for t in got)
        rows = range(first, last + 1)
        need = {j // tile for j in range(kvlen) if any(visible(p, j, window, sinks) for p in (rows if len(rows) < 40 else (
            first, last, *rng.sample(list(rows), 20))))}
        assert need <= set(got), (first, last, kvlen, window, sinks, tile)
        if last < 0 or kvlen == 0:
            assert got == []
    # a window keeps a long cache's walk short, and the largest values do not overflow
    assert key_tiles(lib, 100000, 100000, 100001, 64, 4, 32) == [0, 3123, 3124, 3125]
    assert key_tiles(lib, 2 ** 31 - 2, 2 ** 31 - 2, 2 ** 31 - 1, 1, 0, 64) == [(2 ** 31 - 2) // 64]


def test_items_cover_every_block(lib):
    """A block's key tiles never exceed what its items were counted for, and items of all
    requests stay within the grid's bound."""
    rng = random.Random(2)
    for _ in range(400):
        bm, tile = rng.choice([(16, 32), (16, 64), (64, 64), (128, 64)])
        group = rng.choice([1, 2, 3, 4, 5, 8, 16, 71])
        window, sinks = rng.choice([0, rng.randint(1, 300)]), rng.choice([0, 4, rng.randint(0, 130)])
        requests = []
        for _ in range(rng.randint(1, 6)):
            kvlen = rng.randint(0, 700)
            requests.append((rng.randint(0, min(kvlen + 2, 90)), kvlen))
        plans, shift = [], rng.choice([0, 0, 1, 3])
        for qlen, kvlen in requests:
            blocks = ctypes.c_int()
            tiles = lib.split(qlen, kvlen, group, bm, window, sinks, tile, ctypes.byref(blocks))
            assert blocks.value == -(-qlen * group // bm)
            for b in range(blocks.value):
                r0, r1 = b * bm, min((b + 1) * bm, qlen * group) - 1
                base = kvlen - qlen
                assert len(key_tiles(lib, base + r0 // group, base + r1 // group, kvlen, window, sinks, tile)) <= tiles
            plans.append((blocks.value, tiles))
        total = 0
        for b, t in plans:
            total = lib.add(total, lib.work(b, t, shift))
        target, least = rng.randint(1, 40), rng.choice([1, 2, 4])
        per = lib.per_item(total, shift, target, least)
        items = sum(lib.items(b, t, per) for b, t in plans)
        assert per >= least and items <= target + sum(b for b, _ in plans)
        assert all(lib.chunks(b, t, per) * per >= t for b, t in plans)
        for _, t in plans:
            c = lib.chunks(1, t, per)
            assert t <= lib.even(t, c) * c and (c == 1 or lib.even(t, c) <= per)
        rows = sum(q for q, _ in requests) * group
        assert sum(b for b, _ in plans) <= min(rows, rows // bm + len(requests))
    assert lib.even(0, 1) == 0 and lib.even(2 ** 31 - 1, 1) == 2 ** 31 - 1 and lib.even(7, 3) == 3
    assert lib.chunks(1, 0, 4) == 1 and lib.chunks(1, 2 ** 31 - 1, 2 ** 31 - 1) == 1


def test_sums_of_broken_requests_do_not_overflow(lib):
    most = 0x3fffffff
    assert lib.work(2 ** 27, 2 ** 26, 0) == most and lib.work(8192, 2 ** 26, 10) == 8192 * 2 ** 16
    assert lib.items(2 ** 27, 2 ** 26, 1) == most and lib.add(most, most) == most and lib.add(most, 5) == most
    assert lib.per_item(most, 0, 1, 2) == most and lib.per_item(most, 20, 1, 2) == most
    assert lib.per_item(0, 0, 300, 4) == 4 and lib.per_item(8192 * 2 ** 16, 10, 320, 4) == most  # (-> 1.7e9 tiles)
    assert lib.per_item(2 ** 20, 10, 320, 4) == -(-2 ** 20 // 320) * 1024


def test_lines_of_the_merge_stay_inside(lib):
    """The table's line of a block that no item filled holds anything."""
    assert lib.line(0, 4, 0, 16, 4, 16, 16) and lib.line(3, 1, 16, 0, 4, 16, 16)
    for bad in [(-1, 2, 0, 16), (0, 5, 0, 16), (3, 2, 0, 16), (0, -1, 0, 16), (0, 4, -1, 16), (0, 4, 1, 16), (0, 4, 0, 17),
                (0, 4, 0, -1), (2**31 - 1, 2**31 - 1, 0, 16), (-2**31, 2, 0, 16), (0, 2, 2**31 - 1, 16)]:
        assert not lib.line(*bad, 4, 16, 16), bad
