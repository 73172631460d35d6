"""CPU: the paged attention's grid and workspace hold the pieces that its wavefronts
find, with the kernel's own constants (paged_plan.h compiled for the host)."""
from __future__ import annotations

import ctypes as C
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "scope_amd", "libscope_amd.so")
needs_lib = pytest.mark.skipif(not os.path.exists(LIB), reason="libscope_amd.so not built")

PLAN = r'''
#include "%s/scope_amd/csrc/paged_plan.h"
using namespace scope;
extern "C" {
void sizes(int B, int Hkv, int D, int bs, int MP, int Hq, int maxkv, int64_t* o) {
  const SplitSizes s = split_sizes(B, Hkv, D, bs, MP, Hq, maxkv);
  o[0] = s.pieces, o[1] = s.slots, o[2] = s.tiles_cap, o[3] = s.split, o[4] = kMostPieces;
}
// as every wavefront finds its piece: the batch's sum, then the sequences' pieces in order; returns
// the pieces, or -1 where one is not a range of its sequence's tiles or they do not cover them
int64_t found(int B, int D, int64_t cap, const int32_t* lens, const int32_t* first, int pieces, int* most) {
  int64_t total = 0, n_all = 0;
  int lo;
  for (int b = 0; b < B; ++b) total += seq_tiles(lens[b], first[b], cap, &lo);
  const int64_t piece = piece_tiles(total, pieces, kPieceTiles, piece_turn(D));
  *most = 0;
  for (int b = 0; b < B; ++b) {
    const int tiles = seq_tiles(lens[b], first[b], cap, &lo), n = seq_pieces(tiles, piece);
    int at = lo;
    for (int i = 0; i < n; ++i) {
      int t0, t1;
      piece_range(lo, tiles, n, i, &t0, &t1);
      if (t0 != at || t1 < t0) return -1;
      at = t1;
    }
    if (at != lo + tiles) return -1;
    n_all += n;
    *most = n > *most ? n : *most;
  }
  return n_all;
}
int rows_each(int64_t N) { return append_rows(N); }
int list_range(int tiles_cap, int pieces) {
  int at = 0;
  for (int i = 0; i < pieces; ++i) {
    int t0, t1;
    piece_range(0, tiles_cap, pieces, i, &t0, &t1);
    if (t0 != at || t1 < t0) return 0;
    at = t1;
  }
  return at == tiles_cap;
}
}
'''


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(PLAN % ROOT)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    str(d / "plan.cpp"), "-o", str(d / "plan.so")], check=True)
    lib = C.CDLL(str(d / "plan.so"))
    lib.found.restype, lib.found.argtypes = C.c_int64, [C.c_int, C.c_int, C.c_int64, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p]
    lib.rows_each.restype, lib.rows_each.argtypes = C.c_int, [C.c_int64]
    lib.sizes.restype, lib.sizes.argtypes = None, [C.c_int] * 7 + [C.c_void_p]
    return lib


def sizes(plan, *a):
    o = (C.c_int64 * 5)()
    plan.sizes(*a, o)
    return tuple(o)


def drawn(r):
    Hkv, G = r.choice([1, 2, 3, 8, 64, 4096]), r.choice([1, 4, 8, 15, 16, 17, 33, 128])
    bs = r.choice([16, 32, 64, 128, 256])
    MP = r.choice([1, 2, 3, 4, 9, 1027, 8192, (2 ** 31 - 32) // bs])
    return r.choice([1, 1, 2, 3, 5, 64, 65, 200, 3000]), Hkv, r.choice([64, 128, 256]), bs, MP, Hkv * G


@pytest.mark.parametrize("seed", range(120))
def test_slots_hold_every_piece_that_is_found(plan, seed):
    r = random.Random(seed)
    B, Hkv, D, bs, MP, Hq = drawn(r)
    pieces, slots, cap, split, most = sizes(plan, B, Hkv, D, bs, MP, Hq, 0)
    assert cap == -(-MP * bs // 32) and pieces >= 1 and (split or (pieces == 1 and slots == B))
    for kind in range(4):
        top = MP * bs
        lens = [{0: top, 1: r.randint(0, top), 2: int(top ** r.random()), 3: r.choice([0, 0, 0, top, 2 ** 31 - 1, -3])}[kind]
                for _ in range(B)]
        first = [0 if kind != 2 else r.choice([0, n // 2, n - 1, n + 5, -9]) for n in lens]
        n = C.c_int()
        got = plan.found(B, D, top, (C.c_int32 * B)(*lens), (C.c_int32 * B)(*first), pieces, C.byref(n))
        assert B <= got <= slots, f"{got} pieces in {slots} slots"
        assert n.value <= most and (split or n.value == 1)


@pytest.mark.parametrize("seed", range(60))
def test_lists_have_a_slot_for_every_piece(plan, seed):
    r = random.Random(seed)
    B, Hkv, D, bs, MP, Hq = drawn(r)
    maxkv = r.choice([1, 2, 3, 9, 64, 1000, (2 ** 31 - 1) // bs])
    pieces, slots, cap, split, most = sizes(plan, B, Hkv, D, bs, MP, Hq, maxkv)
    assert cap == -(-maxkv * bs // 32) and slots == pieces * B and 1 <= pieces <= most and bool(split) == (pieces > 1)
    assert plan.list_range(cap, pieces)


@needs_lib
@pytest.mark.parametrize("seed", range(60))
def test_the_workspace_holds_the_slots(plan, seed):
    """Partial rows and sums of every slot, the plan, and with a mass every tile's sums."""
    from scope_amd import _lib

    lib = _lib.load()
    r = random.Random(seed)
    B, Hkv, D, bs, MP, Hq = drawn(r)
    for maxkv in (0, 9):
        _, slots, cap, split, _ = sizes(plan, B, Hkv, D, bs, MP, Hq, maxkv)
        up = lambda x: -(-x // 16) * 16  # noqa: E731
        want = up(4 * slots * Hq * D) + up(8 * slots * Hq) + up(8 * B) if split else 0
        c = _lib.PagedCache(B, Hkv, D, bs, MP)
        assert lib.scope_paged_attn_workspace_bytes(C.byref(c), Hq, maxkv, 0) == want
        want += up(4 * B * Hq) + up(4 * B * Hq * cap * (2 if bs == 16 else 1))
        assert lib.scope_paged_attn_workspace_bytes(C.byref(c), Hq, maxkv, 1) == want


def test_appended_rows_fit_a_grid(plan):
    """A launch holds less than 2^32 work-items; a wavefront places up to 64 rows."""
    edges = [1, 8191, 8192, 2 ** 27 - 8, 2 ** 27 - 7, 2 ** 27, 2 ** 28, 2 ** 29 - 1, 2 ** 30 + 1, 2 ** 31 - 1]
    for n in edges + [random.Random(i).randint(1, 2 ** 31 - 1) for i in range(200)]:
        rows = plan.rows_each(n)
        assert 1 <= rows <= 64 and -(-n // (4 * rows)) * 256 < 2 ** 32
    assert [plan.rows_each(n) for n in (8191, 8192, 2 ** 27 - 8, 2 ** 27 - 7)] == [1, 2, 2, 4]
