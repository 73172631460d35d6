"""CPU: the plan gives the wavefronts of these cases as many tiles as their tests are about."""
from __future__ import annotations

import os
import subprocess

import pytest

from tests.paged_fp4_tiles import FORMS, KINDS

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PLAN = r'''
#include <stdio.h>
#include <stdlib.h>
#include "%s/scope_amd/csrc/paged_plan.h"
using namespace scope;
// B Hkv Hq D bs MP maxkv resident, then B lengths and B first positions -> the pieces of each sequence and the tiles of
// its longest one
int main(int argc, char** argv) {
  int at = 1;
  const auto next = [&]() { return atoi(argv[at++]); };
  const int B = next(), Hkv = next(), Hq = next(), D = next(), bs = next(), MP = next(), maxkv = next(), resident = next();
  const SplitSizes s = split_sizes(B, Hkv, D, bs, MP, Hq, maxkv);
  const int cols = Hkv * ((Hq / Hkv + 15) / 16);
  int64_t total = 0;
  int lo, lens[64], first[64];
  for (int b = 0; b < B; ++b) lens[b] = next();
  for (int b = 0; b < B; ++b) first[b] = next();
  for (int b = 0; b < B; ++b) total += seq_tiles(lens[b], first[b], (int64_t)MP * bs, &lo);
  const int w = pieces_wanted4(total, cols, B, resident), n = w < s.pieces ? w : s.pieces;
  const int64_t piece = piece_tiles(total, n, kPieceTiles, piece_turn(D));
  for (int b = 0; b < B; ++b) {
    const int tiles = maxkv ? (int)s.tiles_cap : seq_tiles(lens[b], first[b], (int64_t)MP * bs, &lo);
    const int m = maxkv ? s.pieces : seq_pieces(tiles, piece);
    int longest = 0;
    for (int i = 0; i < m; ++i) {
      int t0, t1;
      piece_range(0, tiles, m, i, &t0, &t1);
      if (t1 - t0 > longest) longest = t1 - t0;
    }
    printf("%%d %%d\n", m, longest);
  }
  return 0;
}'''


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(PLAN % ROOT)
    subprocess.run(["g++", "-O1", "-std=c++17", str(d / "plan.cpp"), "-o", str(d / "plan")], check=True)

    def of(*numbers):
        out = subprocess.run([str(d / "plan"), *map(str, numbers)], check=True, capture_output=True, text=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]

    return of


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D,G,bs,dtype", FORMS)
def test_wavefronts_have_that_many_tiles(plan, kind, D, G, bs, dtype):
    k = KINDS[kind]
    B, MP, L = len(k["lens"]), max(-(-n // bs) for n in k["lens"]) + 1, -(-k["listed"] // bs) if "listed" in k else 0
    for resident in (256, 512, 768, 1024):
        got = plan(B, k["Hkv"], k["Hkv"] * G, D, bs, MP, L, resident, *k["lens"], *k.get("first", [0] * B))
        pieces, longest = zip(*got)
        assert max(-(-t // 4) for t in longest) >= k["most"] if G <= 16 or "pieces" not in k else True, got
        assert max(pieces) == (k.get("pieces", 1) if G <= 16 else 1), got
        if kind in ("ragged", "windows", "rising", "absent", "lists"):  # looked up more than once
            assert max(longest) > 256
        if kind == "ragged":  # wavefronts with none, with one and with every number up to five, before the long one
            assert sorted({-(-(t - w) // 4) for t in longest[:-1] for w in range(4)}) == [0, 1, 2, 3, 4, 5]
