// How the attention over a paged cache is cut into pieces: plain integer
// functions of the host and the device.
//
// Keys are taken 32 at a time (a tile: the depth of one 16x16x32 product).  A
// sequence's tiles run from the one of its first seen position to the one of
// its last.  Sequences of very different lengths share the device evenly when
// every piece has about the same number of tiles: the piece length follows
// from the batch's sum, each sequence takes as many pieces as it needs.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define SCOPE_HD __host__ __device__ __forceinline__
#else
#define SCOPE_HD inline
#endif

namespace scope {

constexpr int kTileKeys = 32;

// wavefronts of a piece's workgroup, which take its tiles in turn
constexpr int kAttnWaves = 4;

// A piece's least tiles: short rows wait less in more pieces (1100 positions of 8
// heads 10.0 us with 2, 12.2 with 4, 15.2 with 16; lists of nine blocks of 128 8.2,
// 8.6 and 11.3).
constexpr int kPieceTiles = 2;

// Workgroups aimed at.  The pieces of a ragged batch are not equal, and smaller ones
// even out its end (64 query heads over 24 sequences of 9k to 65k: 1536 272 us, 1024
// 281, 768 313; 48 windows of 4096 at D = 64 54.1 and 57.3; 32 sequences to 16k 58.9
// and 59.7; two to eight sequences of one length, which the host cannot tell, the
// other way by 0.5 to 3%).  One sequence's are equal (131k positions: 1024 93.5 us,
// 1536 96.0; 16k 22.8 and 23.9), and at D = 256 the partial rows are longer (16
// sequences to 16k: 1024 107 us, 1536 114; in whole turns of the wavefronts, which
// change nothing elsewhere, 102).
constexpr int kMostPieces = 1536;
SCOPE_HD int pieces_wanted(int B, int D) { return B == 1 || D == 256 ? 1024 : kMostPieces; }
SCOPE_HD int piece_turn(int D) { return D == 256 ? kAttnWaves : 1; }

// positions that a sequence of `len` holds in a table row of `cap`
SCOPE_HD int64_t seq_end(int64_t len, int64_t cap) { return len < 0 ? 0 : len < cap ? len : cap; }

// tiles of the seen positions [first, end); *lo: the first one
SCOPE_HD int seq_tiles(int64_t len, int64_t first, int64_t cap, int* lo) {
  const int64_t end = seq_end(len, cap);
  const int64_t from = first > 0 ? first : 0;
  *lo = 0;
  if (from >= end) return 0;
  *lo = static_cast<int>(from / kTileKeys);
  return static_cast<int>((end + kTileKeys - 1) / kTileKeys) - *lo;
}

// tiles of a piece at most, for a batch of `total` tiles and about `pieces` of them:
// `least`, or a multiple of `turn` above it (piece_range evens out a sequence's)
SCOPE_HD int64_t piece_tiles(int64_t total, int pieces, int least, int turn) {
  const int64_t c = (total + pieces - 1) / pieces, d = (c + turn - 1) / turn * turn;
  return c > least ? d : least;
}

// pieces of a sequence (one at least: it writes the zeros of an empty row).
// Over a batch they sum to at most `pieces` + its sequences; one sequence takes
// at most `pieces`.
SCOPE_HD int seq_pieces(int tiles, int64_t piece) {
  const int n = tiles <= piece ? 1 : static_cast<int>((tiles + piece - 1) / piece);
  return n;
}

// The pieces aimed at and the slots of a (key head, group of 16 query heads): what
// the grid and the workspace are made for.  With lists (of maxkv entries; 0: none)
// every list is cut into `pieces`.
struct SplitSizes {
  int pieces, slots;
  int64_t tiles_cap;  // tiles of a full table row (list)
  bool split;         // some sequence may take more than one piece
};
SCOPE_HD SplitSizes split_sizes(int B, int Hkv, int D, int bs, int MP, int Hq, int maxkv) {
  SplitSizes s;
  const int G = Hq / Hkv, ng = (G + 15) / 16, want = pieces_wanted(B, D);
  s.tiles_cap = (static_cast<int64_t>(maxkv ? maxkv : MP) * bs + kTileKeys - 1) / kTileKeys;
  const int64_t cols = static_cast<int64_t>(Hkv) * ng * (maxkv ? B : 1);
  const int64_t most = (s.tiles_cap + kPieceTiles - 1) / kPieceTiles;  // the shortest pieces of a full row
  const int64_t share = (want + cols - 1) / cols, pieces = maxkv && most < share ? most : share;
  s.split = most > 1 && pieces > 1;
  s.pieces = s.split ? static_cast<int>(pieces) : 1;
  // (the pieces of a batch are no more than those aimed at and one a sequence, nor
  // than the shortest ones that its table rows hold)
  const int64_t ragged = s.pieces + B < most * B ? s.pieces + B : most * B;
  s.slots = maxkv ? s.pieces * B : s.split ? static_cast<int>(ragged) : B;
  return s;
}

// tiles [*t0, *t1) of piece i of n
SCOPE_HD void piece_range(int lo, int tiles, int n, int i, int* t0, int* t1) {
  const int per = (tiles + n - 1) / n, a = per * i, b = per * (i + 1);
  *t0 = lo + (a < tiles ? a : tiles);
  *t1 = lo + (b < tiles ? b : tiles);
}

// page of block lb of a sequence, -1 where it has none
SCOPE_HD int64_t block_page(const int32_t* row, int MP, int64_t lb, int64_t P) {
  if (lb < 0 || lb >= MP) return -1;
  const int64_t page = row[lb];
  return page >= 0 && page < P ? page : -1;
}

// work-items that one dimension of a grid holds
constexpr int64_t kGridItems = (static_cast<int64_t>(1) << 32) - 1;

// rows of a wavefront that appends N of them, four wavefronts a workgroup: one while
// that leaves the device wavefronts to spare, two from 8192 on, and as many as the
// grid needs (up to 64, for 2^31 - 1)
SCOPE_HD int append_rows(int64_t N) {
  int rows = N >= 8192 ? 2 : 1;
  while ((N + 4 * rows - 1) / (4 * rows) * 256 > kGridItems) rows *= 2;
  return rows;
}

// where row i of the new ones goes: its sequence in *b and its position, -1 for
// a row of no sequence.  cu [B + 1] or null (row i to sequence i); whatever cu
// holds, *b stays in [0, B).
SCOPE_HD int64_t row_position(const int32_t* cu, const int32_t* lens, int B, int64_t i, int* b) {
  if (!cu) {
    *b = static_cast<int>(i);
    return static_cast<int64_t>(lens[i]);
  }
  int lo = 0, hi = B;  // the last b in [0, B) with cu[b] <= i, if cu does not decrease
  while (lo + 1 < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= i)
      lo = mid;
    else
      hi = mid;
  }
  *b = lo;
  if (i < cu[lo] || i >= cu[lo + 1]) return -1;
  return static_cast<int64_t>(lens[lo]) + (i - cu[lo]);
}

}  // namespace scope
