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

// tiles of a piece, for a batch of `total` tiles and about `pieces` of them: a
// multiple of `turn`, `least` at least
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
