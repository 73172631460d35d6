// What the kernels of the paged cache share, over 16-bit and 8-bit pages (paged.hip)
// and over 4-bit ones (paged4.hip): steps over a wavefront's registers, the pieces
// of a batch, and the end of a piece.
#pragma once

#include <type_traits>

#include "attn_common.h"
#include "paged_plan.h"

namespace scope {

__device__ __forceinline__ float half_to_f32(uint16_t h) { return static_cast<float>(__builtin_bit_cast(_Float16, h)); }
__device__ __forceinline__ uint16_t f32_to_half(float f) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f)); }

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

// op over a wavefront in six steps on neighbouring lanes' registers (row shifts by
// 1, 2, 4, 8, then the rows' last lanes to the rows behind them): lane l gets the
// result over lanes 0 .. l.  A step costs a few cycles, one through LDS some sixty.
template <int CTRL, int ROWS, class Op>
__device__ __forceinline__ uint32_t lane_step(uint32_t v, uint32_t none, Op op) {
  return op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(static_cast<int>(none), static_cast<int>(v), CTRL, ROWS, 0xf, false)));
}
template <class Op>
__device__ __forceinline__ uint32_t lane_prefix(uint32_t v, uint32_t none, Op op) {
  v = lane_step<0x111, 0xf>(v, none, op);
  v = lane_step<0x112, 0xf>(v, none, op);
  v = lane_step<0x114, 0xf>(v, none, op);
  v = lane_step<0x118, 0xf>(v, none, op);
  v = lane_step<0x142, 0xa>(v, none, op);
  return lane_step<0x143, 0xc>(v, none, op);
}
__device__ __forceinline__ uint32_t add_u32(uint32_t a, uint32_t b) { return a + b; }
__device__ __forceinline__ uint32_t add_f32(uint32_t a, uint32_t b) {
  return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
}
__device__ __forceinline__ uint32_t max_f32(uint32_t a, uint32_t b) {
  return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
}
// op over the four lanes l % 16 + 16 k, or over two of them (k = 0, 1 and 2, 3): rows
// of 16 lanes and halves of 32 exchanged between two copies
template <class Op>
__device__ __forceinline__ float over_rows2(float v, Op op) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(op(r[0], r[1]));
}
template <class Op>
__device__ __forceinline__ float over_rows(float v, Op op) {
  const uint32_t x = __float_as_uint(over_rows2(v, op));
  const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return __uint_as_float(op(r[0], r[1]));
}
// the sums over lanes 0 .. l of a count
__device__ __forceinline__ int prefix_of(int v) { return static_cast<int>(lane_prefix(static_cast<uint32_t>(v), 0u, add_u32)); }

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint4 load_past(const uint4* p) {
  return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p)));
}
__device__ __forceinline__ void store_past(uint8_t* p, uint2 x) {
  __builtin_nontemporal_store(__builtin_bit_cast(u32x2_t, x), reinterpret_cast<u32x2_t*>(p));
}
__device__ __forceinline__ void store_past(uint16_t* p, uint4 x) {
  __builtin_nontemporal_store(__builtin_bit_cast(u32x4_t, x), reinterpret_cast<u32x4_t*>(p));
}

// ---- attention of one new token -------------------------------------------------
struct PagedAttnArgs {
  int Hq, maxkv;
  float scale;
  int64_t q_sb, q_sh;
  const uint16_t* q;
  const void* k_pages;
  const void* v_pages;
  const void* k_scale;  // of e4m3 pages [Hkv] fp32, of 4-bit ones their bytes
  const void* v_scale;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* first;
  const int32_t* kv_num;
  const int32_t* kv_idx;
  float* mass;
  uint16_t* out;
  float* lse;
};

// Workgroups of kAttnWaves wavefronts, one for each piece of the batch (paged_plan.h) and
// column (key head, group of 16 query heads): blockIdx.x and blockIdx.y over 16-bit and
// 8-bit pages; over 4-bit ones the columns of a piece come one after the other.
constexpr int kAttnThreads = 64 * kAttnWaves;

struct AttnSplit {
  int pieces, slots;   // pieces aimed at and slots of a (key head, group); with lists: pieces of every list
  int64_t tiles_cap;   // tiles of a full table row (list)
  float* po;           // [slots][Hq][D] partial P·V, unnormalised
  float* pml;          // [slots][Hq][2] their maxima (log2 units) and sums
  int2* plan;          // [B] (pieces, first slot) of each sequence
  float* lse2;         // [B][Hq] log2 of the whole sums of rows in one piece, for the mass
  float* tile_lse;     // [B][Hq][tiles_cap][halves] log2 of each tile's (half tile's) sum, for the mass
};

// piece i of n of sequence b: its tiles, and the sequence's first slot; the sequence's
// length and first position, as they were given
struct Piece {
  int b, t0, t1, i, n, slot, len, first;
};

// The piece of this workgroup, found by every wavefront for itself: the batch's
// tiles are summed, then the sequences' numbers of pieces.  false: there is none.
// wanted(tiles of the batch): how many pieces they are cut into, about.
template <class Wanted>
__device__ __forceinline__ bool find_piece(const scope_paged_cache& c, const PagedAttnArgs& a, int x, int turn, Wanted wanted,
                                           Piece& p) {
  const int lane = threadIdx.x & 63;
  const int64_t cap = static_cast<int64_t>(c.MP) * c.bs;
  const auto tiles_of = [&](int b, int* lo, int* len, int* first) {
    *lo = *len = *first = 0;
    if (b >= c.B) return 0;
    *len = a.lens[b];
    if (a.first) *first = a.first[b];
    return seq_tiles(*len, *first, cap, lo);
  };
  int lo0, len0, first0;
  const int tiles0 = tiles_of(lane, &lo0, &len0, &first0);
  // (64 sequences of less than 2^26 tiles: their sum fits 32 bits)
  int64_t total = static_cast<uint32_t>(__builtin_amdgcn_readlane(prefix_of(tiles0), 63));
  for (int b0 = 64; b0 < c.B; b0 += 64) {
    int lo, len, first;
    total += static_cast<uint32_t>(__builtin_amdgcn_readlane(prefix_of(tiles_of(b0 + lane, &lo, &len, &first)), 63));
  }
  const int64_t piece = piece_tiles(total, wanted(total), kPieceTiles, turn);
  int before = 0;
  for (int b0 = 0; b0 < c.B; b0 += 64) {
    int lo = lo0, len = len0, first = first0;
    const int tiles = b0 ? tiles_of(b0 + lane, &lo, &len, &first) : tiles0;
    const int n = b0 + lane < c.B ? seq_pieces(tiles, piece) : 0;
    const int upto = prefix_of(n);
    const uint64_t hit = __ballot(x < before + upto);
    if (hit) {
      const int at = __ffsll(static_cast<unsigned long long>(hit)) - 1;
      p.b = b0 + at;
      p.n = __builtin_amdgcn_readlane(n, at);
      p.slot = before + __builtin_amdgcn_readlane(upto, at) - p.n;
      p.i = x - p.slot;
      p.len = __builtin_amdgcn_readlane(len, at);
      p.first = __builtin_amdgcn_readlane(first, at);
      piece_range(__builtin_amdgcn_readlane(lo, at), __builtin_amdgcn_readlane(tiles, at), p.n, p.i, &p.t0, &p.t1);
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// two 16-bit values, rounded to nearest even
template <int TYPE>
__device__ __forceinline__ uint32_t round2(float lo, float hi) {
  if constexpr (TYPE == SCOPE_BF16) {
    return cvt_pk_bf16(lo, hi);
  } else {
    f16x2_t v;
    v[0] = static_cast<_Float16>(lo);
    v[1] = static_cast<_Float16>(hi);
    return __builtin_bit_cast(uint32_t, v);
  }
}

// the halves of a word of two 16-bit values
template <int TYPE>
__device__ __forceinline__ float low_half(uint32_t w) {
  return TYPE == SCOPE_BF16 ? __uint_as_float(w << 16) : half_to_f32(static_cast<uint16_t>(w));
}
template <int TYPE>
__device__ __forceinline__ float high_half(uint32_t w) {
  return TYPE == SCOPE_BF16 ? __uint_as_float(w & 0xffff0000u) : half_to_f32(static_cast<uint16_t>(w >> 16));
}

// The end of a piece: the wavefronts' maxima and sums (relative to those) in sm, sl
// [waves][16] and their outputs in so [waves][nq][D], in LDS, are joined and written, to
// the result where the piece is a sequence's only one.  vs: a factor on the outputs.
struct Shares {
  float *sm, *sl, *so;
};
__device__ __forceinline__ Shares shares_of(float* lds) { return {lds, lds + kAttnWaves * 16, lds + kAttnWaves * 32}; }

template <int TYPE, int D>
__device__ __forceinline__ void join_shares(const PagedAttnArgs& a, const AttnSplit& s, const Piece& p, int h0, int nq, float vs,
                                            const Shares& z) {
  const int b = p.b;
  for (int i = threadIdx.x; i < nq * D; i += kAttnThreads) {
    const int q = i / D, d = i % D, h = h0 + q;
    float M = z.sm[q];
#pragma unroll
    for (int w = 1; w < kAttnWaves; ++w) M = fmaxf(M, z.sm[w * 16 + q]);
    float L = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kAttnWaves; ++w) {
      // (a sum of 0 is a share without keys; a NaN stays one, whatever its maximum)
      const float f = z.sl[w * 16 + q] == 0.f ? 0.f : __builtin_amdgcn_exp2f(z.sm[w * 16 + q] - M);
      L += f * z.sl[w * 16 + q];
      o += f * z.so[(w * nq + q) * D + d];
    }
    if (p.n == 1) {
      const float y = L == 0.f ? 0.f : o / L * vs;
      a.out[(static_cast<int64_t>(b) * a.Hq + h) * D + d] = TYPE == SCOPE_FP16 ? f32_to_half(y) : f32_to_bf16(y);
      if (d == 0) {
        const float e = L == 0.f ? -INFINITY : M + __builtin_amdgcn_logf(L);
        a.lse[static_cast<int64_t>(b) * a.Hq + h] = e * kLn2;
        if (s.lse2) s.lse2[static_cast<int64_t>(b) * a.Hq + h] = e;
      }
    } else {
      const int64_t at = static_cast<int64_t>(p.slot + p.i) * a.Hq + h;
      s.po[at * D + d] = o;
      if (d == 0) {
        s.pml[2 * at] = M;
        s.pml[2 * at + 1] = L;
      }
    }
  }
}

inline bool aligned16(const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; }

// of paged.hip
int check_cache(const scope_paged_cache* c, const void* k_pages, const void* v_pages, const char* fn);
// The checks of an attention call beside those of its pages, and its pieces in *s.
int check_attn(const scope_paged_cache& c, const PagedAttnArgs& a, void* work, AttnSplit* s, const char* fn);
// What follows the pieces' kernel; v_scale: the factors [Hkv] of joined outputs, or null.
int launch_paged_finish(const scope_paged_cache& c, const PagedAttnArgs& a, const float* v_scale, const AttnSplit& s, hipStream_t st);

}  // namespace scope
