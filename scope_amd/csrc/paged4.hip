// The paged cache in 4 bits: rows quantised as they are written, the attention of
// one new token over such pages, and rows read back out of pages of any type.
//
// A row's D features go in groups of 32 to e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and
// their negatives), two a byte with the even feature in the low nibble, and one e8m0
// byte a group that stands for 2^(byte - 127), 255 for NaN: the MXFP4 format of the
// Open Compute Project, which gfx950 converts in one instruction for two values.
// Pages are [P][Hkv][bs][D/2] bytes (any page, head and row strides), scales
// [P][Hkv][bs][D/32] (any page and head strides).
#include <math.h>

#include <algorithm>

#include "paged_attn.h"

namespace scope {

namespace {
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));

// the lane's value and those of the other lanes of its quad, op over all four
template <class Op>
__device__ __forceinline__ uint32_t over_quad(uint32_t v, Op op) {
  v = op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0xb1, 0xf, 0xf, true)));
  return op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x4e, 0xf, 0xf, true)));
}
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a), __builtin_bit_cast(u16x2_t, b)));
}

// the scale of an e8m0 byte, as the conversions take it: they read bits 23 .. 30 alone
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }
}  // namespace

// ---- rows in and out -----------------------------------------------------------
// N rows of Hkv·D / 8 chunks of eight features, `rows` of them to a wavefront, chunks
// dealt to its lanes in turn: lane r < rows finds the place of row i0 + r.
struct MoveArgs {
  int64_t N;
  int rows, chunks, skip_rows, skip_chunks;  // 64 = skip_rows · chunks + skip_chunks
  const int32_t* cu;
  const int32_t* table;
};

// page (-1: none) and slot of row i, `from` [B] (NULL: 0) the position of a sequence's
// first one, `to` [B] (NULL: the table's end) the end of its positions
__device__ __forceinline__ int2 row_place(const scope_paged_cache& c, const MoveArgs& m, const int32_t* from, const int32_t* to,
                                          int64_t i) {
  int b;
  const int64_t pos = row_position(m.cu, from, c.B, i, &b), cap = static_cast<int64_t>(c.MP) * c.bs;
  if (pos < 0 || pos >= (to ? seq_end(to[b], cap) : cap)) return make_int2(-1, 0);
  const int64_t page = block_page(m.table + static_cast<int64_t>(b) * c.MP, c.MP, pos / c.bs, c.P);
  return make_int2(static_cast<int>(page), static_cast<int>(pos % c.bs));
}

// f(row of the wavefront, chunk, page, slot) for every chunk of this wavefront's n rows
// that has a lane; places: those that row_place gave the first n lanes.
template <class F>
__device__ __forceinline__ void each_chunk(const MoveArgs& m, int n, int2 places, F f) {
  const int lane = threadIdx.x & 63;
  int r = lane / m.chunks, e = lane % m.chunks;
  for (int at = 0; at < n * m.chunks; at += 64) {  // (all lanes go on to the end: others take their places from them)
    const int page = __shfl(places.x, min(r, 63)), slot = __shfl(places.y, min(r, 63));
    if (r < n) f(r, e, page, slot);
    r += m.skip_rows;
    e += m.skip_chunks;
    if (e >= m.chunks) {
      e -= m.chunks;
      ++r;
    }
  }
}

// Rows written: a quad of lanes has a group of 32 features, so that its largest value
// takes two steps in registers, and every lane moves 16 bytes in and 4 out.  Bound by
// memory: 65539 rows of 8 heads of 128 (340 MB) 66.5 us, 5.1 TB/s, as a large copy (four
// rows a wavefront instead of two, or none passing the caches, 5 to 20 us more).
struct Append4Args {
  int64_t k_sn, k_sh, v_sn, v_sh;
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* lens;
  uint8_t* k_pages;
  uint8_t* v_pages;
  uint8_t* k_scale;
  uint8_t* v_scale;
};

// Eight values of a group of 32 that a quad of lanes holds as e2m1 codes; *byte: its
// scale.  With 2^x the power of two below the largest |value| a the scale is 2^(x - 2),
// or 2^(x - 1) where a >= 1.75 · 2^x: a is at most 7 of it, which becomes 6, so that no
// value is off by more than half a step of the grid (codes are rounded to nearest
// even).  Adding a quarter to a's significand carries into its exponent just there.
// The scale stays where all codes of it are finite in the rows' type and no code is
// subnormal in fp32; larger values become 6 of it, smaller ones 0.  A group with an
// infinity or a NaN gets the scale NaN and codes 0.
template <int TYPE>
__device__ __forceinline__ uint32_t e2m1x8(const uint4& u, uint32_t* byte) {
  constexpr uint32_t kAbs = 0x7fff7fffu, kInf = TYPE == SCOPE_FP16 ? 0x7c00u : 0x7f80u, kTop = TYPE == SCOPE_FP16 ? 140 : 252;
  uint32_t m = max_u16x2(max_u16x2(u.x & kAbs, u.y & kAbs), max_u16x2(u.z & kAbs, u.w & kAbs));
  m = over_quad(m, max_u16x2);
  m = max(m & 0xffffu, m >> 16);
  if (m >= kInf) {
    *byte = 255;
    return 0;
  }
  const float a = TYPE == SCOPE_FP16 ? half_to_f32(static_cast<uint16_t>(m)) : bf16_to_f32(static_cast<uint16_t>(m));
  const uint32_t e = (__float_as_uint(a) + 0x200000u) >> 23;
  *byte = min(max(e, 4u) - 2u, kTop);
  const float s = scale_of(*byte);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  uint32_t o = 0;
  if constexpr (TYPE == SCOPE_FP16) {
    o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, __builtin_bit_cast(f16x2_t, w[0]), s, 0);
    o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, __builtin_bit_cast(f16x2_t, w[1]), s, 1);
    o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, __builtin_bit_cast(f16x2_t, w[2]), s, 2);
    o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, __builtin_bit_cast(f16x2_t, w[3]), s, 3);
  } else {
    o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(bf16x2_t, w[0]), s, 0);
    o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(bf16x2_t, w[1]), s, 1);
    o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(bf16x2_t, w[2]), s, 2);
    o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(bf16x2_t, w[3]), s, 3);
  }
  return o;
}

template <int TYPE>
__global__ __launch_bounds__(256) void paged_append4_kernel(scope_paged_cache c, scope_paged_scales z, MoveArgs m, Append4Args a) {
  const int lane = threadIdx.x & 63;
  const int64_t i0 = (static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6)) * m.rows;
  int2 place = make_int2(-1, 0);
  if (lane < m.rows && i0 + lane < m.N) place = row_place(c, m, a.lens, nullptr, i0 + lane);
  const int dshift = __builtin_ctz(c.D) - 3;
  const int n = static_cast<int>(min(static_cast<int64_t>(m.rows), m.N - i0));
  each_chunk(m, n, place, [&](int r, int e, int page, int slot) {
    if (page < 0) return;  // (a quad of lanes has one row: its chunks are a multiple of eight)
    const int h = e >> dshift, d = (e & ((1 << dshift) - 1)) * 8;
    const uint4 xk = load_past(reinterpret_cast<const uint4*>(a.k + (i0 + r) * a.k_sn + h * a.k_sh + d));
    const uint4 xv = load_past(reinterpret_cast<const uint4*>(a.v + (i0 + r) * a.v_sn + h * a.v_sh + d));
    uint32_t bk, bv;
    const uint32_t ck = e2m1x8<TYPE>(xk, &bk), cv = e2m1x8<TYPE>(xv, &bv);
    *reinterpret_cast<uint32_t*>(a.k_pages + page * c.k_sp + h * c.k_sh + slot * c.k_sr + d / 2) = ck;
    *reinterpret_cast<uint32_t*>(a.v_pages + page * c.v_sp + h * c.v_sh + slot * c.v_sr + d / 2) = cv;
    if ((lane & 3) == 0) {
      const int at = slot * (c.D / 32) + d / 32;
      a.k_scale[page * z.k_sp + h * z.k_sh + at] = static_cast<uint8_t>(bk);
      a.v_scale[page * z.v_sp + h * z.v_sh + at] = static_cast<uint8_t>(bv);
    }
  });
}

// Rows read: 16 bytes out a lane, past the caches (131072 rows of 4 bits 149 -> 140 us, 4.9
// TB/s; 24k of e4m3 38.5 -> 26.6; one row a wavefront 142, K and V by workgroups of their
// own 158).
struct ReadArgs {
  const int32_t* lens;
  const int32_t* first;
  const void* k_pages;
  const void* v_pages;
  const void* k_scale;
  const void* v_scale;
  uint16_t* k;
  uint16_t* v;
};

enum { kPages16 = 0, kPages8 = 1, kPages4 = 2 };

// eight features of a row of pages, from `at` elements (bytes of 4-bit pages) on
template <int KIND, int TYPE>
__device__ __forceinline__ uint4 read8(const void* pages, int64_t at, float scale) {
  if constexpr (KIND == kPages16) {
    return *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(pages) + at);
  } else {
    uint32_t o[4];
    if constexpr (KIND == kPages8) {
      const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(pages) + at);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const auto x = i % 2 ? __builtin_amdgcn_cvt_pk_f32_fp8(i / 2 ? w.y : w.x, true) : __builtin_amdgcn_cvt_pk_f32_fp8(i / 2 ? w.y : w.x, false);
        o[i] = round2<TYPE>(x[0] * scale, x[1] * scale);
      }
    } else {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(pages) + at);
      const auto put = [&](int i, auto x) { o[i] = round2<TYPE>(x[0], x[1]); };
      if constexpr (TYPE == SCOPE_BF16) {  // (exact)
        o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
        o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
        o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
        o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
      } else {
        put(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0));
        put(1, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1));
        put(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2));
        put(3, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3));
      }
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
  }
}

template <int KIND, int TYPE>
__global__ __launch_bounds__(256) void paged_read_kernel(scope_paged_cache c, scope_paged_scales z, MoveArgs m, ReadArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t i0 = (static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6)) * m.rows;
  int2 place = make_int2(-1, 0);
  if (lane < m.rows && i0 + lane < m.N) place = row_place(c, m, a.first, a.lens, i0 + lane);
  const int dshift = __builtin_ctz(c.D) - 3;
  const int n = static_cast<int>(min(static_cast<int64_t>(m.rows), m.N - i0));
  each_chunk(m, n, place, [&](int r, int e, int page, int slot) {
    const int h = e >> dshift, d = (e & ((1 << dshift) - 1)) * 8;
    uint4 xk = make_uint4(0, 0, 0, 0), xv = xk;
    if (page >= 0) {
      float sk = 1.f, sv = 1.f;
      if constexpr (KIND == kPages8) {
        if (a.k_scale) sk = static_cast<const float*>(a.k_scale)[h];
        if (a.v_scale) sv = static_cast<const float*>(a.v_scale)[h];
      }
      if constexpr (KIND == kPages4) {
        const int at = slot * (c.D / 32) + d / 32;
        sk = scale_of(static_cast<const uint8_t*>(a.k_scale)[page * z.k_sp + h * z.k_sh + at]);
        sv = scale_of(static_cast<const uint8_t*>(a.v_scale)[page * z.v_sp + h * z.v_sh + at]);
      }
      const int dd = KIND == kPages4 ? d / 2 : d;
      xk = read8<KIND, TYPE>(a.k_pages, page * c.k_sp + h * c.k_sh + slot * c.k_sr + dd, sk);
      xv = read8<KIND, TYPE>(a.v_pages, page * c.v_sp + h * c.v_sh + slot * c.v_sr + dd, sv);
    }
    const int64_t to = (i0 + r) * c.Hkv * c.D + e * 8;
    store_past(a.k + to, xk);
    store_past(a.v + to, xv);
  });
}

// ---- attention of one new token -------------------------------------------------
typedef const __attribute__((address_space(1))) char* bytes_t;  // in device memory
template <class T>
__device__ __forceinline__ T read_as(bytes_t p) {
  return *(const __attribute__((address_space(1))) T*)p;  // (an address-space cast needs a C-style cast)
}
// past the caches
template <class T>
__device__ __forceinline__ T read_once(bytes_t p) {
  return __builtin_nontemporal_load((const __attribute__((address_space(1))) T*)p);
}

template <int D>
struct Tile4 {  // a lane's share of 32 keys and their scales
  static constexpr int VE = D / 16 < 8 ? D / 16 : 8;  // features in a row of V
  static constexpr int NH = D / (16 * VE);            // (in halves)
  static constexpr int KW = D == 64 ? 2 : 4;          // words in a row of K
  static constexpr int NK = D / (32 * KW);            // (parts of it)
  static constexpr int SB = D / 32;                   // bytes of a row's scales
  typedef uint32_t Row __attribute__((ext_vector_type(KW)));
  Row k[2][NK];
  uint32_t ks[2][NK];
  uint32_t v[NH][8];
  uint32_t vs[2 * SB];
};

// The tiles, the split, the running maximum and the join are those of the attention over
// 16-bit pages (paged.hip); what differs:
//   S^T = K·Q^T   K's codes become bf16 with their scale, two in one instruction, which is
//                 exact, and are operand A; a q in fp16 is the sum of two bf16 values.
//   O^T = V^T·P^T a conversion gives a position's two neighbouring features in one word,
//                 the operand wants two positions of one feature there.  Instead of
//                 transposing (32 v_perm a tile), a product runs over 16 positions with
//                 both features as its depth, operand B holding the probability in the
//                 half of the one and 0 in that of the other: columns 0 .. 7 the even
//                 features' outputs of the group's heads, 8 .. 15 the odd ones'.  Groups
//                 of more than 8 heads (WIDE) take two products.  WIDE for 8 heads too: 16
//                 sequences to 32k at D = 128 43 -> 50 us, at D = 256 74 -> 82.
//                 A probability is the sum of three bf16 values, the upper halves of what
//                 is left of it: all of its 24 bits, so that the product is fp32's.
// Bound by memory while a wavefront has tiles enough: 24 sequences of 9k to 65k with 64
// query heads (798 MB) 155 us, 5.1 TB/s with the launch behind it.  Below that the start
// counts (four dependent loads from the lengths to the first row, some 5 us) and the second
// launch (4.5 us): 131k positions with weights (143 MB) 33.1 us, of which the kernel 29.5; at
// D = 64 the vector units are busy 66% of the time (48 windows of 4096, 62 MB: 26 us).
// The next tile's loads are under way while one is worked on: a tile has a quarter of the
// bytes of 16-bit rows and as many instructions (131k positions 46.6 -> 32.8 us).  Two
// tiles ahead 31.4 us for 30.3 at D = 64, spilling elsewhere.  WIDE at D = 256 has no
// registers for it: with one wavefront a SIMD 138 us (16 sequences to 32k), with two that
// load as they go 94.
// K passes the caches where its rows are long enough (24 sequences 176 -> 164 us, 131k
// positions 40.4 -> 35.1, V alone 173 and 35.1, both 167 and 38.4; pages of 16 30.3 ->
// 31.4, D = 64 32.0 -> 32.8).
// K's codes as they are in the scaled product of 4-bit and 8-bit operands, q in e4m3
// parts, saves 32 conversions a tile and changed nothing there; forming the parts took
// 1.2 us (nine blocks a head 5.4 -> 6.6, 48 windows 27.2 -> 30.4).
constexpr int attn4_waves(int D, bool wide) {  // wavefronts a SIMD that the registers are cut to
  // (D = 64: with 3 windows 30.4 -> 31.8 us, 8 sequences to 60k 56 -> 61; WIDE at D = 128
  // with 3 29.0 -> 30.5 and fp16 spills)
  return D == 256 || (wide && D == 128) ? 2 : D == 64 && !wide ? 4 : 3;
}

// SMALL: pages of 16 positions, two a tile (other pages' addresses are scalars).
template <int TYPE, int D, bool WIDE, bool SMALL>
__global__ __launch_bounds__(kAttnThreads, attn4_waves(D, WIDE)) void paged_attn4_kernel(scope_paged_cache c, scope_paged_scales z,
                                                                                         PagedAttnArgs a, AttnSplit s) {
  using Tile = Tile4<D>;
  constexpr int VE = Tile::VE, NH = Tile::NH, KW = Tile::KW, NK = Tile::NK, SB = Tile::SB;
  constexpr int NP2 = VE / 2;                     // pairs of features of a lane in a row of V
  constexpr int NJ = D / 32;                      // products over D
  constexpr int NQ = TYPE == SCOPE_FP16 ? 2 : 1;  // bf16 values whose sum is one of q
  constexpr int NP = 3;                           // bf16 values whose sum is a probability
  constexpr int NC = WIDE ? 2 : 1;                // products for even and odd features
  constexpr bool kPast = !SMALL && D >= 128;      // K passes the caches
  constexpr bool kAhead = !(WIDE && D == 256);    // the next tile's loads are under way
  extern __shared__ float lds[];
  // (what is the same for a wavefront is told to the compiler: scalar registers, branches and addresses)
  const auto same = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  const int lane = threadIdx.x & 63, wave = same(threadIdx.x >> 6), g4 = lane >> 4, c16 = lane & 15;
  const int G = a.Hq / c.Hkv, ng = (G + 15) / 16;
  // the columns of one piece start together, and pieces that there are not last
  const uint32_t cols = gridDim.y, id = blockIdx.y * gridDim.x + blockIdx.x;  // (less than 2^17 slots and 2^13 columns)
  const int slot = same(id / cols), column = same(id % cols);
  const int hk = column / ng, cg = column % ng, nq = min(16, G - 16 * cg);
  const int h0 = hk * G + 16 * cg;                // first query head
  const int col = WIDE ? c16 : c16 & 7;           // this lane's
  const bool lists = a.kv_idx != nullptr;
  Piece p;
  int n_list = 0;
  if (lists) {
    // pieces of one length for every list, so that the list is read without waiting for its number
    p.b = slot / s.pieces;
    p.i = slot % s.pieces;
    p.n = s.pieces;
    p.slot = p.b * s.pieces;
    p.len = a.lens[p.b];
    p.first = a.first ? a.first[p.b] : 0;
    n_list = min(max(a.kv_num[static_cast<int64_t>(p.b) * c.Hkv + hk], 0), a.maxkv);
    piece_range(0, static_cast<int>(s.tiles_cap), p.n, p.i, &p.t0, &p.t1);
  } else {
    const auto wanted = [&](int64_t total) { return min(s.pieces, pieces_wanted4(total, cols, c.B, kUnits * attn4_waves(D, WIDE))); };
    if (!find_piece(c, a, slot, piece_turn(D), wanted, p)) return;
  }
  p.b = same(p.b);
  p.i = same(p.i);
  p.n = same(p.n);
  p.slot = same(p.slot);
  p.t0 = same(p.t0);
  p.t1 = same(p.t1);
  const int b = p.b;
  if (s.plan && column == 0 && p.i == 0 && threadIdx.x == 0) s.plan[b] = make_int2(p.n, p.slot);
  const int64_t cap = static_cast<int64_t>(c.MP) * c.bs;
  const int end = same(static_cast<int>(seq_end(p.len, cap))), low = same(max(p.first, 0));
  const int32_t* row = a.table + static_cast<int64_t>(b) * c.MP;
  const int32_t* list = lists ? a.kv_idx + (static_cast<int64_t>(b) * c.Hkv + hk) * a.maxkv : nullptr;
  const int shift = __builtin_ctz(c.bs);

  // Q^T: column c is query head h0 + col.  Scores are taken times the scale's size, q
  // with its sign (0 where it is 0), so that the largest product is the largest score.
  const float c_log2 = a.scale == 0.f ? 1.f : fabsf(a.scale) * kLog2e;
  const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u, keep = a.scale == 0.f ? 0u : ~0u;
  uint4 qf[NQ][NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int d = D == 64 ? g4 * 16 + j * 8 : (j / 4) * 128 + g4 * 32 + (j % 4) * 8;
    uint4 u = make_uint4(0, 0, 0, 0);
    if (col < nq) u = *reinterpret_cast<const uint4*>(a.q + b * a.q_sb + (h0 + col) * a.q_sh + d);
    const uint32_t w[4] = {(u.x ^ flip) & keep, (u.y ^ flip) & keep, (u.z ^ flip) & keep, (u.w ^ flip) & keep};
    if constexpr (TYPE == SCOPE_BF16) {
      qf[0][j] = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = low_half<SCOPE_FP16>(w[i]), y = high_half<SCOPE_FP16>(w[i]);
        hi[i] = round2<SCOPE_BF16>(x, y);
        lo[i] = round2<SCOPE_BF16>(x - low_half<SCOPE_BF16>(hi[i]), y - high_half<SCOPE_BF16>(hi[i]));
      }
      qf[0][j] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      qf[1][j] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
  }

  f32x4_t acc[NC][NH * NP2];
#pragma unroll
  for (int n = 0; n < NC; ++n)
#pragma unroll
    for (int i = 0; i < NH * NP2; ++i) acc[n][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // the maximum so far, what the probabilities are taken relative to, their sum
  float m = -INFINITY, ref = 0.f, l = 0.f;

  const bytes_t kbase = (bytes_t)a.k_pages + hk * c.k_sh;
  const bytes_t vbase = (bytes_t)a.v_pages + hk * c.v_sh;
  const bytes_t ksbase = (bytes_t)a.k_scale + hk * z.k_sh;
  const bytes_t vsbase = (bytes_t)a.v_scale + hk * z.v_sh;
  // operand A of the scores: row m is key 8 (m / 4) + 4 i + m % 4 of the tile in product i
  const int krow = (c16 >> 2) * 8 + (c16 & 3), vrow = g4 * 8;
  const int krow_in = SMALL ? krow & 15 : krow, vrow_in = SMALL ? vrow & 15 : vrow;
  // (row strides are less than 2^26 bytes)
  const uint32_t koff = krow_in * static_cast<uint32_t>(c.k_sr) + g4 * (KW * 4);
  const uint32_t voff = vrow_in * static_cast<uint32_t>(c.v_sr) + c16 * (VE / 2);
  const uint32_t ksoff = krow_in * SB + (D == 64 ? g4 >> 1 : g4), vsoff = vrow_in * SB;
  // where the byte of this lane's features is among a row's (a word's): rotated by this, it is at bit 23
  const int vturn = (8 * (D == 64 ? c16 >> 3 : c16 >> 2) + 9) & 31;
  // a probability's upper half in the half of a word that this lane's column takes (bytes of 0 beside it)
  const uint32_t half = c16 < 8 ? 0x0c0c0706u : 0x07060c0cu;

  // pages and blocks of this wavefront's next 64 tiles, one a lane (two where a tile is two pages)
  int pg0 = -1, pg1 = -1, lb0 = 0, lb1 = 0;
  const auto resolve = [&](int t) __attribute__((always_inline)) {
    const auto one = [&](int64_t e, int& lb) -> int {  // entry e of the list, or block e
      const int64_t blk = !lists ? e : e < a.maxkv ? list[e] : -1;
      const int64_t page = block_page(row, c.MP, blk, c.P);
      lb = page < 0 ? 0 : static_cast<int>(blk);
      return lists && e >= n_list ? -1 : static_cast<int>(page);
    };
    pg0 = pg1 = -1;
    lb0 = lb1 = 0;
    if (t < p.t1) {
      const int64_t e = (static_cast<int64_t>(t) * kTileKeys) >> shift;
      pg0 = one(e, lb0);
      if constexpr (SMALL) pg1 = one(e + 1, lb1);
    }
  };
  struct Where {  // a tile's pages (-1: none), their first positions in it, its first row in its page
    int page0, page1, pos0, pos1, r0;
  };
  int u = 0;
  const auto where = [&](int t) __attribute__((always_inline)) {  // of tile t, entry u of the 64
    Where w;
    w.page0 = __builtin_amdgcn_readlane(pg0, u);
    w.page1 = SMALL ? __builtin_amdgcn_readlane(pg1, u) : w.page0;
    w.r0 = SMALL ? 0 : (t * kTileKeys) & (c.bs - 1);
    w.pos0 = (__builtin_amdgcn_readlane(lb0, u) << shift) + w.r0;
    w.pos1 = SMALL ? __builtin_amdgcn_readlane(lb1, u) << shift : w.pos0 + 16;
    return w;
  };

  const auto put_sum = [&](int t, float x) {  // log2 of tile t's sum (of this lane's half of it)
    if (c16 < nq && (g4 & (SMALL ? 1 : 3)) == 0)
      s.tile_lse[((static_cast<int64_t>(b) * a.Hq + h0 + c16) * s.tiles_cap + t) * (SMALL ? 2 : 1) + (SMALL ? g4 >> 1 : 0)] = x;
  };
  int t = p.t0 + wave;
  const auto seek = [&]() __attribute__((always_inline)) {  // from tile t on to one that has a page
    while (t < p.t1) {
      if (u == 64) {
        resolve(t + lane * kAttnWaves);
        u = 0;
      }
      if (__builtin_amdgcn_readlane(pg0, u) >= 0 || (SMALL && __builtin_amdgcn_readlane(pg1, u) >= 0)) return;
      if (s.tile_lse) put_sum(t, -INFINITY);
      t += kAttnWaves;
      ++u;
    }
  };

  const auto load = [&](const Where& w, Tile& x) __attribute__((always_inline)) {
    // (a scalar address and a lane's offset as the loads take them, which the compiler would
    // otherwise add up in registers that earlier loads are still on their way to)
    const auto row = [](bytes_t p) __attribute__((always_inline)) {
      if constexpr (!SMALL) asm("" : "+s"(p));
      return p;
    };
    const auto off = [](uint32_t x) __attribute__((always_inline)) {
      if constexpr (!SMALL) asm volatile("" : "+v"(x));
      return x;
    };
    const uint32_t ko = off(koff), kso = off(ksoff), vo = off(voff), vso = off(vsoff);
    const auto get = [&](bytes_t kr, bytes_t vr, bytes_t ksr, bytes_t vsr) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bytes_t r = row(kr + 4 * i * c.k_sr);
#pragma unroll
        for (int j = 0; j < NK; ++j)
          x.k[i][j] = kPast ? read_once<typename Tile::Row>(r + ko + j * 64) : read_as<typename Tile::Row>(r + ko + j * 64);
      }
      ksr = row(ksr);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NK; ++j) x.ks[i][j] = read_as<uint8_t>(ksr + kso + 4 * i * SB + 4 * j);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bytes_t r = row(vr + i * c.v_sr);
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          if constexpr (VE == 4)
            x.v[h][i] = read_as<uint16_t>(r + vo);
          else
            x.v[h][i] = read_as<uint32_t>(r + vo + h * 64);
        }
      }
      vsr = row(vsr);
#pragma unroll
      for (int i = 0; i < SB / 2; ++i) {
        const u32x4_t q = read_as<u32x4_t>(vsr + vso + 16 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) x.vs[4 * i + j] = q[j];
      }
    };
    if constexpr (!SMALL) {
      const int64_t page = max(w.page0, 0);
      get(kbase + page * c.k_sp + w.r0 * c.k_sr, vbase + page * c.v_sp + w.r0 * c.v_sr, ksbase + page * z.k_sp + w.r0 * SB,
          vsbase + page * z.v_sp + w.r0 * SB);
    } else {
      const int64_t kp = max(krow >= 16 ? w.page1 : w.page0, 0), vp = max(vrow >= 16 ? w.page1 : w.page0, 0);
      get(kbase + kp * c.k_sp, vbase + vp * c.v_sp, ksbase + kp * z.k_sp, vsbase + vp * z.v_sp);
    }
  };

  const auto compute = [&](int t, const Where& w, Tile& y) __attribute__((always_inline)) {
    // keys outside [low, end) and of no page are not seen: most tiles have none
    const bool whole = w.page0 >= 0 && w.page1 >= 0 && w.pos0 >= low && w.pos0 + 16 <= end && w.pos1 >= low && w.pos1 + 16 <= end;
    int from = 0, to = 8;  // of the lane's eight keys
    if (!whole) {
      const bool back = vrow >= 16;
      const int page = back ? w.page1 : w.page0, pos = (back ? w.pos1 : w.pos0) + (vrow & 15);
      from = page < 0 ? 8 : low - pos;  // (positions and lengths are at least 0: no overflow)
      to = end - pos;
      // a row of V that is not seen may hold anything, and 0 times NaN is NaN
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool see = i >= from && i < to;
#pragma unroll
        for (int h = 0; h < NH; ++h) y.v[h][i] = see ? y.v[h][i] : 0u;
        if constexpr (D == 64) {
          y.vs[i / 2] &= see ? ~0u : i % 2 ? 0xffffu : 0xffff0000u;
        } else {
#pragma unroll
          for (int h = 0; h < NH; ++h) y.vs[NH * i + h] = see ? y.vs[NH * i + h] : 0u;
        }
      }
    }
    // scores
    f32x4_t sc[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) sc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t x = y.k[i][j / KW][j % KW];
        const float f = scale_of(y.ks[i][j / KW]);
        const uint4 kk = make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, f, 0)),
                                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, f, 1)),
                                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, f, 2)),
                                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, f, 3)));
#pragma unroll
        for (int k = 0; k < NQ; ++k) sc[i] = mfma16(kk, qf[k][j], sc[i]);
      }
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = sc[i >> 2][i & 3];
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = i >= from && i < to ? x[i] : -INFINITY;
    }
    float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]))) * c_log2;
    if (__any(top > m + 8.f)) {
      top = over_rows(top, max_f32);
      const float mn = fmaxf(m, top), f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      l *= f;
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int i = 0; i < NH * NP2; ++i) acc[n][i] *= f;
      m = mn;
      ref = m == -INFINITY ? 0.f : m;
    }
    float lt = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], c_log2, -ref));
      lt += x[i];
    }
    l += lt;
    if (s.tile_lse) {
      lt = SMALL ? over_rows2(lt, add_f32) : over_rows(lt, add_f32);
      put_sum(t, ref + __builtin_amdgcn_logf(lt));
    }
    // four rows of V at a time: the probabilities as a sum of bf16 values each (the upper
    // half of what is left of them), and their products with the rows' features, in pairs
#pragma unroll
    for (int r = 0; r < 8; r += 4) {
      uint32_t pw[NC][NP][4];
#pragma unroll
      for (int k = 0; k < NP; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t bits = __float_as_uint(x[r + i]), hi = bits & 0xffff0000u;
          if constexpr (WIDE) {
            pw[0][k][i] = bits >> 16;
            pw[1][k][i] = hi;
          } else {
            pw[0][k][i] = __builtin_amdgcn_perm(bits, 0u, half);
          }
          x[r + i] -= __uint_as_float(hi);
        }
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t sw = D == 64 ? y.vs[(r + i) / 2] >> (16 * (i % 2)) : y.vs[NH * (r + i) + h];
          f[i] = __uint_as_float(__builtin_amdgcn_alignbit(sw, sw, vturn));
        }
        const auto pair = [&](auto at) __attribute__((always_inline)) {  // pair `at` of the features
          constexpr int e = decltype(at)::value;
          uint32_t o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            o[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(y.v[h][r + i], f[i], e));
          const uint4 vt = make_uint4(o[0], o[1], o[2], o[3]);
#pragma unroll
          for (int n = 0; n < NC; ++n)
#pragma unroll
            for (int k = 0; k < NP; ++k)
              acc[n][h * NP2 + e] = mfma16(vt, make_uint4(pw[n][k][0], pw[n][k][1], pw[n][k][2], pw[n][k][3]), acc[n][h * NP2 + e]);
        };
        pair(std::integral_constant<int, 0>{});
        pair(std::integral_constant<int, 1>{});
        if constexpr (NP2 == 4) {
          pair(std::integral_constant<int, 2>{});
          pair(std::integral_constant<int, 3>{});
        }
      }
    }
  };

  resolve(p.t0 + wave + lane * kAttnWaves);
  if (lists) p.t1 = min(p.t1, same(static_cast<int>((static_cast<int64_t>(n_list) * c.bs + kTileKeys - 1) / kTileKeys)));
  // Two tiles in turn: one's loads are under way while the other is worked on.  (Behind the
  // last one it is loaded once more: loads on one side of a branch would be waited for at
  // its end with all that are under way.)
  seek();
  if constexpr (!kAhead) {
    while (t < p.t1) {
      Tile x;
      const Where w = where(t);
      load(w, x);
      __builtin_amdgcn_sched_barrier(0);
      compute(t, w, x);
      t += kAttnWaves;
      ++u;
      seek();
    }
  } else if (t < p.t1) {
    Tile x, y;
    Where wx = where(t), wy;
    int tx = t, ty;
    bool last = true;  // x is still to be worked on behind the loop
    load(wx, x);
    t += kAttnWaves;
    ++u;
    seek();
    while (t < p.t1) {
      wy = where(t);
      ty = t;
      load(wy, y);
      __builtin_amdgcn_sched_barrier(0);
      compute(tx, wx, x);
      t += kAttnWaves;
      ++u;
      seek();
      wx = wy;
      if (t < p.t1) wx = where(t);
      tx = t;
      load(wx, x);
      __builtin_amdgcn_sched_barrier(0);
      compute(ty, wy, y);
      if (tx >= p.t1) {
        last = false;
        break;
      }
      t += kAttnWaves;
      ++u;
      seek();
    }
    if (last) compute(tx, wx, x);
  }

  l = over_rows(l, add_f32);
  const Shares sh = shares_of(lds);
  if (g4 == 0) {
    sh.sm[wave * 16 + c16] = m == -INFINITY ? m : ref;
    sh.sl[wave * 16 + c16] = l;
  }
  if (col < nq) {
    float* o = sh.so + (wave * nq + col) * D + g4 * 4 * VE + (WIDE ? 0 : c16 >> 3);
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int j = 0; j < NP2; ++j) o[h * 128 + r * VE + 2 * j + n] = acc[n][h * NP2 + j][r];
  }
  __syncthreads();
  join_shares<TYPE, D>(a, s, p, h0, nq, 1.f, sh);
}

namespace {
int check_scales(const scope_paged_cache* c, const scope_paged_scales* z, const void* k_scale, const void* v_scale, const char* fn) {
  SCOPE_REQUIRE(z && k_scale && v_scale, "%s: null scales", fn);
  SCOPE_REQUIRE(z->k_sp % 16 == 0 && z->k_sh % 16 == 0 && z->v_sp % 16 == 0 && z->v_sh % 16 == 0 && aligned16(k_scale) &&
                    aligned16(v_scale),
                "%s: the scales of a page's head must be 16-byte aligned", fn);
  constexpr int64_t kMost = 1 << 26;  // (the attention's lanes count 32 rows in 32 bits)
  SCOPE_REQUIRE(c->k_sr >= 0 && c->k_sr < kMost && c->v_sr >= 0 && c->v_sr < kMost, "%s: the pages' rows must be less than 2^26 bytes apart", fn);
  return SCOPE_OK;
}

// pages of bytes as check_cache knows them
scope_paged_cache in_bytes(const scope_paged_cache& c) {
  scope_paged_cache x = c;
  x.fp8 = 1;
  return x;
}

MoveArgs move_args(const scope_paged_cache& c, int64_t N, const int32_t* cu, const int32_t* table) {
  const int chunks = c.Hkv * (c.D / 8);
  return MoveArgs{N, moved_rows(N, chunks), chunks, 64 / chunks, 64 % chunks, cu, table};
}
}  // namespace

}  // namespace scope

using namespace scope;

extern "C" {

int scope_paged_append_fp4(const scope_paged_cache* c, const scope_paged_scales* z, int64_t N, const uint16_t* k, int64_t k_sn,
                           int64_t k_sh, const uint16_t* v, int64_t v_sn, int64_t v_sh, const int32_t* cu, const int32_t* table,
                           const int32_t* lens, void* k_scale, void* v_scale, void* k_pages, void* v_pages, void* stream) {
  const char* fn = "scope_paged_append_fp4";
  SCOPE_REQUIRE(c, "%s: null cache", fn);
  const scope_paged_cache bytes = in_bytes(*c);
  if (int rc = check_cache(&bytes, k_pages, v_pages, fn)) return rc;
  if (int rc = check_scales(c, z, k_scale, v_scale, fn)) return rc;
  SCOPE_REQUIRE(N >= 0 && N <= INT32_MAX, "%s: %lld rows (0 .. 2^31 - 1)", fn, (long long)N);
  SCOPE_REQUIRE(cu || N <= c->B, "%s: %lld rows for %d sequences need cu", fn, (long long)N, c->B);
  if (N == 0) return SCOPE_OK;
  SCOPE_REQUIRE(k && v && table && lens, "%s: null pointer", fn);
  SCOPE_REQUIRE(aligned16(k) && aligned16(v) && k_sn % 8 == 0 && k_sh % 8 == 0 && v_sn % 8 == 0 && v_sh % 8 == 0,
                "%s: the rows of k and v must be 16-byte aligned", fn);
  const MoveArgs m = move_args(*c, N, cu, table);
  const Append4Args a{k_sn, k_sh, v_sn, v_sh, k, v, lens, static_cast<uint8_t*>(k_pages), static_cast<uint8_t*>(v_pages),
                      static_cast<uint8_t*>(k_scale), static_cast<uint8_t*>(v_scale)};
  const dim3 grid(ceil_div(N, 4 * m.rows)), block(256);
  if (c->type == SCOPE_BF16)
    hipLaunchKernelGGL(paged_append4_kernel<SCOPE_BF16>, grid, block, 0, as_stream(stream), bytes, *z, m, a);
  else
    hipLaunchKernelGGL(paged_append4_kernel<SCOPE_FP16>, grid, block, 0, as_stream(stream), bytes, *z, m, a);
  return check_launch("paged_append4_kernel");
}

int scope_paged_read(const scope_paged_cache* c, const scope_paged_scales* z, int64_t N, const int32_t* cu, const int32_t* table,
                     const int32_t* lens, const int32_t* first, const void* k_scale, const void* v_scale, const void* k_pages,
                     const void* v_pages, uint16_t* k, uint16_t* v, void* stream) {
  const char* fn = "scope_paged_read";
  SCOPE_REQUIRE(c, "%s: null cache", fn);
  const scope_paged_cache as = z ? in_bytes(*c) : *c;
  if (int rc = check_cache(&as, k_pages, v_pages, fn)) return rc;
  if (z)
    if (int rc = check_scales(c, z, k_scale, v_scale, fn)) return rc;
  SCOPE_REQUIRE(N >= 0 && N <= INT32_MAX, "%s: %lld rows (0 .. 2^31 - 1)", fn, (long long)N);
  SCOPE_REQUIRE(cu || N <= c->B, "%s: %lld rows for %d sequences need cu", fn, (long long)N, c->B);
  if (N == 0) return SCOPE_OK;
  SCOPE_REQUIRE(table && lens && k && v, "%s: null pointer", fn);
  SCOPE_REQUIRE(aligned16(k) && aligned16(v), "%s: k and v must be 16-byte aligned", fn);
  const MoveArgs m = move_args(*c, N, cu, table);
  const ReadArgs a{lens, first, k_pages, v_pages, k_scale, v_scale, k, v};
  const scope_paged_scales none{};
  const dim3 grid(ceil_div(N, 4 * m.rows)), block(256);
  hipStream_t st = as_stream(stream);
  const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, st, as, z ? *z : none, m, a); };
  if (z)
    c->type == SCOPE_BF16 ? launch(paged_read_kernel<kPages4, SCOPE_BF16>) : launch(paged_read_kernel<kPages4, SCOPE_FP16>);
  else if (c->fp8)
    c->type == SCOPE_BF16 ? launch(paged_read_kernel<kPages8, SCOPE_BF16>) : launch(paged_read_kernel<kPages8, SCOPE_FP16>);
  else  // (16-bit values are moved as they are)
    launch(paged_read_kernel<kPages16, SCOPE_BF16>);
  return check_launch("paged_read_kernel");
}

int scope_paged_decode_attn_fp4(const scope_paged_cache* c, const scope_paged_scales* z, int Hq, int maxkv, float scale,
                                const uint16_t* q, int64_t q_sb, int64_t q_sh, const void* k_pages, const void* v_pages,
                                const void* k_scale, const void* v_scale, const int32_t* table, const int32_t* lens,
                                const int32_t* first, const int32_t* kv_num, const int32_t* kv_idx, float* mass, void* work,
                                uint16_t* out, float* lse, void* stream) {
  const char* fn = "scope_paged_decode_attn_fp4";
  SCOPE_REQUIRE(c, "%s: null cache", fn);
  const scope_paged_cache bytes = in_bytes(*c);
  if (int rc = check_cache(&bytes, k_pages, v_pages, fn)) return rc;
  if (int rc = check_scales(c, z, k_scale, v_scale, fn)) return rc;
  const PagedAttnArgs a{Hq,      maxkv, scale, q_sb,  q_sh,   q,      k_pages, v_pages, k_scale,
                        v_scale, table, lens,  first, kv_num, kv_idx, mass,    out,     lse};
  AttnSplit s;
  if (int rc = check_attn(bytes, a, work, &s, fn)) return rc;
  const int G = Hq / c->Hkv, ng = (G + 15) / 16;
  const dim3 grid(s.slots, c->Hkv * ng);
  const size_t lds = sizeof(float) * kAttnWaves * (32 + static_cast<size_t>(std::min(G, 16)) * c->D);
  hipStream_t st = as_stream(stream);
  const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kAttnThreads), lds, st, bytes, *z, a, s); };
  const auto of_sizes = [&](auto type, auto wide, auto small) {
    constexpr int T = decltype(type)::value;
    constexpr bool W = decltype(wide)::value, S = decltype(small)::value;
    if (c->D == 64)
      launch(paged_attn4_kernel<T, 64, W, S>);
    else if (c->D == 128)
      launch(paged_attn4_kernel<T, 128, W, S>);
    else
      launch(paged_attn4_kernel<T, 256, W, S>);
  };
  using std::false_type, std::true_type;
  const auto of_width = [&](auto type, auto small) { G > 8 ? of_sizes(type, true_type{}, small) : of_sizes(type, false_type{}, small); };
  const auto of_type = [&](auto type) { c->bs == 16 ? of_width(type, true_type{}) : of_width(type, false_type{}); };
  c->type == SCOPE_BF16 ? of_type(std::integral_constant<int, SCOPE_BF16>{}) : of_type(std::integral_constant<int, SCOPE_FP16>{});
  if (int rc = check_launch("paged_attn4_kernel")) return rc;
  return launch_paged_finish(bytes, a, nullptr, s, st);
}

}  // extern "C"
