// The paged key-value cache of a decode loop: rows of new tokens written to
// their pages, the attention of one new token per sequence over its pages,
// and the choice of the pages that leave when the cache is over its budget.
//
// Pages are [P][Hkv][bs][D] (any page, head and row strides); row b of the
// table [B][MP] names the page of each block of bs positions of sequence b.
// An entry outside [0, P) is a block without a page (not there yet, or
// evicted): nothing is written to it and no key of it is seen.
#include <math.h>

#include <algorithm>

#include "paged_attn.h"

namespace scope {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// the sum and the largest over all lanes
__device__ __forceinline__ float sum_of(float v) {
  return __uint_as_float(__builtin_amdgcn_readlane(lane_prefix(__float_as_uint(v), 0u, add_f32), 63));
}
__device__ __forceinline__ float max_of(float v) {
  return __uint_as_float(__builtin_amdgcn_readlane(lane_prefix(__float_as_uint(v), 0xff800000u, max_f32), 63));
}

// ---- append ------------------------------------------------------------------
// Row i of the N new ones belongs to the sequence b with cu[b] <= i < cu[b + 1]
// (row i to sequence i without cu) and goes to position lens[b] + i - cu[b].
// Bound by memory: a wavefront takes `rows` rows; lane r finds the place of its
// r-th row (a search, two loads), so the chain of loads is paid once for all of
// them, then every row moves 16 bytes a lane.  65539 rows of 8 heads of 128: into
// e4m3 77 us, 5.2 TB/s, as a large copy (one row a wavefront 86, eight 88; 82
// with loads and stores through the caches); 16-bit pages 105 us, 5.1 TB/s
// (there past the caches 108).
struct AppendArgs {
  int64_t N, k_sn, k_sh, v_sn, v_sh;
  int rows;
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* cu;
  const int32_t* table;
  const int32_t* lens;
  const float* k_scale;
  const float* v_scale;
  void* k_pages;
  void* v_pages;
};

// 1 / s where the quotient x / s may be formed by it (quotient below), else 0: for
// scales in 2^-60 .. 2^60 whose significand is not all ones
__device__ __forceinline__ float quotient_factor(float s) {
  return s >= 0x1p-60f && s <= 0x1p60f && (__float_as_uint(s) & 0x7fffffu) != 0x7fffffu ? 1.f / s : 0.f;
}

// The fp32 quotient x / s of a 16-bit x, rounded to nearest as a division rounds
// it, as far as e4m3 can tell.  With r = 1 / s to nearest, q = x·r is next to the
// quotient, and one residual step q + r·(x - q·s) gives it to nearest (Markstein's
// division; the residual is exact while it does not fall below 2^-126, as for
// |q| >= 2^-20 and these scales it does not).  Quotients below that are 0 in e4m3
// and keep their sign without the step; those past every finite e4m3, infinities
// and NaN need none.  A few instructions for the division's ten.
__device__ __forceinline__ float quotient(float x, float s, float r) {
  if (r == 0.f) return x / s;
  const float q = x * r;
  const float a = fabsf(q);
  return a >= 0x1p-20f && a < 0x1p20f ? __builtin_fmaf(__builtin_fmaf(-q, s, x), r, q) : q;
}

// eight 16-bit values as e4m3 of x / s: cut to the largest finite value, rounded
// to nearest even; NaN stays NaN
template <int TYPE>
__device__ __forceinline__ uint2 e4m3x8(const uint4& u, float s, float r) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint16_t h = static_cast<uint16_t>(i % 2 ? w[i / 2] >> 16 : w[i / 2]);
    const float q = quotient(TYPE == SCOPE_FP16 ? half_to_f32(h) : bf16_to_f32(h), s, r);
    f[i] = q > 448.f ? 448.f : q < -448.f ? -448.f : q;
  }
  uint32_t o[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    o[i] = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i], f[4 * i + 1], 0, false);
    o[i] = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2], f[4 * i + 3], o[i], true);
  }
  return make_uint2(o[0], o[1]);
}

template <int TYPE, bool FP8>
__global__ __launch_bounds__(256) void paged_append_kernel(scope_paged_cache c, AppendArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t i0 = (static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6)) * a.rows;
  // lane r: page (-1: the row is not written) and slot of row i0 + r
  int page_l = -1, slot_l = 0;
  if (lane < a.rows && i0 + lane < a.N) {
    int b;
    const int64_t pos = row_position(a.cu, a.lens, c.B, i0 + lane, &b);
    if (pos >= 0 && pos < static_cast<int64_t>(c.MP) * c.bs) {
      page_l = static_cast<int>(block_page(a.table + static_cast<int64_t>(b) * c.MP, c.MP, pos / c.bs, c.P));
      slot_l = static_cast<int>(pos % c.bs);
    }
  }
  const int chunks = c.Hkv * c.D / 8, dshift = __builtin_ctz(c.D) - 3;
  for (int r = 0; r < a.rows; ++r) {
    const int page = __builtin_amdgcn_readlane(page_l, r), slot = __builtin_amdgcn_readlane(slot_l, r);
    if (page < 0) continue;
    const uint16_t* ks = a.k + (i0 + r) * a.k_sn;
    const uint16_t* vs = a.v + (i0 + r) * a.v_sn;
    const int64_t ko = static_cast<int64_t>(page) * c.k_sp + slot * c.k_sr, vo = static_cast<int64_t>(page) * c.v_sp + slot * c.v_sr;
    for (int e = lane; e < chunks; e += 64) {
      const int h = e >> dshift, d = (e & ((1 << dshift) - 1)) * 8;
      const uint4* kp = reinterpret_cast<const uint4*>(ks + h * a.k_sh + d);
      const uint4* vp = reinterpret_cast<const uint4*>(vs + h * a.v_sh + d);
      const int64_t ok = ko + h * c.k_sh + d, ov = vo + h * c.v_sh + d;
      if constexpr (FP8) {
        const float sk = a.k_scale ? a.k_scale[h] : 1.f, sv = a.v_scale ? a.v_scale[h] : 1.f;
        const uint4 xk = load_past(kp), xv = load_past(vp);
        store_past(static_cast<uint8_t*>(a.k_pages) + ok, e4m3x8<TYPE>(xk, sk, quotient_factor(sk)));
        store_past(static_cast<uint8_t*>(a.v_pages) + ov, e4m3x8<TYPE>(xv, sv, quotient_factor(sv)));
      } else {
        const uint4 xk = *kp, xv = *vp;
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.k_pages) + ok) = xk;
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.v_pages) + ov) = xv;
      }
    }
  }
}

// ---- attention of one new token -------------------------------------------------
// the largest 16-bit values below two positive numbers (0 below 0)
template <int TYPE>
__device__ __forceinline__ uint32_t below2(float lo, float hi) {
  const uint32_t a = __builtin_elementwise_sub_sat(__float_as_uint(lo), 1u), b = __builtin_elementwise_sub_sat(__float_as_uint(hi), 1u);
  if constexpr (TYPE == SCOPE_BF16)
    return pack_hi16(a, b);
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(__uint_as_float(a), __uint_as_float(b)));
}

template <int N>
struct Words {
  uint32_t w[N];
};

// N words that are read once: they are not kept in the caches in front of others
template <int N>
__device__ __forceinline__ Words<N> load_once(const char* p) {
  Words<N> x;
  if constexpr (N == 1) {
    x.w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
  } else {
    typedef uint32_t words_t __attribute__((ext_vector_type(N), aligned(4)));
    const words_t v = __builtin_nontemporal_load(reinterpret_cast<const words_t*>(p));
#pragma unroll
    for (int i = 0; i < N; ++i) x.w[i] = v[i];
  }
  return x;
}

template <int TYPE>
__device__ __forceinline__ f32x4_t mfma_16(const uint4& a, const uint4& b, const f32x4_t& acc) {
  if constexpr (TYPE == SCOPE_BF16) {
    return mfma16(a, b, acc);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), acc, 0, 0, 0);
  }
}

// two e4m3 bytes as 16-bit values (exact)
template <int TYPE, bool HI>
__device__ __forceinline__ uint32_t widen2(uint32_t w) {
  if constexpr (TYPE == SCOPE_BF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
}

// The attention of one new token.  For a tile of 32 keys and 16 query heads of
// one key head (those past the group are zero), with lane l, g = l / 16, c = l % 16:
//   S^T = K·Q^T   two products; operand A's row m is key 8(m/4) + 4t + m%4 of
//                 the tile in product t, so that lane l holds of query c the
//                 scores of the eight keys 8g .. 8g+7;
//   O^T = V^T·P^T the same eight probabilities are operand B without moving;
//                 operand A takes for feature f = VE·m + j (product j) the
//                 eight keys' values, an 8 x VE transposition of 16-bit values
//                 within the lane (v_perm) of rows loaded 16 lanes wide.
// So K and V go from memory to the matrix units through registers alone, and a
// query's maximum, sum and outputs stay in the lanes of its column.  Scores are
// scaled into log2 units in fp32; the maximum that the probabilities are taken
// relative to moves only when a score passes it by more than 8 (p <= 256 until
// then, no loss in floating point).  For the product with V, whose instruction
// takes 16-bit operands, a probability is the sum of 16-bit values: three in bf16
// (two, off by 2^-17 of it, were 1% faster in e4m3 and no faster in bf16), two in
// fp16.  All but the last are the largest below what is left, so that none is
// negative, nor 0 unless the probability is small (bf16 2^-100, fp16 2^-15 of its
// tile's largest): an infinite value of V stays one.  That leaves an error of 2^-23
// (bf16), 2^-21 (fp16) of a probability.  e4m3 has no infinities: rounded to nearest,
// 2^-27 and 2^-23.
// fp16 has no exponents for the small weights of a long cache (below 2^-25 a key
// would count in the sum and not in the output: behind one key that takes nearly all
// of the weight, 131k others 17.4 nats lower came out as 0).  There the
// probabilities are taken relative to each tile's own largest, which becomes 2^14 to
// 2^15, and sums and outputs follow by powers of two: a key is off by no more than
// 2^-39 of its tile's largest (half of fp16's smallest step), all of them by 2^-34 of
// the sum.  That costs up to 1% (48 windows of 4096 at D = 64 53.8 us either way, 32
// sequences to 16k at D = 128 58.8 -> 59.1); a tile's product of its own, joined by an
// fp32 factor, spills at D = 128 (79.7).
// Bound by memory: 131k positions of 8 heads of 128 in bf16 (537 MB) in 87 us,
// 6.2 TB/s, where reading alone takes 80; 24 sequences of 9k to 65k in e4m3 (1.5
// GB) 5.5 TB/s with the launch behind it.  Groups of more than 16 query heads read K
// and V once for every 16 (8 sequences of 60k on one key head: 16 heads 59 us, 32 87,
// 64 145).  V passes the caches (131k positions with the launch behind it 96 us,
// through them 105); K does not (the same 96 past them, but 1100 positions 10.0 ->
// 10.7 us).  More in flight (two tiles at once, the next one's loads ahead) changed
// nothing.
constexpr int attn_waves(int D, bool fp8) {  // wavefronts a SIMD that the registers are cut to
  // (D = 256 needs 256 registers and a few more in 16 bits: one wavefront 107 us, two
  // that spill 113; in e4m3 two 58, one 75)
  return D == 64 ? 4 : D == 128 ? 3 : fp8 ? 2 : 1;
}

// fp16: log2 of a tile's largest probability (less than 15), and how far below the
// largest so far a tile is taken as it is (deeper, its keys are off by up to 2^-99 of
// the sum; the sums stay below 2^(15 + 60 + 31), the outputs 2^16 times that)
constexpr float kTopBits = 14.f, kMostBelow = 60.f;

// 16-bit values whose sum is a probability in the product with V
constexpr int prob_parts(int type) { return type == SCOPE_FP16 ? 2 : 3; }

template <int TYPE, bool FP8, int D>
__global__ __launch_bounds__(kAttnThreads, attn_waves(D, FP8)) void paged_attn_kernel(scope_paged_cache c, PagedAttnArgs a, AttnSplit s) {
  constexpr int NJ = D / 32;                     // products over D
  constexpr int VE = D / 16 < 8 ? D / 16 : 8;    // features of a lane in a row of V
  constexpr int NH = D / (16 * VE);              // rows of V in halves
  constexpr int ES = FP8 ? 1 : 2;                // bytes of an element
  constexpr int KV = FP8 ? NJ / 2 : NJ;          // 16-byte loads of a row of K a lane
  constexpr int VW = VE * ES / 4;                // words of a lane in a row of V
  extern __shared__ float lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g4 = lane >> 4, c16 = lane & 15;
  const int G = a.Hq / c.Hkv, ng = (G + 15) / 16;
  const int hk = blockIdx.y / ng, cg = blockIdx.y % ng, nq = min(16, G - 16 * cg);
  const int h0 = hk * G + 16 * cg;  // first query head
  const bool lists = a.kv_idx != nullptr;
  Piece p;
  int n_list = 0;
  if (lists) {
    // pieces of one length for every list, so that the list is read without waiting for its number
    p.b = blockIdx.x / s.pieces;
    p.i = blockIdx.x % s.pieces;
    p.n = s.pieces;
    p.slot = p.b * s.pieces;
    n_list = min(max(a.kv_num[static_cast<int64_t>(p.b) * c.Hkv + hk], 0), a.maxkv);
    piece_range(0, static_cast<int>(s.tiles_cap), p.n, p.i, &p.t0, &p.t1);
  } else if (!find_piece(c, a, blockIdx.x, piece_turn(D), [&](int64_t) { return s.pieces; }, p)) {
    return;
  }
  const int b = p.b;
  if (s.plan && blockIdx.y == 0 && p.i == 0 && threadIdx.x == 0) s.plan[b] = make_int2(p.n, p.slot);
  const int64_t cap = static_cast<int64_t>(c.MP) * c.bs;
  const int end = static_cast<int>(seq_end(a.lens[b], cap)), low = a.first ? max(a.first[b], 0) : 0;
  const int32_t* row = a.table + static_cast<int64_t>(b) * c.MP;
  const int32_t* list = lists ? a.kv_idx + (static_cast<int64_t>(b) * c.Hkv + hk) * a.maxkv : nullptr;
  const int shift = __builtin_ctz(c.bs);
  const bool small = c.bs == 16;  // a tile is two pages

  // Q^T: column c is query head h0 + c
  uint4 qf[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int d = FP8 ? (j / 2) * 64 + g4 * 16 + (j % 2) * 8 : j * 32 + g4 * 8;
    qf[j] = make_uint4(0, 0, 0, 0);
    if (c16 < nq) qf[j] = *reinterpret_cast<const uint4*>(a.q + b * a.q_sb + (h0 + c16) * a.q_sh + d);
  }
  const float to_log2 = a.scale * kLog2e * (a.k_scale ? static_cast<const float*>(a.k_scale)[hk] : 1.f);

  f32x4_t acc[NH * VE];
#pragma unroll
  for (int i = 0; i < NH * VE; ++i) acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // the maximum so far, what the probabilities are taken relative to, their sum
  float m = -INFINITY, ref = 0.f, l = 0.f;

  const char* kbase = static_cast<const char*>(a.k_pages) + hk * c.k_sh * ES;
  const char* vbase = static_cast<const char*>(a.v_pages) + hk * c.v_sh * ES;
  const int krow = (c16 >> 2) * 8 + (c16 & 3), vrow = g4 * 8;
  const int64_t koff = ((small ? krow & 15 : krow) * c.k_sr + g4 * (16 / ES)) * ES;
  const int64_t voff = ((small ? vrow & 15 : vrow) * c.v_sr + c16 * VE) * ES;

  // pages and blocks of this wavefront's next 64 tiles, one a lane (two where a tile is two pages)
  int pg0 = -1, pg1 = -1, lb0 = 0, lb1 = 0;
  const auto resolve = [&](int t) {
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
      if (small) pg1 = one(e + 1, lb1);
    }
  };

  resolve(p.t0 + wave + lane * kAttnWaves);
  if (lists) p.t1 = min(p.t1, static_cast<int>((static_cast<int64_t>(n_list) * c.bs + kTileKeys - 1) / kTileKeys));
  int u = 0;
  for (int t = p.t0 + wave; t < p.t1; t += kAttnWaves, ++u) {
    if (u == 64) {
      resolve(t + lane * kAttnWaves);
      u = 0;
    }
    const int page0 = __builtin_amdgcn_readlane(pg0, u), page1 = small ? __builtin_amdgcn_readlane(pg1, u) : page0;
    const auto put_sum = [&](float x) {  // log2 of the tile's sum (of this lane's half of it)
      if (c16 < nq && (g4 & (small ? 1 : 3)) == 0)
        s.tile_lse[(((static_cast<int64_t>(b) * a.Hq + h0 + c16) * s.tiles_cap + t) << small) + (small ? g4 >> 1 : 0)] = x;
    };
    if (page0 < 0 && page1 < 0) {  // nothing to see
      if (s.tile_lse) put_sum(-INFINITY);
      continue;
    }
    const int r0 = small ? 0 : (t * kTileKeys) & (c.bs - 1);  // the tile's first row in its page
    // this lane's rows of K (product operand) and of V (and of the scores)
    const int kp = small && krow >= 16 ? page1 : page0, vp = small && vrow >= 16 ? page1 : page0;
    const char* kr = kbase + (static_cast<int64_t>(max(kp, 0)) * c.k_sp + r0 * c.k_sr) * ES + koff;
    const char* vr = vbase + (static_cast<int64_t>(max(vp, 0)) * c.v_sp + r0 * c.v_sr) * ES + voff;
    uint4 kf[2][KV];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < KV; ++j) kf[i][j] = *reinterpret_cast<const uint4*>(kr + 4 * i * c.k_sr * ES + j * 64);
    Words<VW> vf[NH][8];
    const auto load_v = [&](int h) {
#pragma unroll
      for (int i = 0; i < 8; ++i) vf[h][i] = load_once<VW>(vr + (i * c.v_sr + h * 128) * ES);
    };
    load_v(0);
    __builtin_amdgcn_sched_barrier(0);  // all loads are under way before the first is waited for

    // scores
    f32x4_t sc[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      sc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        if constexpr (FP8) {
          const uint4 w = kf[i][j / 2];
          const uint32_t x = j % 2 ? w.z : w.x, y = j % 2 ? w.w : w.y;
          sc[i] = mfma_16<TYPE>(make_uint4(widen2<TYPE, false>(x), widen2<TYPE, true>(x), widen2<TYPE, false>(y),
                                           widen2<TYPE, true>(y)), qf[j], sc[i]);
        } else {
          sc[i] = mfma_16<TYPE>(kf[i][j], qf[j], sc[i]);
        }
      }
    }
    if constexpr (NH > 1) {  // D = 256: into K's registers, which are free by now
      __builtin_amdgcn_sched_barrier(0);
      load_v(1);
    }
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = sc[i >> 2][i & 3] * to_log2;
    // the lane's first key; keys outside [low, end) and of no page are not seen
    const int lbl = small && vrow >= 16 ? __builtin_amdgcn_readlane(lb1, u) : __builtin_amdgcn_readlane(lb0, u);
    const int64_t pos = static_cast<int64_t>(lbl) * c.bs + r0 + (small ? vrow & 15 : vrow);
    const int from = vp < 0 ? 8 : static_cast<int>(min(max(low - pos, static_cast<int64_t>(0)), static_cast<int64_t>(8)));
    const int to = static_cast<int>(min(max(end - pos, static_cast<int64_t>(0)), static_cast<int64_t>(8)));
    if (__any(from > 0 || to < 8)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool see = i >= from && i < to;
        x[i] = see ? x[i] : -INFINITY;
        // (a row that is not seen may hold anything, and 0 times NaN is NaN)
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
          for (int w = 0; w < VW; ++w) vf[h][i].w[w] = see ? vf[h][i].w[w] : 0u;
      }
    }
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, x[i]);
    const auto rescale = [&](float f) {
      l *= f;
#pragma unroll
      for (int i = 0; i < NH * VE; ++i) acc[i] *= f;
    };
    if constexpr (TYPE == SCOPE_FP16) {
      top = over_rows(top, max_f32);
      const float mn = fmaxf(m, top), to = floorf(fmaxf(top, mn - kMostBelow)) - kTopBits;
      if (mn != -INFINITY) {
        rescale(m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ref - to));
        ref = to;
        m = mn;
      }
    } else if (__any(top > m + 8.f)) {
      top = over_rows(top, max_f32);
      const float mn = fmaxf(m, top);
      rescale(mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn));
      m = mn;
      ref = m == -INFINITY ? 0.f : m;
    }
    float lt = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = __builtin_amdgcn_exp2f(x[i] - ref);
      lt += x[i];
    }
    l += lt;
    if (s.tile_lse) {
      lt = small ? over_rows2(lt, add_f32) : over_rows(lt, add_f32);
      put_sum(ref + __builtin_amdgcn_logf(lt));
    }
    // the probabilities as a sum of 16-bit values each
    constexpr int NP = prob_parts(TYPE);
    uint4 pf[NP];
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = k + 1 < NP && !FP8 ? below2<TYPE>(x[2 * i], x[2 * i + 1]) : round2<TYPE>(x[2 * i], x[2 * i + 1]);
        x[2 * i] -= low_half<TYPE>(w[i]);
        x[2 * i + 1] -= high_half<TYPE>(w[i]);
      }
      pf[k] = make_uint4(w[0], w[1], w[2], w[3]);
    }
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      if constexpr (NH > 1) __builtin_amdgcn_sched_barrier(0);  // (or registers spill: e4m3 59 us, this way 55.5)
      uint32_t v[8][VE / 2];  // the eight rows as 16-bit pairs of neighbouring features
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int w = 0; w < VE / 2; ++w) {
          if constexpr (FP8)
            v[i][w] = w % 2 ? widen2<TYPE, true>(vf[h][i].w[w / 2]) : widen2<TYPE, false>(vf[h][i].w[w / 2]);
          else
            v[i][w] = vf[h][i].w[w];
        }
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        uint32_t op[4];
#pragma unroll
        for (int w = 0; w < 4; ++w)
          op[w] = j % 2 ? pack_hi16(v[2 * w][j / 2], v[2 * w + 1][j / 2]) : pack_lo16(v[2 * w][j / 2], v[2 * w + 1][j / 2]);
        const uint4 vt = make_uint4(op[0], op[1], op[2], op[3]);
#pragma unroll
        for (int k = 0; k < NP; ++k) acc[h * VE + j] = mfma_16<TYPE>(vt, pf[k], acc[h * VE + j]);
      }
    }
  }

  // the wavefronts' shares: maxima and sums, then the outputs of the group's queries
  l = over_rows(l, add_f32);
  const Shares z = shares_of(lds);
  if (g4 == 0) {
    z.sm[wave * 16 + c16] = m == -INFINITY ? m : ref;
    z.sl[wave * 16 + c16] = l;
  }
  if (c16 < nq) {
    float* o = z.so + (wave * nq + c16) * D + g4 * 4 * VE;
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < VE; j += 4)
          *reinterpret_cast<float4*>(o + h * 128 + r * VE + j) = make_float4(
              acc[h * VE + j][r], acc[h * VE + j + 1][r], acc[h * VE + j + 2][r], acc[h * VE + j + 3][r]);
  }
  __syncthreads();
  join_shares<TYPE, D>(a, s, p, h0, nq, a.v_scale ? static_cast<const float*>(a.v_scale)[hk] : 1.f, z);
}

// (maximum, sum relative to it) of a row from its n pieces' (maximum, sum) pairs,
// `step` floats apart: by one wavefront, the same in every lane; the first pair
// of each lane is read once.
__device__ __forceinline__ float2 join_sums(const float* ml, int n, int64_t step) {
  const int lane = threadIdx.x & 63;
  float m0 = -INFINITY, l0 = 0.f;
  if (lane < n) {
    m0 = ml[lane * step];
    l0 = ml[lane * step + 1];
  }
  float M = m0;
  for (int i = lane + 64; i < n; i += 64) M = fmaxf(M, ml[i * step]);
  M = max_of(M);
  float L = l0 == 0.f ? 0.f : __builtin_amdgcn_exp2f(m0 - M) * l0;
  for (int i = lane + 64; i < n; i += 64) {
    const float li = ml[i * step + 1];
    L += li == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml[i * step] - M) * li;
  }
  return make_float2(M, sum_of(L));
}

// What follows the pieces, for (sequence, key head) (blockIdx.z, blockIdx.y).
// The first G workgroups join the pieces of a query head of the group each, sixteen
// bytes of the output row a thread, the pieces shared out over groups of threads.
// With a mass, the others add 256 blocks' probabilities each, formed from their
// tiles' sums and the rows' whole ones, a block a thread, its heads and tiles in
// order.  Both in one launch: a second one costs more than the sums joined anew
// (4.7 us).
template <int D>
__global__ __launch_bounds__(256) void paged_finish_kernel(scope_paged_cache c, PagedAttnArgs a, AttnSplit s) {
  const int b = blockIdx.z, hk = blockIdx.y, G = a.Hq / c.Hkv;
  const int x = static_cast<int>(blockIdx.x) - (s.po ? G : 0);  // < 0: joins, else adds blocks
  const bool lists = a.kv_idx != nullptr;
  constexpr int LD = D / 4, NG = 256 / LD;
  __shared__ float w[kMostPieces], so[NG][D];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int2 plan = make_int2(1, 0);
  if (s.po) plan = lists ? make_int2(s.pieces, b * s.pieces) : s.plan[b];
  // (lengths that another stream changes under a call leave any plan: it stays among the slots)
  plan.y = min(max(plan.y, 0), s.slots - 1);
  const int n = min(min(max(plan.x, 1), s.slots - plan.y), kMostPieces);
  const int64_t step = 2ll * a.Hq;
  const float* ml0 = s.pml + (static_cast<int64_t>(plan.y) * a.Hq + hk * G) * 2;  // of the group's first head
  if (x < 0) {
    if (n == 1) return;  // written by its only piece
    const int g = x + G, h = hk * G + g;
    const float* ml = ml0 + 2 * g;
    const int dl = tid % LD, grp = tid / LD;
    const float* po = s.po + (static_cast<int64_t>(plan.y) * a.Hq + h) * D + 4 * dl;
    const int64_t row = static_cast<int64_t>(a.Hq) * D;
    // the first rows of each group are under way while the sums are formed
    constexpr int EARLY = 4;
    float4 v[EARLY];
#pragma unroll
    for (int k = 0; k < EARLY; ++k) v[k] = *reinterpret_cast<const float4*>(po + min(grp + k * NG, n - 1) * row);
    const float2 ML = join_sums(ml, n, step);
    for (int i = tid; i < n; i += 256) w[i] = ml[i * step + 1] == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml[i * step] - ML.x);
    __syncthreads();
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    const auto add = [&](const float4& r, float f) {
      acc.x += f * r.x;
      acc.y += f * r.y;
      acc.z += f * r.z;
      acc.w += f * r.w;
    };
#pragma unroll
    for (int k = 0; k < EARLY; ++k)
      if (grp + k * NG < n) add(v[k], w[grp + k * NG]);
#pragma unroll 4
    for (int i = grp + EARLY * NG; i < n; i += NG) add(*reinterpret_cast<const float4*>(po + i * row), w[i]);
    *reinterpret_cast<float4*>(&so[grp][4 * dl]) = acc;
    __syncthreads();
    if (tid < D) {
      float o = 0.f;
#pragma unroll
      for (int i = 0; i < NG; ++i) o += so[i][tid];
      const float y = ML.y == 0.f ? 0.f : o / ML.y * (a.v_scale ? static_cast<const float*>(a.v_scale)[hk] : 1.f);
      a.out[(static_cast<int64_t>(b) * a.Hq + h) * D + tid] = c.type == SCOPE_FP16 ? f32_to_half(y) : f32_to_bf16(y);
      if (tid == 0)
        a.lse[static_cast<int64_t>(b) * a.Hq + h] = ML.y == 0.f ? -INFINITY : (ML.x + __builtin_amdgcn_logf(ML.y)) * kLn2;
    }
    return;
  }
  const int blocks = lists ? a.maxkv : c.MP;
  const int64_t e = static_cast<int64_t>(x) * 256 + tid, bh = static_cast<int64_t>(b) * c.Hkv + hk;
  int64_t lb = -1;
  int lo = 0;
  int64_t hi;
  if (lists) {
    const int num = min(max(a.kv_num[bh], 0), a.maxkv);
    if (e < num) lb = a.kv_idx[bh * a.maxkv + e];
    hi = (static_cast<int64_t>(num) * c.bs + kTileKeys - 1) / kTileKeys;
  } else {
    if (e < blocks) lb = e;
    hi = seq_tiles(a.lens[b], a.first ? a.first[b] : 0, static_cast<int64_t>(c.MP) * c.bs, &lo);
    hi += lo;
  }
  // the block's tiles (half tiles of blocks of 16) among those that were formed
  const int halves = c.bs == 16 ? 2 : 1, per = c.bs == 16 ? 1 : c.bs / kTileKeys;
  const int64_t u0 = max(e * per, static_cast<int64_t>(lo) * halves), u1 = min((e + 1) * per, hi * halves);
  const bool live = lb >= 0 && lb < c.MP && u0 < u1;
  float sum = 0.f;
  for (int g0 = 0; g0 < G; g0 += 256) {
    __syncthreads();
    const int ng = min(256, G - g0);
    for (int g = wave; g < ng; g += 4) {  // log2 of the heads' whole sums
      float all;
      if (n > 1) {
        const float2 ML = join_sums(ml0 + 2 * (g0 + g), n, step);
        all = ML.y == 0.f ? -INFINITY : ML.x + __builtin_amdgcn_logf(ML.y);
      } else {
        all = s.lse2[static_cast<int64_t>(b) * a.Hq + hk * G + g0 + g];
      }
      if (lane == 0) w[g] = all;
    }
    __syncthreads();
    for (int g = 0; g < ng && live; ++g) {
      const float all = w[g];
      if (all == -INFINITY) continue;
      const float* t = s.tile_lse + (static_cast<int64_t>(b) * a.Hq + hk * G + g0 + g) * s.tiles_cap * halves;
      for (int64_t u = u0; u < u1; ++u) sum += __builtin_amdgcn_exp2f(t[u] - all);
    }
  }
  if (!live) return;
  // (a list may name a block once; an atomic for the lists that break this)
  if (lists)
    atomicAdd(a.mass + bh * c.MP + lb, sum);
  else
    a.mass[bh * c.MP + lb] += sum;
}

// ---- eviction -----------------------------------------------------------------
struct EvictArgs {
  int B, Hkv, MP, bs, window, n_global;
  const int32_t* table;
  const float* mass;
  const int32_t* lens;
  const int32_t* budget;
  int32_t* table_out;
  int32_t* freed;
  int32_t* n_freed;
};

// A total order of the accumulated weights: unsigned keys that compare as the
// floats do, -0 as +0, NaN above them, and above all a block that may not go.
constexpr uint32_t kKeyNaN = 0xfffffffeu, kKeyStays = 0xffffffffu;
__device__ __forceinline__ uint32_t weight_key(float f) {
  if (f != f) return kKeyNaN;
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

// One workgroup per sequence, K blocks a thread (block i = 1024·k + thread) with
// their keys in registers, so that mass is read once.  The n-th smallest key is
// found in three digits of 11, 11 and 10 bits: the keys that agree with the
// digits found so far are counted by their next one in LDS, and the digit is
// where the running count passes n.  Blocks with a smaller key go, of those with
// the same key the first ones.  Bound by latency: one sequence of 1027 blocks and
// 8 heads 6.3 us (10.8 with the key found two bits at a time by ballots), 64 of
// 8192 blocks 14.5 us for 15 MB (a workgroup a sequence; 37.6 with the ballots
// and 16 loads a thread under way instead of 32), one of 16384 20.4, of 16385 38.7
// and of 65536 72 us (64 blocks a thread).
constexpr int kEvictThreads = 1024, kEvictWaves = kEvictThreads / 64;

constexpr int kDigit = 11, kBins = 1 << kDigit;

// counts[k·16 + wavefront] = the set flags before that group of 64 blocks, in the
// blocks' order; returns the sum of all.  counts: K·16 + 1 ints of LDS.
template <int K, class Flag>
__device__ __forceinline__ int prefix_flags(Flag flag, int* counts) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int n = __popcll(__ballot(flag(k)));
    if (lane == 0) counts[k * kEvictWaves + wave] = n;
  }
  __syncthreads();
  if (wave == 0) {  // K·16 counts, K/4 neighbouring ones a lane
    constexpr int N = K * kEvictWaves, PER = N < 64 ? 1 : N / 64;
    int v[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      v[i] = lane * PER + i < N ? counts[lane * PER + i] : 0;
      sum += v[i];
    }
    const int upto = prefix_of(sum);
    int at = upto - sum;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (lane * PER + i < N) counts[lane * PER + i] = at;
      at += v[i];
    }
    if (lane == 63) counts[N] = upto;
  }
  __syncthreads();
  return counts[K * kEvictWaves];
}

template <int K>
__global__ __launch_bounds__(kEvictThreads) void paged_evict_kernel(EvictArgs a) {
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t base = static_cast<int64_t>(b) * a.MP;
  __shared__ int counts[K * kEvictWaves + 1];
  __shared__ int bins[kBins], totals[2 * kEvictWaves], found[2];
  const int64_t len = a.lens[b];
  const int n = len <= 0 ? 0 : static_cast<int>(min((len + a.bs - 1) / a.bs, static_cast<int64_t>(a.MP)));
  uint32_t key[K];
  int held = 0, may = 0;  // of the wavefront
  // KG blocks and eight heads at a time, so that their loads are under way
  // together (block indices past the row are cut to it, and left out of the keys)
  constexpr int KG = K < 4 ? K : 4;
  const float* mass = a.mass + static_cast<int64_t>(b) * a.Hkv * a.MP;
#pragma unroll
  for (int g = 0; g < K; g += KG) {
#pragma unroll
    for (int k = 0; k < KG; ++k) key[g + k] = kKeyStays;
    if (g * kEvictThreads >= n) continue;
    int id[KG];
    double sum[KG];
    uint32_t at[KG];
#pragma unroll
    for (int k = 0; k < KG; ++k) {
      at[k] = min((g + k) * kEvictThreads + tid, a.MP - 1);
      id[k] = a.table[base + at[k]];
      sum[k] = 0.0;
    }
    int h = 0;
    for (; h + 8 <= a.Hkv; h += 8) {
      float f[8][KG];
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int k = 0; k < KG; ++k) f[j][k] = (mass + static_cast<int64_t>(h + j) * a.MP)[at[k]];
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int k = 0; k < KG; ++k) sum[k] += f[j][k];
    }
    for (; h < a.Hkv; ++h)
#pragma unroll
      for (int k = 0; k < KG; ++k) sum[k] += (mass + static_cast<int64_t>(h) * a.MP)[at[k]];
#pragma unroll
    for (int k = 0; k < KG; ++k) {
      const int i = (g + k) * kEvictThreads + tid;
      const bool here = i < n && id[k] >= 0, can = here && i >= a.n_global && i < n - a.window;
      held += __popcll(__ballot(here));
      may += __popcll(__ballot(can));
      if (can) key[g + k] = weight_key(static_cast<float>(sum[k]));
    }
  }
  if (lane == 0) {
    totals[wave] = held;
    totals[kEvictWaves + wave] = may;
  }
  __syncthreads();
  held = may = 0;
#pragma unroll
  for (int w = 0; w < kEvictWaves; ++w) {
    held += totals[w];
    may += totals[kEvictWaves + w];
  }
  const int n_drop = min(max(held - max(a.budget[b], 0), 0), may);
  uint64_t go = 0;  // bit k: block k of this thread
  if (n_drop > 0) {
    uint32_t cut = 0;  // the n_drop-th smallest key, its digits from the top
    int below = 0;     // keys below it
    static_assert(kBins == 2 * kEvictThreads, "two bins a thread");
#pragma unroll
    for (int digit = 0; digit < 3; ++digit) {
      const int low = digit == 0 ? 21 : digit == 1 ? 10 : 0, width = digit == 2 ? 10 : kDigit, top = low + width;
      bins[2 * tid] = bins[2 * tid + 1] = 0;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (key[k] != kKeyStays && (digit == 0 || key[k] >> (top & 31) == cut >> (top & 31)))
          atomicAdd(&bins[key[k] >> low & ((1 << width) - 1)], 1);
      __syncthreads();
      const int b0 = bins[2 * tid], b1 = bins[2 * tid + 1], upto = prefix_of(b0 + b1);
      if (lane == 63) totals[wave] = upto;
      __syncthreads();
      int before = below + upto - b0 - b1;
#pragma unroll
      for (int w = 0; w < kEvictWaves; ++w) before += w < wave ? totals[w] : 0;
      if (before < n_drop && n_drop <= before + b0 + b1) {  // one thread
        const bool second = n_drop > before + b0;
        found[0] = 2 * tid + second;
        found[1] = before + (second ? b0 : 0);
      }
      __syncthreads();
      cut |= static_cast<uint32_t>(found[0]) << low;
      below = found[1];
    }
    prefix_flags<K>([&](int k) { return key[k] == cut; }, counts);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const uint64_t same = __ballot(key[k] == cut);
      const int rank = below + counts[k * kEvictWaves + wave] + __popcll(same & ((1ull << lane) - 1));
      if (key[k] < cut || (key[k] == cut && rank < n_drop)) go |= 1ull << k;
    }
  }
  // ids in the blocks' order
  const int all = prefix_flags<K>([&](int k) { return go >> k & 1; }, counts);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = k * kEvictThreads + tid;
    const bool mine = go >> k & 1;
    const uint64_t gone = __ballot(mine);
    if (i < a.MP) {
      const int id = a.table[base + i];  // (this thread alone writes table_out's entry, which may be this one)
      if (mine) a.freed[base + counts[k * kEvictWaves + wave] + __popcll(gone & ((1ull << lane) - 1))] = id;
      a.table_out[base + i] = mine ? -1 : id;
    }
  }
  for (int i = all + tid; i < a.MP; i += kEvictThreads) a.freed[base + i] = -1;
  if (tid == 0) a.n_freed[b] = all;
}

int check_cache(const scope_paged_cache* c, const void* k_pages, const void* v_pages, const char* fn) {
  SCOPE_REQUIRE(c, "%s: null cache", fn);
  SCOPE_REQUIRE(c->D == 64 || c->D == 128 || c->D == 256, "%s: head dim must be 64, 128 or 256, got %d", fn, c->D);
  SCOPE_REQUIRE(c->bs == 16 || c->bs == 32 || c->bs == 64 || c->bs == 128 || c->bs == 256,
                "%s: page size must be 16, 32, 64, 128 or 256, got %d", fn, c->bs);
  SCOPE_REQUIRE(c->type == SCOPE_BF16 || c->type == SCOPE_FP16, "%s: unknown type %d", fn, c->type);
  SCOPE_REQUIRE(c->B >= 1 && c->B <= 65535 && c->Hkv >= 1 && c->Hkv <= 4096 && c->P >= 1,
                "%s: bad sizes B=%d (1 .. 65535), Hkv=%d (1 .. 4096), P=%lld (at least 1)", fn, c->B, c->Hkv, (long long)c->P);
  // (less than 2^26 tiles a row: the plan sums 64 rows in 32 bits)
  SCOPE_REQUIRE(c->MP >= 1 && static_cast<int64_t>(c->MP) * c->bs <= INT32_MAX - (kTileKeys - 1),
                "%s: a table row of %d pages of %d positions (1 .. 2^31 - 32 positions)", fn, c->MP, c->bs);
  const int al = c->fp8 ? 16 : 8;  // elements of 16 bytes
  SCOPE_REQUIRE(k_pages && v_pages, "%s: null pages", fn);
  SCOPE_REQUIRE(c->k_sp % al == 0 && c->k_sh % al == 0 && c->k_sr % al == 0 && c->v_sp % al == 0 && c->v_sh % al == 0 &&
                    c->v_sr % al == 0 && aligned16(k_pages) && aligned16(v_pages),
                "%s: the rows of the pages must be 16-byte aligned", fn);
  return SCOPE_OK;
}

namespace {
// The pieces of a call and its workspace (laid out in `work` where s is given);
// returns its bytes.
int64_t plan_split(const scope_paged_cache& c, int Hq, int maxkv, bool with_mass, AttnSplit* out, void* work) {
  const SplitSizes z = split_sizes(c.B, c.Hkv, c.D, c.bs, c.MP, Hq, maxkv);
  AttnSplit s{};
  s.pieces = z.pieces;
  s.slots = z.slots;
  s.tiles_cap = z.tiles_cap;
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    char* p = work ? static_cast<char*>(work) + at : nullptr;
    at += (bytes + 15) & ~static_cast<int64_t>(15);
    return p;
  };
  if (z.split) {
    s.po = reinterpret_cast<float*>(take(4ll * s.slots * Hq * c.D));
    s.pml = reinterpret_cast<float*>(take(8ll * s.slots * Hq));
    s.plan = reinterpret_cast<int2*>(take(8ll * c.B));
  }
  if (with_mass) {
    s.lse2 = reinterpret_cast<float*>(take(4ll * c.B * Hq));
    s.tile_lse = reinterpret_cast<float*>(take(4ll * c.B * Hq * s.tiles_cap * (c.bs == 16 ? 2 : 1)));
  }
  if (out) *out = s;
  return at;
}
}  // namespace

int check_attn(const scope_paged_cache& c, const PagedAttnArgs& a, void* work, AttnSplit* s, const char* fn) {
  SCOPE_REQUIRE(a.Hq >= 1 && a.Hq <= 65535 && a.Hq % c.Hkv == 0, "%s: Hq=%d must be a multiple of Hkv=%d, at most 65535", fn,
                a.Hq, c.Hkv);
  SCOPE_REQUIRE((a.kv_num != nullptr) == (a.kv_idx != nullptr) &&
                    (a.kv_idx ? a.maxkv >= 1 && static_cast<int64_t>(a.maxkv) * c.bs <= INT32_MAX : a.maxkv == 0),
                "%s: kv_num and kv_idx come together, with 1 .. 2^31 / bs entries (maxkv=%d; 0 without lists)", fn, a.maxkv);
  SCOPE_REQUIRE(a.q && a.table && a.lens && a.out && a.lse, "%s: null pointer", fn);
  SCOPE_REQUIRE(plan_split(c, a.Hq, a.maxkv, a.mass != nullptr, s, work) == 0 || work, "%s: null pointer (the workspace)", fn);
  SCOPE_REQUIRE(aligned16(a.q) && aligned16(work) && a.q_sb % 8 == 0 && a.q_sh % 8 == 0,
                "%s: the rows of q and the workspace must be 16-byte aligned", fn);
  return SCOPE_OK;
}

int launch_paged_finish(const scope_paged_cache& c, const PagedAttnArgs& args, const float* v_scale, const AttnSplit& s, hipStream_t st) {
  if (!s.po && !args.mass) return SCOPE_OK;  // every sequence is one piece
  PagedAttnArgs a = args;
  a.v_scale = v_scale;
  const int G = a.Hq / c.Hkv, blocks = a.kv_idx ? a.maxkv : c.MP;
  const dim3 fg((s.po ? G : 0) + (a.mass ? ceil_div(blocks, 256) : 0), c.Hkv, c.B);
  if (c.D == 64)
    hipLaunchKernelGGL(paged_finish_kernel<64>, fg, dim3(256), 0, st, c, a, s);
  else if (c.D == 128)
    hipLaunchKernelGGL(paged_finish_kernel<128>, fg, dim3(256), 0, st, c, a, s);
  else
    hipLaunchKernelGGL(paged_finish_kernel<256>, fg, dim3(256), 0, st, c, a, s);
  return check_launch("paged_finish_kernel");
}

}  // namespace scope

using namespace scope;

extern "C" {

int scope_paged_append(const scope_paged_cache* c, int64_t N, const uint16_t* k, int64_t k_sn, int64_t k_sh,
                       const uint16_t* v, int64_t v_sn, int64_t v_sh, const int32_t* cu, const int32_t* table,
                       const int32_t* lens, const float* k_scale, const float* v_scale, void* k_pages, void* v_pages,
                       void* stream) {
  const char* fn = "scope_paged_append";
  if (int rc = check_cache(c, k_pages, v_pages, fn)) return rc;
  SCOPE_REQUIRE(N >= 0 && N <= INT32_MAX, "%s: %lld rows (0 .. 2^31 - 1)", fn, (long long)N);
  SCOPE_REQUIRE(cu || N <= c->B, "%s: %lld rows for %d sequences need cu", fn, (long long)N, c->B);
  if (N == 0) return SCOPE_OK;
  SCOPE_REQUIRE(k && v && table && lens, "%s: null pointer", fn);
  SCOPE_REQUIRE(aligned16(k) && aligned16(v) && k_sn % 8 == 0 && k_sh % 8 == 0 && v_sn % 8 == 0 && v_sh % 8 == 0,
                "%s: the rows of k and v must be 16-byte aligned", fn);
  const int rows = append_rows(N);
  const AppendArgs a{N, k_sn, k_sh, v_sn, v_sh, rows, k, v, cu, table, lens, k_scale, v_scale, k_pages, v_pages};
  const dim3 grid(ceil_div(N, 4 * rows)), block(256);
  hipStream_t st = as_stream(stream);
  if (!c->fp8)  // (16-bit values are moved as they are)
    hipLaunchKernelGGL((paged_append_kernel<SCOPE_BF16, false>), grid, block, 0, st, *c, a);
  else if (c->type == SCOPE_BF16)
    hipLaunchKernelGGL((paged_append_kernel<SCOPE_BF16, true>), grid, block, 0, st, *c, a);
  else
    hipLaunchKernelGGL((paged_append_kernel<SCOPE_FP16, true>), grid, block, 0, st, *c, a);
  return check_launch("paged_append_kernel");
}

int64_t scope_paged_attn_workspace_bytes(const scope_paged_cache* c, int Hq, int maxkv, int with_mass) {
  if (!c || c->B < 1 || c->MP < 1 || c->bs < 1 || c->D < 1 || c->Hkv < 1 || Hq < 1 || Hq % c->Hkv || maxkv < 0) return 0;
  return plan_split(*c, Hq, maxkv, with_mass != 0, nullptr, nullptr);
}

int scope_paged_decode_attn(const scope_paged_cache* c, int Hq, int maxkv, float scale, const uint16_t* q, int64_t q_sb,
                            int64_t q_sh, const void* k_pages, const void* v_pages, const float* k_scale,
                            const float* v_scale, const int32_t* table, const int32_t* lens, const int32_t* first,
                            const int32_t* kv_num, const int32_t* kv_idx, float* mass, void* work, uint16_t* out,
                            float* lse, void* stream) {
  const char* fn = "scope_paged_decode_attn";
  if (int rc = check_cache(c, k_pages, v_pages, fn)) return rc;
  const PagedAttnArgs a{Hq,    maxkv, scale, q_sb,   q_sh,   q,    k_pages, v_pages, k_scale,
                        v_scale, table, lens,  first, kv_num, kv_idx, mass, out,     lse};
  AttnSplit s;
  if (int rc = check_attn(*c, a, work, &s, fn)) return rc;
  const int G = Hq / c->Hkv, ng = (G + 15) / 16;
  const dim3 grid(s.slots, c->Hkv * ng);
  const size_t lds = sizeof(float) * kAttnWaves * (32 + static_cast<size_t>(std::min(G, 16)) * c->D);
  hipStream_t st = as_stream(stream);
  const auto launch = [&](auto type, auto fp8) {
    constexpr int T = decltype(type)::value;
    constexpr bool F = decltype(fp8)::value;
    if (c->D == 64)
      hipLaunchKernelGGL((paged_attn_kernel<T, F, 64>), grid, dim3(kAttnThreads), lds, st, *c, a, s);
    else if (c->D == 128)
      hipLaunchKernelGGL((paged_attn_kernel<T, F, 128>), grid, dim3(kAttnThreads), lds, st, *c, a, s);
    else
      hipLaunchKernelGGL((paged_attn_kernel<T, F, 256>), grid, dim3(kAttnThreads), lds, st, *c, a, s);
  };
  using std::integral_constant;
  if (c->type == SCOPE_BF16)
    c->fp8 ? launch(integral_constant<int, SCOPE_BF16>{}, integral_constant<bool, true>{})
           : launch(integral_constant<int, SCOPE_BF16>{}, integral_constant<bool, false>{});
  else
    c->fp8 ? launch(integral_constant<int, SCOPE_FP16>{}, integral_constant<bool, true>{})
           : launch(integral_constant<int, SCOPE_FP16>{}, integral_constant<bool, false>{});
  if (int rc = check_launch("paged_attn_kernel")) return rc;
  return launch_paged_finish(*c, a, v_scale, s, st);
}

int scope_paged_evict(int B, int Hkv, int MP, int bs, int window, int n_global, const int32_t* table, const float* mass,
                      const int32_t* lens, const int32_t* budget, int32_t* table_out, int32_t* freed, int32_t* n_freed,
                      void* stream) {
  const char* fn = "scope_paged_evict";
  SCOPE_REQUIRE(B >= 1 && B <= 65535 && Hkv >= 1 && MP >= 1 && MP <= SCOPE_PAGED_EVICT_MAX_PAGES && bs >= 1,
                "%s: bad sizes B=%d (1 .. 65535), Hkv=%d, MP=%d (1 .. %d), bs=%d", fn, B, Hkv, MP, SCOPE_PAGED_EVICT_MAX_PAGES, bs);
  SCOPE_REQUIRE(window >= 1 && n_global >= 0, "%s: window=%d must be at least 1 (the page being written stays), n_global=%d at least 0",
                fn, window, n_global);
  SCOPE_REQUIRE(table && mass && lens && budget && table_out && freed && n_freed, "%s: null pointer", fn);
  const EvictArgs a{B, Hkv, MP, bs, window, n_global, table, mass, lens, budget, table_out, freed, n_freed};
  const dim3 grid(B), block(kEvictThreads);
  hipStream_t st = as_stream(stream);
  const int k = ceil_div(MP, kEvictThreads);
  if (k <= 1)
    hipLaunchKernelGGL(paged_evict_kernel<1>, grid, block, 0, st, a);
  else if (k <= 2)
    hipLaunchKernelGGL(paged_evict_kernel<2>, grid, block, 0, st, a);
  else if (k <= 4)
    hipLaunchKernelGGL(paged_evict_kernel<4>, grid, block, 0, st, a);
  else if (k <= 8)
    hipLaunchKernelGGL(paged_evict_kernel<8>, grid, block, 0, st, a);
  else if (k <= 16)
    hipLaunchKernelGGL(paged_evict_kernel<16>, grid, block, 0, st, a);
  else
    hipLaunchKernelGGL(paged_evict_kernel<64>, grid, block, 0, st, a);
  return check_launch("paged_evict_kernel");
}

}  // extern "C"
