// The paged key-value cache of a decode loop: rows of new tokens written to
// their pages, the attention of one new token per sequence over its pages,
// and the choice of the pages that leave when the cache is over its budget.
//
// Pages are [P][Hkv][bs][D] (any page, head and row strides); row b of the
// table [B][MP] names the page of each block of bs positions of sequence b.
// An entry outside [0, P) is a block without a page (not there yet, or
// evicted): nothing is written to it and no key of it is seen.
#include <math.h>

#include "common.h"

namespace scope {

namespace {
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float half_to_f32(uint16_t h) { return static_cast<float>(__builtin_bit_cast(_Float16, h)); }
__device__ __forceinline__ uint16_t f32_to_half(float f) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f)); }

// positions that sequence b holds: its length cut to the table's, the first one seen
__device__ __forceinline__ int64_t seq_end(const scope_paged_cache& c, const int32_t* lens, int b) {
  const int64_t n = lens[b], cap = static_cast<int64_t>(c.MP) * c.bs;
  return n < 0 ? 0 : n < cap ? n : cap;
}

// two floats from two e4m3 bytes (the low two, or the high two, of w)
template <bool HI>
__device__ __forceinline__ float2 e4m3x2(uint32_t w) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  const f32x2_t f = __builtin_amdgcn_cvt_pk_f32_fp8(w, HI);
  return make_float2(f[0], f[1]);
}
}  // namespace

// ---- append ------------------------------------------------------------------
// Row i of the N new ones belongs to the sequence b with cu[b] <= i < cu[b + 1]
// (row i to sequence i without cu) and goes to position lens[b] + i - cu[b].
// One wavefront per row.
struct AppendArgs {
  int64_t N, k_sn, k_sh, v_sn, v_sh;
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

// the e4m3 byte of x / s: the quotient cut to the largest finite value, then
// rounded to nearest even (one rounding each; NaN stays NaN)
__device__ __forceinline__ uint8_t to_e4m3(float x, float s) {
  const float q = x / s;
  const float y = q > 448.f ? 448.f : q < -448.f ? -448.f : q;
  return static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false) & 0xff);
}

__global__ __launch_bounds__(256) void paged_append_kernel(scope_paged_cache c, AppendArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (i >= a.N) return;
  int b = static_cast<int>(i);
  int64_t pos = 0;
  if (a.cu) {
    int lo = 0, hi = c.B;  // the last b in [0, B) with cu[b] <= i
    while (lo + 1 < hi) {
      const int mid = (lo + hi) >> 1;
      if (a.cu[mid] <= i) lo = mid; else hi = mid;
    }
    b = lo;
    if (i < a.cu[b] || i >= a.cu[b + 1]) return;  // a row of no sequence
    pos = i - a.cu[b];
  }
  pos += a.lens[b];
  if (pos < 0 || pos >= static_cast<int64_t>(c.MP) * c.bs) return;
  const int64_t page = a.table[static_cast<int64_t>(b) * c.MP + pos / c.bs];
  if (page < 0 || page >= c.P) return;
  const int64_t r = pos % c.bs;
  for (int e = lane; e < c.Hkv * c.D; e += 64) {
    const int h = e / c.D, d = e % c.D;
    const uint16_t xk = a.k[i * a.k_sn + h * a.k_sh + d], xv = a.v[i * a.v_sn + h * a.v_sh + d];
    const int64_t ok = page * c.k_sp + h * c.k_sh + r * c.k_sr + d, ov = page * c.v_sp + h * c.v_sh + r * c.v_sr + d;
    if (c.fp8) {
      const float fk = c.type == SCOPE_FP16 ? half_to_f32(xk) : bf16_to_f32(xk);
      const float fv = c.type == SCOPE_FP16 ? half_to_f32(xv) : bf16_to_f32(xv);
      static_cast<uint8_t*>(a.k_pages)[ok] = to_e4m3(fk, a.k_scale ? a.k_scale[h] : 1.f);
      static_cast<uint8_t*>(a.v_pages)[ov] = to_e4m3(fv, a.v_scale ? a.v_scale[h] : 1.f);
    } else {
      static_cast<uint16_t*>(a.k_pages)[ok] = xk;
      static_cast<uint16_t*>(a.v_pages)[ov] = xv;
    }
  }
}

// ---- attention of one new token -------------------------------------------------
struct PagedAttnArgs {
  int Hq, maxkv;
  float scale;
  int64_t q_sb, q_sh;
  const uint16_t* q;
  const void* k_pages;
  const void* v_pages;
  const float* k_scale;
  const float* v_scale;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* first;
  const int32_t* kv_num;
  const int32_t* kv_idx;
  float* mass;
  uint16_t* out;
  float* lse;
};

__device__ __forceinline__ float paged_value(const scope_paged_cache& c, const void* pages, int64_t off) {
  if (c.fp8) return e4m3x2<false>(static_cast<const uint8_t*>(pages)[off]).x;
  const uint16_t x = static_cast<const uint16_t*>(pages)[off];
  return c.type == SCOPE_FP16 ? half_to_f32(x) : bf16_to_f32(x);
}

// One workgroup per (sequence, key head), its wavefronts taking keys in turn
// with the running maximum and sum of a softmax, merged at the end; then, for
// the mass, the probabilities of every page's keys once more.
constexpr int kSimpleWaves = 16;

__global__ __launch_bounds__(64 * kSimpleWaves) void paged_attn_simple_kernel(scope_paged_cache c, PagedAttnArgs a) {
  const int b = blockIdx.x, hk = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int G = a.Hq / c.Hkv, per = c.D / 64;
  __shared__ float sm[kSimpleWaves], sl[kSimpleWaves], so[kSimpleWaves][256], s_lse;
  const int64_t end = seq_end(c, a.lens, b);
  const int64_t low = a.first ? max(a.first[b], 0) : 0;
  const int64_t row = static_cast<int64_t>(b) * c.Hkv + hk;
  const int n = a.kv_idx ? min(max(a.kv_num[row], 0), a.maxkv) : static_cast<int>((end + c.bs - 1) / c.bs);
  const float ks = a.k_scale ? a.k_scale[hk] : 1.f, vs = a.v_scale ? a.v_scale[hk] : 1.f;
  for (int g = 0; g < G; ++g) {
    const int h = hk * G + g;
    float qv[4];
    for (int i = 0; i < per; ++i) {
      const uint16_t x = a.q[b * a.q_sb + h * a.q_sh + lane * per + i];
      qv[i] = (c.type == SCOPE_FP16 ? half_to_f32(x) : bf16_to_f32(x)) * (a.scale * kLog2e * ks);
    }
    const auto page_of = [&](int e, int64_t& lb) -> int64_t {
      lb = a.kv_idx ? a.kv_idx[row * a.maxkv + e] : e;
      if (lb < 0 || lb >= c.MP) return -1;
      const int64_t page = a.table[static_cast<int64_t>(b) * c.MP + lb];
      return page < c.P ? page : -1;
    };
    const auto score = [&](int64_t page, int r) {
      float s = 0.f;
      for (int i = 0; i < per; ++i)
        s = fmaf(paged_value(c, a.k_pages, page * c.k_sp + hk * c.k_sh + r * c.k_sr + lane * per + i), qv[i], s);
      for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, kWave);
      return s;
    };
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int e = 0; e < n; ++e) {
      int64_t lb;
      const int64_t page = page_of(e, lb);
      if (page < 0) continue;
      for (int r = wave; r < c.bs; r += kSimpleWaves) {
        const int64_t j = lb * c.bs + r;
        if (j < low || j >= end) continue;
        const float s = score(page, r);
        const float mn = !(s <= m) ? s : m;  // NaN stays
        const float keep = m == -INFINITY ? 0.f : exp2f(m - mn), pr = s == -INFINITY ? 0.f : exp2f(s - mn);
        l = l * keep + pr;
        for (int i = 0; i < per; ++i)
          o[i] = o[i] * keep + pr * paged_value(c, a.v_pages, page * c.v_sp + hk * c.v_sh + r * c.v_sr + lane * per + i);
        m = mn;
      }
    }
    if (lane == 0) {
      sm[wave] = m;
      sl[wave] = l;
    }
    for (int i = 0; i < per; ++i) so[wave][lane * per + i] = o[i];
    __syncthreads();
    float M = -INFINITY, L = 0.f;
    for (int w = 0; w < kSimpleWaves; ++w) M = !(sm[w] <= M) ? sm[w] : M;
    for (int w = 0; w < kSimpleWaves; ++w) L += sm[w] == -INFINITY ? 0.f : exp2f(sm[w] - M) * sl[w];
    for (int d = threadIdx.x; d < c.D; d += blockDim.x) {
      float acc = 0.f;
      for (int w = 0; w < kSimpleWaves; ++w) acc += sm[w] == -INFINITY ? 0.f : exp2f(sm[w] - M) * so[w][d];
      const float y = L == 0.f ? 0.f : acc / L * vs;
      a.out[(static_cast<int64_t>(b) * a.Hq + h) * c.D + d] = c.type == SCOPE_FP16 ? f32_to_half(y) : f32_to_bf16(y);
    }
    const float lse2 = L == 0.f ? -INFINITY : M + log2f(L);
    if (threadIdx.x == 0) {
      a.lse[static_cast<int64_t>(b) * a.Hq + h] = lse2 * kLn2;
      s_lse = lse2;
    }
    __syncthreads();
    if (a.mass) {
      for (int e = wave; e < n; e += kSimpleWaves) {
        int64_t lb;
        const int64_t page = page_of(e, lb);
        if (page < 0) continue;
        float w = 0.f;
        for (int r = 0; r < c.bs; ++r) {
          const int64_t j = lb * c.bs + r;
          if (j < low || j >= end) continue;
          w += exp2f(score(page, r) - s_lse);
        }
        if (lane == 0 && w != 0.f) a.mass[row * c.MP + lb] += w;
      }
    }
    __syncthreads();
  }
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
// floats do, -0 as +0, NaN above everything.
__device__ __forceinline__ uint32_t weight_key(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

// One workgroup per sequence.  The number of candidate pages with a smaller
// key, or the same key and a smaller index, is a page's rank; the first ones
// go.  The keys sit in the freed row until the ids replace them.
constexpr int kEvictThreads = 1024;

__device__ __forceinline__ int block_sum(int v, int* red) {
  v = wave_sum_i32(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  int s = 0;
  for (int w = 0; w < kEvictThreads / 64; ++w) s += red[w];
  return s;
}

__global__ __launch_bounds__(kEvictThreads) void paged_evict_kernel(EvictArgs a) {
  const int b = blockIdx.x, tid = threadIdx.x;
  const int64_t base = static_cast<int64_t>(b) * a.MP;
  __shared__ int red[kEvictThreads / 64];
  const int64_t len = a.lens[b];
  const int n = len <= 0 ? 0 : static_cast<int>(min((len + a.bs - 1) / a.bs, static_cast<int64_t>(a.MP)));
  int held = 0, may = 0;
  for (int i = tid; i < n; i += kEvictThreads) {
    const bool here = a.table[base + i] >= 0;
    held += here;
    may += here && i >= a.n_global && i < n - a.window;
  }
  held = block_sum(held, red);
  may = block_sum(may, red);
  const int over = held - max(a.budget[b], 0);
  const int n_drop = min(max(over, 0), may);
  const auto key_of = [&](int i) -> uint64_t {  // above every weight where the page may not go
    if (i < a.n_global || i >= n - a.window || a.table[base + i] < 0) return ~0ull;
    double s = 0.0;
    for (int h = 0; h < a.Hkv; ++h) s += a.mass[(static_cast<int64_t>(b) * a.Hkv + h) * a.MP + i];
    return static_cast<uint64_t>(weight_key(static_cast<float>(s))) << 31 | static_cast<uint32_t>(i);
  };
  // the n_drop-th smallest (key, index), bit by bit: pages at or below it go
  uint64_t cut = 0;
  if (n_drop > 0) {
    for (int bit = 62; bit >= 0; --bit) {
      const uint64_t probe = cut | 1ull << bit;
      int below = 0;
      for (int i = tid; i < n; i += kEvictThreads) below += key_of(i) < probe;
      if (block_sum(below, red) < n_drop) cut = probe;
    }
  }
  // ids in the pages' order
  int done = 0;
  for (int i0 = 0; i0 < a.MP; i0 += kEvictThreads) {
    const int i = i0 + tid;
    const int id = i < a.MP ? a.table[base + i] : -1;
    const bool go = n_drop > 0 && i < n && key_of(i) <= cut;
    const uint64_t ballot = __ballot(go);
    __syncthreads();
    if ((tid & 63) == 0) red[tid >> 6] = __popcll(ballot);
    __syncthreads();
    int at = done + __popcll(ballot & ((1ull << (tid & 63)) - 1));
    int all = 0;
    for (int w = 0; w < kEvictThreads / 64; ++w) {
      if (w < (tid >> 6)) at += red[w];
      all += red[w];
    }
    if (go) a.freed[base + at] = id;
    if (i < a.MP) a.table_out[base + i] = go ? -1 : id;
    done += all;
  }
  for (int i = done + tid; i < a.MP; i += kEvictThreads) a.freed[base + i] = -1;
  if (tid == 0) a.n_freed[b] = done;
}

namespace {
bool aligned16(const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; }

int check_cache(const scope_paged_cache* c, const void* k_pages, const void* v_pages, const char* fn) {
  SCOPE_REQUIRE(c, "%s: null cache", fn);
  SCOPE_REQUIRE(c->D == 64 || c->D == 128 || c->D == 256, "%s: head dim must be 64, 128 or 256, got %d", fn, c->D);
  SCOPE_REQUIRE(c->bs == 16 || c->bs == 32 || c->bs == 64 || c->bs == 128 || c->bs == 256,
                "%s: page size must be 16, 32, 64, 128 or 256, got %d", fn, c->bs);
  SCOPE_REQUIRE(c->type == SCOPE_BF16 || c->type == SCOPE_FP16, "%s: unknown type %d", fn, c->type);
  SCOPE_REQUIRE(c->B >= 1 && c->B <= 65535 && c->Hkv >= 1 && c->Hkv <= 4096 && c->P >= 1,
                "%s: bad sizes B=%d (1 .. 65535), Hkv=%d (1 .. 4096), P=%lld (at least 1)", fn, c->B, c->Hkv, (long long)c->P);
  SCOPE_REQUIRE(c->MP >= 1 && static_cast<int64_t>(c->MP) * c->bs <= INT32_MAX,
                "%s: a table row of %d pages of %d positions (1 .. 2^31 - 1 positions)", fn, c->MP, c->bs);
  const int al = c->fp8 ? 16 : 8;  // elements of 16 bytes
  SCOPE_REQUIRE(k_pages && v_pages, "%s: null pages", fn);
  SCOPE_REQUIRE(c->k_sp % al == 0 && c->k_sh % al == 0 && c->k_sr % al == 0 && c->v_sp % al == 0 && c->v_sh % al == 0 &&
                    c->v_sr % al == 0 && aligned16(k_pages) && aligned16(v_pages),
                "%s: the rows of the pages must be 16-byte aligned", fn);
  return SCOPE_OK;
}
}  // namespace

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
  const AppendArgs a{N, k_sn, k_sh, v_sn, v_sh, k, v, cu, table, lens, k_scale, v_scale, k_pages, v_pages};
  hipLaunchKernelGGL(paged_append_kernel, dim3(ceil_div(N, 4)), dim3(256), 0, as_stream(stream), *c, a);
  return check_launch("paged_append_kernel");
}

int64_t scope_paged_attn_workspace_bytes(const scope_paged_cache* c, int Hq, int maxkv, int with_mass) { return 16; }

int scope_paged_decode_attn(const scope_paged_cache* c, int Hq, int maxkv, float scale, const uint16_t* q, int64_t q_sb,
                            int64_t q_sh, const void* k_pages, const void* v_pages, const float* k_scale,
                            const float* v_scale, const int32_t* table, const int32_t* lens, const int32_t* first,
                            const int32_t* kv_num, const int32_t* kv_idx, float* mass, void* work, uint16_t* out,
                            float* lse, void* stream) {
  const char* fn = "scope_paged_decode_attn";
  if (int rc = check_cache(c, k_pages, v_pages, fn)) return rc;
  SCOPE_REQUIRE(Hq >= 1 && Hq <= 65535 && Hq % c->Hkv == 0, "%s: Hq=%d must be a multiple of Hkv=%d, at most 65535", fn, Hq,
                c->Hkv);
  SCOPE_REQUIRE((kv_num != nullptr) == (kv_idx != nullptr) && (!kv_idx || maxkv >= 1),
                "%s: kv_num and kv_idx come together, with maxkv >= 1 (got %d)", fn, maxkv);
  SCOPE_REQUIRE(q && table && lens && out && lse, "%s: null pointer", fn);
  SCOPE_REQUIRE(aligned16(q) && q_sb % 8 == 0 && q_sh % 8 == 0, "%s: the rows of q must be 16-byte aligned", fn);
  const PagedAttnArgs a{Hq,    maxkv, scale, q_sb,   q_sh,   q,    k_pages, v_pages, k_scale,
                        v_scale, table, lens,  first, kv_num, kv_idx, mass, out,     lse};
  hipLaunchKernelGGL(paged_attn_simple_kernel, dim3(c->B, c->Hkv), dim3(64 * kSimpleWaves), 0, as_stream(stream), *c, a);
  return check_launch("paged_attn_simple_kernel");
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
  hipLaunchKernelGGL(paged_evict_kernel, dim3(B), dim3(kEvictThreads), 0, as_stream(stream), a);
  return check_launch("paged_evict_kernel");
}

}  // extern "C"
