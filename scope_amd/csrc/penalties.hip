// Penalties, biases and grammar bits on the logits of a step of the token loop.
//
// For sequence b with history tokens[b][first .. len): seen(v) says whether v
// occurs in it, c(v) how often at positions from n_prompt on.  In this order,
// every step in fp32 (no contraction: each is a tensor operation's rounding):
//   z := seen ? (z > 0 ? z / r : z · r) : z
//   z := z - frequency · c;   z := z - presence · [c > 0]
//   z := z + bias;  z := z / temperature;  z := -inf where the word's bit is 0
#include <math.h>

#include <type_traits>

#include "common.h"

namespace scope {

namespace {
constexpr int kPenWords = 8;  // of a thread
constexpr int kXcds = 8;
// Room for up to this many tokens, or one row, takes 512 threads (4096 words) a
// workgroup, whose waits are shorter (128 rows of 50304 words, histories to 8192,
// everything on: 16.7 us, with 1024 threads 18.3; one row of 50257 words with room
// for 131k and 1152 of them held 4.35 against 5.25, all of them held 16.1 against
// 17.2).  Longer histories of several rows are read by fewer workgroups with 1024,
// and those of a row follow each other on one XCD, so that its history comes into
// one L2 (16 rows of 100003 words, histories of 60k to 131k: 19.0 us; on all XCDs
// 22.1, with 512 threads 26.3).  The host does not know the lengths: two to 32 rows
// with such room take up to 1 us longer than with 512 threads while they hold little
// of it (8 rows of 1152 5.4 against 4.6, 2 rows of 20000 7.3 against 6.4) and 5 to 6
// less where it is full (8 rows of 131k 17.6 against 23.6).
constexpr int64_t kLongHistory = 16384;
}  // namespace

struct PenaltyArgs {
  const void* logits;
  const void* tokens;
  const void* lens;
  const int32_t* first;
  const int32_t* n_prompt;
  const float* repetition;
  const float* presence;
  const float* frequency;
  const float* temperature;
  const float* bias;
  const int32_t* mask;
  void* out;
};

// N values at any address their type allows (16 bytes a load)
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Packed {
  T x[N];
};

template <int TYPE>
__device__ __forceinline__ float logit_in(uint32_t raw) {
  if constexpr (TYPE == SCOPE_FP32) return __uint_as_float(raw);
  if constexpr (TYPE == SCOPE_FP16) return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(raw)));
  return bf16_to_f32(static_cast<uint16_t>(raw));
}
template <int TYPE>
__device__ __forceinline__ auto logit_out(float f) {
  if constexpr (TYPE == SCOPE_FP32)
    return __float_as_uint(f);
  else if constexpr (TYPE == SCOPE_FP16)
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f));
  else
    return f32_to_bf16(f);
}

// A workgroup holds the counters of its words in LDS (bit 31: seen, the rest: c)
// and reads the whole history, its tokens 16 bytes a load and four loads under
// way; its logits, bias and bits are loaded before that, so one latency covers
// both.
template <int TYPE, class Token, int THREADS>
__global__ __launch_bounds__(THREADS, 2048 / THREADS) void logit_penalties_kernel(scope_penalty_params p, PenaltyArgs a) {
  using Logit = typename std::conditional<TYPE == SCOPE_FP32, uint32_t, uint16_t>::type;
  constexpr int PT = 16 / sizeof(Token), UNR = 4, TILE = THREADS * kPenWords, XCDS = THREADS == 1024 ? kXcds : 1;
  __shared__ __attribute__((aligned(16))) uint32_t count[TILE + kWave];  // (and a place a lane for words of other tiles)
  const int tid = threadIdx.x;
  // (workgroups go round the XCDs)
  const int tiles = static_cast<int>((p.V + TILE - 1) / TILE), slot = blockIdx.x / XCDS;
  const int64_t b = static_cast<int64_t>(slot / tiles) * XCDS + blockIdx.x % XCDS;
  const int64_t v0 = static_cast<int64_t>(slot % tiles) * TILE;
  if (b >= p.B) return;
  const int nv = static_cast<int>(min(static_cast<int64_t>(TILE), p.V - v0));
  const int w0 = tid * kPenWords, mine = min(max(nv - w0, 0), kPenWords);  // this thread's words
  const int64_t len = p.lens64 ? static_cast<const int64_t*>(a.lens)[b] : static_cast<const int32_t*>(a.lens)[b];
  const int64_t end = min(len, p.T), from = a.first ? max(a.first[b], 0) : 0, cut = a.n_prompt ? a.n_prompt[b] : 0;
  const float r = a.repetition ? a.repetition[b] : p.repetition, f = a.frequency ? a.frequency[b] : p.frequency;
  const float pr = a.presence ? a.presence[b] : p.presence, te = a.temperature ? a.temperature[b] : p.temperature;
  const Logit* zin = static_cast<const Logit*>(a.logits) + b * p.z_sb + v0 + w0;
  const float* bin = a.bias ? a.bias + b * p.bias_sb + v0 + w0 : nullptr;
  Packed<Logit, kPenWords> z;
  Packed<float, kPenWords> bias;
  uint32_t bits = ~0u;
  if (mine == kPenWords) {
    z = *reinterpret_cast<const Packed<Logit, kPenWords>*>(zin);
    if (bin) bias = *reinterpret_cast<const Packed<float, kPenWords>*>(bin);
  } else {
#pragma unroll
    for (int i = 0; i < kPenWords; ++i) {
      z.x[i] = i < mine ? zin[i] : Logit{0};
      bias.x[i] = bin && i < mine ? bin[i] : 0.f;
    }
  }
  if (a.mask && mine > 0) bits = static_cast<uint32_t>(a.mask[b * p.mask_sb + (v0 + w0) / 32]) >> (w0 % 32);
#pragma unroll
  for (int i = 0; i < kPenWords; i += 4) *reinterpret_cast<uint4*>(&count[i * THREADS + 4 * tid]) = make_uint4(0, 0, 0, 0);
  __syncthreads();
  const Token* tokens = static_cast<const Token*>(a.tokens) + b * p.tok_sb;
  // A token's counter, or the lane's own place past them: a token of another tile
  // or outside the vocabulary costs no branch.  (Words past V in the last tile
  // have counters that nothing reads.)
  const auto counter = [&](Token token) {
    const uint32_t w = static_cast<uint32_t>(token) - static_cast<uint32_t>(v0);
    return min(sizeof(Token) == 8 && static_cast<uint64_t>(token) >> 32 ? ~0u : w, static_cast<uint32_t>(TILE + tid % kWave));
  };
  const auto add = [&](Token token, bool counts) {
    if (counts)
      atomicAdd(&count[counter(token)], 1u);
    else
      atomicOr(&count[counter(token)], 0x80000000u);
  };
  constexpr int STEP = THREADS * PT;
  const auto within = [](int64_t x) { return static_cast<int>(max(min(x, static_cast<int64_t>(1) << 30), -(static_cast<int64_t>(1) << 30))); };
  if (end - from >= PT) {
    for (int64_t base = from; base < end; base += UNR * STEP) {
      // places relative to base: the history's last load, and the first token that counts
      const int last = within(end - base) - PT, first_new = within(cut - base);
      Packed<Token, PT> t[UNR];
      // (loads past the history's last are moved back to it, and only their new
      // tokens count; no load under a branch, which would wait for those before it)
#pragma unroll
      for (int u = 0; u < UNR; ++u) t[u] = *reinterpret_cast<const Packed<Token, PT>*>(tokens + base + min(u * STEP + tid * PT, last));
      if (last + PT >= UNR * STEP && (first_new <= 0 || first_new >= UNR * STEP)) {
        // within the history, and on one side of n_prompt
        if (first_new <= 0) {
#pragma unroll
          for (int u = 0; u < UNR; ++u)
#pragma unroll
            for (int k = 0; k < PT; ++k) atomicAdd(&count[counter(t[u].x[k])], 1u);
        } else {
#pragma unroll
          for (int u = 0; u < UNR; ++u)
#pragma unroll
            for (int k = 0; k < PT; ++k) atomicOr(&count[counter(t[u].x[k])], 0x80000000u);
        }
        continue;
      }
#pragma unroll
      for (int u = 0; u < UNR; ++u)
        if (u * STEP < last + PT) {
          const int j = u * STEP + tid * PT, at = min(j, last);
#pragma unroll
          for (int k = 0; k < PT; ++k)
            if (at + k >= j) add(t[u].x[k], at + k >= first_new);
        }
    }
  } else if (from + tid < end) {
    add(tokens[from + tid], from + tid >= cut);
  }
  __syncthreads();
  if (mine == 0) return;
  uint32_t n[kPenWords];
#pragma unroll
  for (int i = 0; i < kPenWords; i += 4) {
    const uint4 q = *reinterpret_cast<const uint4*>(&count[w0 + i]);
    n[i] = q.x;
    n[i + 1] = q.y;
    n[i + 2] = q.z;
    n[i + 3] = q.w;
  }
  Packed<Logit, kPenWords> o;
#pragma unroll
  for (int i = 0; i < kPenWords; ++i) {
    float y = logit_in<TYPE>(z.x[i]);
    if (n[i]) {
      const float c = static_cast<float>(n[i] & 0x7fffffffu);
      y = y > 0.f ? y / r : y * r;
      if (c > 0.f) {
        y = y - f * c;
        y = y - pr;
      }
    }
    if (bin) y = y + bias.x[i];
    if (te != 1.f) y = y / te;  // (a quotient by 1 is the number itself)
    o.x[i] = logit_out<TYPE>(bits >> i & 1 ? y : -INFINITY);
  }
  Logit* zout = static_cast<Logit*>(a.out) + b * p.o_sb + v0 + w0;
  if (mine == kPenWords) {
    *reinterpret_cast<Packed<Logit, kPenWords>*>(zout) = o;
  } else {
#pragma unroll
    for (int i = 0; i < kPenWords; ++i)
      if (i < mine) zout[i] = o.x[i];
  }
}

}  // namespace scope

using namespace scope;

extern "C" int scope_logit_penalties(const scope_penalty_params* p, const void* logits, const void* tokens, const void* lens,
                                     const int32_t* first, const int32_t* n_prompt, const float* repetition,
                                     const float* presence, const float* frequency, const float* temperature,
                                     const float* bias, const int32_t* mask, void* out, void* stream) {
  const char* fn = "scope_logit_penalties";
  SCOPE_REQUIRE(p && p->B >= 1 && p->B <= 65535 && p->V >= 1 && p->V <= INT32_MAX && p->T >= 0 && p->T <= INT32_MAX,
                "%s: sizes B (1 .. 65535), V (1 .. 2^31 - 1) and T (0 .. 2^31 - 1) out of range", fn);
  SCOPE_REQUIRE(p->type == SCOPE_BF16 || p->type == SCOPE_FP16 || p->type == SCOPE_FP32, "%s: unknown type %d", fn, p->type);
  SCOPE_REQUIRE(logits && out && lens && (tokens || p->T == 0), "%s: null pointer", fn);
  const PenaltyArgs a{logits, tokens, lens, first, n_prompt, repetition, presence, frequency, temperature, bias, mask, out};
  const bool lng = p->T > kLongHistory && p->B > 1;
  const int threads = lng ? 1024 : 512, rows = lng ? ceil_div(p->B, kXcds) * kXcds : p->B;
  const int64_t groups = static_cast<int64_t>(rows) * ceil_div(p->V, threads * kPenWords);
  // (a grid holds less than 2^32 work-items)
  SCOPE_REQUIRE(groups * threads <= UINT32_MAX, "%s: %d rows of %lld words are more than one launch holds (about 2^35 in all)", fn,
                p->B, (long long)p->V);
  const dim3 grid(static_cast<uint32_t>(groups)), block(threads);
  hipStream_t st = as_stream(stream);
  const auto launch = [&](auto type) {
    constexpr int T = decltype(type)::value;
    if (p->tokens64 && lng)
      hipLaunchKernelGGL((logit_penalties_kernel<T, int64_t, 1024>), grid, block, 0, st, *p, a);
    else if (p->tokens64)
      hipLaunchKernelGGL((logit_penalties_kernel<T, int64_t, 512>), grid, block, 0, st, *p, a);
    else if (lng)
      hipLaunchKernelGGL((logit_penalties_kernel<T, int32_t, 1024>), grid, block, 0, st, *p, a);
    else
      hipLaunchKernelGGL((logit_penalties_kernel<T, int32_t, 512>), grid, block, 0, st, *p, a);
  };
  if (p->type == SCOPE_FP32)
    launch(std::integral_constant<int, SCOPE_FP32>{});
  else if (p->type == SCOPE_FP16)
    launch(std::integral_constant<int, SCOPE_FP16>{});
  else
    launch(std::integral_constant<int, SCOPE_BF16>{});
  return check_launch("logit_penalties_kernel");
}
