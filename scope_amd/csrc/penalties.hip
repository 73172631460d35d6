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
constexpr int kPenThreads = 1024;
constexpr int kPenWords = 8;  // of a thread
constexpr int kPenTile = kPenThreads * kPenWords;
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
// both.  8192 words a workgroup: with fewer, more workgroups read the same
// history, which is what bounds long ones.
template <int TYPE, class Token>
__global__ __launch_bounds__(kPenThreads) void logit_penalties_kernel(scope_penalty_params p, PenaltyArgs a) {
  using Logit = typename std::conditional<TYPE == SCOPE_FP32, uint32_t, uint16_t>::type;
  constexpr int PT = 16 / sizeof(Token), UNR = 4;
  __shared__ __attribute__((aligned(16))) uint32_t count[kPenTile];
  const int tid = threadIdx.x;
  const int64_t b = blockIdx.y, v0 = static_cast<int64_t>(blockIdx.x) * kPenTile;
  const int nv = static_cast<int>(min(static_cast<int64_t>(kPenTile), p.V - v0));
  const int w0 = tid * kPenWords, mine = min(max(nv - w0, 0), kPenWords);  // this thread's words
  const int64_t len = p.lens64 ? static_cast<const int64_t*>(a.lens)[b] : static_cast<const int32_t*>(a.lens)[b];
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
  for (int i = 0; i < kPenWords; i += 4) *reinterpret_cast<uint4*>(&count[i * kPenThreads + 4 * tid]) = make_uint4(0, 0, 0, 0);
  __syncthreads();
  const int64_t end = min(len, p.T), from = a.first ? max(a.first[b], 0) : 0, cut = a.n_prompt ? a.n_prompt[b] : 0;
  const Token* tokens = static_cast<const Token*>(a.tokens) + b * p.tok_sb;
  for (int64_t j0 = from + tid * PT; j0 - tid * PT < end; j0 += static_cast<int64_t>(kPenThreads) * PT * UNR) {
    Packed<Token, PT> t[UNR];
#pragma unroll
    for (int u = 0; u < UNR; ++u) {
      const int64_t j = j0 + static_cast<int64_t>(u) * kPenThreads * PT;
      if (j + PT <= end) {
        t[u] = *reinterpret_cast<const Packed<Token, PT>*>(tokens + j);
      } else {
#pragma unroll
        for (int k = 0; k < PT; ++k) t[u].x[k] = j + k < end ? tokens[j + k] : Token{-1};
      }
    }
#pragma unroll
    for (int u = 0; u < UNR; ++u) {
      const int64_t j = j0 + static_cast<int64_t>(u) * kPenThreads * PT;
#pragma unroll
      for (int k = 0; k < PT; ++k) {
        // (a token outside the vocabulary, and a place past the history, are no words of any tile)
        const uint64_t w = static_cast<uint64_t>(static_cast<int64_t>(t[u].x[k]) - v0);
        if (w >= static_cast<uint64_t>(nv)) continue;
        if (j + k >= cut)
          atomicAdd(&count[w], 1u);
        else
          atomicOr(&count[w], 0x80000000u);
      }
    }
  }
  __syncthreads();
  if (mine == 0) return;
  const float r = a.repetition ? a.repetition[b] : p.repetition, f = a.frequency ? a.frequency[b] : p.frequency;
  const float pr = a.presence ? a.presence[b] : p.presence, te = a.temperature ? a.temperature[b] : p.temperature;
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
  const dim3 grid(ceil_div(p->V, kPenTile), p->B), block(kPenThreads);
  const auto launch = [&](auto type) {
    constexpr int T = decltype(type)::value;
    if (p->tokens64)
      hipLaunchKernelGGL((logit_penalties_kernel<T, int64_t>), grid, block, 0, as_stream(stream), *p, a);
    else
      hipLaunchKernelGGL((logit_penalties_kernel<T, int32_t>), grid, block, 0, as_stream(stream), *p, a);
  };
  if (p->type == SCOPE_FP32)
    launch(std::integral_constant<int, SCOPE_FP32>{});
  else if (p->type == SCOPE_FP16)
    launch(std::integral_constant<int, SCOPE_FP16>{});
  else
    launch(std::integral_constant<int, SCOPE_BF16>{});
  return check_launch("logit_penalties_kernel");
}
