// Penalties, biases and grammar bits on the logits of a step of the token loop.
//
// For sequence b with history tokens[b][first .. len): seen(v) says whether v
// occurs in it, c(v) how often at positions from n_prompt on.  In this order,
// every step in fp32 (no contraction: each is a tensor operation's rounding):
//   z := seen ? (z > 0 ? z / r : z · r) : z
//   z := z - frequency · c;   z := z - presence · [c > 0]
//   z := z + bias;  z := z / temperature;  z := -inf where the word's bit is 0
#include <math.h>

#include "common.h"

namespace scope {

namespace {
constexpr int kPenTile = 4096;  // words of a workgroup
constexpr int kPenThreads = 1024;
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

__device__ __forceinline__ float logit_in(const void* p, int64_t i, int type) {
  if (type == SCOPE_FP32) return static_cast<const float*>(p)[i];
  const uint16_t x = static_cast<const uint16_t*>(p)[i];
  return type == SCOPE_FP16 ? static_cast<float>(__builtin_bit_cast(_Float16, x)) : bf16_to_f32(x);
}
__device__ __forceinline__ void logit_out(void* p, int64_t i, int type, float f) {
  if (type == SCOPE_FP32)
    static_cast<float*>(p)[i] = f;
  else
    static_cast<uint16_t*>(p)[i] = type == SCOPE_FP16 ? __builtin_bit_cast(uint16_t, static_cast<_Float16>(f)) : f32_to_bf16(f);
}

// A workgroup holds the counts of its words in LDS and reads the whole history.
// Bit 31 of a word's counter: seen; the rest: c.
__global__ __launch_bounds__(kPenThreads) void logit_penalties_kernel(scope_penalty_params p, PenaltyArgs a) {
  __shared__ uint32_t count[kPenTile];
  const int64_t b = blockIdx.y, v0 = static_cast<int64_t>(blockIdx.x) * kPenTile;
  const int64_t nv = min(static_cast<int64_t>(kPenTile), p.V - v0);
  for (int i = threadIdx.x; i < kPenTile; i += kPenThreads) count[i] = 0;
  __syncthreads();
  const int64_t len = p.lens64 ? static_cast<const int64_t*>(a.lens)[b] : static_cast<const int32_t*>(a.lens)[b];
  const int64_t end = min(len, p.T), from = a.first ? max(a.first[b], 0) : 0, cut = a.n_prompt ? a.n_prompt[b] : 0;
  for (int64_t j = from + threadIdx.x; j < end; j += kPenThreads) {
    const int64_t t = p.tokens64 ? static_cast<const int64_t*>(a.tokens)[b * p.tok_sb + j]
                                 : static_cast<const int32_t*>(a.tokens)[b * p.tok_sb + j];
    if (t < v0 || t - v0 >= nv) continue;
    atomicOr(&count[t - v0], 0x80000000u);
    if (j >= cut) atomicAdd(&count[t - v0], 1u);
  }
  __syncthreads();
  const float r = a.repetition ? a.repetition[b] : p.repetition, f = a.frequency ? a.frequency[b] : p.frequency;
  const float pr = a.presence ? a.presence[b] : p.presence, te = a.temperature ? a.temperature[b] : p.temperature;
  for (int i = threadIdx.x; i < nv; i += kPenThreads) {
    const int64_t v = v0 + i;
    const uint32_t n = count[i];
    float z = logit_in(a.logits, b * p.z_sb + v, p.type);
    if (n) {
      const float c = static_cast<float>(n & 0x7fffffffu);
      z = z > 0.f ? z / r : z * r;
      if (c > 0.f) {
        z = z - f * c;
        z = z - pr;
      }
    }
    if (a.bias) z = z + a.bias[b * p.bias_sb + v];
    z = z / te;
    if (a.mask && !((a.mask[b * p.mask_sb + v / 32] >> (v % 32)) & 1)) z = -INFINITY;
    logit_out(a.out, b * p.o_sb + v, p.type, z);
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
  hipLaunchKernelGGL(logit_penalties_kernel, dim3(ceil_div(p->V, kPenTile), p->B), dim3(kPenThreads), 0, as_stream(stream), *p,
                     a);
  return check_launch("logit_penalties_kernel");
}
