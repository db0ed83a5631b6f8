// Log probabilities of given tokens, the entropy and the most likely tokens of
// rows of logits.
//
// With m = max x and s = sum e^(x - m) a token's log probability is
// x - m - ln s and the entropy ln s - sum (x - m) e^(x - m) / s.
#include "hb_internal.h"

namespace hb {
namespace {

constexpr uint32_t kThreads = 256;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// Larger logits, and of equal ones lower columns, have larger keys; a NaN the
// least.
__device__ __forceinline__ uint64_t KeyOf(float x, uint32_t column) {
  const uint32_t bits = __float_as_uint(x + 0.f);  // -0 as 0
  const uint32_t order = x != x ? 0u : bits & 0x80000000u ? ~bits : bits | 0x80000000u;
  return (uint64_t)order << 32 | (uint32_t)~column;
}

template <class T>
__global__ __launch_bounds__(kThreads) void LogprobsKernel(const LogprobsArgs a) {
  __shared__ float f[kThreads / 64];
  __shared__ uint64_t keys[kThreads / 64];
  const uint32_t row = blockIdx.x, tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  const T* const x = static_cast<const T*>(a.logits) + row * a.stride;
  const float c = a.scale * kLog2e;  // in powers of two from here on
  auto sum = [&](float v) {
    for (uint32_t d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    __syncthreads();
    if (lane == 0) f[wave] = v;
    __syncthreads();
    return f[0] + f[1] + f[2] + f[3];
  };
  float m = -__builtin_inff();
  for (uint32_t i = tid; i < a.vocab; i += kThreads) m = fmaxf(m, (float)x[i]);
  for (uint32_t d = 1; d < 64; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
  if (lane == 0) f[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3]));
  const float ref = m == -__builtin_inff() ? 0.f : m;
  float l = 0.f, w = 0.f;
  for (uint32_t i = tid; i < a.vocab; i += kThreads) {
    const float d = ((float)x[i] - ref) * c, p = __builtin_amdgcn_exp2f(d);
    l += p;
    w += p * fmaxf(d, -1e4f);
  }
  l = sum(l);
  w = sum(w);
  const float log = l == 0.f ? 0.f : __builtin_amdgcn_logf(l);
  auto logprob = [&](float logit) {
    return l == 0.f ? -__builtin_inff() : ((logit - ref) * c - log) * kLn2;
  };
  if (tid == 0) {
    if (a.tokens != nullptr) {
      const int32_t t = a.tokens[row];
      a.logprobs[row] = t < 0 ? 0.f
                        : (uint32_t)t >= a.vocab ? __builtin_nanf("")
                                                 : logprob((float)x[t]);
    }
    if (a.entropy != nullptr) a.entropy[row] = l == 0.f ? 0.f : (log - w / l) * kLn2;
  }
  uint64_t below = ~0ull;
  for (uint32_t k = 0; k < a.top; ++k) {
    uint64_t best = 0;
    for (uint32_t i = tid; i < a.vocab; i += kThreads) {
      const uint64_t key = KeyOf((float)x[i], i);
      if (key < below) best = max(best, key);
    }
    for (uint32_t d = 1; d < 64; d *= 2) best = max(best, (uint64_t)__shfl_xor((unsigned long long)best, d));
    __syncthreads();
    if (lane == 0) keys[wave] = best;
    __syncthreads();
    best = max(max(keys[0], keys[1]), max(keys[2], keys[3]));
    below = best;
    if (tid == 0) {
      const uint32_t column = ~(uint32_t)best;
      a.top_ids[(uint64_t)row * a.top + k] = (int32_t)column;
      a.top_logprobs[(uint64_t)row * a.top + k] = logprob((float)x[column]);
    }
  }
}

}  // namespace

hipError_t LaunchLogprobs(const LogprobsArgs& a, Workspace&, hipStream_t stream) {
  switch (a.type) {
    case HB_TYPE_F32: LogprobsKernel<float><<<a.rows, kThreads, 0, stream>>>(a); break;
    case HB_TYPE_BF16: LogprobsKernel<__bf16><<<a.rows, kThreads, 0, stream>>>(a); break;
    default: LogprobsKernel<_Float16><<<a.rows, kThreads, 0, stream>>>(a);
  }
  return hipGetLastError();
}

}  // namespace hb
