// Attention over the paged 8-bit cache.
#include <cmath>

#include "hb_internal.h"
#include "hb_kv.h"

namespace hb {
namespace {

constexpr uint32_t kThreads = 256;
constexpr float kLog2e = 1.44269504088896340736f;

// A wave a row: its lanes share the columns, keys come one after another.
template <class T, uint32_t D>
__global__ __launch_bounds__(kThreads) void AttnKernel(const AttnArgs a) {
  constexpr uint32_t kCols = D / 64;
  const uint32_t lane = threadIdx.x % 64, group = a.q_heads / a.heads;
  const uint64_t unit =
      (uint64_t)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t qh = (uint32_t)(unit % a.q_heads), head = qh / group;
  const uint64_t rest = unit / a.q_heads;
  const uint32_t i = (uint32_t)(rest % a.max_new);
  const uint64_t b = rest / a.max_new;
  if (b >= a.batch) return;
  const KvSpan span =
      KvRequest(a.cu[b], a.cu[b + 1], a.kv_lens[b], a.prefix ? a.prefix[b] : 0, a.tokens,
                a.max_new, (uint64_t)a.columns * a.groups * 32);
  if (i >= span.rows) return;
  const int32_t pos = span.total - span.count + (int32_t)i;
  const int32_t lead = KvLead(span.prefix, a.sinks, pos, span.total);
  const int64_t lo = a.window > 0 ? (int64_t)pos + 1 - a.window : 0;
  const KvWalk walk = KvRecords(pos, pos, span.total, lead, a.window);
  const T* const q = static_cast<const T*>(a.q) + (uint64_t)(span.first + i) * a.q_token +
                     (uint64_t)qh * a.q_head + lane * kCols;
  float x[kCols], o[kCols], m = -__builtin_inff(), l = 0.f;
  for (uint32_t c = 0; c < kCols; ++c) {
    x[c] = (float)q[c];
    o[c] = 0.f;
  }
  for (uint32_t r = 0; r < walk.count; ++r) {
    const uint32_t index = KvWalkRecord(walk, r);
    uint64_t record;
    if (!KvRecord(a.table + b * a.table_stride, a.columns, index, head, a.pages, a.heads, a.groups,
                  &record))
      continue;
    const uint8_t* const from = a.cache + record * Kv8RecordBytes(D);
    const float ks = __uint_as_float((uint32_t)from[Kv8Scale(D, 0)] << 23);
    const float vs = __uint_as_float((uint32_t)from[Kv8Scale(D, 1)] << 23);
    for (uint32_t t = 0; t < 32; ++t) {
      const int32_t key = (int32_t)(32 * index + t);
      if (key >= span.total || !((key <= pos && key >= lo) || key < lead)) continue;
      float s = 0.f;
      for (uint32_t c = 0; c < kCols; ++c)
        s = fmaf(x[c],
                 __builtin_amdgcn_cvt_f32_fp8((int)from[Kv8KCode(D, t, lane * kCols + c)], 0) * ks,
                 s);
      for (uint32_t d = 1; d < 64; d *= 2) s += __shfl_xor(s, d);
      s *= a.scale;
      if (a.cap > 0.f) s = a.cap * tanhf(s / a.cap);
      s *= kLog2e;
      const float top = fmaxf(m, s);
      const float f = top == m ? 1.f : __builtin_amdgcn_exp2f(m - top);
      const float p = s == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(s - top);
      m = top;
      l = fmaf(l, f, p);
      for (uint32_t c = 0; c < kCols; ++c)
        o[c] = fmaf(o[c], f,
                    p * (__builtin_amdgcn_cvt_f32_fp8((int)from[Kv8VCode(D, t, lane * kCols + c)],
                                                      0) * vs));
    }
  }
  T* const out = static_cast<T*>(a.out) + (uint64_t)(span.first + i) * a.out_token +
                 (uint64_t)qh * a.out_head + lane * kCols;
  for (uint32_t c = 0; c < kCols; ++c) out[c] = (T)(l == 0.f ? 0.f : o[c] / l);
}

template <class T>
hipError_t LaunchType(const AttnArgs& a, uint32_t grid, hipStream_t s) {
  switch (a.dim) {
    case 64: AttnKernel<T, 64><<<grid, kThreads, 0, s>>>(a); break;
    case 128: AttnKernel<T, 128><<<grid, kThreads, 0, s>>>(a); break;
    default: AttnKernel<T, 256><<<grid, kThreads, 0, s>>>(a);
  }
  return hipGetLastError();
}

}  // namespace

AttnWay WayOfAttention8(const AttnArgs&) {
  AttnWay how{};
  how.way = HB_KV_WAY_ROWS;
  how.splits = 1;
  return how;
}

hipError_t LaunchAttention8(const AttnArgs& a, Workspace&, hipStream_t stream) {
  const uint64_t waves = (uint64_t)a.batch * a.max_new * a.q_heads;
  if (waves > 0x7FFFFFFFu) return hipErrorInvalidValue;
  const uint32_t grid = (uint32_t)((waves + kThreads / 64 - 1) / (kThreads / 64));
  switch (a.type) {
    case HB_TYPE_F32: return LaunchType<float>(a, grid, stream);
    case HB_TYPE_BF16: return LaunchType<__bf16>(a, grid, stream);
    default: return LaunchType<_Float16>(a, grid, stream);
  }
}

}  // namespace hb
