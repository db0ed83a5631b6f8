// K and V rows into the 8-bit paged cache and back out: E4M3 codes with one
// scale for the 32 tokens of a block and a head.
#include <algorithm>

#include "hb_internal.h"
#include "hb_kv.h"

namespace hb {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kThreads = 256;

// 2^(byte - 127) as a float, byte 0 to 246 (0 stands beside zeros only).
__device__ __forceinline__ float ScaleOf(uint32_t byte) { return __uint_as_float(byte << 23); }
// 2^(127 - byte), byte 10 to 246.
__device__ __forceinline__ float Unscale(uint32_t byte) { return __uint_as_float((254 - byte) << 23); }

__device__ __forceinline__ uint32_t WaveMax(uint32_t x) {
#pragma unroll
  for (uint32_t d = 1; d < 64; d *= 2) x = max(x, (uint32_t)__shfl_xor((int)x, (int)d));
  return x;
}

// The code of x times a power of two, nearest even; past 448 that.
__device__ __forceinline__ uint8_t Code(float x) {
  x = __builtin_amdgcn_fmed3f(x, -448.f, 448.f);
  return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(x, x, 0, false);
}
__device__ __forceinline__ float Value(uint8_t code, float scale) {
  return __builtin_amdgcn_cvt_f32_fp8((int)code, 0) * scale;
}

// A wave takes a run of rows (of neighbouring slots within a block) and a
// head: the runs' first rows find them, waves of other rows end at once.
template <class T, uint32_t dim>
__global__ __launch_bounds__(kThreads) void AppendKernel(const KvRowsArgs g) {
  constexpr uint32_t kCols = dim / 64;
  const uint32_t lane = threadIdx.x % 64;
  const uint64_t wave =
      (uint64_t)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t head = (uint32_t)(wave % g.heads);
  const uint64_t row = wave / g.heads;
  if (row >= g.tokens) return;
  // slots of the row before, its own and 62 after it, a lane each
  int32_t slot = -1;
  if (row + lane >= 1 && row + lane - 1 < g.tokens) slot = g.slots[row + lane - 1];
  const int32_t mine = __builtin_amdgcn_readlane(slot, 1);
  uint64_t record;
  uint32_t t0;
  if (!KvSlot(mine, g.pages, g.heads, g.groups, &record, &t0)) return;
  if (t0 > 0 && __builtin_amdgcn_readlane(slot, 0) == mine - 1) return;  // within a run
  const bool follows = lane >= 1 && (int64_t)slot == (int64_t)mine + lane - 1 && t0 + lane <= 32;
  const uint32_t count =
      (uint32_t)__builtin_ctzll(~(__builtin_amdgcn_ballot_w64(follows) >> 1));
  uint8_t* const to =
      g.cache + (record + (uint64_t)head * g.groups) * Kv8RecordBytes(dim);
  const uint32_t col0 = lane * kCols;
  const T* const k = static_cast<const T*>(g.k) + row * g.k_token + head * g.k_head + col0;
  const T* const v = static_cast<const T*>(g.v) + row * g.v_token + head * g.v_head + col0;
  uint32_t bad = 0, k_top = 0, v_top = 0;
  for (uint32_t t = 0; t < count; ++t) {
    uint32_t kt = 0, vt = 0;
    for (uint32_t c = 0; c < kCols; ++c) {
      kt = max(kt, __float_as_uint((float)k[t * g.k_token + c]) & 0x7FFFFFFFu);
      vt = max(vt, __float_as_uint((float)v[t * g.v_token + c]) & 0x7FFFFFFFu);
    }
    if (__builtin_amdgcn_ballot_w64(max(kt, vt) >= 0x7F800000u) != 0) {
      bad |= 1u << t;
      continue;
    }
    k_top = max(k_top, kt);
    v_top = max(v_top, vt);
  }
  const uint32_t had_k = t0 > 0 ? to[Kv8Scale(dim, 0)] : 0, had_v = t0 > 0 ? to[Kv8Scale(dim, 1)] : 0;
  const uint32_t ks = max(had_k, Kv8ScaleOf(WaveMax(k_top)));
  const uint32_t vs = max(had_v, Kv8ScaleOf(WaveMax(v_top)));
  if (ks > had_k && had_k > 0) {
    const float f = ScaleOf(had_k) * Unscale(ks);
    for (uint32_t t = 0; t < t0; ++t)
      for (uint32_t c = 0; c < kCols; ++c) {
        uint8_t* const at = to + Kv8KCode(dim, t, col0 + c);
        if ((*at & 0x7F) != 0x7F) *at = Code(Value(*at, f));
      }
  }
  if (vs > had_v && had_v > 0) {
    const float f = ScaleOf(had_v) * Unscale(vs);
    for (uint32_t t = 0; t < t0; ++t)
      for (uint32_t c = 0; c < kCols; ++c) {
        uint8_t* const at = to + Kv8VCode(dim, t, col0 + c);
        *at = Code(Value(*at, f));
      }
  }
  const float ku = ks > 0 ? Unscale(ks) : 0.f, vu = vs > 0 ? Unscale(vs) : 0.f;
  for (uint32_t t = 0; t < count; ++t) {
    const bool b = bad >> t & 1;
    for (uint32_t c = 0; c < kCols; ++c) {
      to[Kv8KCode(dim, t0 + t, col0 + c)] = b ? 0x7F : Code((float)k[t * g.k_token + c] * ku);
      to[Kv8VCode(dim, t0 + t, col0 + c)] = b ? 0 : Code((float)v[t * g.v_token + c] * vu);
    }
  }
  if (lane == 0) {
    to[Kv8Scale(dim, 0)] = (uint8_t)ks;
    to[Kv8Scale(dim, 1)] = (uint8_t)vs;
  }
}

// The stored values of slots: a wave a token and head.
template <class T, uint32_t dim>
__global__ __launch_bounds__(kThreads) void ReadKernel(const KvRowsArgs g) {
  constexpr uint32_t kCols = dim / 64;
  const uint32_t lane = threadIdx.x % 64;
  const uint64_t wave =
      (uint64_t)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t head = (uint32_t)(wave % g.heads);
  const uint64_t row = wave / g.heads;
  if (row >= g.tokens) return;
  T* const k = static_cast<T*>(g.k_out) + row * g.k_token + head * g.k_head + lane * kCols;
  T* const v = static_cast<T*>(g.v_out) + row * g.v_token + head * g.v_head + lane * kCols;
  uint64_t record;
  uint32_t t;
  const bool there = KvSlot(g.slots[row], g.pages, g.heads, g.groups, &record, &t);
  const uint8_t* const from =
      g.cache + (there ? record + (uint64_t)head * g.groups : 0) * Kv8RecordBytes(dim);
  const float ks = ScaleOf(from[Kv8Scale(dim, 0)]), vs = ScaleOf(from[Kv8Scale(dim, 1)]);
  for (uint32_t c = 0; c < kCols; ++c) {
    k[c] = (T)(there ? Value(from[Kv8KCode(dim, t, lane * kCols + c)], ks) : 0.f);
    v[c] = (T)(there ? Value(from[Kv8VCode(dim, t, lane * kCols + c)], vs) : 0.f);
  }
}

template <class T, uint32_t dim>
hipError_t LaunchOf(const KvRowsArgs& a, bool read, hipStream_t s) {
  const uint64_t waves = (uint64_t)a.tokens * a.heads;
  const uint32_t grid = (uint32_t)((waves + kThreads / 64 - 1) / (kThreads / 64));
  if (read) ReadKernel<T, dim><<<grid, kThreads, 0, s>>>(a);
  else AppendKernel<T, dim><<<grid, kThreads, 0, s>>>(a);
  return hipGetLastError();
}

template <class T>
hipError_t LaunchType(const KvRowsArgs& a, bool read, hipStream_t s) {
  switch (a.dim) {
    case 64: return LaunchOf<T, 64>(a, read, s);
    case 128: return LaunchOf<T, 128>(a, read, s);
    case 256: return LaunchOf<T, 256>(a, read, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t LaunchKv8Rows(const KvRowsArgs& a, bool read, hipStream_t stream) {
  switch (a.type) {
    case HB_TYPE_F32: return LaunchType<float>(a, read, stream);
    case HB_TYPE_BF16: return LaunchType<__bf16>(a, read, stream);
    default: return LaunchType<_Float16>(a, read, stream);
  }
}

}  // namespace hb
