// K and V rows into the 8-bit paged cache and back out: E4M3 codes with one
// scale for the 32 tokens of a block and a head.
#include <algorithm>

#include "hb_internal.h"
#include "hb_kv.h"
#include "hb_lanes.h"

namespace hb {
namespace {

constexpr uint32_t kThreads = 256, kWaves = kThreads / 64;

// 2^(byte - 127), byte 0 to 246 (0 stands beside zeros only).
__device__ __forceinline__ float ScaleOf(uint32_t byte) { return __uint_as_float(byte << 23); }
// 2^(127 - byte), byte 10 to 246.
__device__ __forceinline__ float Unscale(uint32_t byte) { return __uint_as_float((254 - byte) << 23); }

__device__ __forceinline__ uint32_t WaveMax(uint32_t x) {
#pragma unroll
  for (uint32_t d = 1; d < 64; d *= 2) x = max(x, (uint32_t)__shfl_xor((int)x, (int)d));
  return x;
}

// Four values as codes, the first in the lowest byte: nearest even, past 448
// that.
__device__ __forceinline__ uint32_t Codes(float a, float b, float c, float d) {
  a = __builtin_amdgcn_fmed3f(a, -448.f, 448.f);
  b = __builtin_amdgcn_fmed3f(b, -448.f, 448.f);
  c = __builtin_amdgcn_fmed3f(c, -448.f, 448.f);
  d = __builtin_amdgcn_fmed3f(d, -448.f, 448.f);
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}
// Four codes times f <= 1, which nothing passes 448 by and NaN stays in.
__device__ __forceinline__ uint32_t Again(uint32_t codes, float f) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false);
  const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a[0] * f, a[1] * f, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(b[0] * f, b[1] * f, lo, true);
}

template <class T>
__device__ __forceinline__ void Load4(const T* x, bool vec, float* y) {
  typedef typename Four<T>::type V;
  if (vec) {
    const V v = *reinterpret_cast<const V*>(x);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = (float)v[j];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = (float)x[j];
  }
}

// A workgroup takes the runs that begin in `window` neighbouring rows, of one
// head, one after another (a run: rows whose slots are neighbours within a
// block): 4 columns of 2, 4 or 8 tokens a thread, all of a run in registers
// between its maximum and its codes.  A run that is a whole block leaves through
// LDS in the record's order, 16 bytes a store; of others a token's own bytes,
// which lie all over the record.  Memory bounds it: 16,001 tokens of 5 heads of 64
// in fp32, 41 MB read and 10 written, 12.3 us = 4.2 TB/s (95 with a wave a run and
// a byte a store); 64 single tokens of 8 heads of 128, bf16, 4.8 us, the chain from
// their slots over rows and scales to the stores.
template <class T, uint32_t dim>
__global__ __launch_bounds__(kThreads) void AppendKernel(const KvRowsArgs g) {
  constexpr uint32_t kRow = dim / 4, kGroups = kThreads / kRow, kRows = 32 / kGroups;
  __shared__ __align__(16) uint8_t image[64 * dim];
  __shared__ uint32_t tops[kWaves][2], scales;
  const uint32_t tid = threadIdx.x, lane = tid % 64;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const uint32_t head = blockIdx.x % g.heads;
  const uint32_t row0 = (blockIdx.x / g.heads + g.first) * g.window;
  const uint32_t group = tid / kRow, col = tid % kRow * 4;
  // slots of the row before the window's and of 63 rows from there, a lane each
  const uint64_t at = (uint64_t)row0 + lane;
  const int32_t slot = at >= 1 && at - 1 < g.tokens ? g.slots[at - 1] : -1;
  const int32_t before = __shfl_up(slot, 1);
  const bool goes_on = lane > 0 && slot % 32 != 0 && slot > 0 && before == slot - 1;
  uint64_t record;
  uint32_t t0;
  const bool there = KvSlot(slot, g.pages, g.heads, g.groups, &record, &t0);
  const uint64_t on = __builtin_amdgcn_ballot_w64(goes_on);
  uint64_t starts = __builtin_amdgcn_ballot_w64(there && !goes_on && lane > 0 && lane <= g.window);
  for (; starts != 0; starts &= starts - 1) {
    const uint32_t l = (uint32_t)__builtin_ctzll(starts);
    const uint32_t row = row0 + l - 1;
    const uint32_t count = 1 + (uint32_t)__builtin_ctzll(~(on >> (l + 1)));
    (void)KvSlot(__builtin_amdgcn_readlane(slot, (int)l), g.pages, g.heads, g.groups, &record, &t0);
    uint8_t* const to = g.cache + (record + (uint64_t)head * g.groups) * Kv8RecordBytes(dim);
    uint32_t had = 0;  // one thread's, so that all see the same whatever others write
    if (tid == 0 && t0 > 0) had = *reinterpret_cast<const uint16_t*>(to + Kv8Scale(dim, 0));
    float k[kRows][4], v[kRows][4];
    // a whole block's thread has tokens that are neighbours, whose V codes are
    // too; of a few tokens every group of threads has some
    const auto token = [&](uint32_t i) {
      return count == 32 ? group * kRows + i : i * kGroups + group;
    };
#pragma unroll
    for (uint32_t i = 0; i < kRows; ++i) {
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) k[i][j] = v[i][j] = 0.f;
      const uint32_t t = token(i);
      if (t >= count) continue;
      const uint64_t r = row + t;
      Load4(static_cast<const T*>(g.k) + r * g.k_token + head * g.k_head + col, g.vec, k[i]);
      Load4(static_cast<const T*>(g.v) + r * g.v_token + head * g.v_head + col, g.vec, v[i]);
    }
    uint32_t bad = 0, k_top = 0, v_top = 0;
#pragma unroll
    for (uint32_t i = 0; i < kRows; ++i) {
      uint32_t kt = 0, vt = 0;
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        kt = max(kt, __float_as_uint(k[i][j]) & 0x7FFFFFFFu);
        vt = max(vt, __float_as_uint(v[i][j]) & 0x7FFFFFFFu);
      }
      // a row's threads are lanes of one wave
      const uint64_t odd = __builtin_amdgcn_ballot_w64(max(kt, vt) >= 0x7F800000u);
      const uint64_t mine = (~0ull >> (64 - kRow)) << (lane / kRow * kRow);
      if ((odd & mine) != 0) {
        bad |= 1u << i;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) k[i][j] = v[i][j] = 0.f;
      } else {
        k_top = max(k_top, kt);
        v_top = max(v_top, vt);
      }
    }
    k_top = WaveMax(k_top);
    v_top = WaveMax(v_top);
    if (lane == 0) {
      tops[wave][0] = k_top;
      tops[wave][1] = v_top;
    }
    if (tid == 0) scales = had;
    __syncthreads();
    had = scales;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) {
      k_top = max(k_top, tops[w][0]);
      v_top = max(v_top, tops[w][1]);
    }
    const uint32_t had_k = had & 255u, had_v = had >> 8;
    const uint32_t ks = max(had_k, Kv8ScaleOf(k_top)), vs = max(had_v, Kv8ScaleOf(v_top));
    const float ku = ks > 0 ? Unscale(ks) : 0.f, vu = vs > 0 ? Unscale(vs) : 0.f;
    if (count == 32) {
#pragma unroll
      for (uint32_t i = 0; i < kRows; ++i) {
        const uint32_t codes = Codes(k[i][0] * ku, k[i][1] * ku, k[i][2] * ku, k[i][3] * ku);
        *reinterpret_cast<uint32_t*>(image + Kv8KCode(dim, group * kRows + i, col)) =
            bad >> i & 1 ? 0x7F7F7F7Fu : codes;
      }
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        uint8_t* const y = image + Kv8VCode(dim, group * kRows, col + j);
        if constexpr (kRows == 2) {
          *reinterpret_cast<uint16_t*>(y) =
              (uint16_t)Codes(v[0][j] * vu, v[1][j] * vu, 0.f, 0.f);
        } else {
#pragma unroll
          for (uint32_t i = 0; i < kRows; i += 4)  // 4 tokens on: the next lanes' piece
            *reinterpret_cast<uint32_t*>(image + Kv8VCode(dim, group * kRows + i, col + j)) =
                Codes(v[i][j] * vu, v[(i + 1) % kRows][j] * vu, v[(i + 2) % kRows][j] * vu,
                      v[(i + 3) % kRows][j] * vu);
        }
      }
      __syncthreads();
#pragma unroll
      for (uint32_t p = 0; p < 64 * dim; p += kThreads * 16)
        *reinterpret_cast<u32x4*>(to + p + tid * 16) =
            *reinterpret_cast<const u32x4*>(image + p + tid * 16);
    } else {
      // earlier tokens' codes where the scale grows, in 16-byte pieces
      const bool k_grows = ks > had_k && had_k > 0, v_grows = vs > had_v && had_v > 0;
      if (k_grows || v_grows) {
        for (uint32_t p = tid; p < 4 * dim; p += kThreads) {
          const bool is_k = p < 2 * dim;
          if (!(is_k ? k_grows : v_grows)) continue;
          const float f = is_k ? ScaleOf(had_k) * Unscale(ks) : ScaleOf(had_v) * Unscale(vs);
          u32x4* const piece = reinterpret_cast<u32x4*>(to) + p;
          u32x4 x = *piece;
#pragma unroll
          for (uint32_t j = 0; j < 4; ++j) {
            const uint32_t y = Again(x[j], f);
            if (is_k) {  // a piece is of one token
              const uint32_t t = p / 64 / (dim / 64) * 16 + p % 16;
              if (t < t0) x[j] = y;
            } else {  // a word is of four
              const uint32_t t = j % 2 * 16 + p % 64 / 16 * 4;
              const uint32_t keep = t + 4 <= t0 ? ~0u : t >= t0 ? 0u : (1u << (8 * (t0 - t))) - 1;
              x[j] = (y & keep) | (x[j] & ~keep);
            }
          }
          *piece = x;
        }
        __syncthreads();  // before the new tokens' bytes
      }
#pragma unroll
      for (uint32_t i = 0; i < kRows; ++i) {
        const uint32_t t = token(i);
        if (t >= count) continue;
        const uint32_t codes = Codes(k[i][0] * ku, k[i][1] * ku, k[i][2] * ku, k[i][3] * ku);
        *reinterpret_cast<uint32_t*>(to + Kv8KCode(dim, t0 + t, col)) =
            bad >> i & 1 ? 0x7F7F7F7Fu : codes;
        const uint32_t values = Codes(v[i][0] * vu, v[i][1] * vu, v[i][2] * vu, v[i][3] * vu);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
          to[Kv8VCode(dim, t0 + t, col + j)] = (uint8_t)(values >> (8 * j));
      }
    }
    if (tid == 0)
      *reinterpret_cast<uint16_t*>(to + Kv8Scale(dim, 0)) = (uint16_t)(ks | vs << 8);
    __syncthreads();  // image, tops and scales have been read
  }
}

template <class T>
__device__ __forceinline__ void Store4(T* to, bool vec, uint32_t codes, float scale) {
  typedef typename Four<T>::type V;
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false);
  const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
  const float y[4] = {a[0] * scale, a[1] * scale, b[0] * scale, b[1] * scale};
  if (vec) {
    V v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (T)y[j];
    *reinterpret_cast<V*>(to) = v;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) to[j] = (T)y[j];
  }
}

// The stored values of slots, 4 columns of 4 neighbouring rows a thread.  Where
// their slots are neighbours too, from a multiple of 4 on, a column's four V codes
// are a word; else each is a load of its own.  The rows above back to fp32, 10 MB
// read and 41 written, 10.6 us = 4.8 TB/s (12.1 with loads of their own).
template <class T, uint32_t dim>
__global__ __launch_bounds__(kThreads) void ReadKernel(const KvRowsArgs g) {
  constexpr uint32_t kRow = dim / 4, kGroups = kThreads / kRow, kEach = 4;
  const uint32_t head = blockIdx.x % g.heads, col = threadIdx.x % kRow * 4;
  const uint64_t row0 =
      (uint64_t)(blockIdx.x / g.heads + g.first) * (kGroups * kEach) + threadIdx.x / kRow * kEach;
  uint32_t k[kEach], v[kEach], scales[kEach], t[kEach];
  int32_t slot[kEach];
  const uint8_t* from[kEach];
  bool there[kEach], four = true;
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i) slot[i] = row0 + i < g.tokens ? g.slots[row0 + i] : -1;
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i) {
    uint64_t record;
    there[i] = KvSlot(slot[i], g.pages, g.heads, g.groups, &record, &t[i]);
    from[i] = g.cache + (there[i] ? record + (uint64_t)head * g.groups : 0) * Kv8RecordBytes(dim);
    four = four && there[i] && slot[i] == slot[0] + (int32_t)i;
  }
  four = four && slot[0] % 4 == 0;
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i) {
    k[i] = v[i] = scales[i] = 0;
    if (!there[i]) continue;
    k[i] = *reinterpret_cast<const uint32_t*>(from[i] + Kv8KCode(dim, t[i], col));
    scales[i] = *reinterpret_cast<const uint16_t*>(from[i] + Kv8Scale(dim, 0));
  }
  if (four) {
    uint32_t w[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j)
      w[j] = *reinterpret_cast<const uint32_t*>(from[0] + Kv8VCode(dim, t[0], col + j));
    // from a column's tokens to a token's columns
    const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u);  // tokens 0, 1
    const uint32_t b = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);  // tokens 2, 3
    const uint32_t d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    v[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    v[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    v[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
    v[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
      if (!there[i]) continue;
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j)
        v[i] |= (uint32_t)from[i][Kv8VCode(dim, t[i], col + j)] << (8 * j);
    }
  }
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i) {
    const uint64_t row = row0 + i;
    if (row >= g.tokens) continue;
    Store4(static_cast<T*>(g.k_out) + row * g.k_token + head * g.k_head + col, g.vec, k[i],
           ScaleOf(scales[i] & 255u));
    Store4(static_cast<T*>(g.v_out) + row * g.v_token + head * g.v_head + col, g.vec, v[i],
           ScaleOf(scales[i] >> 8));
  }
}

template <class T, uint32_t dim>
hipError_t LaunchOf(KvRowsArgs& a, bool read, hipStream_t s) {
  if (read) {
    constexpr uint32_t kRows = kThreads / (dim / 4) * 4;
    return LaunchRowGroups(a, (a.tokens + kRows - 1) / kRows, [&](uint32_t grid) {
      ReadKernel<T, dim><<<grid, kThreads, 0, s>>>(a);
    });
  }
  // eight workgroups a CU, of a block's rows at most
  const uint64_t rows = (uint64_t)a.tokens * a.heads / (8 * (uint64_t)DeviceCus());
  a.window = (uint32_t)std::min<uint64_t>(32, std::max<uint64_t>(1, rows));
  return LaunchRowGroups(a, (a.tokens + a.window - 1) / a.window, [&](uint32_t grid) {
    AppendKernel<T, dim><<<grid, kThreads, 0, s>>>(a);
  });
}

template <class T>
hipError_t LaunchType(KvRowsArgs& a, bool read, hipStream_t s) {
  switch (a.dim) {
    case 64: return LaunchOf<T, 64>(a, read, s);
    case 128: return LaunchOf<T, 128>(a, read, s);
    case 256: return LaunchOf<T, 256>(a, read, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t LaunchKv8Rows(const KvRowsArgs& in, bool read, hipStream_t stream) {
  KvRowsArgs a = in;
  a.vec = KvRowsAligned(a, read);
  switch (a.type) {
    case HB_TYPE_F32: return LaunchType<float>(a, read, stream);
    case HB_TYPE_BF16: return LaunchType<__bf16>(a, read, stream);
    default: return LaunchType<_Float16>(a, read, stream);
  }
}

}  // namespace hb
