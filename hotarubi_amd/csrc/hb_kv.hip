// Serving operators around the paged MXFP4 cache: the step plan (block
// tables, slots and positions on the device), the per-head norm with the
// rotation by position, and K and V rows into the cache and back out.
#include <algorithm>

#include "hb_internal.h"
#include "hb_kv.h"

namespace hb {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

template <class T>
struct Four;
template <>
struct Four<float> {
  typedef f32x4 type;
};
template <>
struct Four<__bf16> {
  typedef bf16x4 type;
};
template <>
struct Four<_Float16> {
  typedef f16x4 type;
};

constexpr uint32_t kThreads = 256;

// ------------------------------------------------------------------- plan --

// Inclusive sum over the workgroup's threads; *total the sum of all.  `part`
// holds a value per wave.
__device__ __forceinline__ int64_t BlockSum(int64_t x, int64_t* part, int64_t* total) {
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  for (uint32_t d = 1; d < 64; d *= 2) {
    const int64_t y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();  // the values of an earlier call have been read
  if (lane == 63) part[wave] = x;
  __syncthreads();
  int64_t sum = 0;
  for (uint32_t w = 0; w < kThreads / 64; ++w) {
    if (w < wave) x += part[w];
    sum += part[w];
  }
  *total = sum;
  return x;
}

// Pages of `tokens` tokens.
__device__ __forceinline__ uint32_t Pages(uint32_t tokens, uint32_t page) {
  return tokens / page + (tokens % page != 0 ? 1u : 0u);
}

// Two sums over the requests (tokens, then the pages of those that fit), then
// a thread per token: its request by bisection, its position, its slot, and
// the table entry where it is the first token of a new page.  Every workgroup
// makes the sums for itself, which is less than a launch or a wait between
// workgroups would cost: requests come in chunks, each thread taking
// kPlanEach neighbours, and the tokens of a chunk go round over the
// workgroups.  No workgroup reads what another writes: new pages come from
// the free list, entries of older ones are not written.  What bounds it is
// the chain of loads, sums and bisection, so a thread takes as few requests
// and tokens as there are: 64 requests of a token or few 3.9 us (5.6 with four
// requests a thread), 512 requests of 38,912 tokens 6.1 us (10.0 with four and
// four tokens a thread).
template <uint32_t kPlanEach>
__global__ __launch_bounds__(kThreads) void PlanKernel(const PlanArgs a) {
  constexpr uint32_t kPlanChunk = kPlanEach * kThreads;
  __shared__ int64_t part[kThreads / 64];
  __shared__ int64_t ends[kPlanChunk], first[kPlanChunk];  // tokens; pages before
  __shared__ int32_t have_len[kPlanChunk];
  __shared__ uint8_t fine[kPlanChunk];
  __shared__ uint32_t status[2];
  const uint32_t tid = threadIdx.x;
  const uint32_t page = a.page;
  const int64_t free_count = max(0, min(*a.free_count, (int32_t)a.free_size));
  int64_t tokens = 0, pages = 0;
  if (tid < 2) status[tid] = 0;  // (the sums' barriers come before its use)
  for (uint32_t base = 0; base < a.batch; base += kPlanChunk) {
    const uint32_t chunk = min(kPlanChunk, a.batch - base);
    uint32_t len[kPlanEach], more[kPlanEach], need[kPlanEach];
    int64_t sum = 0, total;
    for (uint32_t j = 0; j < kPlanEach; ++j) {
      const uint32_t i = tid * kPlanEach + j;
      len[j] = i < chunk ? (uint32_t)max(0, a.lens[base + i]) : 0u;
      more[j] = i < chunk ? (uint32_t)max(0, a.new_tokens[base + i]) : 0u;
      sum += more[j];
    }
    int64_t at = tokens + BlockSum(sum, part, &total) - sum;
    const int64_t chunk_end = tokens + total;
    sum = 0;
    uint32_t fits = 0;
    for (uint32_t j = 0; j < kPlanEach; ++j) {
      const uint32_t i = tid * kPlanEach + j;
      at += more[j];
      const uint32_t used = Pages(len[j], page), want = Pages(len[j] + more[j], page);
      const bool f = want <= a.columns && at <= a.size && len[j] + more[j] <= 0x7FFFFFFFu;
      need[j] = f ? want - used : 0;
      fits |= (uint32_t)f << j;
      sum += need[j];
      if (i < chunk) {
        ends[i] = at;
        have_len[i] = (int32_t)len[j];
        if (blockIdx.x == 0) a.cu[base + i + 1] = (int32_t)at;
      }
    }
    int64_t stop = pages + BlockSum(sum, part, &total) - sum;
    pages += total;
    uint32_t ok_pages = 0, bad = 0;
    for (uint32_t j = 0; j < kPlanEach; ++j) {
      const uint32_t i = tid * kPlanEach + j;
      stop += need[j];
      const bool ok = (fits >> j & 1) != 0 && (need[j] == 0 || stop <= free_count);
      if (i < chunk) {
        first[i] = stop - need[j];
        fine[i] = ok;
        ok_pages += ok ? need[j] : 0;
        bad += ok ? 0 : 1;
        if (blockIdx.x == 0) a.kv_lens[base + i] = (int32_t)(ok ? len[j] + more[j] : len[j]);
      }
    }
    // whole numbers, so the order of these does not matter
    if (blockIdx.x == 0 && ok_pages > 0) atomicAdd(&status[0], ok_pages);
    if (blockIdx.x == 0 && bad > 0) atomicAdd(&status[1], bad);
    __syncthreads();
    const int64_t last = min(chunk_end, (int64_t)a.size);
    for (int64_t t = tokens + blockIdx.x * kThreads + tid; t < last;
         t += (int64_t)gridDim.x * kThreads) {
      uint32_t lo = 0, hi = chunk - 1;  // the first request whose tokens end past t
      while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (ends[mid] > t) hi = mid;
        else lo = mid + 1;
      }
      const int64_t begin = lo > 0 ? ends[lo - 1] : tokens;
      // below 2^32: the request's tokens are within `size`, or its slot is not
      // looked up
      const uint32_t pos = (uint32_t)have_len[lo] + (uint32_t)(t - begin);
      int64_t slot = -1;
      if (fine[lo]) {
        const uint32_t col = pos / page, used = Pages((uint32_t)have_len[lo], page);
        int32_t* const row = a.table + (uint64_t)(base + lo) * a.table_stride;
        int32_t p;
        if (col >= used) {
          const int64_t i = free_count - 1 - first[lo] - (col - used);
          p = a.free_pages[i];
          if (pos % page == 0) row[col] = p;
        } else {
          p = row[col];
        }
        if (p >= 0) slot = (int64_t)p * page + pos % page;
        if (slot > 0x7FFFFFFF) slot = -1;
      }
      a.slots[t] = (int32_t)slot;
      a.positions[t] = (int32_t)pos;
    }
    tokens = chunk_end;
    __syncthreads();  // the chunk's LDS has been read
  }
  for (int64_t t = tokens + blockIdx.x * kThreads + tid; t < a.size;
       t += (int64_t)gridDim.x * kThreads) {
    a.slots[t] = -1;
    a.positions[t] = -1;
  }
  __syncthreads();  // status, also where there was no request
  if (blockIdx.x == 0 && tid == 0) {
    a.cu[0] = 0;
    a.status[0] = (int32_t)status[0];
    a.status[1] = (int32_t)status[1];
  }
}

// ------------------------------------------------------------------- rope --

// cos and sin of 2 pi r.  r is reduced to an eighth of a turn around its
// quadrant in 64 bits; on |x| <= pi/4 the Taylor series to x^9 and x^10 is off
// by less than 2^-29.
__device__ __forceinline__ void Turn(double r, float* c, float* s) {
  r -= rint(r);
  const double q = rint(4.0 * r);
  const float x = (float)((r - 0.25 * q) * 6.283185307179586476925);
  const float y = x * x;
  float u = fmaf(y, 1.f / 362880.f, -1.f / 5040.f);
  u = fmaf(y, u, 1.f / 120.f);
  u = fmaf(y, u, -1.f / 6.f);
  const float si = fmaf(x * y, u, x);
  float v = fmaf(y, -1.f / 3628800.f, 1.f / 40320.f);
  v = fmaf(y, v, -1.f / 720.f);
  v = fmaf(y, v, 1.f / 24.f);
  v = fmaf(y, v, -0.5f);
  const float co = fmaf(y, v, 1.f);
  const int k = (int)q & 3;
  const float a = k & 1 ? si : co, b = k & 1 ? co : si;
  *c = k == 1 || k == 2 ? -a : a;
  *s = k >= 2 ? -b : b;
}

// Sum over the `lanes` (8, 16, 32 or 64) neighbouring lanes that hold a head.
__device__ __forceinline__ float HeadSum(float x, uint32_t lanes) {
#define HB_DPP_ADD(ctrl) \
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), ctrl, 0xF, 0xF, false))
  HB_DPP_ADD(0xB1);   // xor 1
  HB_DPP_ADD(0x4E);   // xor 2
  HB_DPP_ADD(0x141);  // the other four of eight
  if (lanes > 8) HB_DPP_ADD(0x140);  // the other eight of sixteen
#undef HB_DPP_ADD
  if (lanes > 16) x += __shfl_xor(x, 16);
  if (lanes > 32) x += __shfl_xor(x, 32);
  return x;
}

// A lane's four pairs of elements of a head: pair p of the first rot / 2 is
// what a rotation turns (p and p + rot/2, or 2p and 2p + 1), the others are
// the rest of the head, cut in halves or in neighbours too.
struct Pairs {
  uint32_t a, b, step;  // elements a + step j, b + step j
};
template <bool neighbours>
__device__ __forceinline__ Pairs PairsOf(uint32_t p, uint32_t dim, uint32_t rot) {
  if (neighbours) return {2 * p, 2 * p + 1, 2};
  const uint32_t half = rot / 2;
  if (p < half) return {p, p + half, 1};
  return {rot + p - half, rot + p - half + (dim - rot) / 2, 1};
}

template <class T, bool vec, bool neighbours>
__device__ __forceinline__ void LoadPairs(const T* x, uint32_t p, const RopeArgs& g, float* a,
                                          float* b) {
  typedef typename Four<T>::type V;
  if (vec) {
    const Pairs at = PairsOf<neighbours>(p, g.dim, g.rot);
    const V lo = *reinterpret_cast<const V*>(x + at.a);
    const V hi = *reinterpret_cast<const V*>(x + (neighbours ? at.a + 4 : at.b));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      a[j] = neighbours ? (j < 2 ? (float)lo[2 * j % 4] : (float)hi[2 * j % 4]) : (float)lo[j];
      b[j] = neighbours ? (j < 2 ? (float)lo[(2 * j + 1) % 4] : (float)hi[(2 * j + 1) % 4])
                        : (float)hi[j];
    }
  } else {
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      a[j] = b[j] = 0.f;
      if (p + j < g.dim / 2) {
        const Pairs at = PairsOf<neighbours>(p + j, g.dim, g.rot);
        a[j] = (float)x[at.a];
        b[j] = (float)x[at.b];
      }
    }
  }
}

template <class T, bool vec, bool neighbours>
__device__ __forceinline__ void StorePairs(T* x, uint32_t p, const RopeArgs& g, const float* a,
                                           const float* b) {
  typedef typename Four<T>::type V;
  if (vec) {
    const Pairs at = PairsOf<neighbours>(p, g.dim, g.rot);
    V lo, hi;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      lo[j] = (T)(neighbours ? (j % 2 ? b[j / 2] : a[j / 2]) : a[j]);
      hi[j] = (T)(neighbours ? (j % 2 ? b[2 + j / 2] : a[2 + j / 2]) : b[j]);
    }
    *reinterpret_cast<V*>(x + at.a) = lo;
    *reinterpret_cast<V*>(x + (neighbours ? at.a + 4 : at.b)) = hi;
  } else {
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      if (p + j < g.dim / 2) {
        const Pairs at = PairsOf<neighbours>(p + j, g.dim, g.rot);
        x[at.a] = (T)a[j];
        x[at.b] = (T)b[j];
      }
    }
  }
}

// y = x gamma / sqrt(mean(x^2) + eps) of every query and key head, then each
// pair of its first rot elements turned by position x frequency: one read and
// one write of the rows.  A lane holds four pairs, so 8 to 64 lanes hold a
// head and a wave several; the pairs, and with them the cosines and sines, are
// the same for every head, so a wave computes a token's angles once, a lane
// each (64 bits), while its first heads load, passes them through LDS and
// takes the token's heads one after another (angles made by every lane for
// itself took 37 us where this takes 32).  `parts` waves share a token where
// tokens are few.  Memory bounds it: 8,192 tokens of 32 + 8 heads of 128 in
// bf16, 168 MB, 32 us = 5.2 TB/s; 16 tokens of 20 heads of 64 3.9 us, latency.
template <class T, bool vec, bool neighbours>
__global__ __launch_bounds__(kThreads) void RopeKernel(const RopeArgs g) {
  constexpr uint32_t kBatch = 2;  // heads of a lane in flight
  __shared__ float turns[kThreads / 64][256][2];
  const uint32_t lane = threadIdx.x % 64;
  const uint32_t in = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t wave = blockIdx.x * (kThreads / 64) + in;
  const uint32_t token = wave / g.parts, part = wave % g.parts;
  if (token >= g.tokens) return;
  const uint32_t per = 64 / g.lanes, p = lane % g.lanes * 4, half = g.rot / 2;
  const uint32_t heads = g.q_heads + g.k_heads;
  const bool holds = p < g.dim / 2;
  const uint32_t step = per * g.parts;
  float a[kBatch][4], b[kBatch][4];
  auto load = [&](uint32_t h0) {
#pragma unroll
    for (uint32_t u = 0; u < kBatch; ++u) {
      const uint32_t h = h0 + u * step;
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) a[u][j] = b[u][j] = 0.f;
      if (h < heads && holds) {
        const bool is_q = h < g.q_heads;
        const T* x = is_q ? static_cast<const T*>(g.q) + token * g.q_token + h * g.q_head
                          : static_cast<const T*>(g.k) + token * g.k_token +
                                (h - g.q_heads) * g.k_head;
        LoadPairs<T, vec, neighbours>(x, p, g, a[u], b[u]);
      }
    }
  };
  uint32_t h0 = part * per + lane / g.lanes;
  load(h0);
  for (uint32_t i = lane; i < half; i += 64) {
    const uint32_t axis = (i >= g.sections[0] ? 1u : 0u) + (i >= g.sections[1] ? 1u : 0u);
    const double turn = g.inv_freq[i] * 0.15915494309189533577;
    Turn((double)g.positions[axis * g.position_stride + token] * turn, &turns[in][i][0],
         &turns[in][i][1]);
  }
  float gq[8], gk[8];
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    gq[j] = gq[4 + j] = gk[j] = gk[4 + j] = 1.f;
    if (p + j < g.dim / 2) {
      const Pairs at = PairsOf<neighbours>(p + j, g.dim, g.rot);
      if (g.gamma_q) {
        gq[j] = g.gamma_q[at.a];
        gq[4 + j] = g.gamma_q[at.b];
      }
      if (g.gamma_k) {
        gk[j] = g.gamma_k[at.a];
        gk[4 + j] = g.gamma_k[at.b];
      }
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  float c[4], s[4];
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    const bool turned = p + j < half;
    c[j] = turned ? turns[in][p + j][0] : 1.f;
    s[j] = turned ? turns[in][p + j][1] : 0.f;
  }
  const float inv_dim = 1.f / (float)g.dim;
  while (h0 < heads) {
#pragma unroll
    for (uint32_t u = 0; u < kBatch; ++u) {
      const uint32_t h = h0 + u * step;
      const bool is_q = h < g.q_heads;
      if (is_q ? g.gamma_q != nullptr : g.gamma_k != nullptr) {
        float sum = 0.f;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
          sum = fmaf(a[u][j], a[u][j], fmaf(b[u][j], b[u][j], sum));
        sum = HeadSum(sum, g.lanes);
        const float r = __builtin_amdgcn_rsqf(fmaf(sum, inv_dim, g.eps));
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
          a[u][j] *= r * (is_q ? gq[j] : gk[j]);
          b[u][j] *= r * (is_q ? gq[4 + j] : gk[4 + j]);
        }
      }
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        // past rot each element is left alone: a turn by 0 would carry an
        // infinity or NaN to the other one of its pair
        const bool turned = p + j < half;
        const float x = a[u][j], y = b[u][j];
        a[u][j] = turned ? fmaf(x, c[j], -(y * s[j])) : x;
        b[u][j] = turned ? fmaf(y, c[j], x * s[j]) : y;
      }
      if (h < heads && holds) {
        T* y = is_q ? static_cast<T*>(g.q_out) + token * g.q_out_token + h * g.q_out_head
                    : static_cast<T*>(g.k_out) + token * g.k_out_token +
                          (h - g.q_heads) * g.k_out_head;
        StorePairs<T, vec, neighbours>(y, p, g, a[u], b[u]);
      }
    }
    h0 += step * kBatch;
    load(h0);
  }
}

// ------------------------------------------------------------ cache rows --

template <class T>
__device__ __forceinline__ void Load8(const T* x, bool vec, float* y) {
  typedef typename Four<T>::type V;
  if (vec) {
    const V lo = reinterpret_cast<const V*>(x)[0], hi = reinterpret_cast<const V*>(x)[1];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = (float)(j < 4 ? lo[j % 4] : hi[j % 4]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = (float)x[j];
  }
}

// Largest over the four lanes of a 32-column block.
__device__ __forceinline__ uint32_t QuadMax(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xF, 0xF, false));
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, false));
}

// Eight values of a block as E2M1 codes (nearest even, saturated), value j in
// nibble j, and the block's scale byte: exponent floor(log2 max) - 2 within
// [-126, 125], 0 for a block of zeros.
__device__ __forceinline__ uint32_t Encode8(const float* x, uint32_t* scale) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[j]) & 0x7FFFFFFFu);
  top = QuadMax(top);
  // a subnormal maximum's field is 0: below the clamp as the exponent is
  const int32_t e = (int32_t)(top >> 23) - 129;
  *scale = top == 0 ? 127u : (uint32_t)(127 + min(max(e, -126), 125));
  const float unit = __uint_as_float(*scale << 23);
  uint32_t code = 0;
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[0], x[1], unit, 0);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[2], x[3], unit, 1);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[4], x[5], unit, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[6], x[7], unit, 3);
}

// Eight columns' V codes: one run of bytes where a lane of the reading wave
// holds 8 columns or more, two where it holds 4.
__device__ __forceinline__ void StoreV(uint8_t* record, uint32_t dim, uint32_t t, uint32_t col,
                                       uint32_t code) {
  if (dim == 64) {
    *reinterpret_cast<uint16_t*>(record + KvVCode(64, t, col)) = (uint16_t)code;
    *reinterpret_cast<uint16_t*>(record + KvVCode(64, t, col + 4)) = (uint16_t)(code >> 16);
  } else {
    *reinterpret_cast<uint32_t*>(record + KvVCode(dim, t, col)) = code;
  }
}
__device__ __forceinline__ uint32_t LoadV(const uint8_t* record, uint32_t dim, uint32_t t,
                                          uint32_t col) {
  if (dim == 64) {
    const uint32_t lo = *reinterpret_cast<const uint16_t*>(record + KvVCode(64, t, col));
    return lo | (uint32_t)*reinterpret_cast<const uint16_t*>(record + KvVCode(64, t, col + 4))
                    << 16;
  }
  return *reinterpret_cast<const uint32_t*>(record + KvVCode(dim, t, col));
}

// K and V rows of one token and head into the cache: 8 columns of both a
// lane, so 8, 16 or 32 lanes hold a head and four a block.  A workgroup takes
// neighbouring tokens of one head: where their slots are neighbours too, as
// in a prompt, a record's bytes of several tokens leave in one store (a token's
// own lie 2 to 16 bytes long all over the record).  A row with an infinity or
// NaN in K or V is stored as NaN keys and zero values.  Memory bounds it:
// 16,001 tokens of 5 heads of 64 in fp32, 41 MB read and 6 MB written, 9.3 us =
// 5.0 TB/s (13.2 with a token's heads side by side); 64 tokens of 8 heads 3 us.
template <uint32_t dim>
struct RowLanes {
  static constexpr uint32_t kLanes = dim / 8, kTokens = kThreads / kLanes;
  uint32_t token, head, col;
  __device__ __forceinline__ explicit RowLanes(uint32_t heads) {
    head = blockIdx.x % heads;
    token = blockIdx.x / heads * kTokens + threadIdx.x / kLanes;
    col = threadIdx.x % kLanes * 8;
  }
};
template <class T, uint32_t dim>
__global__ __launch_bounds__(kThreads) void AppendKernel(const KvRowsArgs g) {
  const RowLanes<dim> at(g.heads);
  constexpr uint32_t kLanes = RowLanes<dim>::kLanes;
  float k[8] = {}, v[8] = {};
  int32_t slot = -1;
  if (at.token < g.tokens) {
    slot = g.slots[at.token];
    Load8(static_cast<const T*>(g.k) + at.token * g.k_token + at.head * g.k_head + at.col, g.vec,
          k);
    Load8(static_cast<const T*>(g.v) + at.token * g.v_token + at.head * g.v_head + at.col, g.vec,
          v);
  }
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    top = max(top, max(__float_as_uint(k[j]) & 0x7FFFFFFFu, __float_as_uint(v[j]) & 0x7FFFFFFFu));
  const uint64_t odd = __builtin_amdgcn_ballot_w64(top >= 0x7F800000u);
  const uint64_t mine = (~0ull >> (64 - kLanes)) << (threadIdx.x % 64 / kLanes * kLanes);
  const bool bad = (odd & mine) != 0;
  if (bad) {
#pragma unroll
    for (int j = 0; j < 8; ++j) k[j] = v[j] = 0.f;
  }
  uint32_t ks, vs;
  const uint32_t kc = Encode8(k, &ks), vc = Encode8(v, &vs);
  uint64_t record;
  uint32_t t;
  if (!KvSlot(slot, g.pages, g.heads, g.groups, &record, &t)) return;
  uint8_t* const to = g.cache + (record + (uint64_t)at.head * g.groups) * KvRecordBytes(dim);
  *reinterpret_cast<uint32_t*>(to + KvKCode(dim, t, at.col)) = kc;
  StoreV(to, dim, t, at.col, vc);
  if (at.col % 32 == 0) {
    to[KvKScale(dim, t, at.col)] = bad ? 255 : (uint8_t)ks;
    to[KvVScale(dim, t, at.col)] = (uint8_t)vs;
  }
}

// Eight codes as values of type T.
template <class T>
__device__ __forceinline__ void Decode8(uint32_t code, uint32_t scale, T* y) {
  const float s = __uint_as_float(scale << 23);
#define HB_PAIR(i)                                                                          \
  if constexpr (sizeof(T) == 4) {                                                           \
    const f32x2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, s, i);                   \
    y[2 * i] = p[0];                                                                        \
    y[2 * i + 1] = p[1];                                                                    \
  } else if constexpr (__is_same(T, __bf16)) {                                              \
    const bf16x2 p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, s, i);                 \
    y[2 * i] = p[0];                                                                        \
    y[2 * i + 1] = p[1];                                                                    \
  } else {                                                                                  \
    const f16x2 p = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code, s, i);                   \
    y[2 * i] = p[0];                                                                        \
    y[2 * i + 1] = p[1];                                                                    \
  }
  HB_PAIR(0)
  HB_PAIR(1)
  HB_PAIR(2)
  HB_PAIR(3)
#undef HB_PAIR
}

template <class T>
__device__ __forceinline__ void Store8(T* to, bool vec, const T* y) {
  typedef typename Four<T>::type V;
  if (vec) {
    V lo, hi;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      lo[j] = y[j];
      hi[j] = y[4 + j];
    }
    reinterpret_cast<V*>(to)[0] = lo;
    reinterpret_cast<V*>(to)[1] = hi;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) to[j] = y[j];
  }
}

// The stored values of slots, on AppendKernel's lanes: codes times scales are
// exact in all three types wherever the type's range holds them.  Memory
// bounds it: the rows above back to fp32 in 11.9 us, 4.0 TB/s.
template <class T, uint32_t dim>
__global__ __launch_bounds__(kThreads) void ReadKernel(const KvRowsArgs g) {
  const RowLanes<dim> at(g.heads);
  if (at.token >= g.tokens) return;
  uint64_t record;
  uint32_t t;
  uint32_t kc = 0, vc = 0, ks = 127, vs = 127;
  if (KvSlot(g.slots[at.token], g.pages, g.heads, g.groups, &record, &t)) {
    const uint8_t* from = g.cache + (record + (uint64_t)at.head * g.groups) * KvRecordBytes(dim);
    kc = *reinterpret_cast<const uint32_t*>(from + KvKCode(dim, t, at.col));
    vc = LoadV(from, dim, t, at.col);
    ks = from[KvKScale(dim, t, at.col)];
    vs = from[KvVScale(dim, t, at.col)];
  }
  T y[8];
  Decode8(kc, ks, y);
  Store8(static_cast<T*>(g.k_out) + at.token * g.k_token + at.head * g.k_head + at.col, g.vec, y);
  Decode8(vc, vs, y);
  Store8(static_cast<T*>(g.v_out) + at.token * g.v_token + at.head * g.v_head + at.col, g.vec, y);
}

template <class T>
hipError_t LaunchRopeOf(const RopeArgs& a, bool vec, uint32_t grid, hipStream_t s) {
  if (vec && a.neighbours) RopeKernel<T, true, true><<<grid, kThreads, 0, s>>>(a);
  else if (vec) RopeKernel<T, true, false><<<grid, kThreads, 0, s>>>(a);
  else if (a.neighbours) RopeKernel<T, false, true><<<grid, kThreads, 0, s>>>(a);
  else RopeKernel<T, false, false><<<grid, kThreads, 0, s>>>(a);
  return hipGetLastError();
}

template <class T>
hipError_t LaunchKvRowsOf(const KvRowsArgs& a, bool read, uint32_t grid, hipStream_t s) {
#define HB_ROWS_DIM(d)                                                   \
  case d:                                                                \
    if (read) ReadKernel<T, d><<<grid, kThreads, 0, s>>>(a);             \
    else AppendKernel<T, d><<<grid, kThreads, 0, s>>>(a);                \
    break;
  switch (a.dim) {
    HB_ROWS_DIM(64)
    HB_ROWS_DIM(128)
    HB_ROWS_DIM(256)
    default: return hipErrorInvalidValue;
  }
#undef HB_ROWS_DIM
  return hipGetLastError();
}

}  // namespace

hipError_t LaunchPlan(const PlanArgs& a, hipStream_t stream) {
  const uint32_t grid = std::min(256u, std::max(1u, (a.size + kThreads - 1) / kThreads));
  if (a.batch <= kThreads) PlanKernel<1><<<grid, kThreads, 0, stream>>>(a);
  else if (a.batch <= 2 * kThreads) PlanKernel<2><<<grid, kThreads, 0, stream>>>(a);
  else PlanKernel<4><<<grid, kThreads, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t LaunchRope(const RopeArgs& in, hipStream_t stream) {
  RopeArgs a = in;
  a.lanes = 8;
  while (a.lanes * 8 < a.dim) a.lanes *= 2;
  const uint32_t steps = (a.q_heads + a.k_heads + 64 / a.lanes - 1) / (64 / a.lanes);
  // about 16 waves a CU, as far as the heads go
  const uint32_t want = 16 * (uint32_t)DeviceCus();
  a.parts = std::max(1u, std::min(steps, want / std::max(1u, a.tokens)));
  const uint64_t waves = (uint64_t)a.tokens * a.parts;
  const uint32_t grid = (uint32_t)((waves + kThreads / 64 - 1) / (kThreads / 64));
  const uint32_t size = a.type == HB_TYPE_F32 ? 4 : 2;
  const uint64_t strides = a.q_token | a.q_head | a.k_token | a.k_head | a.q_out_token |
                           a.q_out_head | a.k_out_token | a.k_out_head;
  const uintptr_t bases = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) |
                          reinterpret_cast<uintptr_t>(a.q_out) |
                          reinterpret_cast<uintptr_t>(a.k_out);
  const bool vec = strides % 4 == 0 && bases % (4 * size) == 0 && a.dim % 8 == 0 &&
                   (a.neighbours || (a.rot % 8 == 0 && (a.dim - a.rot) % 8 == 0));
  switch (a.type) {
    case HB_TYPE_F32: return LaunchRopeOf<float>(a, vec, grid, stream);
    case HB_TYPE_BF16: return LaunchRopeOf<__bf16>(a, vec, grid, stream);
    default: return LaunchRopeOf<_Float16>(a, vec, grid, stream);
  }
}

hipError_t LaunchKvRows(const KvRowsArgs& in, bool read, hipStream_t stream) {
  KvRowsArgs a = in;
  const uint32_t size = a.type == HB_TYPE_F32 ? 4 : 2;
  const uint64_t strides = a.k_token | a.k_head | a.v_token | a.v_head;
  const uintptr_t bases =
      read ? reinterpret_cast<uintptr_t>(a.k_out) | reinterpret_cast<uintptr_t>(a.v_out)
           : reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v);
  a.vec = strides % 4 == 0 && bases % (4 * size) == 0;
  const uint32_t tokens = kThreads / (a.dim / 8);  // of a workgroup
  const uint32_t grid = (a.tokens + tokens - 1) / tokens * a.heads;
  switch (a.type) {
    case HB_TYPE_F32: return LaunchKvRowsOf<float>(a, read, grid, stream);
    case HB_TYPE_BF16: return LaunchKvRowsOf<__bf16>(a, read, grid, stream);
    default: return LaunchKvRowsOf<_Float16>(a, read, grid, stream);
  }
}

}  // namespace hb
