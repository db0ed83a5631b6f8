// Log probabilities of given tokens, the entropy and the most likely tokens of
// rows of logits, one pass over them.
//
// With c = scale log2 e, m the running maximum, t = x - m, l = sum 2^(c t) and
// w = sum t 2^(c t), a token's log probability is scale t - ln l and the entropy
// ln l - scale w / l.  Parts with maxima m1, m2 meet at m = max as
// l = sum l_i f_i, w = sum (w_i + (m_i - m) l_i) f_i, f_i = 2^(c (m_i - m)).  The
// difference comes before the product, so that logits of any size have one.
//
// The most likely tokens: every lane keeps the maxima of its stretches of the
// row in LDS.  `top` logits reach the `top`-th largest of the lanes' largest or two
// largest maxima, so that (its upper 16 bits) is a bound, and only stretches that
// reach it are read again, all at once; their logits go into a list of sorted 64-bit
// keys, one a lane, 64 of them at a time.  (64 likeliest tokens want all lanes of
// one each: 200 rows of 100,001 in fp32 64 us, 40 with two.)
//
// About 10 vector instructions a logit, four of an exponential's slots among them,
// for 2 or 4 bytes: memory bounds long rows, 4,096 of 65,537 bf16 logits with the 5
// likeliest 115 us = 4.7 TB/s (a reading of them once at what the card copies at
// is 105; without the likeliest tokens 105), 2,048 of 65,537 in fp32 107 us = 5.0.
// Of short calls the waves' chain does: 8 rows of 50,001 fp32 logits, 20 each,
// 9.0 us and 5.4 for the join.
#include <algorithm>

#include "hb_internal.h"
#include "hb_lanes.h"

namespace hb {
namespace {

constexpr uint32_t kThreads = 256, kWaves = kThreads / 64;
constexpr uint32_t kLoads = 2;  // 16-byte loads of a lane's batch
constexpr uint32_t kStretches = 24;
// Likeliest tokens up to which a lane's largest maximum makes the bound: 2,000 rows
// of 50,001 bf16 logits with 20 each 51.5 us, 52.1 with two maxima a lane, but with
// 32 54.3 and 54.0, with 64 108 and 70.
constexpr uint32_t kOfOne = 24;
// Parts of a row and the keys that are joined of them: 9 x 161,526 fp32, 32 each, 17.4
// us, 21.1 with 40 parts of 32 keys, 19.2 with 8.
constexpr uint32_t kMostParts = 64, kJoined = 512;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// Values of a 16-byte load, as fp32.
template <class T>
struct Packed;
template <>
struct Packed<float> {
  static constexpr uint32_t kCount = 4, kLowest = 0xFF800000u;
  static __device__ __forceinline__ float At(u32x4 x, uint32_t i) { return __uint_as_float(x[i]); }
};
template <>
struct Packed<__bf16> {
  static constexpr uint32_t kCount = 8, kLowest = 0xFF80FF80u;
  static __device__ __forceinline__ float At(u32x4 x, uint32_t i) {
    return __uint_as_float(i % 2 ? x[i / 2] & 0xFFFF0000u : x[i / 2] << 16);
  }
};
template <>
struct Packed<_Float16> {
  static constexpr uint32_t kCount = 8, kLowest = 0xFC00FC00u;
  static __device__ __forceinline__ float At(u32x4 x, uint32_t i) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(x[i / 2] >> (i % 2 * 16)));
  }
};

// Larger logits have larger orders, a NaN 0; of equal logits lower columns have
// larger keys.
__device__ __forceinline__ uint32_t OrderOf(float x) {
  const uint32_t bits = __float_as_uint(x + 0.f);  // -0 as 0
  return x != x ? 0u : (int32_t)bits < 0 ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ uint64_t KeyOf(float x, uint32_t column) {
  return (uint64_t)OrderOf(x) << 32 | (uint32_t)~column;
}
__device__ __forceinline__ float LogitOf(uint64_t key) {
  const uint32_t order = (uint32_t)(key >> 32);
  return __uint_as_float((int32_t)order < 0 ? order ^ 0x80000000u : ~order);
}

// (fmaxf would make sure of quiet NaNs first)
__device__ __forceinline__ float AtLeast(float x, float least) {
  float y;
  asm("v_max_f32 %0, %1, %2" : "=v"(y) : "v"(x), "v"(least));
  return y;
}

// What t may be down to in w, where its weight is 0.
constexpr float kFar = -3e38f;

struct Sums {
  float m, l, w;  // m: -inf where nothing was seen
};
__device__ __forceinline__ float Reference(float m) { return m == -__builtin_inff() ? 0.f : m; }
// w under a maximum that is `less` further up, f = 2^(c less); in this order no
// product passes fp32.
__device__ __forceinline__ float Moved(const Sums& a, float less, float f) {
  return f == 0.f ? 0.f : a.w * f + fmaxf(less, kFar) * (a.l * f);
}
__device__ __forceinline__ Sums Joined(const Sums& a, const Sums& b, float c) {
  Sums y;
  y.m = fmaxf(a.m, b.m);
  const float ref = Reference(y.m);
  // (nothing seen: l and w are 0; two +inf give NaN, as they should)
  const float da = a.m == -__builtin_inff() ? 0.f : a.m - ref;
  const float db = b.m == -__builtin_inff() ? 0.f : b.m - ref;
  const float fa = __builtin_amdgcn_exp2f(c * da), fb = __builtin_amdgcn_exp2f(c * db);
  y.l = a.l * fa + b.l * fb;
  y.w = Moved(a, da, fa) + Moved(b, db, fb);
  return y;
}
// Over the wave, in every lane: within 4, 8 and 16 lanes, then across those.
template <class Op>
__device__ __forceinline__ float OverWave(float x, Op&& op) {
#define HB_DPP(ctrl) \
  x = op(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), ctrl, 0xF, 0xF, false)))
  HB_DPP(0xB1);   // xor 1
  HB_DPP(0x4E);   // xor 2
  HB_DPP(0x141);  // the other four of eight
  HB_DPP(0x140);  // the other eight of sixteen
#undef HB_DPP
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ Sums JoinedOverWave(const Sums& s, float c) {
  Sums y;
  y.m = OverWave(s.m, [](float a, float b) { return fmaxf(a, b); });
  const float less = s.m == -__builtin_inff() ? 0.f : s.m - Reference(y.m);
  const float f = __builtin_amdgcn_exp2f(c * less);
  const auto add = [](float a, float b) { return a + b; };
  y.l = OverWave(s.l * f, add);
  y.w = OverWave(Moved(s, less, f), add);
  return y;
}

__device__ __forceinline__ uint64_t ReadLane(uint64_t x, uint32_t lane) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, (int)lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), (int)lane);
  return (uint64_t)hi << 32 | lo;
}

// The largest order of 16 upper bits that k of the lanes' reach (two a lane, or
// one), found bit by bit.
template <bool two_each>
__device__ __forceinline__ uint32_t Reached(uint32_t first, uint32_t second, uint32_t k) {
  uint32_t least = 0;
#pragma unroll
  for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit /= 2) {
    const uint64_t one = __builtin_amdgcn_ballot_w64(first >= (least | bit));
    const uint64_t two =
        two_each ? __builtin_amdgcn_ballot_w64(second >= (least | bit)) : 0;
    if ((uint32_t)(__builtin_popcountll(one) + __builtin_popcountll(two)) >= k) least |= bit;
  }
  return least;
}

// A sorted list and up to 64 keys that it does not have, one a lane, 0 for none
// (`some` lanes have one), as a list of the largest 64: every key's place is the
// number of keys above it.  Through `lds`, 64 keys of the wave's own.
__device__ __forceinline__ uint64_t With(uint64_t list, uint32_t listed, uint64_t key,
                                         uint64_t some, volatile uint64_t* lds) {
  const uint32_t lane = threadIdx.x % 64;
  uint32_t key_place = 0, list_place = lane;
  for (uint64_t left = some; left != 0; left &= left - 1) {
    const uint64_t one = ReadLane(key, (uint32_t)__builtin_ctzll(left));
    key_place += one > key;
    list_place += one > list;
  }
  for (uint32_t i = 0; i < listed; ++i) key_place += ReadLane(list, i) > key;
  lds[lane] = 0;
  WaveFence();
  if (list != 0 && list_place < 64) lds[list_place] = list;
  if (key != 0 && key_place < 64) lds[key_place] = key;
  WaveFence();
  const uint64_t y = lds[lane];
  WaveFence();
  return y;
}

// Keys of `other` (k of them, falling) that are above `key`.
__device__ __forceinline__ uint32_t Above(const uint64_t* other, uint32_t k, uint64_t key) {
  uint32_t n = 0;
#pragma unroll
  for (uint32_t step = 64; step > 0; step /= 2)
    if (n + step <= k && other[n + step - 1] > key) n += step;
  return n;
}
// `count` lists of k falling keys become one, in pairs: a key's place is its own
// in its list and the number of keys above it in the other.  Lists of fewer keys
// end in zeros.
__device__ __forceinline__ const uint64_t* Merged(uint64_t* lists, uint64_t* other, uint32_t count,
                                                  uint32_t k) {
  while (count > 1) {
    const uint32_t left = (count + 1) / 2;
    for (uint32_t i = threadIdx.x; i < left * k; i += kThreads) other[i] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < count * k; i += kThreads) {
      const uint32_t list = i / k, pair = list ^ 1;
      const uint64_t key = lists[i];
      uint32_t place = i % k;
      if (pair < count) place += Above(lists + pair * k, k, key);
      if (place < k && key != 0) other[list / 2 * k + place] = key;
    }
    __syncthreads();
    uint64_t* const t = lists;
    lists = other;
    other = t;
    count = left;
  }
  return lists;
}

// A row's given token, -1 for none, and its logit: asked for before the row is
// read, as two loads that wait for one another.
template <class T>
struct Given {
  int32_t token = -1;
  float logit = 0.f;
  __device__ __forceinline__ Given(const LogprobsArgs& a, uint32_t row) {
    if (a.tokens == nullptr) return;
    token = a.tokens[row];
    if (token >= 0 && (uint32_t)token < a.vocab)
      logit = (float)static_cast<const T*>(a.logits)[row * a.stride + (uint32_t)token];
  }
};

// What goes out for a row, from its sums and its keys, one a lane of a wave.
template <class T>
__device__ __forceinline__ void Finish(const LogprobsArgs& a, uint32_t row, const Given<T>& given,
                                       Sums s, uint64_t key) {
  const T* const x = static_cast<const T*>(a.logits) + row * a.stride;
  const float inf = __builtin_inff(), ref = Reference(s.m);
  const float log = s.l == 0.f ? 0.f : __builtin_amdgcn_logf(s.l) * kLn2;
  const auto logprob = [&](float logit) {
    if (s.l == 0.f) return -inf;
    const float t = logit - ref;
    // (by halves where the difference passes fp32 and the scale may bring it back;
    // such a term is 0 in the sums)
    return t == -inf ? fmaf(0.5f * logit - 0.5f * ref, 2.f * a.scale, -log)
                     : fmaf(t, a.scale, -log);
  };
  const uint32_t lane = threadIdx.x % 64;
  if (lane == 0) {
    if (a.tokens != nullptr)
      a.logprobs[row] = given.token < 0                     ? 0.f
                        : (uint32_t)given.token >= a.vocab ? __builtin_nanf("")
                                                            : logprob(given.logit);
    if (a.entropy != nullptr) a.entropy[row] = s.l == 0.f ? 0.f : fmaf(-a.scale, s.w / s.l, log);
  }
  if (a.top == 0) return;
  const uint64_t at = (uint64_t)row * a.top;
  if (lane < a.top && key != 0) {
    a.top_ids[at + lane] = (int32_t)~(uint32_t)key;
    a.top_logprobs[at + lane] = logprob(LogitOf(key));
  }
  // fewer numbers than were asked for: the first NaNs
  uint32_t found = (uint32_t)__builtin_popcountll(
      __builtin_amdgcn_ballot_w64(lane < a.top && key != 0));
  for (uint64_t base = 0; found < a.top && base < a.vocab; base += 64) {
    const bool odd = base + lane < a.vocab && (float)x[base + lane] != (float)x[base + lane];
    const uint64_t all = __builtin_amdgcn_ballot_w64(odd);
    const uint32_t place = found + (uint32_t)__builtin_popcountll(all & ((1ull << lane) - 1));
    if (odd && place < a.top) {
      a.top_ids[at + place] = (int32_t)(base + lane);
      a.top_logprobs[at + place] = __builtin_nanf("");
    }
    found += (uint32_t)__builtin_popcountll(all);
  }
}

// A part of a row in the workspace.
__device__ __forceinline__ uint64_t* PartAt(const LogprobsArgs& a, uint64_t unit) {
  return reinterpret_cast<uint64_t*>(a.ws) + unit * (a.top + 2);
}

// kW waves take a part of a row, batches of it in turn, the next one's loads
// under way while a batch is summed up.
template <class T, uint32_t kW>
__global__ __launch_bounds__(kThreads, 8) void LogprobsKernel(const LogprobsArgs a) {
  typedef Packed<T> P;
  union Lds {
    uint16_t maxima[kWaves][kStretches][64];  // orders' upper halves
    uint64_t lists[2][kWaves * 64];
  };
  __shared__ Lds lds;
  __shared__ uint16_t again[kWaves][128];  // stretches to be read again
  __shared__ uint64_t keys[kWaves][128];   // and keys that wait for the list
  __shared__ Sums sums[kWaves];
  __shared__ uint32_t bound, odd;
  const uint32_t lane = threadIdx.x % 64;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), mine = wave % kW;
  const uint32_t unit = blockIdx.x * (kWaves / kW) + wave / kW;
  if (kW == 1 && unit >= a.rows * a.parts) return;
  const uint32_t row = unit / a.parts, part = unit % a.parts;
  const T* const x = static_cast<const T*>(a.logits) + row * a.stride;
  // 16-byte pieces from the one that the row begins in
  const uint32_t skew = (uint32_t)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
  const uint64_t last = skew + (uint64_t)a.vocab;
  const uint32_t pieces = (uint32_t)((last + P::kCount - 1) / P::kCount);
  const uint32_t each = (pieces + a.parts - 1) / a.parts;
  const uint32_t begin = min(pieces, part * each), end = min(pieces, begin + each);
  if (kW > 1) {
    if (threadIdx.x == 0) bound = odd = 0;
    __syncthreads();
  }
  auto piece_of = [&](uint32_t batch, uint32_t u, uint32_t of) {
    return (uint64_t)begin + ((uint64_t)batch * kLoads + u) * 64 + of;
  };
  auto load = [&](uint64_t i) {
    u32x4 y = {P::kLowest, P::kLowest, P::kLowest, P::kLowest};
    if (i >= end) return y;
    const uint64_t at = i * P::kCount;  // of its first value, from `skew` before the row
    if (at >= skew && at + P::kCount <= last) return *reinterpret_cast<const u32x4*>(x + (at - skew));
#pragma unroll
    for (uint32_t j = 0; j < P::kCount; ++j) {  // the row's ends
      if (at + j < skew || at + j >= last) continue;
      const T one = x[at + j - skew];
      if constexpr (sizeof(T) == 4) {
        y[j] = __builtin_bit_cast(uint32_t, one);
      } else {
        const uint32_t bits = __builtin_bit_cast(uint16_t, one);
        y[j / 2] = j % 2 ? (y[j / 2] & 0xFFFFu) | bits << 16 : (y[j / 2] & 0xFFFF0000u) | bits;
      }
    }
    return y;
  };
  const float c = a.scale * kLog2e;
  const uint32_t batches = (end - begin + kLoads * 64 - 1) / (kLoads * 64);
  // batches of a stretch
  const uint32_t run = (((batches + kW - 1) / kW) + kStretches - 1) / kStretches;
  Sums s{-__builtin_inff(), 0.f, 0.f};
  float high = -__builtin_inff();
  uint32_t stretch = 0, in = 0;
  const Given<T> given(a, row);
  u32x4 now[kLoads], next[kLoads];
#pragma unroll
  for (uint32_t u = 0; u < kLoads; ++u) now[u] = load(piece_of(mine, u, lane));
#pragma unroll 1
  for (uint32_t batch = mine; batch < batches; batch += kW) {
    if (batch + kW < batches) {
#pragma unroll
      for (uint32_t u = 0; u < kLoads; ++u) next[u] = load(piece_of(batch + kW, u, lane));
    }
    float top = -__builtin_inff();
#pragma unroll
    for (uint32_t u = 0; u < kLoads; ++u)
#pragma unroll
      for (uint32_t j = 0; j < P::kCount; j += 2)
        top = Max3(top, P::At(now[u], j), P::At(now[u], j + 1));
    if (top > s.m) {
      if (s.m != -__builtin_inff()) {
        const float less = s.m - top, f = __builtin_amdgcn_exp2f(c * less);
        s.w = Moved(s, less, f);
        s.l *= f;
      }
      s.m = top;
    }
    const float ref = Reference(s.m);
#pragma unroll
    for (uint32_t u = 0; u < kLoads; ++u)
#pragma unroll
      for (uint32_t j = 0; j < P::kCount; ++j) {
        const float t = P::At(now[u], j) - ref, p = __builtin_amdgcn_exp2f(c * t);
        s.l += p;
        s.w = fmaf(p, AtLeast(t, kFar), s.w);
      }
    if (a.top > 0) {
      high = fmaxf(high, top);
      if (++in == run || batch + kW >= batches) {
        lds.maxima[wave][stretch][lane] = (uint16_t)(OrderOf(high) >> 16);
        high = -__builtin_inff();
        in = 0;
        ++stretch;
      }
    }
#pragma unroll
    for (uint32_t u = 0; u < kLoads; ++u) now[u] = next[u];
  }
  uint64_t list = 0;
  if (a.top > 0) {
    uint32_t least;
    if (a.top > kOfOne) {
      // the lane's two largest maxima (here, as registers in the loop above are dear)
      uint32_t first = 0, second = 0;
      for (uint32_t i = 0; i < stretch; ++i) {
        const uint32_t one = lds.maxima[wave][i][lane];
        second = max(second, min(first, one));
        first = max(first, one);
      }
      least = Reached<true>(first << 16, second << 16, a.top);
    } else {
      least = Reached<false>(OrderOf(s.m), 0, a.top);
    }
    // a signalling NaN may have hidden what came before it from a maximum
    bool all = __builtin_amdgcn_ballot_w64(s.l != s.l) != 0;
    if (kW > 1) {
      if (lane == 0) {
        atomicMax(&bound, least);
        if (all) atomicOr(&odd, 1u);
      }
      __syncthreads();
      least = bound;
      all = odd != 0;
    } else {
      WaveFence();
    }
    uint64_t last_key = 0;
    uint32_t listed = 0, waiting = 0;
    auto take_keys = [&]() {  // the keys that wait, up to 64
      const uint32_t take = min(waiting, 64u);
      WaveFence();
      uint64_t key = lane < take ? keys[wave][lane] : 0;
      const uint64_t rest = 64 + lane < waiting ? keys[wave][64 + lane] : 0;
      WaveFence();
      if (64 + lane < waiting) keys[wave][lane] = rest;
      waiting -= take;
      if (key <= last_key) key = 0;
      const uint64_t some = __builtin_amdgcn_ballot_w64(key != 0);
      if (some == 0) return;
      list = With(list, listed, key, some, &keys[wave][64]);
      listed = min(listed + (uint32_t)__builtin_popcountll(some), a.top);
      last_key = ReadLane(list, a.top - 1);
    };
    uint32_t found = 0, next_stretch = 0;
    const uint64_t below = (1ull << lane) - 1;
    while (true) {
      while (found < 64 && next_stretch < stretch) {
        const bool flag = all || lds.maxima[wave][next_stretch][lane] >= least >> 16;
        const uint64_t some = __builtin_amdgcn_ballot_w64(flag);
        if (flag)
          again[wave][found + (uint32_t)__builtin_popcountll(some & below)] =
              (uint16_t)(next_stretch * 64 + lane);
        found += (uint32_t)__builtin_popcountll(some);
        ++next_stretch;
      }
      if (found == 0) break;
      WaveFence();
      const uint32_t take = min(found, 64u);
      const uint32_t one = lane < take ? again[wave][lane] : 0;
      const uint32_t rest = 64 + lane < found ? again[wave][64 + lane] : 0;
      WaveFence();
      if (64 + lane < found) again[wave][lane] = (uint16_t)rest;
      found -= take;
#pragma unroll 1
      for (uint32_t g = 0; g < run; ++g) {
        const uint32_t batch = mine + (one / 64 * run + g) * kW;
        // (both loads at once cost registers that eight waves a SIMD do not have:
        // 217 us for 117 over 4,096 rows of 65,537)
#pragma unroll 1
        for (uint32_t u = 0; u < kLoads; ++u) {
          const uint64_t i = piece_of(batch, u, one % 64);
          const bool there = lane < take && batch < batches && i < end;
          const u32x4 y = load(there ? i : end);
#pragma unroll
          for (uint32_t j = 0; j < P::kCount; ++j) {
            const uint64_t at = i * P::kCount + j - skew;
            uint64_t key = there && at < a.vocab ? KeyOf(P::At(y, j), (uint32_t)at) : 0;
            if ((uint32_t)(key >> 32) < max(least, 1u)) key = 0;
            if (key <= last_key) key = 0;
            const uint64_t some = __builtin_amdgcn_ballot_w64(key != 0);
            if (some == 0) continue;
            if (key != 0)
              keys[wave][waiting + (uint32_t)__builtin_popcountll(some & below)] = key;
            waiting += (uint32_t)__builtin_popcountll(some);
            if (waiting >= 64) take_keys();
          }
        }
      }
    }
    if (waiting > 0) take_keys();
  }
  s = JoinedOverWave(s, c);
  if (kW > 1) {
    if (lane == 0) sums[wave] = s;
    __syncthreads();  // the maxima have been read
    if (lane < a.top) lds.lists[0][wave * a.top + lane] = list;
    __syncthreads();
    s = Joined(Joined(sums[0], sums[1], c), Joined(sums[2], sums[3], c), c);
    const uint64_t* const best = Merged(lds.lists[0], lds.lists[1], kWaves, a.top);
    if (wave > 0) return;
    list = lane < a.top ? best[lane] : 0;
  }
  if (a.parts == 1) {
    Finish<T>(a, row, given, s, list);
    return;
  }
  uint64_t* const to = PartAt(a, unit);
  if (lane < a.top) to[lane] = list;
  if (lane == 0) {
    to[a.top] = (uint64_t)__float_as_uint(s.l) << 32 | __float_as_uint(s.m);
    to[a.top + 1] = __float_as_uint(s.w);
  }
}

// A row's parts.  A launch of its own: with the last of a row's workgroups joining
// them, which takes fences across the chip's L2s, 8 rows of 50,001 took 15.6 us for
// 13.7, 64 of 128,000 40 for 19.
template <class T>
__global__ __launch_bounds__(kThreads) void JoinKernel(const LogprobsArgs a) {
  __shared__ uint64_t lists[2][kJoined];
  __shared__ Sums sums;
  const uint32_t row = blockIdx.x, tid = threadIdx.x;
  const uint64_t* const from = PartAt(a, (uint64_t)row * a.parts);
  const Given<T> given(a, row);
  for (uint32_t i = tid; i < a.parts * a.top; i += kThreads)
    lists[0][i] = from[i / a.top * (a.top + 2) + i % a.top];
  if (tid < 64) {
    Sums s{-__builtin_inff(), 0.f, 0.f};
    if (tid < a.parts) {
      const uint64_t* const x = from + tid * (a.top + 2) + a.top;
      s = Sums{__uint_as_float((uint32_t)x[0]), __uint_as_float((uint32_t)(x[0] >> 32)),
               __uint_as_float((uint32_t)x[1])};
    }
    s = JoinedOverWave(s, a.scale * kLog2e);
    if (tid == 0) sums = s;
  }
  __syncthreads();
  const uint64_t* const keys = Merged(lists[0], lists[1], a.parts, a.top);
  if (tid < 64) Finish<T>(a, row, given, sums, tid < a.top ? keys[tid] : 0);
}

template <class T>
hipError_t LaunchType(LogprobsArgs& a, Workspace& ws, hipStream_t stream) {
  // A row a wave where there are rows enough that its end is not what waits:
  // 4,096 rows of 1,000 bf16 logits 9 us (20 with four waves a row), 2,000 of
  // 8,192 14 (19), 4,500 of 16,000 38 (47), 4,096 of 65,537 115 (126), but 1,024
  // of 32,000 35 (23), 2,048 of 65,537 75 (59), and 4,096 of 65,537 in fp32 208
  // (199).  Between: 3,200 of 65,537 bf16 109 (101), 3,600 111 (114).  Over 82 such
  // calls, 1,024 to 8,192 rows of 2,000 to 128,000, the choice is within 10% of the
  // other, and mostly the better.
  const uint64_t cus = (uint64_t)DeviceCus();
  const bool alone = a.rows >= 4 * cus && (a.vocab * sizeof(T) <= 16384 ||
                                           (a.rows >= 16 * cus && sizeof(T) == 2));
  // four workgroups a CU, of two batches a wave at least (8 x 50,001 fp32, 20
  // each: 14.3 us; 15.2 with one, 14.6 with four)
  const uint64_t per = 2 * kLoads * 64 * kWaves * Packed<T>::kCount;
  const uint64_t want = (4 * cus + a.rows - 1) / a.rows;
  static_assert(kJoined / 64 >= 8, "parts of the most likeliest tokens");
  const uint64_t few = kJoined / std::max(1u, a.top);
  a.parts = (uint32_t)std::min<uint64_t>({want, (a.vocab + per - 1) / per, kMostParts, few});
  if (a.parts > 1) {
    const hipError_t err =
        GrowWorkspace(ws, (size_t)a.rows * a.parts * (a.top + 2) * sizeof(uint64_t), stream);
    if (err != hipSuccess) return err;
    a.ws = ws.ptr + kSplitCounters;
  }
  if (alone)
    LogprobsKernel<T, 1><<<(a.rows * a.parts + kWaves - 1) / kWaves, kThreads, 0, stream>>>(a);
  else
    LogprobsKernel<T, kWaves><<<a.rows * a.parts, kThreads, 0, stream>>>(a);
  if (a.parts > 1) JoinKernel<T><<<a.rows, kThreads, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t LaunchLogprobs(const LogprobsArgs& in, Workspace& ws, hipStream_t stream) {
  LogprobsArgs a = in;
  switch (a.type) {
    case HB_TYPE_F32: return LaunchType<float>(a, ws, stream);
    case HB_TYPE_BF16: return LaunchType<__bf16>(a, ws, stream);
    default: return LaunchType<_Float16>(a, ws, stream);
  }
}

}  // namespace hb
