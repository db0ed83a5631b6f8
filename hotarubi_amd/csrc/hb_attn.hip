// Attention over the paged MXFP4 cache.
//
// Rows of one request and K/V head (new tokens x the query heads that share
// it) in tiles of 16, keys in records of 32.  With A = K and B = Q^T the
// matrix cores give S^T: lane (g, n) = 16 g + n holds the scores of row n
// for tokens 4g .. 4g+3 and 16+4g .. 16+4g+3, which is where the B operand of
// O^T = V^T P^T wants them, so P goes from the softmax to the next product in
// the same registers, with no trip through LDS; the record's layout gives the
// lane its K and V codes for both products as they lie.
#include <algorithm>
#include <cmath>

#include "hb_internal.h"
#include "hb_kv.h"
#include "hb_ring.h"

namespace hb {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <uint32_t parts>
struct TypeOf;  // the tensors' type by the bf16 parts that hold its values exactly
template <>
struct TypeOf<1> {
  typedef __bf16 type;
  typedef bf16x4 four;
};
template <>
struct TypeOf<2> {
  typedef _Float16 type;
  typedef f16x4 four;
};
template <>
struct TypeOf<3> {
  typedef float type;
  typedef f32x4 four;
};

constexpr uint32_t kWaves = 4, kThreads = 64 * kWaves;
constexpr float kLog2e = 1.44269504088896340736f;
// A row's maximum moves once a score passes it by this much (in powers of
// two): between moves P is at most 2^8, and nothing is rescaled.
constexpr float kSlack = 8.f, kLift = 7.f;

// ---------------------------------------------------------------- records --

template <uint32_t D>
struct Record {
  u32x4 k[D / 64], v[D / 64];
  uint32_t ks[D == 256 ? 2 : 1];  // scale bytes of tokens n, 16 + n of the lane's block(s)
  uint32_t vs[2];                 // scale bytes of the lane's 8 tokens
};

// Records go from memory into LDS by direct loads, kDepth of them under way or
// waiting per wave (a ring of its own, no barrier): what a CU needs in flight
// to draw its share of HBM is 40 KB or more, which registers do not hold.
template <uint32_t D>
struct Ring {
  static constexpr uint32_t kSlot = D == 64 ? 2304 : 34 * D;  // whole loads
  static constexpr uint32_t kOps = D / 32 + (D == 256 ? 2 : 1);
  static constexpr uint32_t kDepth = D == 64 ? 7 : D == 128 ? 4 : 2;
};
template <uint32_t D>
__device__ __forceinline__ void FetchRecord(const uint8_t* base, uint32_t lds) {
  const uint32_t lane = threadIdx.x % 64;
#pragma unroll
  for (uint32_t c = 0; c < D / 32; ++c) ring::Dma16(base + c * 1024, lane * 16, lds + c * 1024);
  // 2 D bytes of scales; the upper lanes repeat the lower ones' where that is
  // half a load
  ring::Dma4(base + 32 * D, (D == 64 ? lane % 32 : lane) * 4, lds + 32 * D);
  if (D == 256) ring::Dma4(base + 32 * D + 256, lane * 4, lds + 32 * D + 256);
}
template <uint32_t D>
__device__ __forceinline__ void ReadKeys(const uint8_t* slot, Record<D>& r) {
  const uint32_t lane = threadIdx.x % 64, g = lane / 16, n = lane % 16;
#pragma unroll
  for (uint32_t c = 0; c < D / 64; ++c)
    r.k[c] = *reinterpret_cast<const u32x4*>(slot + c * 1024 + lane * 16);
  const uint32_t block = D == 256 ? 2 * g : g * D / 128;
  r.ks[0] = *reinterpret_cast<const uint16_t*>(slot + 32 * D + block * 32 + n * 2);
  if (D == 256)
    r.ks[D == 256] = *reinterpret_cast<const uint16_t*>(slot + 32 * D + block * 32 + 32 + n * 2);
}
template <uint32_t D>
__device__ __forceinline__ void ReadValues(const uint8_t* slot, Record<D>& r) {
  const uint32_t lane = threadIdx.x % 64, g = lane / 16, n = lane % 16;
#pragma unroll
  for (uint32_t c = 0; c < D / 64; ++c)
    r.v[c] = *reinterpret_cast<const u32x4*>(slot + 16 * D + c * 1024 + lane * 16);
  const uint2 vs = *reinterpret_cast<const uint2*>(slot + 33 * D + n * D / 512 * 32 + g * 8);
  r.vs[0] = vs.x;
  r.vs[1] = vs.y;
}

__device__ __forceinline__ float ScaleOf(uint32_t bytes, uint32_t i) {
  return __uint_as_float(((bytes >> (8 * i)) & 255u) << 23);
}

// Two codes, byte `sel` of a word, as bf16 values (exact: E2M1 on any E8M0).
template <int sel>
__device__ __forceinline__ uint32_t Two(uint32_t word, float scale) {
  return __builtin_bit_cast(uint32_t,
                            __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, sel));
}
// Operand of K: tokens 16 tile + n, the lane's columns 8 s .. 8 s + 7.
template <uint32_t D>
__device__ __forceinline__ bf16x8 KeyOperand(const Record<D>& r, uint32_t tile, uint32_t s) {
  const uint32_t word = tile * (D / 32) + s;
  const uint32_t w = r.k[word / 4][word % 4];
  const float scale = ScaleOf(r.ks[D == 256 ? s / 4 : 0], tile);
  u32x4 x;
  x[0] = Two<0>(w, scale);
  x[1] = Two<1>(w, scale);
  x[2] = Two<2>(w, scale);
  x[3] = Two<3>(w, scale);
  return __builtin_bit_cast(bf16x8, x);
}

// P V in f16 for the 16-bit types: P's error is then below the output's
// rounding (2^-12 of each weight against bf16's 2^-9), and V is exact in f16
// wherever its scale bytes lie in [104, 140] (0.5 x 2^-23 .. 6 x 2^13).  Other
// records take V in bf16 and each f16 weight as two bf16 parts.  fp32 takes three bf16 parts of P.
template <bool half>
struct Value;
template <>
struct Value<true> {
  typedef f16x8 type;
};
template <>
struct Value<false> {
  typedef bf16x8 type;
};
// Nonzero where one of the 4 bytes lies outside [104, 140].
__device__ __forceinline__ uint32_t OutsideHalf(uint32_t x) {
  const uint32_t low = x & 0x7F7F7F7Fu;
  return (((low + 0x73737373u) & x) | ~((low + 0x18181818u) | x)) & 0x80808080u;
}

template <int sel, bool half>
__device__ __forceinline__ uint32_t TwoAs(uint32_t word, float scale) {
  if constexpr (half)
    return __builtin_bit_cast(uint32_t,
                              __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, sel));
  else
    return Two<sel>(word, scale);
}
template <bool half>
__device__ __forceinline__ uint32_t TwoOf(uint32_t word, float scale, uint32_t sel) {
  switch (sel) {  // the instruction's byte is an immediate: folded where sel is known
    case 0: return TwoAs<0, half>(word, scale);
    case 1: return TwoAs<1, half>(word, scale);
    case 2: return TwoAs<2, half>(word, scale);
    default: return TwoAs<3, half>(word, scale);
  }
}

// Operands of V^T for the lane's columns 2 i and 2 i + 1 (rows c of column
// tiles 2 i and 2 i + 1) over the record's 32 tokens.  A byte holds two columns
// of one token, so two conversions meet in two byte permutes.
template <uint32_t D, bool half>
__device__ __forceinline__ void ValueOperands(const Record<D>& r, uint32_t i,
                                              typename Value<half>::type* even,
                                              typename Value<half>::type* odd) {
  typedef typename Value<half>::type V;
  uint32_t x[8];
#pragma unroll
  for (uint32_t j = 0; j < 8; ++j) {
    const uint32_t byte = j * (D / 32) + i;
    x[j] = TwoOf<half>(r.v[byte / 16][byte / 4 % 4], ScaleOf(r.vs[j / 4], j % 4), byte % 4);
  }
  u32x4 lo, hi;
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    lo[j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x05040100u);
    hi[j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x07060302u);
  }
  *even = __builtin_bit_cast(V, lo);
  *odd = __builtin_bit_cast(V, hi);
}
__device__ __forceinline__ f32x4 Product(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 Product(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// fp32 values as bf16 parts: one part rounds to nearest; two or three cut 8
// bits each, so three are exact and two leave at most 2^-16 of the value.
template <uint32_t parts>
__device__ __forceinline__ void ToParts(const float* x, bf16x8* out) {
  if constexpr (parts == 1) {
#pragma unroll
    for (int j = 0; j < 8; ++j) out[0][j] = (__bf16)x[j];
  } else {
    float rest[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) rest[j] = x[j];
#pragma unroll
    for (uint32_t p = 0; p < parts; ++p) {
      u32x4 w;
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        const uint32_t lo = __float_as_uint(rest[2 * j]), hi = __float_as_uint(rest[2 * j + 1]);
        w[j] = __builtin_amdgcn_perm(hi, lo, 0x07060302u);
        rest[2 * j] -= __uint_as_float(lo & 0xFFFF0000u);
        rest[2 * j + 1] -= __uint_as_float(hi & 0xFFFF0000u);
      }
      out[p] = __builtin_bit_cast(bf16x8, w);
    }
  }
}

// Over the four lanes that share a row (n, 16 + n, 32 + n, 48 + n).
__device__ __forceinline__ float RowMax(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float RowSum(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// ------------------------------------------------------------------ rows --

// What a lane's row sees: keys lo .. hi and those below pre.
struct Sight {
  int32_t lo, hi, pre;
};
__device__ __forceinline__ Sight SightOf(const KvSpan& s, uint32_t token, bool valid,
                                         uint32_t window) {
  Sight v;
  const int32_t pos = s.total - s.count + (int32_t)token;
  v.hi = valid ? min(pos, s.total - 1) : -1;
  v.lo = window > 0 && (int64_t)pos + 1 > (int64_t)window ? pos + 1 - (int32_t)window : 0;
  v.pre = valid ? s.prefix : 0;
  return v;
}

// 8 elements of a query row, zeros past the rows.
template <uint32_t parts>
__device__ __forceinline__ void LoadQuery(const AttnArgs& a, uint64_t at, bool valid, bool vec,
                                          bf16x8* out) {
  typedef typename TypeOf<parts>::type T;
  typedef typename TypeOf<parts>::four V;
  const T* x = static_cast<const T*>(a.q) + at;
  float y[8] = {};
  if (valid && vec) {
    const V lo = reinterpret_cast<const V*>(x)[0], hi = reinterpret_cast<const V*>(x)[1];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = (float)(j < 4 ? lo[j % 4] : hi[j % 4]);
  } else if (valid) {
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = (float)x[j];
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] *= a.sign;
  ToParts<parts>(y, out);
}

template <uint32_t parts>
__device__ __forceinline__ void StoreFour(const AttnArgs& a, uint64_t at, bool vec, f32x4 y) {
  typedef typename TypeOf<parts>::type T;
  typedef typename TypeOf<parts>::four V;
  T* to = static_cast<T*>(a.out) + at;
  V z;
#pragma unroll
  for (int j = 0; j < 4; ++j) z[j] = (T)y[j];
  if (vec) {
    *reinterpret_cast<V*>(to) = z;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) to[j] = z[j];
  }
}

// The state of R tiles of 16 rows on one wave.
template <uint32_t parts, uint32_t D, uint32_t R>
struct Rows {
  bf16x8 q[R][parts][D / 32];
  f32x4 o[R][D / 16];
  float m[R], l[R];
  Sight see[R];
  int32_t see_all, see_from, see_pre;  // every row sees keys see_from .. see_all, and < see_pre
};

// One record: the products of its keys ...
template <uint32_t parts, uint32_t D, uint32_t R>
__device__ __forceinline__ void Scores(const Record<D>& r, const Rows<parts, D, R>& w,
                                       f32x4 (&s)[R][2]) {
#pragma unroll
  for (uint32_t t = 0; t < R; ++t) s[t][0] = s[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (uint32_t i = 0; i < D / 32; ++i) {
#pragma unroll
    for (uint32_t tile = 0; tile < 2; ++tile) {
      const bf16x8 k = KeyOperand<D>(r, tile, i);
#pragma unroll
      for (uint32_t t = 0; t < R; ++t)
#pragma unroll
        for (uint32_t p = parts; p-- > 0;)
          s[t][tile] = Product(k, w.q[t][p][i], s[t][tile]);
    }
  }
}

// ... and the scores' running maximum and sum, and P V.
template <uint32_t parts, uint32_t D, uint32_t R>
__device__ __forceinline__ void Step(const AttnArgs& a, const KvSpan& span, Record<D>& r,
                                     int32_t key0, f32x4 (&s)[R][2], Rows<parts, D, R>& w) {
  const uint32_t g = threadIdx.x % 64 / 16;
  float c = a.scale * kLog2e;  // scores in powers of two: s c
  if (a.cap > 0.f) {           // cap tanh(s scale / cap)
#pragma unroll
    for (uint32_t t = 0; t < R; ++t)
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        float x = s[t][j / 4][j % 4];
        if constexpr (parts == 3) {
          x = a.cap * kLog2e * tanhf(x * a.scale / a.cap);
        } else {
          const float e = __builtin_amdgcn_exp2f(x * (2.f * c / a.cap));
          x = a.cap * kLog2e * fmaf(-2.f, __builtin_amdgcn_rcpf(e + 1.f), 1.f);
        }
        s[t][j / 4][j % 4] = x;
      }
    c = 1.f;
  }
  // Unusual scale bytes of V: a token whose V has a scale of NaN gives NaN
  // scores to the rows that see it and nothing to others (0 x NaN would reach
  // every row of the tile); past the request's end any byte may lie.
  constexpr bool half = parts < 3;
  bool wide = false;
  if (__builtin_amdgcn_ballot_w64((OutsideHalf(r.vs[0]) | OutsideHalf(r.vs[1])) != 0) != 0) {
    uint32_t nan = 0;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      const uint32_t byte = (r.vs[j / 4] >> (8 * (j % 4))) & 255u;
      const int32_t key = key0 + (int32_t)(j / 4 * 16 + 4 * g + j % 4);
      nan |= (uint32_t)(byte == 255u) << j;
      if (byte == 255u || key >= span.total)
        r.vs[j / 4] = (r.vs[j / 4] & ~(255u << (8 * (j % 4)))) | 127u << (8 * (j % 4));
    }
#pragma unroll
    for (uint32_t d = 1; d < 16; d *= 2) nan |= __shfl_xor(nan, d);
#pragma unroll
    for (uint32_t t = 0; t < R; ++t)
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j)
        if (nan >> j & 1) s[t][j / 4][j % 4] = __builtin_nanf("");
    wide = half && __builtin_amdgcn_ballot_w64(
                       (OutsideHalf(r.vs[0]) | OutsideHalf(r.vs[1])) != 0) != 0;
  }
  const bool full = (key0 >= w.see_from && key0 + 31 <= w.see_all) || key0 + 32 <= w.see_pre;
  if (!full) {
#pragma unroll
    for (uint32_t t = 0; t < R; ++t)
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        const int32_t key = key0 + (int32_t)(j / 4 * 16 + 4 * g + j % 4);
        const Sight& v = w.see[t];
        const bool sees = (key >= v.lo && key <= v.hi) || key < v.pre;
        s[t][j / 4][j % 4] = sees ? s[t][j / 4][j % 4] : -__builtin_inff();
      }
  }
  typename Value<half>::type pt[R][half ? 1 : parts];
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (uint32_t t = 0; t < R; ++t) {
    const f32x4 x = s[t][0], y = s[t][1];
    const float top = c * fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])),
                                fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])));
    if (__builtin_amdgcn_ballot_w64(top > w.m[t] + kSlack) != 0) {
      const float m = fmaxf(w.m[t], RowMax(top));
      // rows that have seen nothing yet stay at -inf, with o and l zero
      const float shrink = m == w.m[t] ? 1.f : __builtin_amdgcn_exp2f(w.m[t] - m);
      w.m[t] = m;
      w.l[t] *= shrink;
#pragma unroll
      for (uint32_t i = 0; i < D / 16; ++i) w.o[t][i] *= shrink;
    }
    // weights carry 2^kLift: at most 2^15, and as small as 2^-31 of the
    // maximum before f16 goes subnormal
    const float ref = (w.m[t] == -__builtin_inff() ? 0.f : w.m[t]) - kLift;
    float p[8], sum = 0.f;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      p[j] = __builtin_amdgcn_exp2f(fmaf(j < 4 ? x[j % 4] : y[j % 4], c, -ref));
      sum += p[j];
    }
    w.l[t] += sum;
    if constexpr (half) {
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const f16x2 two = __builtin_convertvector(f32x2{p[j], p[j + 1]}, f16x2);
        pt[t][0][j] = two[0];
        pt[t][0][j + 1] = two[1];
      }
    } else {
      ToParts<parts>(p, pt[t]);
    }
  }
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (half) {
    if (wide) {  // V in bf16, on the two bf16 parts of an f16 weight
#pragma unroll
      for (uint32_t t = 0; t < R; ++t) {
        float p[8];
        bf16x8 part[2];
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = (float)pt[t][0][j];
        ToParts<2>(p, part);
#pragma unroll
        for (uint32_t i = 0; i < D / 32; ++i) {
          bf16x8 v[2];
          ValueOperands<D, false>(r, i, &v[0], &v[1]);
#pragma unroll
          for (uint32_t h = 0; h < 2; ++h) {
            w.o[t][2 * i + h] = Product(v[h], part[1], w.o[t][2 * i + h]);
            w.o[t][2 * i + h] = Product(v[h], part[0], w.o[t][2 * i + h]);
          }
        }
      }
      return;
    }
  }
#pragma unroll
  for (uint32_t i = 0; i < D / 32; ++i) {
    typename Value<half>::type v[2];
    ValueOperands<D, half>(r, i, &v[0], &v[1]);
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
      for (uint32_t t = 0; t < R; ++t)
#pragma unroll
        for (uint32_t p = half ? 1 : parts; p-- > 0;)
          w.o[t][2 * i + h] = Product(v[h], pt[t][p], w.o[t][2 * i + h]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

constexpr uint32_t kNoRecord = 0xFFFFFFFFu;

// The record a wave's lane takes in its turn i.
__device__ __forceinline__ uint32_t PageRecord(const AttnArgs& a, const KvWalk& walk,
                                               const int32_t* row, uint32_t head, uint32_t i,
                                               uint32_t end) {
  uint64_t record;
  if (i >= end || !KvRecord(row, a.columns, KvWalkRecord(walk, i), head, a.pages, a.heads,
                            a.groups, &record))
    return kNoRecord;
  return (uint32_t)record;
}

// A partial result in the workspace: per split of a unit R rows of D sums,
// the maximum and the sum.
template <uint32_t D>
constexpr uint32_t kPartial = D + 4;

// The waves' results of a workgroup, in LDS.
template <uint32_t D, uint32_t R>
struct Merge {
  float o[kWaves][R * 16][D + 4], m[kWaves][R * 16], l[kWaves][R * 16];
};

// split: the workgroup's waves share R tiles of 16 rows and take its records
// in turn; else each wave has R tiles of its own and takes every record.
template <uint32_t parts, uint32_t D, uint32_t R, bool split>
// two workgroups a CU (their rings fill its LDS), so 256 registers a wave
__global__ __launch_bounds__(kThreads, 2) void AttnKernel(const AttnArgs a) {
  const uint32_t lane = threadIdx.x % 64, n = lane % 16, g = lane / 16;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t unit = blockIdx.x / a.splits, part = blockIdx.x % a.splits;
  const uint32_t head = unit % a.heads, rest = unit / a.heads;
  const uint32_t b = rest / a.tiles, tile = a.tiles - 1 - rest % a.tiles;
  const KvSpan span =
      KvRequest(a.cu[b], a.cu[b + 1], a.kv_lens[b], a.prefix ? a.prefix[b] : 0, a.tokens,
                a.max_new, (uint64_t)a.columns * a.groups * 32);
  const uint32_t group = a.q_heads / a.heads, rows = span.rows * group;
  const uint32_t row0 = (split ? tile : tile * kWaves + wave) * R * 16;
  if (row0 >= rows) return;
  const uint32_t last = min(row0 + R * 16, rows) - 1;
  const int32_t base = span.total - span.count;
  const int32_t pos0 = base + (int32_t)(row0 / group), pos1 = base + (int32_t)(last / group);
  const KvWalk walk = KvRecords(pos0, pos1, span.total, span.prefix, a.window);
  const uint32_t begin = part * a.split_records;
  const uint32_t end =
      part + 1 == a.splits ? walk.count : min(walk.count, begin + a.split_records);
  if (part > 0 && begin >= end) return;

  Rows<parts, D, R> w;
  const bool vec = ((a.q_token | a.q_head) % 4 == 0) &&
                   reinterpret_cast<uintptr_t>(a.q) % (4 * sizeof(typename TypeOf<parts>::type)) == 0;
#pragma unroll
  for (uint32_t t = 0; t < R; ++t) {
    const uint32_t row = row0 + t * 16 + n, token = row / group;
    const bool valid = row < rows;
    const uint64_t at = (uint64_t)(span.first + token) * a.q_token +
                        (uint64_t)(head * group + row % group) * a.q_head + g * (D / 4);
#pragma unroll
    for (uint32_t i = 0; i < D / 32; ++i) {
      bf16x8 x[parts];
      LoadQuery<parts>(a, at + 8 * i, valid, vec, x);
#pragma unroll
      for (uint32_t p = 0; p < parts; ++p) w.q[t][p][i] = x[p];
    }
    w.see[t] = SightOf(span, token, valid, a.window);
    w.m[t] = -__builtin_inff();
    w.l[t] = 0.f;
#pragma unroll
    for (uint32_t c = 0; c < D / 16; ++c) w.o[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  w.see_all = min(pos0, span.total - 1);
  w.see_from = SightOf(span, last / group, true, a.window).lo;
  w.see_pre = span.prefix;

  const int32_t* const row = a.table + (uint64_t)b * a.table_stride;
  const uint32_t step = split ? kWaves : 1, first = begin + (split ? wave : 0);
  const uint32_t count = first < end ? (end - first + step - 1) / step : 0;
  typedef Ring<D> Ring;
  constexpr uint32_t kRing = kWaves * Ring::kDepth * Ring::kSlot;
  constexpr uint32_t kMerge = split ? sizeof(Merge<D, R>) : 0;
  __shared__ __align__(16) uint8_t lds[kRing > kMerge ? kRing : kMerge];
  uint8_t* const slots = lds + wave * (Ring::kDepth * Ring::kSlot);
  const uint32_t slots_at =
      (uint32_t) reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)slots);
  // block table entries of 64 records at a time, one a lane; the ring reaches
  // into the next 64
  auto pages = [&](uint32_t i) {
    return PageRecord(a, walk, row, head, first + (i + lane) * step, end);
  };
  uint32_t now = pages(0), after = count > 64 ? pages(64) : kNoRecord;
  uint32_t read_at[Ring::kDepth];
  auto fetch = [&](uint32_t i, uint32_t base, uint32_t slot) {  // base <= i < base + 128
    const uint32_t from = (uint32_t)__builtin_amdgcn_readlane(
        (int)(i - base < 64 ? now : after), (int)((i - base) % 64));
    read_at[slot] = from;
    FetchRecord<D>(a.cache + (from == kNoRecord ? 0 : (uint64_t)from * KvRecordBytes(D)),
                   slots_at + slot * Ring::kSlot);
  };
  asm volatile("" ::: "memory");
#pragma unroll
  for (uint32_t u = 0; u < Ring::kDepth; ++u)
    if (u < count) fetch(u, 0, u);
  for (uint32_t i0 = 0, base = 0; i0 < count; i0 += Ring::kDepth) {
#pragma unroll
    for (uint32_t u = 0; u < Ring::kDepth; ++u) {
      const uint32_t i = i0 + u;
      if (i >= count) break;
      if (i + Ring::kDepth <= count) ring::WaitVm<(Ring::kDepth - 1) * Ring::kOps>();
      else ring::WaitVm<0>();
      asm volatile("" ::: "memory");
      const bool present = read_at[u] != kNoRecord;
      Record<D> r;
      f32x4 s[R][2];
      ReadKeys<D>(slots + u * Ring::kSlot, r);
      ReadValues<D>(slots + u * Ring::kSlot, r);
      ring::WaitLds();  // the slot has been read
      asm volatile("" ::: "memory");
      if (i + Ring::kDepth < count) {
        if (i + Ring::kDepth - base >= 128) {
          base += 64;
          now = after;
          after = pages(base + 64);
        }
        fetch(i + Ring::kDepth, base, u);
      }
      if (present) {
        Scores<parts, D, R>(r, w, s);
        const int32_t key0 = (int32_t)(32 * KvWalkRecord(walk, first + i * step));
        Step<parts, D, R>(a, span, r, key0, s, w);
      }
    }
  }
#pragma unroll
  for (uint32_t t = 0; t < R; ++t) w.l[t] = RowSum(w.l[t]);

  const bool ovec =
      ((a.out_token | a.out_head) % 4 == 0) &&
      reinterpret_cast<uintptr_t>(a.out) % (4 * sizeof(typename TypeOf<parts>::type)) == 0;
  if constexpr (!split) {
#pragma unroll
    for (uint32_t t = 0; t < R; ++t) {
      const uint32_t r = row0 + t * 16 + n;
      if (r >= rows) continue;
      const float inv = w.l[t] == 0.f ? 0.f : 1.f / w.l[t];
      const uint64_t at = (uint64_t)(span.first + r / group) * a.out_token +
                          (uint64_t)(head * group + r % group) * a.out_head + g * (D / 4);
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
        for (uint32_t c = 0; c < D / 16; c += 4) {
          const f32x4 y = {w.o[t][c][i], w.o[t][c + 1][i], w.o[t][c + 2][i], w.o[t][c + 3][i]};
          StoreFour<parts>(a, at + i * (D / 16) + c, ovec, y * inv);
        }
    }
  } else {
    // the waves' sums meet in LDS, in the waves' order
    Merge<D, R>& sum = *reinterpret_cast<Merge<D, R>*>(lds);
    auto& so = sum.o;
    auto& sm = sum.m;
    auto& sl = sum.l;
    __syncthreads();  // every ring has been read
#pragma unroll
    for (uint32_t t = 0; t < R; ++t) {
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
        for (uint32_t c = 0; c < D / 16; c += 4)
          *reinterpret_cast<f32x4*>(&so[wave][t * 16 + n][(4 * g + i) * (D / 16) + c]) =
              f32x4{w.o[t][c][i], w.o[t][c + 1][i], w.o[t][c + 2][i], w.o[t][c + 3][i]};
      if (g == 0) {
        sm[wave][t * 16 + n] = w.m[t];
        sl[wave][t * 16 + n] = w.l[t];
      }
    }
    __syncthreads();
    const uint32_t active =
        a.splits == 1 ? 1u
                      : min(a.splits, max(1u, (walk.count + a.split_records - 1) / a.split_records));
    const uint32_t stored = min(R * 16, a.max_new * group);  // rows a partial has
    for (uint32_t i = threadIdx.x; i < R * 16 * (D / 4); i += kThreads) {
      const uint32_t r = i / (D / 4), c = i % (D / 4) * 4;
      if (row0 + r >= rows) continue;
      float m = sm[0][r];
#pragma unroll
      for (uint32_t k = 1; k < kWaves; ++k) m = fmaxf(m, sm[k][r]);
      const float ref = m == -__builtin_inff() ? 0.f : m;
      float l = 0.f;
      f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (uint32_t k = 0; k < kWaves; ++k) {
        const float f = sm[k][r] == m ? (m == -__builtin_inff() ? 0.f : 1.f)
                                      : __builtin_amdgcn_exp2f(sm[k][r] - ref);
        l += sl[k][r] * f;
        y += *reinterpret_cast<const f32x4*>(&so[k][r][c]) * f;
      }
      if (active == 1) {
        const uint64_t at = (uint64_t)(span.first + (row0 + r) / group) * a.out_token +
                            (uint64_t)(head * group + (row0 + r) % group) * a.out_head + c;
        StoreFour<parts>(a, at, ovec, y * (l == 0.f ? 0.f : 1.f / l));
      } else {
        const uint64_t place = ((uint64_t)b * a.heads + head) * a.tiles + tile;
        float* to = a.ws + ((place * a.splits + part) * stored + r) * kPartial<D>;
        *reinterpret_cast<f32x4*>(to + c) = y;
        if (c == 0) {
          to[D] = m;
          to[D + 1] = l;
        }
      }
    }
  }
}

// The splits of a row in their order: lane groups take every kGroups-th, then
// meet in LDS.
template <uint32_t parts, uint32_t D, uint32_t R>
__global__ __launch_bounds__(kThreads) void JoinKernel(const AttnArgs a) {
  constexpr uint32_t kLanes = D / 4, kGroups = kThreads / kLanes;
  __shared__ float so[kGroups][D], sm[kGroups], sl[kGroups];
  const uint32_t group = a.q_heads / a.heads, stored = min(R * 16, a.max_new * group);
  const uint32_t place = blockIdx.x / stored, r = blockIdx.x % stored;
  const uint32_t tile = place % a.tiles, head = place / a.tiles % a.heads,
                 b = place / a.tiles / a.heads;
  const KvSpan span =
      KvRequest(a.cu[b], a.cu[b + 1], a.kv_lens[b], a.prefix ? a.prefix[b] : 0, a.tokens,
                a.max_new, (uint64_t)a.columns * a.groups * 32);
  const uint32_t rows = span.rows * group, row0 = tile * R * 16;
  if (row0 + r >= rows) return;
  const uint32_t last = min(row0 + R * 16, rows) - 1;
  const int32_t base = span.total - span.count;
  const KvWalk walk = KvRecords(base + (int32_t)(row0 / group), base + (int32_t)(last / group),
                                span.total, span.prefix, a.window);
  const uint32_t active =
      min(a.splits, max(1u, (walk.count + a.split_records - 1) / a.split_records));
  if (active == 1) return;
  const uint32_t lane = threadIdx.x % kLanes, part = threadIdx.x / kLanes;
  const float* from = a.ws + ((uint64_t)place * a.splits * stored + r) * kPartial<D>;
  float m = -__builtin_inff(), l = 0.f;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  for (uint32_t s = part; s < active; s += kGroups) {
    const float* x = from + (uint64_t)s * stored * kPartial<D>;
    const float mx = x[D], lx = x[D + 1];
    const f32x4 yx = *reinterpret_cast<const f32x4*>(x + 4 * lane);
    const float top = fmaxf(m, mx);
    const float f = m == top ? 1.f : __builtin_amdgcn_exp2f(m - top);
    const float fx = mx == top ? 1.f : __builtin_amdgcn_exp2f(mx - top);
    y = y * f + yx * fx;
    l = l * f + lx * fx;
    m = top;
  }
  *reinterpret_cast<f32x4*>(&so[part][4 * lane]) = y;
  if (lane == 0) {
    sm[part] = m;
    sl[part] = l;
  }
  __syncthreads();
  if (part != 0) return;
  float top = sm[0];
  for (uint32_t k = 1; k < kGroups; ++k) top = fmaxf(top, sm[k]);
  l = 0.f;
  y = f32x4{0.f, 0.f, 0.f, 0.f};
  for (uint32_t k = 0; k < kGroups; ++k) {
    const float f = sm[k] == top ? 1.f : __builtin_amdgcn_exp2f(sm[k] - top);
    l += sl[k] * f;
    y += *reinterpret_cast<const f32x4*>(&so[k][4 * lane]) * f;
  }
  const bool ovec =
      ((a.out_token | a.out_head) % 4 == 0) &&
      reinterpret_cast<uintptr_t>(a.out) % (4 * sizeof(typename TypeOf<parts>::type)) == 0;
  const uint64_t at = (uint64_t)(span.first + (row0 + r) / group) * a.out_token +
                      (uint64_t)(head * group + (row0 + r) % group) * a.out_head + 4 * lane;
  StoreFour<parts>(a, at, ovec, y * (l == 0.f ? 0.f : 1.f / l));
}

template <uint32_t parts, uint32_t D, uint32_t R>
hipError_t LaunchOf(AttnArgs& a, Workspace& ws, hipStream_t stream) {
  const uint32_t group = a.q_heads / a.heads;
  const uint64_t rows = (uint64_t)a.max_new * group, tiles = (rows + R * 16 - 1) / (R * 16);
  const uint64_t pairs = (uint64_t)a.batch * a.heads, cus = (uint64_t)DeviceCus();
  if (pairs * ((tiles + kWaves - 1) / kWaves) >= 2 * cus && tiles >= kWaves) {
    a.tiles = (uint32_t)((tiles + kWaves - 1) / kWaves);
    a.splits = 1;
    a.split_records = 1;
    const uint64_t grid = pairs * a.tiles;
    if (grid > 0x7FFFFFFFu) return hipErrorInvalidValue;
    AttnKernel<parts, D, R, false><<<(uint32_t)grid, kThreads, 0, stream>>>(a);
    return hipGetLastError();
  }
  a.tiles = (uint32_t)tiles;
  const uint64_t units = pairs * tiles;
  uint64_t records = ((uint64_t)a.max_kv + 31) / 32;
  if (a.window > 0 && a.prefix == nullptr)
    records = std::min<uint64_t>(records, ((uint64_t)a.window + 16 * R + 62) / 32);
  records = std::max<uint64_t>(records, 1);
  const uint64_t want = std::max<uint64_t>(1, 2 * cus / units);
  const uint64_t most = std::max<uint64_t>(1, records / (2 * kWaves));
  uint64_t splits = std::min(want, most);
  a.split_records = (uint32_t)((records + splits - 1) / splits);
  a.splits = (uint32_t)((records + a.split_records - 1) / a.split_records);
  const uint64_t grid = units * a.splits;
  if (grid > 0x7FFFFFFFu) return hipErrorInvalidValue;
  const uint64_t stored = std::min<uint64_t>(R * 16, rows);
  if (a.splits > 1) {
    const hipError_t err = GrowWorkspace(ws, grid * stored * kPartial<D> * 4, stream);
    if (err != hipSuccess) return err;
    a.ws = ws.ptr + kSplitCounters;
  }
  AttnKernel<parts, D, R, true><<<(uint32_t)grid, kThreads, 0, stream>>>(a);
  if (a.splits > 1)
    JoinKernel<parts, D, R><<<(uint32_t)(units * stored), kThreads, 0, stream>>>(a);
  return hipGetLastError();
}

template <uint32_t parts>
hipError_t LaunchDim(AttnArgs& a, Workspace& ws, hipStream_t stream) {
  const bool two = (uint64_t)a.max_new * (a.q_heads / a.heads) > 16;
  switch (a.dim) {
    case 64: return two ? LaunchOf<parts, 64, 2>(a, ws, stream) : LaunchOf<parts, 64, 1>(a, ws, stream);
    case 128:
      return two ? LaunchOf<parts, 128, 2>(a, ws, stream) : LaunchOf<parts, 128, 1>(a, ws, stream);
    case 256: return LaunchOf<parts, 256, 1>(a, ws, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t LaunchAttention(const AttnArgs& in, Workspace& ws, hipStream_t stream) {
  AttnArgs a = in;
  // scores as |scale| (q sign): the maximum of the products is then that of
  // the scores
  a.sign = a.scale > 0.f ? 1.f : a.scale < 0.f ? -1.f : 0.f;
  a.scale = a.scale == 0.f ? 1.f : std::abs(a.scale);
  switch (a.type) {
    case HB_TYPE_BF16: return LaunchDim<1>(a, ws, stream);
    case HB_TYPE_F16: return LaunchDim<2>(a, ws, stream);
    default: return LaunchDim<3>(a, ws, stream);
  }
}

}  // namespace hb
