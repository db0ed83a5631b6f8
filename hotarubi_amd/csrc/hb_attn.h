// What the attention kernels share: records of the caches as the matrix cores'
// operands, the softmax of a tile, rows and what they see.  Fp4 and Fp8 name the
// records, MXFP4 ones and those of 8 bits.
#pragma once

#include "hb_internal.h"
#include "hb_kv.h"
#include "hb_lanes.h"
#include "hb_ring.h"

namespace hb {
namespace attn {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <uint32_t parts>
struct TypeOf;  // the tensors' type by the bf16 parts that hold its values exactly
template <>
struct TypeOf<1> {
  typedef __bf16 type;
};
template <>
struct TypeOf<2> {
  typedef _Float16 type;
};
template <>
struct TypeOf<3> {
  typedef float type;
};

constexpr float kLog2e = 1.44269504088896340736f;
// A row's maximum moves once a score passes it by this much (in powers of
// two): between moves P is at most 2^8, and nothing is rescaled.
constexpr float kSlack = 8.f, kLift = 7.f;
// What the maximum is set too high by once a wave has met values that sums of
// such weights could carry past fp32: P is below 2^-48 then, 2^31 keys' sum
// below 2^-17, and no value is too large.
constexpr float kRoom = 64.f;

// ---------------------------------------------------------------- records --

struct Fp4 {
  static constexpr bool kSinks = false;
  static constexpr double kSplitRecord = 1;  // (Divide)
  // bf16 parts of q, by the tensors' type
  static constexpr uint32_t Parts(uint32_t parts) { return parts; }
  static constexpr uint32_t Bytes(uint32_t dim) { return KvRecordBytes(dim); }
  static hipError_t Prompt(const AttnArgs& a, Workspace& ws, hipStream_t stream) {
    return LaunchPrompt(a, ws, stream);
  }
};
// E4M3 codes are exact in f16 too, and the scale, one for all keys of the record,
// may go into what their scores are multiplied by: fp16 queries take one product
// (2^33 at most).  bf16 and fp32 ones take keys with the part of their scale that
// is below 1, so that a large query meets small keys and not their codes, and the
// rest of it later, so that large keys' products do not pass fp32 before a small
// `scale` has met them.
struct Fp8 {
  static constexpr bool kSinks = true;
  // what a record costs a split's wave beside an MXFP4 one, whose figures the
  // division's are: of 180 calls (1 to 32 requests of 3 to 1,500 new tokens, the
  // types, D 64 to 256) it divides 22 otherwise than 1 does, 14 of them faster (2 x
  // 1,500 new tokens behind 1,000, 15 heads on 5 of 64, bf16 54 us for 69; 3 x 1,500,
  // 8 heads of 128, fp16 37 for 49), 5 alike, 3 slower (32 x 50 behind 150, 8 heads
  // of 128, fp16 13.0 for 11.1, fp32 17.3 for 12.8)
  static constexpr double kSplitRecord = 0.65;
  static constexpr uint32_t Parts(uint32_t parts) { return parts == 2 ? 1 : parts; }
  static constexpr uint32_t Bytes(uint32_t dim) { return Kv8RecordBytes(dim); }
  static hipError_t Prompt(const AttnArgs& a, Workspace& ws, hipStream_t stream) {
    return LaunchPrompt8(a, ws, stream);
  }
};
// What q and K enter their products as.
template <class F, uint32_t parts>
struct QueryOperand {
  typedef bf16x8 type;
};
template <>
struct QueryOperand<Fp8, 2> {
  typedef f16x8 type;
};

template <class F, uint32_t D>
struct Record;
template <uint32_t D>
struct Record<Fp4, D> {
  u32x4 k[D / 64], v[D / 64];
  uint32_t ks[D == 256 ? 2 : 1];  // scale bytes of tokens n, 16 + n of the lane's block(s)
  uint32_t vs[2];                 // scale bytes of the lane's 8 tokens
};

template <uint32_t D>
struct Record<Fp8, D> {
  u32x4 k[D / 32], v[D / 32];
  uint32_t scales;  // K's byte and V's, the same in all lanes
};

// Records go from memory into LDS by direct loads, kDepth of them under way or
// waiting per wave (a ring of its own, no barrier): what a CU needs in flight
// to draw its share of HBM is 40 KB or more, which registers do not hold.
template <class F, uint32_t D>
struct Ring;
template <uint32_t D>
struct Ring<Fp4, D> {
  static constexpr uint32_t kSlot = D == 64 ? 2304 : 34 * D;  // whole loads
  static constexpr uint32_t kOps = D / 32 + (D == 256 ? 2 : 1);
  static constexpr uint32_t kDepth = D == 64 ? 7 : D == 128 ? 4 : 2;
};
template <uint32_t D>
struct Ring<Fp8, D> {
  static constexpr uint32_t kSlot = 64 * D + 256;
  static constexpr uint32_t kOps = D / 16 + 1;
  static constexpr uint32_t kDepth = D == 64 ? 4 : D == 128 ? 2 : 1;
};
template <class F, uint32_t D>
__device__ __forceinline__ void FetchRecord(const uint8_t* base, uint32_t lds) {
  if constexpr (__is_same(F, Fp8)) {
    const uint32_t lane = threadIdx.x % 64;
#pragma unroll
    for (uint32_t c = 0; c < D / 16; ++c) ring::Dma16(base + c * 1024, lane * 16, lds + c * 1024);
    // the record's last 16 bytes, over and over
    ring::Dma4(base + 64 * D, lane % 4 * 4, lds + 64 * D);
    return;
  }
  const uint32_t lane = threadIdx.x % 64;
#pragma unroll
  for (uint32_t c = 0; c < D / 32; ++c) ring::Dma16(base + c * 1024, lane * 16, lds + c * 1024);
  // 2 D bytes of scales; the upper lanes repeat the lower ones' where that is
  // half a load
  ring::Dma4(base + 32 * D, (D == 64 ? lane % 32 : lane) * 4, lds + 32 * D);
  if (D == 256) ring::Dma4(base + 32 * D + 256, lane * 4, lds + 32 * D + 256);
}
template <uint32_t D>
__device__ __forceinline__ void ReadKeys(const uint8_t* slot, Record<Fp4, D>& r) {
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
__device__ __forceinline__ void ReadValues(const uint8_t* slot, Record<Fp4, D>& r) {
  const uint32_t lane = threadIdx.x % 64, g = lane / 16, n = lane % 16;
#pragma unroll
  for (uint32_t c = 0; c < D / 64; ++c)
    r.v[c] = *reinterpret_cast<const u32x4*>(slot + 16 * D + c * 1024 + lane * 16);
  const uint2 vs = *reinterpret_cast<const uint2*>(slot + 33 * D + n * D / 512 * 32 + g * 8);
  r.vs[0] = vs.x;
  r.vs[1] = vs.y;
}

template <uint32_t D>
__device__ __forceinline__ void ReadKeys(const uint8_t* slot, Record<Fp8, D>& r) {
  const uint32_t lane = threadIdx.x % 64;
#pragma unroll
  for (uint32_t c = 0; c < D / 32; ++c)
    r.k[c] = *reinterpret_cast<const u32x4*>(slot + c * 1024 + lane * 16);
  r.scales = *reinterpret_cast<const uint16_t*>(slot + 64 * D);
}
template <uint32_t D>
__device__ __forceinline__ void ReadValues(const uint8_t* slot, Record<Fp8, D>& r) {
  const uint32_t lane = threadIdx.x % 64;
#pragma unroll
  for (uint32_t c = 0; c < D / 32; ++c)
    r.v[c] = *reinterpret_cast<const u32x4*>(slot + 32 * D + c * 1024 + lane * 16);
}

__device__ __forceinline__ float ScaleOf(uint32_t bytes, uint32_t i) {
  return __uint_as_float(((bytes >> (8 * i)) & 255u) << 23);
}
// Scales of 253 and 254, whose products pass the types' range, count as 255,
// NaN: nonzero where one of the 4 bytes is such a one.
__device__ __forceinline__ uint32_t Nans(uint32_t x) {
  return ((x & 0x7F7F7F7Fu) + 0x03030303u) & x & 0x80808080u;
}

// Two codes, byte `sel` of a word, as bf16 values (exact: E2M1 on E8M0 up to 252).
template <int sel>
__device__ __forceinline__ uint32_t Two(uint32_t word, float scale) {
  return __builtin_bit_cast(uint32_t,
                            __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, sel));
}
// Operand of K: tokens 16 tile + n, the lane's columns 8 s .. 8 s + 7.
template <uint32_t parts, uint32_t D>
__device__ __forceinline__ bf16x8 KeyOperand(const Record<Fp4, D>& r, uint32_t tile, uint32_t s) {
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

// Eight E4M3 codes, two words, as the operand's type (exact where the type's
// range holds code x scale).
template <bool half>
__device__ __forceinline__ u32x4 EightOf(uint32_t lo, uint32_t hi, float scale) {
  u32x4 x;
  if constexpr (half) {
    x[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, false));
    x[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, true));
    x[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, false));
    x[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, true));
  } else {
    x[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
    x[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
    x[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
    x[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
  }
  return x;
}
// 2^(byte - 127); byte 0 stands beside zeros (and NaN keys) only: 1.
__device__ __forceinline__ float Scale8(uint32_t byte) {
  return __uint_as_float((byte == 0 ? 127u : byte) << 23);
}
// K's codes with the part of their scale that is below 1 in bf16 (exact: 2^-9 x
// 2^-117 is normal), bare in f16; KeyExponent is the rest.
template <uint32_t parts, uint32_t D>
__device__ __forceinline__ typename QueryOperand<Fp8, parts>::type KeyOperand(
    const Record<Fp8, D>& r, uint32_t tile, uint32_t s) {
  const uint32_t piece = tile * (D / 32) + s;  // of 8 bytes
  const float scale = parts == 2 ? 1.f : Scale8(min(r.scales & 255u, 127u));
  return __builtin_bit_cast(
      typename QueryOperand<Fp8, parts>::type,
      EightOf<parts == 2>(r.k[piece / 2][piece % 2 * 2], r.k[piece / 2][piece % 2 * 2 + 1],
                          scale));
}

// P V in f16 for the 16-bit types: a weight is off by at most 2^-11 of itself,
// less than bf16's output (2^-8) and as much as fp16's, and V is exact in f16
// wherever its scale bytes lie in [104, 140] (0.5 x 2^-23 .. 6 x 2^13).  Other
// records take V in bf16 and each weight as two bf16 parts (2^-16 of it).  fp32
// takes three bf16 parts of P.
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
// Whether f16 does not hold a record's values, for its scale byte: 2^-9 x 2^-15
// .. 448 x 2^7, or zeros.
__device__ __forceinline__ bool OutsideHalf8(uint32_t byte) {
  return byte != 0 && byte - 112u > 22u;
}
// Nonzero where one of the 4 bytes is 206 or more: values of up to 2^81 do not
// pass fp32 in sums of 2^31 weights of 2^15.
__device__ __forceinline__ uint32_t Large(uint32_t x) {
  return ((x & 0x7F7F7F7Fu) + 0x32323232u) & x & 0x80808080u;
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
__device__ __forceinline__ void ValueOperands(const Record<Fp4, D>& r, uint32_t i,
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
// A column's 8 tokens are neighbours in a record of 8 bits.
template <uint32_t D, bool half>
__device__ __forceinline__ void ValueOperands(const Record<Fp8, D>& r, uint32_t i,
                                              typename Value<half>::type* even,
                                              typename Value<half>::type* odd) {
  typedef typename Value<half>::type V;
  const float scale = Scale8(r.scales >> 8);
  *even = __builtin_bit_cast(V, EightOf<half>(r.v[i][0], r.v[i][1], scale));
  *odd = __builtin_bit_cast(V, EightOf<half>(r.v[i][2], r.v[i][3], scale));
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

// Largest of two, where fmaxf would make sure of quiet NaNs first.
__device__ __forceinline__ float Max2(float a, float b) { return Max3(a, b, b); }
// Of a lane's scores.  The matrix cores' results may be read some cycles after
// their last product only; the compiler keeps its own instructions from them so
// long, but not an asm's, so an addition that reads both results goes first.
__device__ __forceinline__ float MaxOf8(const f32x4 (&s)[2]) {
  const float first = s[0][0] + s[1][0];
  float a, b, c;
  asm("v_max3_f32 %0, %1, %2, %3"
      : "=v"(a) : "v"(s[0][0]), "v"(s[0][1]), "v"(s[0][2]), "v"(first));
  asm("v_max3_f32 %0, %1, %2, %3"
      : "=v"(b) : "v"(s[0][3]), "v"(s[1][0]), "v"(s[1][1]), "v"(first));
  asm("v_max_f32 %0, %1, %2" : "=v"(c) : "v"(s[1][2]), "v"(s[1][3]), "v"(first));
  return Max3(a, b, c);
}

// Over the four lanes that share a row (n, 16 + n, 32 + n, 48 + n).
__device__ __forceinline__ float RowMax(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = Max2(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return Max2(__uint_as_float(b[0]), __uint_as_float(b[1]));
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
template <class F>
__device__ __forceinline__ Sight SightOf(const KvSpan& s, uint32_t token, bool valid,
                                         uint32_t window, uint32_t sinks) {
  Sight v;
  const int32_t pos = s.total - s.count + (int32_t)token;
  v.hi = valid ? min(pos, s.total - 1) : -1;
  v.lo = window > 0 && (int64_t)pos + 1 > (int64_t)window ? pos + 1 - (int32_t)window : 0;
  v.pre = valid ? s.prefix : 0;
  if (F::kSinks && valid) v.pre = KvLead(s.prefix, sinks, pos, s.total);
  return v;
}
// What every row from `token` on sees of the first keys; the rows up to `token`
// see none of them past it but in their windows.
template <class F>
__device__ __forceinline__ int32_t LeadOf(const KvSpan& s, uint32_t token, uint32_t sinks) {
  return F::kSinks ? KvLead(s.prefix, sinks, s.total - s.count + (int32_t)token, s.total)
                   : s.prefix;
}

// Whether q's and out's rows allow loads and stores of four elements.
template <uint32_t parts>
__device__ __forceinline__ bool QueryAligned(const AttnArgs& a) {
  return (a.q_token | a.q_head) % 4 == 0 &&
         reinterpret_cast<uintptr_t>(a.q) % (4 * sizeof(typename TypeOf<parts>::type)) == 0;
}
template <uint32_t parts>
__device__ __forceinline__ bool OutAligned(const AttnArgs& a) {
  return (a.out_token | a.out_head) % 4 == 0 &&
         reinterpret_cast<uintptr_t>(a.out) % (4 * sizeof(typename TypeOf<parts>::type)) == 0;
}

// The lane's D / 4 elements of a query row, as they lie; zeros past the rows.
// The loads of a row are under way together.
template <uint32_t parts, uint32_t D>
struct Query {
  typedef typename TypeOf<parts>::type T;
  typedef typename Four<typename TypeOf<parts>::type>::type V;
  V x[D / 16];
  __device__ __forceinline__ void Load(const AttnArgs& a, uint64_t at, bool valid) {
    const T* from = static_cast<const T*>(a.q) + at;
    const V zero = {(T)0.f, (T)0.f, (T)0.f, (T)0.f};
#pragma unroll
    for (uint32_t i = 0; i < D / 16; ++i) x[i] = zero;
    if (QueryAligned<parts>(a)) {
      if (valid) {
#pragma unroll
        for (uint32_t i = 0; i < D / 16; ++i) x[i] = reinterpret_cast<const V*>(from)[i];
      }
    } else if (valid) {
#pragma unroll
      for (uint32_t i = 0; i < D / 16; ++i)
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) x[i][j] = from[4 * i + j];
    }
  }
  // elements 8 i .. 8 i + 7 as fp32, with the scale's sign
  __device__ __forceinline__ void Eight(const AttnArgs& a, uint32_t i, float* y) const {
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) y[j] = a.sign * (float)x[2 * i + j / 4][j % 4];
  }
  template <class F>
  __device__ __forceinline__ void Parts(const AttnArgs& a, uint32_t i,
                                        typename QueryOperand<F, parts>::type* out) const {
    float y[8];
    Eight(a, i, y);
    if constexpr (F::Parts(parts) == parts) {
      ToParts<parts>(y, out);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) out[0][j] = (_Float16)y[j];
    }
  }
};

// A finished value in the tensors' type: multiplied in fp32, then rounded.  (Left
// to the compiler, fp16 rows are multiplied and rounded by one instruction on
// some of the ways out and by two on others, which differ in the last bit now
// and then: rows would depend on their alignment.)
template <class T>
__device__ __forceinline__ T Rounded(float x) {
  asm("" : "+v"(x));
  return (T)x;
}

template <uint32_t parts>
__device__ __forceinline__ void StoreFour(const AttnArgs& a, uint64_t at, bool vec, f32x4 y) {
  typedef typename TypeOf<parts>::type T;
  typedef typename Four<typename TypeOf<parts>::type>::type V;
  T* to = static_cast<T*>(a.out) + at;
  V z;
#pragma unroll
  for (int j = 0; j < 4; ++j) z[j] = Rounded<T>(y[j]);
  if (vec) {
    *reinterpret_cast<V*>(to) = z;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) to[j] = z[j];
  }
}

// The state of R tiles of 16 rows on one wave.
template <uint32_t D, uint32_t R>
struct State {
  f32x4 o[R][D / 16];
  float m[R], l[R];
  bool large;  // values were met that want kRoom
  bool far;    // a maximum has passed 2^20
  Sight see[R];
  int32_t see_all, see_from, see_pre;  // every row sees keys see_from .. see_all, and < see_pre
};
template <class F, uint32_t parts, uint32_t D, uint32_t R>
struct Rows : State<D, R> {
  typename QueryOperand<F, parts>::type q[R][F::Parts(parts)][D / 32];
};

// A wave's rows: row0 .. of the `rows` rows (token, query head of the group) of
// a request and K/V head; `last` is its last one.
struct RowSet {
  KvSpan span;
  uint32_t group, head, row0, rows, last;
};

// No keys seen yet.
template <class F, uint32_t D, uint32_t R>
__device__ __forceinline__ void Begin(const AttnArgs& a, const RowSet& set, State<D, R>& w) {
  const KvSpan& span = set.span;
#pragma unroll
  for (uint32_t t = 0; t < R; ++t) {
    const uint32_t row = set.row0 + t * 16 + threadIdx.x % 16;
    w.see[t] = SightOf<F>(span, row / set.group, row < set.rows, a.window, a.sinks);
    w.m[t] = -__builtin_inff();
    w.l[t] = 0.f;
#pragma unroll
    for (uint32_t c = 0; c < D / 16; ++c) w.o[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  w.large = w.far = false;
  w.see_all = min(span.total - span.count + (int32_t)(set.row0 / set.group), span.total - 1);
  w.see_from = SightOf<F>(span, set.last / set.group, true, a.window, 0).lo;
  w.see_pre = LeadOf<F>(span, set.row0 / set.group, a.sinks);
}

// Where the lane's columns of tile t's row start in q; false past the rows.
template <uint32_t parts, uint32_t D>
__device__ __forceinline__ bool QueryAt(const AttnArgs& a, const RowSet& set, uint32_t t,
                                        uint64_t* at) {
  const uint32_t row = set.row0 + t * 16 + threadIdx.x % 16;
  *at = (uint64_t)(set.span.first + row / set.group) * a.q_token +
        (uint64_t)(set.head * set.group + row % set.group) * a.q_head +
        threadIdx.x % 64 / 16 * (D / 4);
  return row < set.rows;
}

// The finished rows (l summed over the row's lanes) into out.
template <uint32_t parts, uint32_t D, uint32_t R>
__device__ __forceinline__ void Finish(const AttnArgs& a, const RowSet& set,
                                       const State<D, R>& w) {
  const bool vec = OutAligned<parts>(a);
#pragma unroll
  for (uint32_t t = 0; t < R; ++t) {
    const uint32_t row = set.row0 + t * 16 + threadIdx.x % 16;
    if (row >= set.rows) continue;
    const float inv = w.l[t] == 0.f ? 0.f : 1.f / w.l[t];
    const uint64_t at = (uint64_t)(set.span.first + row / set.group) * a.out_token +
                        (uint64_t)(set.head * set.group + row % set.group) * a.out_head +
                        threadIdx.x % 64 / 16 * (D / 4);
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
      for (uint32_t c = 0; c < D / 16; c += 4) {
        const f32x4 y = {w.o[t][c][i], w.o[t][c + 1][i], w.o[t][c + 2][i], w.o[t][c + 3][i]};
        StoreFour<parts>(a, at + i * (D / 16) + c, vec, y * inv);
      }
  }
}

// One record: the products of its keys ...
template <class F, uint32_t parts, uint32_t D, uint32_t R>
__device__ __forceinline__ void Scores(const Record<F, D>& r, const Rows<F, parts, D, R>& w,
                                       f32x4 (&s)[R][2]) {
#pragma unroll
  for (uint32_t t = 0; t < R; ++t) s[t][0] = s[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (uint32_t i = 0; i < D / 32; ++i) {
#pragma unroll
    for (uint32_t tile = 0; tile < 2; ++tile) {
      const auto k = KeyOperand<parts>(r, tile, i);
#pragma unroll
      for (uint32_t t = 0; t < R; ++t)
#pragma unroll
        for (uint32_t p = F::Parts(parts); p-- > 0;)
          s[t][tile] = Product(k, w.q[t][p][i], s[t][tile]);
    }
  }
}

// tanh(x).  `fine`: to 2^-23 or so of 1, by the odd series to x^13 where 1 - 2 /
// (1 + e^2x) cancels, and a reciprocal with one Newton step elsewhere.
template <bool fine>
__device__ __forceinline__ float Tanh(float x) {
  const float d = 1.f + __builtin_amdgcn_exp2f(x * (2.f * kLog2e));
  float r = __builtin_amdgcn_rcpf(d);
  if constexpr (!fine) return fmaf(-2.f, r, 1.f);
  const float near_one = fmaf(fmaf(-d, r, 1.f), r, r);
  r = d < 1e30f ? near_one : 0.f;  // (inf * 0 in the step)
  const float y = x * x;
  float p = fmaf(y, 21844.f / 6081075.f, -1382.f / 155925.f);
  p = fmaf(y, p, 62.f / 2835.f);
  p = fmaf(y, p, -17.f / 315.f);
  p = fmaf(y, p, 2.f / 15.f);
  p = fmaf(y, p, -1.f / 3.f);
  const float small = fmaf(x * y, p, x), large = fmaf(-2.f, r, 1.f);
  return y < 0.2f ? small : x != x ? x : large;
}

// Scores to powers of two: they are s c with Step's c, capped ones (softcap
// tanh(s scale / softcap)) once Cap has been over them.  The 16-bit types take the
// plain 1 - 2 / (1 + e^2x), off by 2^-22 of the cap, while that is at most
// kPlainCap and the scores so off by 2^-16.
constexpr float kPlainCap = 64.f;
// A key's exponent that a factor without one of its own (AttnArgs) may meet.
constexpr int32_t kNear = 126 - kMostFactor;
template <bool fine, uint32_t R>
__device__ __forceinline__ void Cap(const AttnArgs& a, f32x4 (&s)[R][2], float in) {
  const float out = a.cap * kLog2e;
#pragma unroll
  for (uint32_t t = 0; t < R; ++t)
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j)
      s[t][j / 4][j % 4] = out * Tanh<fine>(in * s[t][j / 4][j % 4]);
}
// What a record's keys lack in their products (KeyOperand), as an exponent.
template <uint32_t parts, uint32_t D>
__device__ __forceinline__ int32_t KeyExponent(const Record<Fp4, D>&) {
  return 0;
}
template <uint32_t parts, uint32_t D>
__device__ __forceinline__ int32_t KeyExponent(const Record<Fp8, D>& r) {
  const int32_t byte = __builtin_amdgcn_readfirstlane((int)(r.scales & 255u));
  return byte == 0 ? 0 : parts == 2 ? byte - 127 : max(byte - 127, 0);
}
// What the products s are multiplied by where scale 2^exponent 2^key may be past
// fp32 (an infinity there makes a NaN of a score of 0, a 0 that of a hidden key's
// -inf): half of the exponent at once, and the rest.  Neither step then leaves fp32
// where both together do not.
template <uint32_t R>
__device__ __forceinline__ float InTwoSteps(const AttnArgs& a, int32_t key, f32x4 (&s)[R][2]) {
  const int32_t all = a.exponent + key + __builtin_amdgcn_frexp_expf(a.scale);
  const int32_t e = min(max(all, -250), 250);  // (past it all products are 0 or past fp32)
  const float half = __builtin_ldexpf(1.f, e / 2);
#pragma unroll
  for (uint32_t t = 0; t < R; ++t)
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) s[t][j / 4][j % 4] *= half;
  return __builtin_ldexpf(__builtin_amdgcn_frexp_mantf(a.scale), e - e / 2);
}

// The record's key of a lane's score j.
__device__ __forceinline__ int32_t KeyOf(int32_t key0, uint32_t j) {
  return key0 + (int32_t)(j / 4 * 16 + threadIdx.x % 64 / 16 * 4 + j % 4);
}

// Zeros for the record's V past `total`.
template <uint32_t D>
__device__ __forceinline__ void DropPast(Record<Fp8, D>& r, int32_t key0, int32_t total) {
  uint32_t keep[2] = {0, 0};
#pragma unroll
  for (uint32_t j = 0; j < 8; ++j)
    if (KeyOf(key0, j) < total) keep[j / 4] |= 255u << (8 * (j % 4));
#pragma unroll
  for (uint32_t c = 0; c < D / 32; ++c)
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) r.v[c][j] &= keep[j % 2];
}

// -inf for the keys a row does not see.
template <uint32_t D, uint32_t R>
__device__ __forceinline__ void Hide(const State<D, R>& w, int32_t key0, f32x4 (&s)[R][2]) {
  if ((key0 >= w.see_from && key0 + 31 <= w.see_all) || key0 + 32 <= w.see_pre) return;
#pragma unroll
  for (uint32_t t = 0; t < R; ++t)
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      const int32_t key = KeyOf(key0, j);
      const Sight& v = w.see[t];
      const bool sees = (key >= v.lo && key <= v.hi) || key < v.pre;
      s[t][j / 4][j % 4] = sees ? s[t][j / 4][j % 4] : -__builtin_inff();
    }
}

// The running maximum of tile t moves where a score passes it by kSlack, and
// what it had so far shrinks.  With `large` it stays kRoom above the scores.
template <uint32_t D, uint32_t R>
__device__ __forceinline__ void Raise(State<D, R>& w, uint32_t t, const f32x4 (&s)[2], float c,
                                      bool large) {
  const float top = c * MaxOf8(s);
  if (__builtin_amdgcn_ballot_w64(top > w.m[t] + (large ? kSlack - kRoom : kSlack)) == 0) return;
  float m = RowMax(top);
  if (large) m += kRoom;
  m = Max2(w.m[t], m);
  // rows that have seen nothing yet stay at -inf, with o and l zero
  const float shrink = m == w.m[t] ? 1.f : __builtin_amdgcn_exp2f(w.m[t] - m);
  w.m[t] = m;
  w.far |= __builtin_amdgcn_ballot_w64(fabsf(m) > 0x1p20f && fabsf(m) < __builtin_inff()) != 0;
  w.l[t] *= shrink;
#pragma unroll
  for (uint32_t i = 0; i < D / 16; ++i) w.o[t][i] *= shrink;
}
// What a row's weights are relative to.
__device__ __forceinline__ float Reference(float m) {
  return kLift - (m == -__builtin_inff() ? 0.f : m);
}
// The record's weights and their sum.  They carry 2^kLift: at most 2^15, and in
// f16 normal down to 2^-21 of the reference, off by 2^-32 of it below that.
// A row whose maximum passes 2^20 takes its scores as the maximum took them, rounded,
// so that the largest is not 2^(half a step of the maximum) of what it should be.
// (The branch takes prompts of up to 4,096 tokens over MXFP4 from 359 to 361 us.)
template <uint32_t D, uint32_t R>
__device__ __forceinline__ void Weights(State<D, R>& w, uint32_t t, const f32x4 (&s)[2], float c,
                                        float* p) {
  const float ref = Reference(w.m[t]);
  float sum = 0.f;
  if (__builtin_expect(w.far, 0)) {
    const float m = w.m[t] == -__builtin_inff() ? 0.f : w.m[t];
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      p[j] = __builtin_amdgcn_exp2f((s[j / 4][j % 4] * c - m) + kLift);
      sum += p[j];
    }
  } else {
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      p[j] = __builtin_amdgcn_exp2f(fmaf(s[j / 4][j % 4], c, ref));
      sum += p[j];
    }
  }
  w.l[t] += sum;
}
__device__ __forceinline__ f16x8 HalfWeights(const float* p) {
  f16x8 y;
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const f16x2 two = __builtin_convertvector(f32x2{p[j], p[j + 1]}, f16x2);
    y[j] = two[0];
    y[j + 1] = two[1];
  }
  return y;
}

// Unusual records, before their scores are hidden from rows; true where V is not
// within f16.
template <bool half, uint32_t D, uint32_t R>
__device__ __forceinline__ bool Unusual(const KvSpan& span, Record<Fp4, D>& r, int32_t key0,
                                        f32x4 (&s)[R][2], State<D, R>& w) {
  // Unusual scale bytes: a token whose K or V has a scale of NaN, or one whose
  // products pass the types' range (253, 254), gives NaN scores to the rows
  // that see it and nothing to others (V's 0 x NaN would reach every row of the
  // tile); past the request's end any byte may lie.
  bool wide = false;
  const uint32_t keys = Nans(r.ks[0] | (D == 256 ? r.ks[D == 256] : 0u) << 16);
  if (__builtin_amdgcn_ballot_w64((OutsideHalf(r.vs[0]) | OutsideHalf(r.vs[1]) | keys) != 0) != 0) {
    uint32_t nan = 0;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      const uint32_t byte = (r.vs[j / 4] >> (8 * (j % 4))) & 255u;
      nan |= (uint32_t)(byte >= 253u) << j;
      if (byte >= 253u || KeyOf(key0, j) >= span.total)
        r.vs[j / 4] = (r.vs[j / 4] & ~(255u << (8 * (j % 4)))) | 127u << (8 * (j % 4));
    }
#pragma unroll
    for (uint32_t d = 1; d < 16; d *= 2) nan |= __shfl_xor(nan, d);
    // K's bytes lie with lane n for tokens n and 16 + n
    uint32_t tokens[2];
#pragma unroll
    for (uint32_t tile = 0; tile < 2; ++tile) {
      uint64_t lanes = __builtin_amdgcn_ballot_w64((keys & (tile ? 0x80008000u : 0x00800080u)) != 0);
      lanes |= lanes >> 32;
      tokens[tile] = (uint32_t)(lanes | lanes >> 16) & 0xFFFFu;
    }
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j)
      nan |= (tokens[j / 4] >> (threadIdx.x % 64 / 16 * 4 + j % 4) & 1u) << j;
#pragma unroll
    for (uint32_t t = 0; t < R; ++t)
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j)
        if (nan >> j & 1) s[t][j / 4][j % 4] = __builtin_nanf("");
    if (__builtin_amdgcn_ballot_w64((Large(r.vs[0]) | Large(r.vs[1])) != 0) != 0)
      w.large = true;
    wide = half && __builtin_amdgcn_ballot_w64(
                       (OutsideHalf(r.vs[0]) | OutsideHalf(r.vs[1])) != 0) != 0;
  }
  return wide;
}
// Records of 8 bits: a NaN key's scores are NaN by themselves and V holds none,
// but past the request's end, where any byte may lie.
template <bool half, uint32_t D, uint32_t R>
__device__ __forceinline__ bool Unusual(const KvSpan& span, Record<Fp8, D>& r, int32_t key0,
                                        f32x4 (&)[R][2], State<D, R>& w) {
  if (key0 + 32 > span.total) DropPast(r, key0, span.total);
  const uint32_t scale = (uint32_t)__builtin_amdgcn_readfirstlane((int)(r.scales >> 8));
  // values of up to 2^81 do not pass fp32 in sums of 2^31 weights of 2^15
  if (scale >= 199u) w.large = true;
  return half && OutsideHalf8(scale);
}

// ... and the scores' running maximum and sum, and P V.
template <class F, uint32_t parts, uint32_t D, uint32_t R>
__device__ __forceinline__ void Step(const AttnArgs& a, const KvSpan& span, Record<F, D>& r,
                                     int32_t key0, f32x4 (&s)[R][2], Rows<F, parts, D, R>& w) {
  const int32_t key = KeyExponent<parts>(r);
  float c = a.scale;
  if (__is_same(F, Fp8)) c *= __uint_as_float((uint32_t)(key + 127) << 23);
  // (one branch, on whole numbers, for what most calls have none of: with two, that
  // the products' end and the softmax lay between, small calls took 1 us longer)
  const bool far = a.exponent != 0 || key < -kNear || key > kNear;
  if (__float_as_uint(a.cap) != 0 || __builtin_expect(far, 0)) {
    if (far) c = InTwoSteps(a, key, s);
    if (a.cap > 0.f) {
      if (parts == 3 || a.cap > kPlainCap) Cap<true, R>(a, s, c);
      else Cap<false, R>(a, s, c);
      c = 1.f;
    }
  }
  constexpr bool half = parts < 3;
  bool wide = Unusual<half>(span, r, key0, s, static_cast<State<D, R>&>(w));
  // weights below 2^-48 are none in f16
  if (half && w.large) wide = true;
  Hide<D, R>(w, key0, s);
  typename Value<half>::type pt[R][half ? 1 : parts];
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (uint32_t t = 0; t < R; ++t) {
    float p[8];
    Raise(static_cast<State<D, R>&>(w), t, s[t], c, w.large);
    Weights(static_cast<State<D, R>&>(w), t, s[t], c, p);
    if constexpr (half) {
      if (wide) {  // V in bf16, on two bf16 parts of a weight
        bf16x8 part[2];
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
      } else {
        pt[t][0] = HalfWeights(p);
      }
    } else {
      ToParts<parts>(p, pt[t]);
    }
  }
  __builtin_amdgcn_sched_barrier(0);
  if (half && wide) return;
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

}  // namespace attn
}  // namespace hb
