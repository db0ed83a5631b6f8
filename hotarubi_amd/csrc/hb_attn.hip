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

#include "hb_attn.h"

namespace hb {
namespace {

using namespace attn;

constexpr uint32_t kWaves = 4, kThreads = 64 * kWaves;

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
// where those do
__global__ __launch_bounds__(kThreads, D == 256 && parts > 1 ? 1 : 2) void AttnKernel(const AttnArgs a) {
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
  const RowSet set{span, group, head, row0, rows, last};
  Begin<D, R>(a, set, w);
  Query<parts, D> query[R];
#pragma unroll
  for (uint32_t t = 0; t < R; ++t) {
    uint64_t at;
    const bool valid = QueryAt<parts, D>(a, set, t, &at);
    query[t].Load(a, at, valid);
  }

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
  uint32_t hidden = 0;  // a bit per slot: no page, the slot holds record 0
  auto fetch = [&](uint32_t i, uint32_t base, uint32_t slot) {  // base <= i < base + 128
    const uint32_t from = (uint32_t)__builtin_amdgcn_readlane(
        (int)(i - base < 64 ? now : after), (int)((i - base) % 64));
    hidden = (hidden & ~(1u << slot)) | (uint32_t)(from == kNoRecord) << slot;
    FetchRecord<D>(a.cache + (from == kNoRecord ? 0 : (uint64_t)from * KvRecordBytes(D)),
                   slots_at + slot * Ring::kSlot);
  };
  asm volatile("" ::: "memory");
#pragma unroll 1
  for (uint32_t u = 0; u < min(count, Ring::kDepth); ++u) fetch(u, 0, u);
  // the queries' loads are under way with the first records'
#pragma unroll
  for (uint32_t t = 0; t < R; ++t)
#pragma unroll
    for (uint32_t i = 0; i < D / 32; ++i) {
      bf16x8 x[parts];
      query[t].Parts(a, i, x);
#pragma unroll
      for (uint32_t p = 0; p < parts; ++p) w.q[t][p][i] = x[p];
    }
  // one copy of the step: what a launch of few records waits for most is its
  // code
#pragma unroll 1
  for (uint32_t i = 0, base = 0, u = 0; i < count; ++i, u = u + 1 == Ring::kDepth ? 0 : u + 1) {
    if (i + Ring::kDepth <= count) ring::WaitVm<(Ring::kDepth - 1) * Ring::kOps>();
    else ring::WaitVm<0>();
    asm volatile("" ::: "memory");
    const bool present = (hidden >> u & 1) == 0;
    Record<D> r;
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
      f32x4 s[R][2];
      Scores<parts, D, R>(r, w, s);
      const int32_t key0 = (int32_t)(32 * KvWalkRecord(walk, first + i * step));
      Step<parts, D, R>(a, span, r, key0, s, w);
    }
  }
#pragma unroll
  for (uint32_t t = 0; t < R; ++t) w.l[t] = RowSum(w.l[t]);

  const bool ovec = OutAligned<parts>(a);
  if constexpr (!split) {
    Finish<parts, D, R>(a, set, w);
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
  const bool ovec = OutAligned<parts>(a);
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
      // (two tiles of three parts take more than 256 registers)
      return two && parts < 3 ? LaunchOf<parts, 128, 2>(a, ws, stream) : LaunchOf<parts, 128, 1>(a, ws, stream);
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
  if (PromptEligible(a)) return LaunchPrompt(a, stream);
  switch (a.type) {
    case HB_TYPE_BF16: return LaunchDim<1>(a, ws, stream);
    case HB_TYPE_F16: return LaunchDim<2>(a, ws, stream);
    default: return LaunchDim<3>(a, ws, stream);
  }
}

}  // namespace hb
