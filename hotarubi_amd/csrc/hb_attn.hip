// Attention over the paged MXFP4 cache.
//
// Rows of one request and K/V head (new tokens x the query heads that share
// it) in tiles of 16, keys in records of 32.  With A = K and B = Q^T the
// matrix cores give S^T: lane (g, n) = 16 g + n holds the scores of row n
// for tokens 4g .. 4g+3 and 16+4g .. 16+4g+3, which is where the B operand of
// O^T = V^T P^T wants them, so P goes from the softmax to the next product in
// the same registers, with no trip through LDS; the record's layout gives the
// lane its K and V codes for both products as they lie.
//
// With o, m and l of a row over the keys so far, a record of scores s (in
// powers of two) makes m' = max(m, max s), o' = o 2^(m - m') + sum 2^(s - m') v
// and l' = l 2^(m - m') + sum 2^(s - m'); parts of a row's keys join by the same
// rule, and out = o / l, or 0 where l = 0.  The cache is read once, 34 D bytes a
// record and head.  Few rows are bound by that: 8 query heads on each of 8 over
// 262,147 keys, D 128, 285 MB, take 51 us and 5 for the join (5.6 TB/s before
// it; the card copies at 4.9, reads and writes together), and 64 requests of
// 1,000 to 8,191 keys, 321 MB, 71 us and 6.  Rows of 32 bits want three products
// where others want one: 32 requests of 50 rows behind 150 keys, 15 heads on 5,
// D 64, take 13.6 us a call in fp32 and 11.1 in bf16.
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

// How a workgroup's waves divide the work:
//   kRows    each wave has R tiles of its own and takes every record
//   kSplits  they share R tiles and take the records of a split of them in turn
//   kShares  the same, over shares of all requests' records that are alike to
//            within one record, whatever the requests' lengths
enum Mode { kRows, kSplits, kShares };

constexpr uint32_t kMaxShared = 256;  // requests of a kShares launch
constexpr uint32_t kLeastShare = 16;  // records
struct Shares {
  uint32_t start[kMaxShared + 1];  // records before request b, over its heads
  uint32_t each[kMaxShared];       // of one of its heads; 1 for a request without keys
  uint32_t part[kThreads / 64];
  uint32_t groups, per, extra;
  __device__ __forceinline__ uint32_t Start(uint32_t group) const {
    return group * per + min(group, extra);
  }
  __device__ __forceinline__ uint32_t GroupOf(uint32_t record) const {
    const uint32_t longer = extra * (per + 1);
    return record < longer ? record / (per + 1) : extra + (record - longer) / per;
  }
};

__device__ __forceinline__ KvSpan SpanOf(const AttnArgs& a, uint32_t b) {
  return KvRequest(a.cu[b], a.cu[b + 1], a.kv_lens[b], a.prefix ? a.prefix[b] : 0, a.tokens,
                   a.max_new, (uint64_t)a.columns * a.groups * 32);
}
// The rows [row0, row0 + count) of a request's, and the records they look at.
__device__ __forceinline__ KvWalk WalkOf(const AttnArgs& a, const KvSpan& span, uint32_t group,
                                         uint32_t row0, uint32_t last) {
  const int32_t base = span.total - span.count;
  return KvRecords(base + (int32_t)(row0 / group), base + (int32_t)(last / group), span.total,
                   span.prefix, a.window);
}

// Every workgroup makes the sums for itself (a thread per request).
__device__ __forceinline__ void ShareOut(const AttnArgs& a, Shares& s) {
  const uint32_t tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  uint32_t n = 0;
  if (tid < a.batch) {
    const KvSpan span = SpanOf(a, tid);
    const uint32_t group = a.q_heads / a.heads, rows = span.rows * group;
    if (rows > 0) n = max(1u, WalkOf(a, span, group, 0, rows - 1).count);
  }
  uint32_t sum = n * a.heads;
  for (uint32_t d = 1; d < 64; d *= 2) {
    const uint32_t x = __shfl_up(sum, d);
    if (lane >= d) sum += x;
  }
  if (lane == 63) s.part[wave] = sum;
  __syncthreads();
  uint32_t total = 0;
  for (uint32_t w = 0; w < kThreads / 64; ++w) {
    if (w < wave) sum += s.part[w];
    total += s.part[w];
  }
  s.start[tid + 1] = sum;
  s.each[tid] = n;
  if (tid == 0) {
    s.start[0] = 0;
    s.groups = max(1u, min(a.splits, total / kLeastShare));
    s.per = total / s.groups;
    s.extra = total % s.groups;
  }
  __syncthreads();
}

// The records [begin, end) of a walk, every `step`-th from `first` on, for the
// wave's rows; `slots` is its ring in LDS.
template <uint32_t parts, uint32_t D, uint32_t R>
__device__ __forceinline__ void TakeRecords(const AttnArgs& a, const RowSet& set, uint32_t b,
                                            const KvWalk& walk, uint32_t first, uint32_t end,
                                            uint32_t step, uint8_t* slots, Rows<parts, D, R>& w) {
  const uint32_t lane = threadIdx.x % 64;
  Begin<D, R>(a, set, w);
  Query<parts, D> query[R];
#pragma unroll
  for (uint32_t t = 0; t < R; ++t) {
    uint64_t at;
    const bool valid = QueryAt<parts, D>(a, set, t, &at);
    query[t].Load(a, at, valid);
  }
  const int32_t* const row = a.table + (uint64_t)b * a.table_stride;
  const uint32_t count = first < end ? (end - first + step - 1) / step : 0;
  typedef Ring<D> Ring;
  const uint32_t slots_at =
      (uint32_t) reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)slots);
  // block table entries of 64 records at a time, one a lane; the ring reaches
  // into the next 64
  auto pages = [&](uint32_t i) {
    return PageRecord(a, walk, row, set.head, first + (i + lane) * step, end);
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
  // one copy of the step: the code is 20 to 70 KB with one per slot
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
      Step<parts, D, R>(a, set.span, r, key0, s, w);
    }
  }
#pragma unroll
  for (uint32_t t = 0; t < R; ++t) w.l[t] = RowSum(w.l[t]);
}

// The waves' results meet in LDS, in the waves' order, and go to out or, where
// the rows have more records elsewhere, to `partial`.
template <uint32_t parts, uint32_t D, uint32_t R>
__device__ __forceinline__ void Meet(const AttnArgs& a, const RowSet& set,
                                     const Rows<parts, D, R>& w, Merge<D, R>& sum,
                                     float* partial) {
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, n = lane % 16, g = lane / 16;
  __syncthreads();  // every ring has been read
#pragma unroll
  for (uint32_t t = 0; t < R; ++t) {
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
      for (uint32_t c = 0; c < D / 16; c += 4)
        *reinterpret_cast<f32x4*>(&sum.o[wave][t * 16 + n][(4 * g + i) * (D / 16) + c]) =
            f32x4{w.o[t][c][i], w.o[t][c + 1][i], w.o[t][c + 2][i], w.o[t][c + 3][i]};
    if (g == 0) {
      sum.m[wave][t * 16 + n] = w.m[t];
      sum.l[wave][t * 16 + n] = w.l[t];
    }
  }
  __syncthreads();
  const bool vec = OutAligned<parts>(a);
  for (uint32_t i = threadIdx.x; i < R * 16 * (D / 4); i += kThreads) {
    const uint32_t r = i / (D / 4), c = i % (D / 4) * 4, row = set.row0 + r;
    if (row >= set.rows) continue;
    float m = sum.m[0][r];
#pragma unroll
    for (uint32_t k = 1; k < kWaves; ++k) m = fmaxf(m, sum.m[k][r]);
    const float ref = m == -__builtin_inff() ? 0.f : m;
    float l = 0.f;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t k = 0; k < kWaves; ++k) {
      const float f = sum.m[k][r] == m ? 1.f : __builtin_amdgcn_exp2f(sum.m[k][r] - ref);
      l += sum.l[k][r] * f;
      y += *reinterpret_cast<const f32x4*>(&sum.o[k][r][c]) * f;
    }
    if (partial == nullptr) {
      const uint64_t at = (uint64_t)(set.span.first + row / set.group) * a.out_token +
                          (uint64_t)(set.head * set.group + row % set.group) * a.out_head + c;
      StoreFour<parts>(a, at, vec, y * (l == 0.f ? 0.f : 1.f / l));
    } else {
      float* to = partial + r * kPartial<D>;
      *reinterpret_cast<f32x4*>(to + c) = y;
      if (c == 0) {
        to[D] = m;
        to[D + 1] = l;
      }
    }
  }
}

// Rows of a partial result: those that a tile has.
template <uint32_t R>
__device__ __forceinline__ uint32_t Stored(const AttnArgs& a) {
  return min(R * 16, a.max_new * (a.q_heads / a.heads));
}

// What a wave waits for is memory or its own chain of products, softmax and
// products (0.7 to 1.8 us a record by itself), so its records come ahead of it
// through a ring of direct loads (the long cache above took 98 us with records
// loaded into registers) and few rows are split over as many workgroups as the
// card holds.  Two of them a CU (their rings fill its LDS), so 256 registers a
// wave where those do.
template <uint32_t parts, uint32_t D, uint32_t R, Mode mode>
__global__ __launch_bounds__(kThreads, D == 256 && parts > 1 ? 1 : 2) void AttnKernel(
    const AttnArgs a) {
  typedef Ring<D> Ring;
  constexpr uint32_t kRing = kWaves * Ring::kDepth * Ring::kSlot;
  constexpr uint32_t kMerge = mode == kRows ? 0 : sizeof(Merge<D, R>);
  __shared__ __align__(16) uint8_t lds[kRing > kMerge ? kRing : kMerge];
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  uint8_t* const slots = lds + wave * (Ring::kDepth * Ring::kSlot);
  const uint32_t group = a.q_heads / a.heads;
  Rows<parts, D, R> w;
  if constexpr (mode != kShares) {
    const uint32_t unit = blockIdx.x / a.splits, part = blockIdx.x % a.splits;
    const uint32_t head = unit % a.heads, rest = unit / a.heads;
    const uint32_t b = rest / a.tiles, tile = a.tiles - 1 - rest % a.tiles;
    const KvSpan span = SpanOf(a, b);
    const uint32_t rows = span.rows * group;
    const uint32_t row0 = (mode == kRows ? tile * kWaves + wave : tile) * R * 16;
    if (row0 >= rows) return;
    const RowSet set{span, group, head, row0, rows, min(row0 + R * 16, rows) - 1};
    const KvWalk walk = WalkOf(a, span, group, row0, set.last);
    if constexpr (mode == kRows) {
      TakeRecords<parts, D, R>(a, set, b, walk, 0, walk.count, 1, slots, w);
      Finish<parts, D, R>(a, set, w);
    } else {
      const uint32_t begin = part * a.split_records;
      const uint32_t end =
          part + 1 == a.splits ? walk.count : min(walk.count, begin + a.split_records);
      if (part > 0 && begin >= end) return;
      TakeRecords<parts, D, R>(a, set, b, walk, begin + wave, end, kWaves, slots, w);
      const bool alone = a.splits == 1 || walk.count <= a.split_records;
      const uint64_t place = ((uint64_t)b * a.heads + head) * a.tiles + tile;
      Meet<parts, D, R>(a, set, w, *reinterpret_cast<Merge<D, R>*>(lds),
                        alone ? nullptr
                              : a.ws + (place * a.splits + part) * Stored<R>(a) * kPartial<D>);
    }
  } else {
    __shared__ Shares shares;
    ShareOut(a, shares);
    const uint32_t share = blockIdx.x;
    if (share >= shares.groups) return;
    const uint32_t stop = __builtin_amdgcn_readfirstlane(shares.Start(share + 1));
    uint32_t at = __builtin_amdgcn_readfirstlane(shares.Start(share));
    uint32_t lo = 0, hi = a.batch - 1;  // the request that record `at` belongs to
    while (lo < hi) {
      const uint32_t mid = (lo + hi) / 2;
      if (__builtin_amdgcn_readfirstlane(shares.start[mid + 1]) > at) hi = mid;
      else lo = mid + 1;
    }
#pragma unroll 1
    for (uint32_t b = lo; at < stop;) {
      const uint32_t n = __builtin_amdgcn_readfirstlane(shares.each[b]);
      const uint32_t in = at - __builtin_amdgcn_readfirstlane(shares.start[b]);
      if (n == 0 || in >= n * a.heads) {
        ++b;
        continue;
      }
      const uint32_t head = in / n, begin = in % n, take = min(n - begin, stop - at);
      const KvSpan span = SpanOf(a, b);
      const uint32_t rows = span.rows * group;
      const RowSet set{span, group, head, 0, rows, rows - 1};
      const KvWalk walk = WalkOf(a, span, group, 0, set.last);
      TakeRecords<parts, D, R>(a, set, b, walk, begin + wave, min(begin + take, walk.count),
                               kWaves, slots, w);
      // a unit's parts lie at its number plus the share's: no two alike
      const uint64_t place = (uint64_t)b * a.heads + head + share;
      Meet<parts, D, R>(a, set, w, *reinterpret_cast<Merge<D, R>*>(lds),
                        take == n ? nullptr : a.ws + place * Stored<R>(a) * kPartial<D>);
      at += take;
      __syncthreads();  // the sums have been read
    }
  }
}

// The parts of a row in their order: lane groups take every kGroups-th, then
// meet in LDS.  A launch of its own, so that no workgroup waits for another; 4.8
// us for 64 rows of 512 parts in all, 6.4 for 2,048 rows: latency.
template <uint32_t parts, uint32_t D, uint32_t R, Mode mode>
__global__ __launch_bounds__(kThreads) void JoinKernel(const AttnArgs a) {
  constexpr uint32_t kLanes = D / 4, kGroups = kThreads / kLanes;
  __shared__ float so[kGroups][D], sl[kGroups];
  const uint32_t group = a.q_heads / a.heads, stored = Stored<R>(a);
  const uint32_t place = blockIdx.x / stored, r = blockIdx.x % stored;
  const uint32_t tile = place % a.tiles, head = place / a.tiles % a.heads,
                 b = place / a.tiles / a.heads;
  const KvSpan span = SpanOf(a, b);
  const uint32_t rows = span.rows * group, row0 = tile * R * 16;
  uint32_t active;
  uint64_t slot;  // of the row's first part
  if constexpr (mode == kShares) {
    __shared__ Shares shares;
    ShareOut(a, shares);
    if (r >= rows) return;
    const uint32_t n = shares.each[b], from = shares.start[b] + head * n;
    const uint32_t first = shares.GroupOf(from);
    active = shares.GroupOf(from + n - 1) - first + 1;
    slot = (uint64_t)place + first;
  } else {
    if (row0 + r >= rows) return;
    const KvWalk walk = WalkOf(a, span, group, row0, min(row0 + R * 16, rows) - 1);
    active = min(a.splits, max(1u, (walk.count + a.split_records - 1) / a.split_records));
    slot = (uint64_t)place * a.splits;
  }
  if (active == 1) return;
  const uint32_t lane = threadIdx.x % kLanes, part = threadIdx.x / kLanes;
  const float* from = a.ws + (slot * stored + r) * kPartial<D>;
  const uint64_t step = (uint64_t)stored * kPartial<D>;
  float m = -__builtin_inff(), l = 0.f;
  // the maximum first (a lane per part), so that the sums do not wait on one
  // another
  for (uint32_t s = threadIdx.x % 64; s < active; s += 64) m = fmaxf(m, from[s * step + D]);
#pragma unroll
  for (uint32_t d = 1; d < 64; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (uint32_t s = part; s < active; s += kGroups) {
    const float* x = from + s * step;
    const float f = x[D] == m ? 1.f : __builtin_amdgcn_exp2f(x[D] - m);
    l += x[D + 1] * f;
    y += *reinterpret_cast<const f32x4*>(x + 4 * lane) * f;
  }
  *reinterpret_cast<f32x4*>(&so[part][4 * lane]) = y;
  if (lane == 0) sl[part] = l;
  __syncthreads();
  if (part != 0) return;
#pragma unroll
  for (uint32_t k = 1; k < kGroups; ++k) {
    l += sl[k];
    y += *reinterpret_cast<const f32x4*>(&so[k][4 * lane]);
  }
  const uint64_t at = (uint64_t)(span.first + (row0 + r) / group) * a.out_token +
                      (uint64_t)(head * group + (row0 + r) % group) * a.out_head + 4 * lane;
  StoreFour<parts>(a, at, OutAligned<parts>(a), y * (l == 0.f ? 0.f : 1.f / l));
}

// What the workspace may hold of opened records (hb_prompt.hip).
constexpr uint64_t kMostOpened = 1ull << 30;

// How a call's work may be divided, and about how long that takes: workgroups
// of a fixed cost and a cost a record, two to a CU, in rounds.  The constants
// are measured ones; what was compared is at Divide.
struct Division {
  enum Way { kByPrompt, kByRows, kBySplits } way;
  uint32_t tiles_of_16;  // of a wave
  uint64_t splits;
  double us;
};

// Call sizes: `pairs` (request, K/V head), `rows` of each, the records of the
// last row (most) and of the middle one (mean).
struct Sizes {
  uint64_t pairs, rows, most, cus;
  double mean, bytes;  // of q and out
  uint32_t dim, parts;
};

double Rounds(const Sizes& z, double groups, double slots, double fixed, double record,
              double share) {
  const double longest = fixed + z.most * share * record, usual = fixed + z.mean * share * record;
  const double rounds = groups / slots;
  return rounds <= 1 ? longest : std::max(longest, (rounds + 0.3) * usual);
}

Division ByPrompt(const Sizes& z, uint64_t tile, uint64_t opened) {
  // us a record of a workgroup with a CU to itself, and how much more beside
  // another
  const double alone = z.dim == 64 ? 0.75 : z.dim == 128 ? 0.62 : 1.25;
  const double more = z.dim == 64 ? 0.6 : z.dim == 128 ? 0.72 : 0;
  const double cus = (double)z.cus, slots = z.dim == 256 ? cus : 2 * cus;
  const double groups = (double)(z.pairs * ((z.rows + tile - 1) / tile));
  const double beside = std::min(1.0, std::max(0.0, groups / cus - 1));
  return {Division::kByPrompt, 0, 1,
          Rounds(z, groups, slots, 7, alone * (1 + beside * more), 1) + z.bytes / 20e6 + 3 +
              (double)opened / 4e6};
}

Division ByWaves(const Sizes& z, Division::Way way, uint32_t tiles_of_16) {
  // us a record of a wave by itself on its SIMD, by type, tiles and head size
  const double alone[3][2][3] = {{{0.72, 0.95, 1.25}, {0.95, 1.35, 0}},
                                 {{0.76, 1.05, 1.5}, {1.05, 1.5, 0}},
                                 {{0.8, 1.15, 1.85}, {1.15, 1.6, 0}}};
  // (one workgroup a CU where its waves take more than 256 registers)
  const double slots = z.dim == 256 && z.parts > 1 ? (double)z.cus : 2.0 * (double)z.cus;
  const uint32_t d = z.dim == 64 ? 0 : z.dim == 128 ? 1 : 2;
  const uint64_t tiles = (z.rows + 16 * tiles_of_16 - 1) / (16 * tiles_of_16);
  const uint64_t units =
      z.pairs * (way == Division::kByRows ? (tiles + kWaves - 1) / kWaves : tiles);
  uint64_t splits = 1;
  if (way == Division::kBySplits) {
    splits = std::max<uint64_t>(1, std::min(2 * z.cus / units, z.most / (2 * kWaves)));
    const uint64_t each = (z.most + splits - 1) / splits;
    splits = (z.most + each - 1) / each;
  }
  const double groups = (double)(units * splits);
  const double beside =
      std::min(slots / (double)z.cus - 1, std::max(0.0, groups / (double)z.cus - 1));
  const double record = alone[z.parts - 1][tiles_of_16 - 1][d] *
                        (1 + beside * (d == 2 ? 0.5 : 0.35));
  const double share = way == Division::kByRows ? 1 : 1.0 / (double)(kWaves * splits);
  return {way, tiles_of_16, splits,
          Rounds(z, groups, slots, (way == Division::kByRows ? 2 : 3) + 3 * tiles_of_16, record,
                 share) +
              (splits > 1 ? 6 : 0) + z.bytes / 8e6};
}

// The shortest.  Measured, us (bf16; prompt / rows / splits; one or two tiles a
// wave): 32 x 50 new tokens behind 150, D 64, 15 on 5 heads: 19 / 12, 15 / 19, 16;
// the same, D 128, 32 on 8: 33 / 28, 23 / 42, 38; 1 x 500 behind 2,000: 65 /
// 71, 90 / 53, 40; 2 x 1,500 behind 1,000: 122 / 200, 152 / 216, 153; 1 x 8
// behind 16,000: 285 / 413, 527 / 17, 22.  Over 60 such calls the choice is
// within 5% of the best for 50, and 1.25 times it at worst.
Division Divide(const AttnArgs& a) {
  Sizes z;
  z.pairs = (uint64_t)a.batch * a.heads;
  z.rows = (uint64_t)a.max_new * (a.q_heads / a.heads);
  z.cus = (uint64_t)DeviceCus();
  z.dim = a.dim;
  z.parts = a.type == HB_TYPE_BF16 ? 1 : a.type == HB_TYPE_F16 ? 2 : 3;
  uint64_t most = ((uint64_t)a.max_kv + 31) / 32;
  double mean = std::max(1.0, ((double)a.max_kv - 0.5 * a.max_new) / 32);
  if (a.window > 0 && a.prefix == nullptr) {
    const uint64_t seen = ((uint64_t)a.window + 94) / 32;
    most = std::min(most, seen);
    mean = std::min(mean, (double)seen);
  }
  z.most = std::max<uint64_t>(most, 1);
  z.mean = mean;
  z.bytes = 2.0 * std::min<double>(a.tokens, (double)a.batch * a.max_new) * a.q_heads * a.dim *
            (z.parts == 3 ? 4 : 2);
  Division best = ByWaves(z, Division::kBySplits, 1);
  const auto take = [&](const Division& d) {
    if (d.us < best.us) best = d;
  };
  if (z.rows > 16 * (kWaves - 1)) take(ByWaves(z, Division::kByRows, 1));
  if (z.rows > 16 && z.dim < 256) {
    take(ByWaves(z, Division::kBySplits, 2));
    if (z.rows > 32 * (kWaves - 1)) take(ByWaves(z, Division::kByRows, 2));
  }
  if (z.parts < 3 && z.rows > 32 && PromptBytes(a) <= kMostOpened)
    take(ByPrompt(z, PromptRows(z.dim), PromptBytes(a)));
  return best;
}

constexpr uint64_t kLeastShared = 64;  // records a CU

template <uint32_t parts, uint32_t D, uint32_t R>
hipError_t LaunchOf(AttnArgs& a, const AttnWay& how, Workspace& ws, hipStream_t stream) {
  const uint64_t rows = (uint64_t)a.max_new * (a.q_heads / a.heads);
  const uint64_t pairs = (uint64_t)a.batch * a.heads, stored = std::min<uint64_t>(R * 16, rows);
  const uint64_t grid = how.way == HB_KV_WAY_SHARES ? how.splits : pairs * how.tiles * how.splits;
  const uint64_t join = how.workspace > 0 ? pairs * how.tiles * stored : 0;
  if (grid > 0x7FFFFFFFu || join > 0x7FFFFFFFu) return hipErrorInvalidValue;
  a.tiles = how.tiles;
  a.splits = how.splits;
  a.split_records = how.split_records;
  if (how.workspace > 0) {
    const hipError_t err = GrowWorkspace(ws, how.workspace, stream);
    if (err != hipSuccess) return err;
    a.ws = ws.ptr + kSplitCounters;
  }
  switch (how.way) {
    case HB_KV_WAY_ROWS:
      AttnKernel<parts, D, R, kRows><<<(uint32_t)grid, kThreads, 0, stream>>>(a);
      break;
    case HB_KV_WAY_SHARES:
      AttnKernel<parts, D, R, kShares><<<(uint32_t)grid, kThreads, 0, stream>>>(a);
      JoinKernel<parts, D, R, kShares><<<(uint32_t)join, kThreads, 0, stream>>>(a);
      break;
    default:
      AttnKernel<parts, D, R, kSplits><<<(uint32_t)grid, kThreads, 0, stream>>>(a);
      if (join > 0) JoinKernel<parts, D, R, kSplits><<<(uint32_t)join, kThreads, 0, stream>>>(a);
  }
  return hipGetLastError();
}

template <uint32_t parts>
hipError_t LaunchDim(AttnArgs& a, const AttnWay& how, Workspace& ws, hipStream_t stream) {
  const bool two = how.tiles_of_16 == 2;
  switch (a.dim) {
    case 64:
      return two ? LaunchOf<parts, 64, 2>(a, how, ws, stream)
                 : LaunchOf<parts, 64, 1>(a, how, ws, stream);
    case 128:
      return two ? LaunchOf<parts, 128, 2>(a, how, ws, stream)
                 : LaunchOf<parts, 128, 1>(a, how, ws, stream);
    default: return LaunchOf<parts, 256, 1>(a, how, ws, stream);
  }
}

}  // namespace

AttnWay WayOfAttention(const AttnArgs& a) {
  const Division best = Divide(a);
  AttnWay how{};
  how.splits = 1;
  const uint64_t rows = (uint64_t)a.max_new * (a.q_heads / a.heads);
  const uint64_t pairs = (uint64_t)a.batch * a.heads, cus = (uint64_t)DeviceCus();
  if (best.way == Division::kByPrompt) {
    how.way = HB_KV_WAY_PROMPT;
    how.tiles_of_16 = PromptTiles(a.dim);
    how.tiles = (uint32_t)((rows + PromptRows(a.dim) - 1) / PromptRows(a.dim));
    how.workspace = PromptBytes(a);
    return how;
  }
  how.tiles_of_16 = best.tiles_of_16;
  const uint32_t of = 16 * how.tiles_of_16;
  const uint64_t tiles = (rows + of - 1) / of;
  if (best.way == Division::kByRows) {
    how.way = HB_KV_WAY_ROWS;
    how.tiles = (uint32_t)((tiles + kWaves - 1) / kWaves);
    return how;
  }
  how.tiles = (uint32_t)tiles;
  uint64_t records = ((uint64_t)a.max_kv + 31) / 32;
  if (a.window > 0 && a.prefix == nullptr)
    records = std::min<uint64_t>(records, ((uint64_t)a.window + of + 62) / 32);
  records = std::max<uint64_t>(records, 1);
  const uint64_t units = pairs * tiles;
  const uint64_t part = std::min<uint64_t>(of, rows) * (a.dim + 4) * 4;  // bytes: kPartial
  // Requests of different lengths, with enough records that the sums over the
  // requests (about 5 us a workgroup) are less than what uneven workgroups
  // leave idle: 64 requests of 1,000 to 8,191 keys 84 us in splits, 72 in shares.
  // (Every record that the tables have room for is counted in 32 bits, whatever
  // kv_lens says.)
  if (tiles == 1 && a.batch > 1 && a.batch <= kMaxShared && units * records >= kLeastShared * cus &&
      units * std::max<uint64_t>((uint64_t)a.columns * a.groups, 1) < 0x7FFFFFFFu) {
    how.way = HB_KV_WAY_SHARES;
    how.splits = (uint32_t)(2 * cus);
    how.workspace = (units + how.splits) * part;
    return how;
  }
  how.way = HB_KV_WAY_SPLITS;
  how.split_records = (uint32_t)((records + best.splits - 1) / best.splits);
  how.splits = (uint32_t)((records + how.split_records - 1) / how.split_records);
  if (how.splits > 1) how.workspace = units * how.splits * part;
  return how;
}

hipError_t LaunchAttention(const AttnArgs& in, Workspace& ws, hipStream_t stream) {
  AttnArgs a = in;
  // scores as |scale| (q sign): the maximum of the products is then that of
  // the scores
  a.sign = a.scale > 0.f ? 1.f : a.scale < 0.f ? -1.f : 0.f;
  a.scale = a.scale == 0.f ? 1.f : std::abs(a.scale);
  // A cap past 2^60 changes no score below 2^48 in 32 bits, and larger scores
  // that differ are 2^24 apart; one below 2^-60 leaves all weights alike.
  if (a.cap > 0x1p60f) {
    a.cap = 0.f;
  } else if (a.cap > 0.f && a.cap < 0x1p-60f) {
    a.cap = a.sign = 0.f;
    a.scale = 1.f;
  }
  const AttnWay how = WayOfAttention(a);
  if (how.way == HB_KV_WAY_PROMPT) return LaunchPrompt(a, ws, stream);
  switch (a.type) {
    case HB_TYPE_BF16: return LaunchDim<1>(a, how, ws, stream);
    case HB_TYPE_F16: return LaunchDim<2>(a, how, ws, stream);
    default: return LaunchDim<3>(a, how, ws, stream);
  }
}

}  // namespace hb
