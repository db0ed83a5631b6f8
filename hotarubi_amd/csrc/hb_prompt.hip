// Attention of many rows over the paged cache: prompts and chunks of them.
//
// Where a record serves many rows the conversion of its codes, not their
// bytes, is what counts (per record and wave 64 conversions and 32 permutes
// beside 32 products): here a launch of its own converts every record that a
// request looks at, once, into the workspace in the order of the matrix cores'
// operands, and the workgroups of all its rows draw them from there straight
// into LDS, for every wave's R tiles of 16 rows.  No one unit bounds
// it: at D 128 a wave's record is 256 cycles of products, about 260 of the
// softmax's 33 vector instructions and 8 exponentials, and 16 KB read from LDS
// (at D 64 the softmax is twice the products).  Three prompts of up to 4,096
// tokens, 32 heads on 8, D 128, bf16, 346 GFLOP, take 13 us for opening and
// 796,000 cycles: 353 us at the 2.27 GHz that an unbroken row of calls settles
// at (366 us a call, 945 TFLOP/s; a large library product reaches 1,231), 398 at
// 2.0 GHz between pauses, up to 486 at 1.64 GHz where such a row begins.  With
// the conversion in each workgroup a call took 454 where it took 366 opened.
// At D 256 one workgroup fills a CU's LDS, so a wave waits on its own chain, 1.3
// us a record: eight chunks of 100 to 256 tokens, fp16, a window of 1,024 and
// capped scores, take 63 us, 13 of them for opening and 7 for the cap.
#include <algorithm>

#include "hb_attn.h"

namespace hb {
namespace {

using namespace attn;

template <uint32_t parts>
struct Operand;  // K and q in the products: both exact in the tensors' type
template <>
struct Operand<1> {
  typedef bf16x8 type;
};
template <>
struct Operand<2> {
  typedef f16x8 type;
};

// Waves of a workgroup, 16-row tiles of a wave, workgroups of a CU (each holds
// two stages of two records in LDS).  Four waves a SIMD hide each other's waits: at D 128
// two workgroups of 8 waves with a tile each took prompts of up to 4,096 tokens
// in 369 us, one of 8 waves with two tiles in 406, one of 16 with one in 379.  At
// D 64 two tiles stay: three workgroups with one took prompts of 4,096 tokens in
// 137 us for 146 (15 heads on 5), but 182 for 171 (32 on 8) and short ones in 47
// for 44.
template <uint32_t D>
struct Shape {
  static constexpr uint32_t kWaves = 8, kTiles = D == 64 ? 2 : 1, kGroups = D == 256 ? 1 : 2;
  static constexpr uint32_t kRows = 16 * kWaves * kTiles;
};

// A record as operands: K [token tile][step][lane][16 B], then V^T [column
// tile][lane][16 B].
template <uint32_t D>
constexpr uint32_t kOpened = 128 * D;

// The place of record r of a request's walk among its opened records.
__device__ __forceinline__ uint32_t OpenedAt(const KvWalk& walk, uint32_t r) {
  return r < walk.head ? r : walk.head + r - walk.from;
}

// A wave a record.  `odd` says where f16 does not hold a scale (K's count for
// f16 queries): the rows that look at it take the general steps.  Tokens past
// the request's end, where any byte may lie, are given a scale of 1.
template <uint32_t parts, uint32_t D>
__global__ __launch_bounds__(256) void OpenKernel(const AttnArgs a) {
  const uint32_t lane = threadIdx.x % 64, n = lane % 16;
  const uint32_t at = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t pair = at / a.opened, i = at % a.opened, b = pair / a.heads;
  if (b >= a.batch) return;
  const KvSpan span =
      KvRequest(a.cu[b], a.cu[b + 1], a.kv_lens[b], a.prefix ? a.prefix[b] : 0, a.tokens,
                a.max_new, (uint64_t)a.columns * a.groups * 32);
  if (span.rows == 0) return;
  const int32_t pos0 = span.total - span.count;
  const KvWalk walk =
      KvRecords(pos0, pos0 + (int32_t)span.rows - 1, span.total, span.prefix, a.window);
  if (i >= walk.count) return;
  uint32_t* const odd = reinterpret_cast<uint32_t*>(a.ws) + at;
  const uint32_t record = __builtin_amdgcn_readfirstlane(PageRecord(
      a, walk, a.table + (uint64_t)b * a.table_stride, pair % a.heads, i, walk.count));
  if (record == kNoRecord) {
    if (lane == 0) *odd = 0;
    return;
  }
  const uint8_t* from = a.cache + (uint64_t)record * KvRecordBytes(D);
  Record<D> r;
  ReadKeys<D>(from, r);
  ReadValues<D>(from, r);
  const int32_t key0 = (int32_t)(32 * KvWalkRecord(walk, i));
  if (key0 + 32 > span.total) {
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j)
      if (KeyOf(key0, j) >= span.total)
        r.vs[j / 4] = (r.vs[j / 4] & ~(255u << (8 * (j % 4)))) | 127u << (8 * (j % 4));
#pragma unroll
    for (uint32_t k = 0; k < (D == 256 ? 2 : 1); ++k) {
      if (key0 + (int32_t)n >= span.total) r.ks[k] = (r.ks[k] & 0xFF00u) | 127u;
      if (key0 + 16 + (int32_t)n >= span.total) r.ks[k] = (r.ks[k] & 0xFFu) | 127u << 8;
    }
  }
  uint32_t outside = OutsideHalf(r.vs[0]) | OutsideHalf(r.vs[1]);
  if constexpr (parts == 2)
    outside |= OutsideHalf(r.ks[0] | (D == 256 ? r.ks[D == 256] : 0x7F7Fu) << 16);
  const uint64_t any = __builtin_amdgcn_ballot_w64(outside != 0);
  if (lane == 0) *odd = any != 0;
  u32x4* const to = reinterpret_cast<u32x4*>(a.opened_at + (uint64_t)at * kOpened<D>) + lane;
#pragma unroll
  for (uint32_t tile = 0; tile < 2; ++tile)
#pragma unroll
    for (uint32_t e = 0; e < D / 32; ++e) {
      const uint32_t word = tile * (D / 32) + e, w = r.k[word / 4][word % 4];
      // (253 and 254 as 255: NaN)
      const uint32_t byte = r.ks[D == 256 ? e / 4 : 0] >> (8 * tile) & 255u;
      const float scale = __uint_as_float((byte >= 253u ? 255u : byte) << 23);
      u32x4 x;
      x[0] = TwoAs<0, parts == 2>(w, scale);
      x[1] = TwoAs<1, parts == 2>(w, scale);
      x[2] = TwoAs<2, parts == 2>(w, scale);
      x[3] = TwoAs<3, parts == 2>(w, scale);
      to[word * 64] = x;
    }
#pragma unroll
  for (uint32_t e = 0; e < D / 32; ++e) {
    f16x8 v[2];
    ValueOperands<D, true>(r, e, &v[0], &v[1]);
    to[(D / 16 + 2 * e) * 64] = __builtin_bit_cast(u32x4, v[0]);
    to[(D / 16 + 2 * e + 1) * 64] = __builtin_bit_cast(u32x4, v[1]);
  }
}

// Rows of q and out pass through LDS, a wave's own part of it: a lane wants the
// D / 4 columns that are its of one row, memory whole rows (64 lines a load
// otherwise, at a line a cycle: 8 us of a workgroup's life).  A row's 16-byte
// pieces are permuted by the row, so that rows do not meet in a bank.
template <uint32_t D>
__device__ __forceinline__ uint32_t PieceAt(uint32_t row, uint32_t piece) {
  return row * (D * 2) + (piece ^ (row % (D / 8))) * 16;
}
template <uint32_t D>
struct RowPiece {  // the lane's piece of its `i`-th row of a tile, in memory's order
  uint32_t row, piece;
  __device__ __forceinline__ explicit RowPiece(uint32_t i) {
    const uint32_t lane = threadIdx.x % 64;
    row = i * (512 / D) + lane / (D / 8);
    piece = lane % (D / 8);
  }
};
template <uint32_t D>
__device__ __forceinline__ uint64_t RowStart(const RowSet& set, uint32_t row, uint64_t token,
                                             uint64_t head) {
  return (uint64_t)(set.span.first + row / set.group) * token +
         (uint64_t)(set.head * set.group + row % set.group) * head;
}
__device__ __forceinline__ bool Whole(const void* base, uint64_t token, uint64_t head) {
  return (token | head) % 8 == 0 && reinterpret_cast<uintptr_t>(base) % 16 == 0;
}
// Ends what the wave's LDS accesses before may still do.
__device__ __forceinline__ void WaveFence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// (`fine`: caps above kPlainCap, in a kernel of their own: beside the plain one
// in the loop, eight chunks with capped scores took 64.9 us for 63.8.)
template <uint32_t parts, uint32_t D, bool fine>
__global__ __launch_bounds__(64 * Shape<D>::kWaves, 2 * Shape<D>::kGroups) void PromptKernel(
    const AttnArgs a) {
  constexpr uint32_t kWaves = Shape<D>::kWaves, R = Shape<D>::kTiles, kSteps = D / 32;
  typedef typename Operand<parts>::type Q;
  struct Stage {
    struct {
      u32x4 k[2][kSteps][64], v[D / 16][64];
    } record[2];
  };
  static_assert(sizeof(Stage) == 2 * kOpened<D>, "records lie as they are opened");
  __shared__ __align__(16) Stage stages[2];

  const uint32_t lane = threadIdx.x % 64, g = lane / 16, n = lane % 16;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  // the tiles with the most keys first, of all requests
  const uint32_t head = blockIdx.x % a.heads, rest = blockIdx.x / a.heads;
  const uint32_t b = rest % a.batch, tile = a.tiles - 1 - rest / a.batch;
  const KvSpan span =
      KvRequest(a.cu[b], a.cu[b + 1], a.kv_lens[b], a.prefix ? a.prefix[b] : 0, a.tokens,
                a.max_new, (uint64_t)a.columns * a.groups * 32);
  const uint32_t group = a.q_heads / a.heads, rows = span.rows * group;
  const uint32_t first_row = tile * kWaves * R * 16;
  if (first_row >= rows) return;
  const uint32_t last_row = min(first_row + kWaves * R * 16, rows) - 1;
  const int32_t base_pos = span.total - span.count;
  const KvWalk walk =
      KvRecords(base_pos + (int32_t)(first_row / group), base_pos + (int32_t)(last_row / group),
                span.total, span.prefix, a.window);

  // a wave past the rows loads its share and computes nothing
  const uint32_t row0 = first_row + wave * R * 16;
  const RowSet set{span, group, head, row0, rows, max(row0, min(row0 + R * 16, rows) - 1)};
  const bool has_rows = row0 < rows;
  State<D, R> w;
  Q q[R][kSteps];
  Begin<D, R>(a, set, w);
  uint8_t* const rows_lds = reinterpret_cast<uint8_t*>(stages) + wave * (R * 16 * D * 2);
  static_assert(kWaves * R * 16 * D * 2 <= sizeof stages, "the rows fit the stages");
  const bool whole = Whole(a.q, a.q_token, a.q_head);
  Query<parts, D> query[R];
  u32x4 piece[R][D / 32];
#pragma unroll
  for (uint32_t t = 0; t < R; ++t) {
    if (whole) {
#pragma unroll
      for (uint32_t i = 0; i < D / 32; ++i) {
        const RowPiece<D> mine(i);
        const uint32_t row = row0 + t * 16 + mine.row;
        piece[t][i] = u32x4{0, 0, 0, 0};
        if (row < rows)
          piece[t][i] = *reinterpret_cast<const u32x4*>(
              static_cast<const typename TypeOf<parts>::type*>(a.q) +
              RowStart<D>(set, row, a.q_token, a.q_head) + mine.piece * 8);
      }
    } else {
      uint64_t at;
      const bool valid = QueryAt<parts, D>(a, set, t, &at);
      query[t].Load(a, at, valid);
    }
  }
  // the keys that any row of the wave sees
  const int32_t wave_hi = base_pos + (int32_t)(set.last / group);
  const int32_t wave_lo = SightOf(span, row0 / group, true, a.window).lo;

  const int32_t* const row = a.table + (uint64_t)b * a.table_stride;
  const uint32_t count = walk.count;
  // the request's opened records; those of pages that are not there, which
  // nothing was written for, are passed over below
  const KvWalk all = KvRecords(base_pos, base_pos + (int32_t)span.rows - 1, span.total,
                               span.prefix, a.window);
  const uint64_t first_opened = ((uint64_t)b * a.heads + head) * a.opened;
  bool slow = all.count > a.opened;
  for (uint32_t i = lane; i < count && !slow; i += 64) {
    const uint32_t r = OpenedAt(all, KvWalkRecord(walk, i));
    slow = reinterpret_cast<const uint32_t*>(a.ws)[first_opened + r] != 0;
  }
  slow = __builtin_amdgcn_ballot_w64(slow) != 0;
  auto key_of = [&](uint32_t i) { return (int32_t)(32 * KvWalkRecord(walk, i)); };
  // Scale bytes that f16 does not hold, or more records than were opened: the
  // rows a tile at a time on the general steps.  (Here, before the loop, so that
  // nothing of this stays in registers through it; and told to be unlikely, so
  // that its code lies behind: short prompts at D 64 36.9 us for 38.2.)
  if (__builtin_expect(slow, 0)) {
#pragma unroll 1
    for (uint32_t t = 0; t < R; ++t) {
      const uint32_t r0 = row0 + t * 16;
      if (r0 >= rows) return;
      const RowSet one{span, group, head, r0, rows, min(r0 + 16, rows) - 1};
      Rows<parts, D, 1> v;
      Begin<D, 1>(a, one, v);
      uint64_t from;
      const bool valid = QueryAt<parts, D>(a, one, 0, &from);
      Query<parts, D> again;
      again.Load(a, from, valid);
#pragma unroll
      for (uint32_t i = 0; i < kSteps; ++i) {
        bf16x8 x[parts];
        again.Parts(a, i, x);
#pragma unroll
        for (uint32_t p = 0; p < parts; ++p) v.q[0][p][i] = x[p];
      }
#pragma unroll 1
      for (uint32_t i = 0; i < count; ++i) {
        const uint32_t record =
            __builtin_amdgcn_readfirstlane(PageRecord(a, walk, row, head, i, count));
        if (record == kNoRecord) continue;
        const uint8_t* at_record = a.cache + (uint64_t)record * KvRecordBytes(D);
        Record<D> r;
        ReadKeys<D>(at_record, r);
        ReadValues<D>(at_record, r);
        f32x4 s[1][2];
        Scores<parts, D, 1>(r, v, s);
        Step<parts, D, 1>(a, span, r, key_of(i), s, v);
      }
      v.l[0] = RowSum(v.l[0]);
      Finish<parts, D, 1>(a, one, v);
    }
    return;
  }
  auto pages = [&](uint32_t i) { return PageRecord(a, walk, row, head, i + lane, count); };
  uint32_t base = 0, now = pages(0), after = count > 64 ? pages(64) : kNoRecord;
  auto hidden = [&](uint32_t i) {  // base <= i < base + 128
    return i >= count || __builtin_amdgcn_readlane((int)(i - base < 64 ? now : after),
                                                   (int)((i - base) % 64)) == (int)kNoRecord;
  };

  if (whole) {
#pragma unroll
    for (uint32_t t = 0; t < R; ++t)
#pragma unroll
      for (uint32_t i = 0; i < D / 32; ++i) {
        const RowPiece<D> mine(i);
        *reinterpret_cast<u32x4*>(rows_lds + t * (32 * D) +
                                  PieceAt<D>(mine.row, mine.piece)) = piece[t][i];
      }
    WaveFence();
#pragma unroll
    for (uint32_t t = 0; t < R; ++t)
#pragma unroll
      for (uint32_t i = 0; i < kSteps; ++i)
        *reinterpret_cast<u32x4*>(&query[t].x[2 * i]) = *reinterpret_cast<const u32x4*>(
            rows_lds + t * (32 * D) + PieceAt<D>(n, g * (D / 32) + i));
  }
#pragma unroll
  for (uint32_t t = 0; t < R; ++t)
#pragma unroll
    for (uint32_t i = 0; i < kSteps; ++i) {
      float y[8];
      query[t].Eight(a, i, y);
#pragma unroll
      for (int j = 0; j < 8; ++j) q[t][i][j] = (typename TypeOf<parts>::type)y[j];
    }
  __syncthreads();  // the rows have left the stages

  // a stage's loads, kOps pieces of 1 KB a wave
  constexpr uint32_t kOps = 2 * kOpened<D> / 1024 / kWaves;
  static_assert(kOps * kWaves * 512 == kOpened<D>, "whole loads");
  const uint32_t stages_at = (uint32_t) reinterpret_cast<uintptr_t>(
      (__attribute__((address_space(3))) uint8_t*)reinterpret_cast<uint8_t*>(stages));
  auto fetch = [&](uint32_t i, uint32_t stage) {
#pragma unroll
    for (uint32_t e = 0; e < kOps; ++e) {
      const uint32_t piece = wave * kOps + e, u = piece / (kOpened<D> / 1024);
      // past the last record the stage holds it twice
      const uint32_t r = OpenedAt(all, KvWalkRecord(walk, min(i + u, count - 1)));
      ring::Dma16(a.opened_at + (first_opened + r) * kOpened<D> +
                      piece % (kOpened<D> / 1024) * 1024,
                  lane * 16, stages_at + stage * (uint32_t)sizeof(Stage) + piece * 1024);
    }
  };
  if (count > 0) fetch(0, 0);
#pragma unroll 1
  for (uint32_t i = 0; i < count; i += 2) {
    const uint32_t in = i / 2 % 2;
    const Stage& stage = stages[in];
    ring::WaitVm<0>();
    ring::WaitLds();
    asm volatile("" ::: "memory");
    // every wave's loads of the stage are there, and its reads of the other
    // are done
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (i + 2 < count) fetch(i + 2, 1 - in);
    if (i + 1 - base >= 128) {
      base += 64;
      now = after;
      after = pages(base + 64);
    }
#pragma unroll
    for (uint32_t u = 0; u < 2; ++u) {
      if (!has_rows || hidden(i + u)) continue;
      const int32_t key0 = key_of(i + u);
      if (!((key0 <= wave_hi && key0 + 31 >= wave_lo) || key0 < span.prefix)) continue;
      f32x4 s[R][2];
#pragma unroll
      for (uint32_t t = 0; t < R; ++t) s[t][0] = s[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (uint32_t e = 0; e < kSteps; ++e)
#pragma unroll
        for (uint32_t k = 0; k < 2; ++k) {
          const Q x = __builtin_bit_cast(Q, stage.record[u].k[k][e][lane]);
#pragma unroll
          for (uint32_t t = 0; t < R; ++t) s[t][k] = Product(x, q[t][e], s[t][k]);
        }
      const float c = PowerOf(a);
      if (a.cap > 0.f) Cap<fine, R>(a, s);
      Hide<D, R>(w, key0, s);
      f16x8 pt[R];
#pragma unroll
      for (uint32_t t = 0; t < R; ++t) {
        float p[8];
        Raise<D, R>(w, t, s[t], c, false);  // (V is within f16 here)
        Weights<D, R>(w, t, s[t], c, p);
        pt[t] = HalfWeights(p);
      }
#pragma unroll
      for (uint32_t e = 0; e < D / 16; ++e) {
        const f16x8 x = __builtin_bit_cast(f16x8, stage.record[u].v[e][lane]);
#pragma unroll
        for (uint32_t t = 0; t < R; ++t) w.o[t][e] = Product(x, pt[t], w.o[t][e]);
      }
    }
  }
#pragma unroll
  for (uint32_t t = 0; t < R; ++t) w.l[t] = RowSum(w.l[t]);
  ring::WaitVm<0>();  // no load into LDS outlives its stage
  if (!Whole(a.out, a.out_token, a.out_head)) {
    if (has_rows) Finish<parts, D, R>(a, set, w);
    return;
  }
  __syncthreads();  // the stages have been read
  typedef typename TypeOf<parts>::four V;
#pragma unroll
  for (uint32_t t = 0; t < R; ++t) {
    const float inv = w.l[t] == 0.f ? 0.f : 1.f / w.l[t];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
      for (uint32_t c = 0; c < D / 16; c += 4) {
        V y;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
          y[j] = Rounded<typename TypeOf<parts>::type>(w.o[t][c + j][i] * inv);
        const uint32_t col = (4 * g + i) * (D / 16) + c;
        *reinterpret_cast<V*>(rows_lds + t * (32 * D) + PieceAt<D>(n, col / 8) + col % 8 * 2) = y;
      }
  }
  WaveFence();
#pragma unroll
  for (uint32_t t = 0; t < R; ++t)
#pragma unroll
    for (uint32_t i = 0; i < D / 32; ++i) {
      const RowPiece<D> mine(i);
      const uint32_t row = row0 + t * 16 + mine.row;
      if (row < rows)
        *reinterpret_cast<u32x4*>(static_cast<typename TypeOf<parts>::type*>(a.out) +
                                  RowStart<D>(set, row, a.out_token, a.out_head) +
                                  mine.piece * 8) = *reinterpret_cast<const u32x4*>(
            rows_lds + t * (32 * D) + PieceAt<D>(mine.row, mine.piece));
    }
}

}  // namespace

uint32_t PromptTiles(uint32_t dim) {
  return dim == 64 ? Shape<64>::kTiles : dim == 128 ? Shape<128>::kTiles : Shape<256>::kTiles;
}
uint32_t PromptRows(uint32_t dim) {
  return dim == 64 ? Shape<64>::kRows : dim == 128 ? Shape<128>::kRows : Shape<256>::kRows;
}

// Records of a request that may be looked at, and the bytes of a launch's
// opened ones.
static uint64_t OpenedRecords(const AttnArgs& a) {
  uint64_t records = ((uint64_t)a.max_kv + 31) / 32;
  if (a.window > 0 && a.prefix == nullptr)
    records = std::min<uint64_t>(records, ((uint64_t)a.window + a.max_new + 62) / 32);
  return std::max<uint64_t>(records, 1);
}
uint64_t PromptBytes(const AttnArgs& a) {
  const uint64_t records = OpenedRecords(a) * a.batch * a.heads;
  return records * 128 * a.dim + (records * 4 + 15) / 16 * 16;
}

template <uint32_t parts, uint32_t D>
static hipError_t LaunchOf(AttnArgs& a, hipStream_t stream) {
  const uint64_t rows = (uint64_t)a.max_new * (a.q_heads / a.heads);
  const uint64_t tiles = (rows + Shape<D>::kRows - 1) / Shape<D>::kRows;
  const uint64_t pairs = (uint64_t)a.batch * a.heads, records = pairs * a.opened;
  const uint64_t grid = tiles * pairs;
  if (grid > 0x7FFFFFFFu || records > 0x7FFFFFFFu) return hipErrorInvalidValue;
  a.tiles = (uint32_t)tiles;
  OpenKernel<parts, D><<<(uint32_t)((records + 3) / 4), 256, 0, stream>>>(a);
  if (a.cap > kPlainCap)
    PromptKernel<parts, D, true><<<(uint32_t)grid, 64 * Shape<D>::kWaves, 0, stream>>>(a);
  else
    PromptKernel<parts, D, false><<<(uint32_t)grid, 64 * Shape<D>::kWaves, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t LaunchPrompt(const AttnArgs& in, Workspace& ws, hipStream_t stream) {
  AttnArgs a = in;
  const hipError_t err = GrowWorkspace(ws, PromptBytes(a), stream);
  if (err != hipSuccess) return err;
  a.opened = (uint32_t)OpenedRecords(a);
  a.ws = ws.ptr + kSplitCounters;  // a word a record, then the records
  a.opened_at = reinterpret_cast<uint8_t*>(a.ws) +
                ((uint64_t)a.opened * a.batch * a.heads * 4 + 15) / 16 * 16;
  const bool half = a.type == HB_TYPE_F16;
  switch (a.dim) {
    case 64: return half ? LaunchOf<2, 64>(a, stream) : LaunchOf<1, 64>(a, stream);
    case 128: return half ? LaunchOf<2, 128>(a, stream) : LaunchOf<1, 128>(a, stream);
    default: return half ? LaunchOf<2, 256>(a, stream) : LaunchOf<1, 256>(a, stream);
  }
}

}  // namespace hb
