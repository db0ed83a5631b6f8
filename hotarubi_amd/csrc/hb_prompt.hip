// Attention of many rows over the paged cache: prompts and chunks of them.
//
// Where a record serves many rows the conversion of its codes, not their
// bytes, is what counts (per record and wave 64 conversions and 32 permutes
// beside 32 products): here a workgroup's waves convert two records together, a
// share each, into LDS in the order of the operands, and every wave reads them
// for its own R tiles of 16 rows.
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

// Waves of a workgroup and 16-row tiles of a wave: two waves a SIMD, so 256
// registers each, of which sums and queries take 6 D / 16 a tile.
template <uint32_t D>
struct Shape {
  static constexpr uint32_t kWaves = D == 64 ? 4 : 8, kTiles = D == 64 ? 4 : D == 128 ? 2 : 1;
  static constexpr uint32_t kRows = 16 * kWaves * kTiles;
};

// A wave's share of a stage (two records), as loaded: kKeys operand blocks of K
// (8 columns a lane of 16 tokens) and kPairs pairs of column tiles of V.
template <uint32_t D>
struct Share {
  static constexpr uint32_t kKeys = D / 8 / Shape<D>::kWaves;
  static constexpr uint32_t kPairs = D / 16 / Shape<D>::kWaves;
  alignas(16) uint32_t k[kKeys];
  uint32_t ks[D == 256 ? 2 : 1];
  u32x4 v[D / 64];
  uint32_t vs[2];
};

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

template <uint32_t parts, uint32_t D>
__global__ __launch_bounds__(64 * Shape<D>::kWaves, 2) void PromptKernel(
    const AttnArgs a) {
  constexpr uint32_t kWaves = Shape<D>::kWaves, R = Shape<D>::kTiles, kSteps = D / 32;
  constexpr uint32_t kKeys = Share<D>::kKeys, kPairs = Share<D>::kPairs;
  constexpr bool half_keys = parts == 2;
  typedef typename Operand<parts>::type Q;
  struct Stage {
    u32x4 k[2][2][kSteps][64], v[2][D / 16][64];
  };
  __shared__ Stage stages[2];
  __shared__ uint32_t odd[2];

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

  // a wave past the rows converts its share and computes nothing
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

  if (threadIdx.x < 2) odd[threadIdx.x] = 0;
  const int32_t* const row = a.table + (uint64_t)b * a.table_stride;
  const uint32_t count = walk.count;
  auto pages = [&](uint32_t i) { return PageRecord(a, walk, row, head, i + lane, count); };
  uint32_t base = 0, now = pages(0), after = count > 64 ? pages(64) : kNoRecord;
  auto place = [&](uint32_t i) {  // base <= i < base + 128
    return i < count ? (uint32_t)__builtin_amdgcn_readlane(
                           (int)(i - base < 64 ? now : after), (int)((i - base) % 64))
                     : kNoRecord;
  };

  // the wave's share: K blocks wave * kKeys .. of [record][token tile][step],
  // V pairs wave * kPairs .. of [record][pair]
  const uint32_t k_record = wave * kKeys / (2 * kSteps), k_tile = wave * kKeys / kSteps % 2,
                 k_step = wave * kKeys % kSteps;
  const uint32_t v_record = wave * kPairs / kSteps, v_pair = wave * kPairs % kSteps;
  Share<D> share;
  uint32_t at[2];
  auto load = [&](uint32_t i) {
    at[0] = place(i);
    at[1] = place(i + 1);
    const uint32_t k_at = k_record ? at[1] : at[0], v_at = v_record ? at[1] : at[0];
    if (k_at != kNoRecord) {
      const uint8_t* from = a.cache + (uint64_t)k_at * KvRecordBytes(D);
      const uint32_t word = k_tile * kSteps + k_step;
      const uint8_t* x = from + word / 4 * 1024 + lane * 16 + word % 4 * 4;
      // within one 16-byte piece
      if constexpr (kKeys == 4) {
        *reinterpret_cast<u32x4*>(share.k) = *reinterpret_cast<const u32x4*>(x);
      } else {
        const uint2 two = *reinterpret_cast<const uint2*>(x);
        share.k[0] = two.x;
        share.k[1] = two.y;
      }
      const uint32_t block = D == 256 ? 2 * g : g * D / 128;
      share.ks[0] = from[32 * D + block * 32 + n * 2 + k_tile];
      if (D == 256) share.ks[D == 256] = from[32 * D + block * 32 + 32 + n * 2 + k_tile];
    }
    if (v_at != kNoRecord) {
      const uint8_t* from = a.cache + (uint64_t)v_at * KvRecordBytes(D);
#pragma unroll
      for (uint32_t c = 0; c < D / 64; ++c)
        share.v[c] = *reinterpret_cast<const u32x4*>(from + 16 * D + c * 1024 + lane * 16);
      const uint2 vs = *reinterpret_cast<const uint2*>(from + 33 * D + n * D / 512 * 32 + g * 8);
      share.vs[0] = vs.x;
      share.vs[1] = vs.y;
    }
  };
  auto key_of = [&](uint32_t i) { return (int32_t)(32 * KvWalkRecord(walk, i)); };

  bool slow = false;
  load(0);
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
  __syncthreads();  // odd
  for (uint32_t i = 0; i < count; i += 2) {
    Stage& stage = stages[i / 2 % 2];
    const uint32_t here[2] = {at[0], at[1]};
    uint32_t bad = 0;
    if (here[k_record] != kNoRecord) {
#pragma unroll
      for (uint32_t j = 0; j < kKeys; ++j) {
        const float scale = __uint_as_float(share.ks[D == 256 ? (k_step + j) / 4 : 0] << 23);
        u32x4 x;
        x[0] = TwoAs<0, half_keys>(share.k[j], scale);
        x[1] = TwoAs<1, half_keys>(share.k[j], scale);
        x[2] = TwoAs<2, half_keys>(share.k[j], scale);
        x[3] = TwoAs<3, half_keys>(share.k[j], scale);
        stage.k[k_record][k_tile][k_step + j][lane] = x;
      }
      if constexpr (half_keys) {
        const bool outside = share.ks[0] - 104 > 36 ||
                             (D == 256 && share.ks[D == 256] - 104 > 36);
        bad |= outside && key_of(i + k_record) + (int32_t)(16 * k_tile + n) < span.total;
      }
    }
    if (here[v_record] != kNoRecord) {
      const int32_t key0 = key_of(i + v_record);
      if (key0 + 32 > span.total) {  // past the request's end any byte may lie
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
          if (KeyOf(key0, j) >= span.total)
            share.vs[j / 4] =
                (share.vs[j / 4] & ~(255u << (8 * (j % 4)))) | 127u << (8 * (j % 4));
      }
      bad |= OutsideHalf(share.vs[0]) | OutsideHalf(share.vs[1]);
#pragma unroll
      for (uint32_t j = 0; j < kPairs; ++j) {
        uint32_t x[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
          // byte e * kSteps + v_pair + j of the lane's, at byte 0 of a word
          uint32_t word;
          if constexpr (D == 64) word = share.v[0][e / 2] >> ((e % 2 * 2 + v_pair) * 8);
          else if constexpr (D == 128) word = share.v[e / 4][e % 4] >> (v_pair * 8);
          else word = (v_pair < 4 ? share.v[e / 2][e % 2 * 2] : share.v[e / 2][e % 2 * 2 + 1]) >> ((v_pair % 4 + j) * 8);
          x[e] = TwoAs<0, true>(word, ScaleOf(share.vs[e / 4], e % 4));
        }
        u32x4 lo, hi;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
          lo[e] = __builtin_amdgcn_perm(x[2 * e + 1], x[2 * e], 0x05040100u);
          hi[e] = __builtin_amdgcn_perm(x[2 * e + 1], x[2 * e], 0x07060302u);
        }
        stage.v[v_record][2 * (v_pair + j)][lane] = lo;
        stage.v[v_record][2 * (v_pair + j) + 1][lane] = hi;
      }
    }
    if (__builtin_amdgcn_ballot_w64(bad != 0) != 0 && lane == 0) odd[i / 2 % 2] = 1;
    if (i + 2 < count) {
      if (i + 4 - base > 128) {
        base += 64;
        now = after;
        after = pages(base + 64);
      }
      load(i + 2);
    }
    __syncthreads();
    if (odd[i / 2 % 2] != 0) {  // the same for every wave: the next stage has a flag of its own
      slow = true;
      break;
    }
#pragma unroll
    for (uint32_t u = 0; u < 2; ++u) {
      if (here[u] == kNoRecord || !has_rows) continue;
      const int32_t key0 = key_of(i + u);
      if (!((key0 <= wave_hi && key0 + 31 >= wave_lo) || key0 < span.prefix)) continue;
      f32x4 s[R][2];
#pragma unroll
      for (uint32_t t = 0; t < R; ++t) s[t][0] = s[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (uint32_t e = 0; e < kSteps; ++e)
#pragma unroll
        for (uint32_t k = 0; k < 2; ++k) {
          const Q x = __builtin_bit_cast(Q, stage.k[u][k][e][lane]);
#pragma unroll
          for (uint32_t t = 0; t < R; ++t) s[t][k] = Product(x, q[t][e], s[t][k]);
        }
      const float c = Capped<parts, R>(a, s);
      Hide<D, R>(w, key0, s);
      f16x8 pt[R];
#pragma unroll
      for (uint32_t t = 0; t < R; ++t) {
        float p[8], shrink;
        Raise<D, R>(w, t, s[t], c, &shrink);
        Weights<D, R>(w, t, s[t], c, p);
        pt[t] = HalfWeights(p);
      }
#pragma unroll
      for (uint32_t e = 0; e < D / 16; ++e) {
        const f16x8 x = __builtin_bit_cast(f16x8, stage.v[u][e][lane]);
#pragma unroll
        for (uint32_t t = 0; t < R; ++t) w.o[t][e] = Product(x, pt[t], w.o[t][e]);
      }
    }
  }
  if (!slow) {
#pragma unroll
    for (uint32_t t = 0; t < R; ++t) w.l[t] = RowSum(w.l[t]);
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
            y[j] = (typename TypeOf<parts>::type)(w.o[t][c + j][i] * inv);
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
    return;
  }
  // scale bytes that f16 does not hold: the rows again, a tile at a time, on
  // the general steps
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
}

}  // namespace

uint32_t PromptRows(uint32_t dim) {
  return dim == 64 ? Shape<64>::kRows : dim == 128 ? Shape<128>::kRows : Shape<256>::kRows;
}

template <uint32_t D>
static hipError_t LaunchDim(AttnArgs& a, hipStream_t stream) {
  const uint64_t rows = (uint64_t)a.max_new * (a.q_heads / a.heads);
  const uint64_t tiles = (rows + Shape<D>::kRows - 1) / Shape<D>::kRows;
  const uint64_t grid = tiles * a.batch * a.heads;
  if (grid > 0x7FFFFFFFu) return hipErrorInvalidValue;
  a.tiles = (uint32_t)tiles;
  if (a.type == HB_TYPE_F16)
    PromptKernel<2, D><<<(uint32_t)grid, 64 * Shape<D>::kWaves, 0, stream>>>(a);
  else
    PromptKernel<1, D><<<(uint32_t)grid, 64 * Shape<D>::kWaves, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t LaunchPrompt(const AttnArgs& in, hipStream_t stream) {
  AttnArgs a = in;
  switch (a.dim) {
    case 64: return LaunchDim<64>(a, stream);
    case 128: return LaunchDim<128>(a, stream);
    default: return LaunchDim<256>(a, stream);
  }
}

}  // namespace hb
