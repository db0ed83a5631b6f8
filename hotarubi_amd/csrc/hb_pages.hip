// Pages of a paged cache that requests share, give back and move: forks, the
// pages of requests that end, renumbering to the front, and the copies that
// these ask for.  A page is in use while a row of the block table names it, so
// there are no counts to keep: marks in LDS, a bit per page, find the pages
// that nothing names.  What they cost is launches and chains of loads: 4 forks of 8
// requests 5.0 us, 96 of 160 5.4; 256 of 512 requests with 17,000 pages end in 12.6
// us, their cache is marked in 10 and renumbered in 5.  The marks are one workgroup's,
// so they grow with the table: 128 of 256 requests with 390,000 entries end in 136
// us, the others' are marked in 38 and renumbered in 13.  The copies are bound by
// memory: 96 pages of 132 KB in two layers, 50 MB read and written, 8.3 us.
#include <algorithm>

#include "hb_internal.h"

namespace hb {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t PagesOf(int32_t tokens, uint32_t page) {
  const uint32_t n = tokens < 0 ? 0u : (uint32_t)tokens;
  return n / page + (n % page != 0 ? 1u : 0u);
}

// Inclusive sum over the workgroup's threads; *total the sum of all.  `part`
// holds a value per wave.
template <uint32_t threads>
__device__ __forceinline__ uint32_t BlockSum(uint32_t x, uint32_t* part, uint32_t* total) {
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  for (uint32_t d = 1; d < 64; d *= 2) {
    const uint32_t y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();  // the values of an earlier call have been read
  if (lane == 63) part[wave] = x;
  __syncthreads();
  uint32_t sum = 0;
  for (uint32_t w = 0; w < threads / 64; ++w) {
    if (w < wave) x += part[w];
    sum += part[w];
  }
  *total = sum;
  return x;
}

// ------------------------------------------------------------------- fork --

constexpr uint32_t kForkThreads = 256, kForkWaves = kForkThreads / 64;
constexpr uint32_t kRowWindow = 8192;  // rows of the table looked at together

// Every workgroup finds for itself which forks are in order (targets that are
// a source, or another's target before them, are not) and sums the pages that
// they want, as the step plan's do; then its waves take forks of their own and
// copy their rows' entries.  Sources are not written, so no workgroup reads
// what another writes.
__global__ __launch_bounds__(kForkThreads) void ForkKernel(const ForkArgs a) {
  __shared__ uint32_t first[kRowWindow], is_source[kRowWindow / 32];
  __shared__ uint32_t bad[kMostForkRows / 32], again[kMostForkRows / 32];
  __shared__ uint32_t place[kForkThreads], part[kForkWaves];
  const uint32_t tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  constexpr uint32_t kNone = 0xFFFFFFFFu;
  // a thread's first fork, which is most often its only one, is loaded once
  const bool any = tid < a.forks;
  const uint32_t source0 = any ? (uint32_t)a.source[tid] : kNone;
  const uint32_t target0 = any ? (uint32_t)a.target[tid] : kNone;
  const uint32_t free_count = (uint32_t)max(0, min(*a.free_count, (int32_t)a.free_size));
  const int32_t len0 = source0 < a.batch ? a.lens[source0] : 0;
  auto source = [&](uint32_t i) { return i == tid ? source0 : (uint32_t)a.source[i]; };
  auto target = [&](uint32_t i) { return i == tid ? target0 : (uint32_t)a.target[i]; };
  for (uint32_t i = tid; i < (a.forks + 31) / 32; i += kForkThreads) bad[i] = again[i] = 0;
  for (uint32_t base = 0; base < a.batch; base += kRowWindow) {
    const uint32_t rows = min(kRowWindow, a.batch - base);
    __syncthreads();  // the window before has been read
    for (uint32_t i = tid; i < rows; i += kForkThreads) first[i] = kNone;
    for (uint32_t i = tid; i < kRowWindow / 32; i += kForkThreads) is_source[i] = 0;
    __syncthreads();
    for (uint32_t i = tid; i < a.forks; i += kForkThreads) {
      const uint32_t s = source(i) - base, t = target(i) - base;
      if (s < rows) atomicOr(&is_source[s / 32], 1u << (s % 32));
      if (t < rows) atomicMin(&first[t], i);
    }
    __syncthreads();
    for (uint32_t i = tid; i < a.forks; i += kForkThreads) {
      const uint32_t t = target(i) - base;
      if (t >= rows) continue;
      if (first[t] != i) atomicOr(&again[i / 32], 1u << (i % 32));
      if (first[t] != i || (is_source[t / 32] >> (t % 32) & 1u))
        atomicOr(&bad[i / 32], 1u << (i % 32));
    }
    // rows that are no target keep their lengths; the others' first fork says
    for (uint32_t i = blockIdx.x * kForkThreads + tid; i < rows; i += gridDim.x * kForkThreads)
      if (first[i] == kNone) a.lens_out[base + i] = a.lens[base + i];
  }
  __syncthreads();
  uint32_t wanted = 0, taken = 0, refused = 0;
  constexpr uint32_t kRefused = 0xFFFFFFFFu, kNoPage = 0xFFFFFFFEu;
  for (uint32_t base = 0; base < a.forks; base += kForkThreads) {
    const uint32_t i = base + tid;
    bool fits = false, need = false;
    if (i < a.forks) {
      const uint32_t s = source(i), t = target(i);
      if (s < a.batch && t < a.batch && !(bad[i / 32] >> (i % 32) & 1u)) {
        const int32_t n = i == tid ? len0 : a.lens[s];
        fits = PagesOf(n, a.page) <= a.columns;
        need = fits && n > 0 && (uint32_t)n % a.page != 0;
      }
    }
    uint32_t total, good, spare;
    const uint32_t stop = wanted + BlockSum<kForkThreads>(need, part, &total);
    const bool ok = fits && (!need || stop <= free_count);
    place[tid] = !ok ? kRefused : need ? free_count - stop : kNoPage;
    BlockSum<kForkThreads>(ok && need, part, &good);
    BlockSum<kForkThreads>(i < a.forks && !ok, part, &spare);
    wanted += total;
    taken += good;
    refused += spare;
    // (the sums' barriers stand between place's writes and its reads)
    const uint32_t chunk = min(kForkThreads, a.forks - base);
    for (uint32_t j = blockIdx.x * kForkWaves + wave; j < chunk; j += gridDim.x * kForkWaves) {
      const uint32_t f = base + j, at = place[j];
      const uint32_t s = (uint32_t)a.source[f], t = (uint32_t)a.target[f];
      int32_t from = -1, to = -1;
      if (at != kRefused) {
        const int32_t n = a.lens[s];
        const uint32_t whole = n > 0 ? (uint32_t)n / a.page : 0u;
        const int32_t* const x = a.table + (uint64_t)s * a.table_stride;
        int32_t* const y = a.table + (uint64_t)t * a.table_stride;
        for (uint32_t c = lane; c < whole; c += 64) y[c] = x[c];
        if (at != kNoPage) {
          from = x[whole];
          to = a.free_pages[at];
          if (lane == 0) y[whole] = to;
        }
      }
      if (lane == 0) {
        a.pairs[2 * (uint64_t)f] = from;
        a.pairs[2 * (uint64_t)f + 1] = to;
        if (t < a.batch && !(again[f / 32] >> (f % 32) & 1u))
          a.lens_out[t] = at != kRefused ? max(0, a.lens[s]) : a.lens[t];
      }
    }
    __syncthreads();  // place has been read
  }
  if (blockIdx.x == 0 && tid == 0) {
    a.status[0] = (int32_t)taken;
    a.status[1] = (int32_t)refused;
  }
}

// ------------------------------------------------------------------- copy --

constexpr uint32_t kCopyThreads = 256;
static_assert(kCopyPiece == kCopyThreads * 16 * 2, "two loads a thread");

// A workgroup takes a piece of a page in one layer, for pairs `stripes` apart:
// it looks at 64 of them at a time, since lists of moves are mostly empty.
__global__ __launch_bounds__(kCopyThreads) void CopyKernel(const CopyArgs a) {
  const uint32_t lane = threadIdx.x % 64;
  const uint32_t stripe = blockIdx.x % a.stripes, slot = blockIdx.x / a.stripes;
  const uint64_t piece = slot % a.pieces;
  uint8_t* const base = a.base + slot / a.pieces * a.layer_bytes + piece * kCopyPiece;
  const uint64_t left = a.page_bytes - piece * kCopyPiece;
  const uint32_t at = threadIdx.x * 16;
  const bool one = at < left, two = at + kCopyPiece / 2 < left;
  for (uint64_t i = stripe; i < a.count; i += 64ull * a.stripes) {
    const uint64_t mine = i + (uint64_t)lane * a.stripes;
    uint32_t from = 0xFFFFFFFFu, to = 0xFFFFFFFFu;
    if (mine < a.count) {
      from = (uint32_t)a.pairs[2 * mine];
      to = (uint32_t)a.pairs[2 * mine + 1];
    }
    uint64_t todo = __builtin_amdgcn_ballot_w64(from < a.pages && to < a.pages && from != to);
    while (todo != 0) {
      const int j = __builtin_ctzll(todo);
      todo &= todo - 1;
      const uint8_t* const x =
          base + (uint32_t)__builtin_amdgcn_readlane((int)from, j) * a.page_bytes + at;
      uint8_t* const y = base + (uint32_t)__builtin_amdgcn_readlane((int)to, j) * a.page_bytes + at;
      u32x4 u, v;
      if (one) u = *reinterpret_cast<const u32x4*>(x);
      if (two) v = *reinterpret_cast<const u32x4*>(x + kCopyPiece / 2);
      if (one) *reinterpret_cast<u32x4*>(y) = u;
      if (two) *reinterpret_cast<u32x4*>(y + kCopyPiece / 2) = v;
    }
  }
}

// --------------------------------------------------------- free, compact --

constexpr uint32_t kMarkThreads = 1024, kMarkWords = kMostPages / 32;

constexpr uint32_t kMarkWaves = kMarkThreads / 64;
// The length of the lane's row among the wave's first 64, which a kernel asks for
// before anything else.
__device__ __forceinline__ int32_t FirstLength(const int32_t* lens, uint32_t batch) {
  const uint32_t mine = threadIdx.x / 64 + threadIdx.x % 64 * kMarkWaves;
  return mine < batch ? lens[mine] : 0;
}
// mark(page, kind) for every entry of a row's pages; which(row), a row a lane, is
// the ballot of the rows' kinds.  A wave takes rows kMarkWaves apart, the lengths
// of 64 of them at once and then the entries of kEach of them, as loads that wait
// for one another are what this takes (512 rows of 8 to 55 pages: the compaction's
// marks 7.8 us, 14.5 with four entries a thread at a time, a length each).
template <class Which, class Mark>
__device__ __forceinline__ void EachEntry(const int32_t* table, const int32_t* lens,
                                          int32_t first_length, uint32_t batch, uint32_t columns,
                                          uint32_t stride, uint32_t page, uint32_t pages,
                                          Which&& which, Mark&& mark) {
  constexpr uint32_t kWaves = kMarkWaves, kEach = 16;
  const uint32_t lane = threadIdx.x % 64;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  for (uint64_t base = wave; base < batch; base += 64 * kWaves) {
    const uint64_t mine = base + (uint64_t)lane * kWaves;
    const int32_t length = base == wave ? first_length : mine < batch ? lens[mine] : 0;
    const uint32_t of = min(columns, PagesOf(length, page));
    const uint32_t rows = (uint32_t)min((uint64_t)64, (batch - base + kWaves - 1) / kWaves);
    const uint64_t marks = which(mine);
    for (uint32_t r = 0; r < rows; r += kEach) {
      uint32_t entry[kEach];
#pragma unroll
      for (uint32_t j = 0; j < kEach; ++j) {
        entry[j] = 0xFFFFFFFFu;
        if (r + j >= rows) continue;  // (the same in all lanes)
        const uint32_t n = (uint32_t)__builtin_amdgcn_readlane((int)of, (int)(r + j));
        if (lane < n)
          entry[j] = (uint32_t)table[(base + (uint64_t)(r + j) * kWaves) * stride + lane];
      }
#pragma unroll
      for (uint32_t j = 0; j < kEach; ++j) {
        if (r + j >= rows) continue;
        if (entry[j] < pages) mark(entry[j], marks >> (r + j) & 1u);
      }
    }
    for (uint32_t r = 0; r < rows; ++r) {  // what is past 64 pages of a row
      const uint32_t n = (uint32_t)__builtin_amdgcn_readlane((int)of, (int)r);
      const uint64_t row = base + (uint64_t)r * kWaves;
      for (uint32_t c = 64; c < n; c += 64 * kEach) {
        uint32_t entry[kEach];
#pragma unroll
        for (uint32_t j = 0; j < kEach; ++j) {
          const uint32_t at = c + j * 64 + lane;
          entry[j] = at < n ? (uint32_t)table[row * stride + at] : 0xFFFFFFFFu;
        }
#pragma unroll
        for (uint32_t j = 0; j < kEach; ++j)
          if (entry[j] < pages) mark(entry[j], marks >> r & 1u);
      }
    }
  }
}

// One workgroup: the marks are a bit per page in its LDS, and a second launch
// or a wait between workgroups would take longer than the table's entries.
__global__ __launch_bounds__(kMarkThreads) void FreeKernel(const FreeArgs a) {
  __shared__ uint32_t kept[kMarkWords], gone[kMarkWords], ends[kMostForkRows / 32];
  __shared__ uint32_t part[kMarkThreads / 64];
  const uint32_t tid = threadIdx.x, words = (a.pages + 31) / 32;
  // what is most often all of the lists, before anything waits
  const int32_t length = FirstLength(a.lens, a.batch);
  const uint32_t end0 = tid < a.count ? (uint32_t)a.rows[tid] : ~0u;
  const uint32_t free0 = tid < a.free_size ? (uint32_t)a.free_pages[tid] : ~0u;
  const int32_t len0 = tid < a.batch ? a.lens[tid] : 0;
  const uint32_t free_count = (uint32_t)max(0, min(*a.free_count, (int32_t)a.free_size));
  for (uint32_t i = tid; i < words; i += kMarkThreads) kept[i] = gone[i] = 0;
  for (uint32_t i = tid; i < (a.batch + 31) / 32; i += kMarkThreads) ends[i] = 0;
  __syncthreads();
  for (uint32_t i = tid; i < a.count; i += kMarkThreads) {
    const uint32_t r = i == tid ? end0 : (uint32_t)a.rows[i];
    if (r < a.batch) atomicOr(&ends[r / 32], 1u << (r % 32));
  }
  for (uint32_t i = tid; i < free_count; i += kMarkThreads) {
    const uint32_t p = i == tid ? free0 : (uint32_t)a.free_pages[i];
    if (p < a.pages) atomicOr(&kept[p / 32], 1u << (p % 32));
  }
  __syncthreads();
  for (uint32_t i = tid; i < a.batch; i += kMarkThreads)
    a.lens_out[i] = ends[i / 32] >> (i % 32) & 1u ? 0 : i == tid ? len0 : a.lens[i];
  EachEntry(a.table, a.lens, length, a.batch, a.columns, a.table_stride, a.page, a.pages,
            [&](uint64_t row) {
              return __builtin_amdgcn_ballot_w64(
                  row < a.batch && (ends[row / 32] >> (row % 32) & 1u) != 0);
            },
            [&](uint32_t p, bool ended) {
              atomicOr((ended ? gone : kept) + p / 32, 1u << (p % 32));
            });
  __syncthreads();
  // the highest page first: thread 0 takes the last words
  const uint32_t each = (words + kMarkThreads - 1) / kMarkThreads;
  uint32_t sum = 0, total;
  for (uint32_t j = 0; j < each; ++j) {
    const uint32_t w = tid * each + j;
    if (w < words) sum += (uint32_t)__builtin_popcount(gone[words - 1 - w] & ~kept[words - 1 - w]);
  }
  uint32_t at = BlockSum<kMarkThreads>(sum, part, &total) - sum;
  const uint32_t room = a.free_size - free_count;
  for (uint32_t j = 0; j < each; ++j) {
    const uint32_t w = tid * each + j;
    if (w >= words) break;
    uint32_t bits = gone[words - 1 - w] & ~kept[words - 1 - w];
    while (bits != 0) {
      const uint32_t b = 31 - (uint32_t)__builtin_clz(bits);
      bits &= ~(1u << b);
      if (at < room) a.free_pages[free_count + at] = (int32_t)((words - 1 - w) * 32 + b);
      ++at;
    }
  }
  if (tid == 0) {
    a.status[0] = (int32_t)min(total, room);
    a.status[1] = (int32_t)(total - min(total, room));
  }
}

// The pages in use: a bit each, and the number of them before each word.
struct Used {
  uint32_t bits[kMarkWords], before[kMarkWords];
  __device__ __forceinline__ bool Has(uint32_t p) const { return bits[p / 32] >> (p % 32) & 1u; }
  __device__ __forceinline__ uint32_t Rank(uint32_t p) const {
    return before[p / 32] + (uint32_t)__builtin_popcount(bits[p / 32] & ((1u << (p % 32)) - 1u));
  }
  // The unused page that `r` unused ones come before (there is one).
  __device__ __forceinline__ uint32_t Hole(uint32_t r, uint32_t words) const {
    uint32_t lo = 0, hi = words - 1;  // the last word that at most r come before
    while (lo < hi) {
      const uint32_t mid = (lo + hi + 1) / 2;
      if (mid * 32 - before[mid] <= r) lo = mid;
      else hi = mid - 1;
    }
    uint32_t left = r - (lo * 32 - before[lo]), unused = ~bits[lo], at = 0;
#pragma unroll
    for (uint32_t half = 16; half > 0; half /= 2) {
      const uint32_t n = (uint32_t)__builtin_popcount(unused & ((1u << half) - 1u));
      if (left >= n) {
        left -= n;
        unused >>= half;
        at += half;
      }
    }
    return lo * 32 + at;
  }
};

// Of `count` pages in use the `stay` below it keep their numbers; the others take
// those of the holes below it, each by its rank: the table, the pairs and the
// list of free pages, an entry a thread.
__device__ __forceinline__ void Renumber(const CompactArgs& a, const Used& used, uint32_t count,
                                         uint32_t stay, uint32_t first, uint32_t step) {
  const uint32_t words = (a.pages + 31) / 32;
  for (uint32_t i = first; i < a.batch * a.columns; i += step) {  // below 2^31
    const uint32_t row = i / a.columns, col = i % a.columns;
    const uint32_t p = (uint32_t)a.table[(uint64_t)row * a.table_stride + col];
    int32_t to = -1;
    if (p < a.pages && col < PagesOf(a.lens[row], a.page))
      to = (int32_t)(p < count ? p : used.Hole(used.Rank(p) - stay, words));
    a.table_out[(uint64_t)row * a.table_out_stride + col] = to;
  }
  for (uint64_t p = count + first; p < a.pages; p += step) {
    if (!used.Has((uint32_t)p)) continue;
    const uint32_t i = used.Rank((uint32_t)p) - stay;
    a.pairs[2 * (uint64_t)i] = (int32_t)p;
    a.pairs[2 * (uint64_t)i + 1] = (int32_t)used.Hole(i, words);
  }
  for (uint64_t i = 2ull * (count - stay) + first; i < 2ull * a.pair_count; i += step)
    a.pairs[i] = -1;
  for (uint64_t i = first; i < a.free_size; i += step)
    a.free_pages[i] = i < a.pages - count ? (int32_t)(a.pages - 1 - (uint32_t)i) : -1;
}

// One workgroup finds the pages in use and, where the lists are short (`whole`),
// renumbers them too; else it leaves what it found in the workspace for as many
// workgroups as the lists want.
__global__ __launch_bounds__(kMarkThreads) void CompactKernel(const CompactArgs a) {
  __shared__ Used used;
  __shared__ uint32_t part[kMarkThreads / 64];
  const uint32_t tid = threadIdx.x, words = (a.pages + 31) / 32;
  const int32_t length = FirstLength(a.lens, a.batch);
  for (uint32_t i = tid; i < words; i += kMarkThreads) used.bits[i] = 0;
  __syncthreads();
  EachEntry(a.table, a.lens, length, a.batch, a.columns, a.table_stride, a.page, a.pages,
            [](uint64_t) { return (uint64_t)0; },
            [&](uint32_t p, bool) { atomicOr(&used.bits[p / 32], 1u << (p % 32)); });
  __syncthreads();
  const uint32_t each = (words + kMarkThreads - 1) / kMarkThreads;
  uint32_t sum = 0, count;
  for (uint32_t j = 0; j < each; ++j) {
    const uint32_t w = tid * each + j;
    if (w < words) sum += (uint32_t)__builtin_popcount(used.bits[w]);
  }
  uint32_t rank = BlockSum<kMarkThreads>(sum, part, &count) - sum;
  for (uint32_t j = 0; j < each; ++j) {
    const uint32_t w = tid * each + j;
    if (w >= words) break;
    used.before[w] = rank;
    rank += (uint32_t)__builtin_popcount(used.bits[w]);
    if (!a.whole) {
      a.found[w] = used.bits[w];
      a.found[words + w] = used.before[w];
    }
  }
  __syncthreads();
  const uint32_t stay = count < a.pages ? used.Rank(count) : count;
  if (tid == 0) {
    a.status[0] = (int32_t)count;
    a.status[1] = (int32_t)(count - stay);
    *a.free_count = (int32_t)(a.pages - count);
  }
  if (a.whole) Renumber(a, used, count, stay, tid, kMarkThreads);
}
__global__ __launch_bounds__(kMarkThreads) void RenumberKernel(const CompactArgs a) {
  __shared__ Used used;
  const uint32_t words = (a.pages + 31) / 32;
  for (uint32_t w = threadIdx.x; w < words; w += kMarkThreads) {
    used.bits[w] = a.found[w];
    used.before[w] = a.found[words + w];
  }
  const uint32_t count = (uint32_t)a.status[0], stay = count - (uint32_t)a.status[1];
  __syncthreads();
  Renumber(a, used, count, stay, blockIdx.x * kMarkThreads + threadIdx.x,
           gridDim.x * kMarkThreads);
}

}  // namespace

hipError_t LaunchFork(const ForkArgs& a, hipStream_t stream) {
  const uint32_t grid = std::min(kForkThreads / kForkWaves,
                                 std::max(1u, (a.forks + kForkWaves - 1) / kForkWaves));
  ForkKernel<<<grid, kForkThreads, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t LaunchCopy(const CopyArgs& in, hipStream_t stream) {
  CopyArgs a = in;
  a.pieces = (a.page_bytes + kCopyPiece - 1) / kCopyPiece;
  const uint64_t slots = a.pieces * a.layers;
  // about 8 workgroups a CU, as far as the pairs go
  const uint64_t want = 8 * (uint64_t)DeviceCus();
  a.stripes = (uint32_t)std::min<uint64_t>(a.count, std::max<uint64_t>(1, want / slots));
  CopyKernel<<<(uint32_t)(slots * a.stripes), kCopyThreads, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t LaunchFree(const FreeArgs& a, hipStream_t stream) {
  FreeKernel<<<1, kMarkThreads, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t LaunchCompact(const CompactArgs& in, Workspace& ws, hipStream_t stream) {
  CompactArgs a = in;
  // Short lists in the same launch: 16,384 numbers are 16 a thread (two of eight
  // requests end, 18.4 us a pass for 21.5).
  const uint64_t numbers = (uint64_t)a.batch * a.columns + a.free_size + 2ull * a.pair_count;
  a.whole = numbers <= 16384;
  if (!a.whole) {
    const size_t words = (a.pages + 31) / 32;
    const hipError_t err = GrowWorkspace(ws, 2 * words * sizeof(uint32_t), stream);
    if (err != hipSuccess) return err;
    a.found = reinterpret_cast<uint32_t*>(ws.ptr + kSplitCounters);
  }
  CompactKernel<<<1, kMarkThreads, 0, stream>>>(a);
  if (!a.whole) {
    const uint64_t groups = (numbers + kMarkThreads - 1) / kMarkThreads;
    RenumberKernel<<<(uint32_t)std::min<uint64_t>((uint64_t)DeviceCus(), groups), kMarkThreads, 0,
                     stream>>>(a);
  }
  return hipGetLastError();
}

}  // namespace hb
