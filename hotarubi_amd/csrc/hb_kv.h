// The paged MXFP4 cache's layout, for the kernels and host code.
//
// A cache is uint8 [pages][heads][groups][34 dim], groups = page_size / 32: a
// record per 32 tokens of one head.  A record holds the K codes (16 dim
// bytes), the V codes (16 dim), the K scales (dim) and the V scales (dim), in
// the order in which one wave's lanes take them (lane 16 g + n, 16 bytes a
// lane and load):
//   K codes   [chunk][g][n][16 B]: lane (g, n) holds, in chunk order, columns
//             [g dim/4, (g + 1) dim/4) of token n, then of token 16 + n: the A
//             operand of K Q^T over its own columns
//   V codes   [chunk][g][c][16 B]: lane (g, c) holds columns
//             [c dim/16, (c + 1) dim/16) of tokens 4g .. 4g+3, then of
//             16+4g .. 16+4g+3: the tokens whose scores the same lane holds
//   K scales  [dim/32][n][2]: tokens n, 16 + n
//   V scales  [dim/32][g][8]: the 8 tokens in the V codes' order
// Even columns are low nibbles (E2M1), scales E8M0 (255: NaN).
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define HB_KV_FN __host__ __device__ __forceinline__
#else
#define HB_KV_FN inline
#endif

namespace hb {

// Bytes of one record.
HB_KV_FN constexpr uint32_t KvRecordBytes(uint32_t dim) { return 34 * dim; }

// Byte offsets within a record, for token t = 0..31 of the record: the byte
// that holds column col (even) of K and V, and the scale bytes of its block.
HB_KV_FN uint32_t KvKCode(uint32_t dim, uint32_t t, uint32_t col) {
  const uint32_t quarter = dim / 4, at = t / 16 * (dim / 8) + col % quarter / 2;
  return at / 16 * 1024 + col / quarter * 256 + t % 16 * 16 + at % 16;
}
HB_KV_FN uint32_t KvVCode(uint32_t dim, uint32_t t, uint32_t col) {
  const uint32_t part = dim / 16, j = t % 4 + t / 16 * 4, g = t % 16 / 4;
  const uint32_t at = j * (dim / 32) + col % part / 2;
  return 16 * dim + at / 16 * 1024 + g * 256 + col / part * 16 + at % 16;
}
HB_KV_FN uint32_t KvKScale(uint32_t dim, uint32_t t, uint32_t col) {
  return 32 * dim + col / 32 * 32 + t % 16 * 2 + t / 16;
}
HB_KV_FN uint32_t KvVScale(uint32_t dim, uint32_t t, uint32_t col) {
  return 33 * dim + col / 32 * 32 + t % 16 / 4 * 8 + t % 4 + t / 16 * 4;
}

// The 8-bit cache's records, 64 dim + 16 bytes: E4M3 codes of K and V in the
// order of the same lanes, and a scale byte for all of K and one for all of V.
//   K codes   [chunk][g][n][16 B]: as above, dim/4 bytes a token
//   V codes   [chunk][g][c][16 B]: lane (g, c) holds columns
//             [c dim/16, (c + 1) dim/16), of each the 8 tokens above: V^T's
//             operand without a permute
// Scale bytes are E8M0, 10 to 246, so that every value is normal in fp32 and
// bf16; 0 where no value but zeros was stored.
HB_KV_FN constexpr uint32_t Kv8RecordBytes(uint32_t dim) { return 64 * dim + 16; }
HB_KV_FN uint32_t Kv8KCode(uint32_t dim, uint32_t t, uint32_t col) {
  const uint32_t quarter = dim / 4, at = t / 16 * quarter + col % quarter;
  return at / 16 * 1024 + col / quarter * 256 + t % 16 * 16 + at % 16;
}
HB_KV_FN uint32_t Kv8VCode(uint32_t dim, uint32_t t, uint32_t col) {
  const uint32_t part = dim / 16, at = col % part * 8 + t % 4 + t / 16 * 4;
  return 32 * dim + at / 16 * 1024 + t % 16 / 4 * 256 + col / part * 16 + at % 16;
}
HB_KV_FN uint32_t Kv8Scale(uint32_t dim, uint32_t v) { return 64 * dim + v; }
// The scale byte of values whose largest has these fp32 bits: the least
// exponent within [-117, 119] that has it at 448 or below.
HB_KV_FN uint32_t Kv8ScaleOf(uint32_t top_bits) {
  if (top_bits == 0) return 0;
  const uint32_t field = (top_bits + 0x1FFFFFu) >> 23;  // one up past 1.75 x 2^n
  return field < 18 ? 10u : field > 254 ? 246u : field - 8;
}

// Record (its index over the whole cache) of head 0 at a slot, and the token
// in it; false for a slot that the cache does not have.
HB_KV_FN bool KvSlot(int32_t slot, uint32_t pages, uint32_t heads, uint32_t groups,
                     uint64_t* record, uint32_t* t) {
  const uint32_t s = (uint32_t)slot, page = s / (32 * groups);
  if (slot < 0 || page >= pages) return false;
  *record = (uint64_t)page * heads * groups + s / 32 % groups;
  *t = s % 32;
  return true;
}

// Record of head `head` that holds keys [32 i, 32 i + 32) of a request whose
// block table row is `row` (`columns` entries); false where the table names no
// page of the cache.
HB_KV_FN bool KvRecord(const int32_t* row, uint32_t columns, uint32_t i, uint32_t head,
                       uint32_t pages, uint32_t heads, uint32_t groups, uint64_t* record) {
  const uint32_t col = i / groups;
  if (col >= columns) return false;
  const uint32_t page = (uint32_t)row[col];
  if (page >= pages) return false;
  *record = ((uint64_t)page * heads + head) * groups + i % groups;
  return true;
}

// A request's rows and keys as the attention kernels take them, every value
// within the tensors whatever cu, kv_lens and prefix hold: rows [first,
// first + rows) of q, `total` keys, row i at position total - count + i,
// where count is what cu says and rows <= count what the launch covers.
struct KvSpan {
  uint32_t first, rows;
  int32_t count, total, prefix;
};
HB_KV_FN KvSpan KvRequest(int32_t cu0, int32_t cu1, int32_t kv_len, int32_t prefix,
                          uint32_t tokens, uint32_t max_new, uint64_t max_keys) {
  KvSpan s;
  s.first = 0;
  s.rows = 0;
  s.count = 0;
  s.total = kv_len < 0 ? 0 : kv_len;
  if ((uint64_t)s.total > max_keys) s.total = (int32_t)max_keys;
  s.prefix = prefix < 0 ? 0 : prefix > s.total ? s.total : prefix;
  if (cu0 < 0 || cu1 <= cu0 || (uint32_t)cu0 >= tokens) return s;
  s.first = (uint32_t)cu0;
  s.count = cu1 - cu0;
  s.rows = (uint32_t)s.count;
  if (s.rows > tokens - s.first) s.rows = tokens - s.first;
  if (s.rows > max_new) s.rows = max_new;
  return s;
}

// Leading keys that a row at position `pos` sees whatever its window: the
// prefix, and of the first `sinks` those up to its own.
HB_KV_FN int32_t KvLead(int32_t prefix, uint32_t sinks, int32_t pos, int32_t total) {
  int64_t lead = (int64_t)pos + 1 < (int64_t)sinks ? (int64_t)pos + 1 : (int64_t)sinks;
  if (lead > total) lead = total;
  return lead > prefix ? (int32_t)lead : prefix;
}

// The records that rows at positions [pos0, pos1] look at, in order:
// `head` records from 0 (the prefix), then those from `from` on, `count` in
// all.  Where the two ranges meet they are one (head = 0).
struct KvWalk {
  uint32_t head, from, count;
};
HB_KV_FN KvWalk KvRecords(int32_t pos0, int32_t pos1, int32_t total, int32_t prefix,
                          uint32_t window) {
  KvWalk w;
  int64_t start = 0;
  if (window > 0 && (int64_t)pos0 + 1 > (int64_t)window) start = (int64_t)pos0 + 1 - window;
  int64_t end = (int64_t)pos1 + 1;
  if (end > total) end = total;
  const uint32_t pre = (uint32_t)((prefix + 31) / 32);
  uint32_t a = 0, b = 0;
  if (end > start) {
    a = (uint32_t)(start / 32);
    b = (uint32_t)((end + 31) / 32);
  }
  if (b == 0 || pre >= a) {  // one range
    w.head = 0;
    w.from = 0;
    w.count = pre > b ? pre : b;
  } else {
    w.head = pre;
    w.from = a;
    w.count = pre + b - a;
  }
  return w;
}
HB_KV_FN uint32_t KvWalkRecord(const KvWalk& w, uint32_t i) {
  return i < w.head ? i : w.from + i - w.head;
}

}  // namespace hb
