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
#include "hb_attn_ways.h"

namespace hb {

AttnWay WayOfAttention(const AttnArgs& a) { return WayOf<Fp4>(a); }
hipError_t LaunchAttention(const AttnArgs& a, Workspace& ws, hipStream_t stream) {
  return Launch<Fp4>(a, ws, stream);
}

}  // namespace hb
