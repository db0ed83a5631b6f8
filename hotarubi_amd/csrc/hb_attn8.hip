// Attention over the paged 8-bit cache: the MXFP4 cache's kernels on records of
// E4M3 codes (hb_attn_ways.h, hb_prompt.hip).
//
// A record is 64 D + 16 bytes for 34 D, and opens with fewer instructions: a
// column's tokens are neighbours in V's codes, so no permutes; K's scale, one for
// the record, goes into what scores are multiplied by where it is 1 or more, and for
// fp16 queries, which so take one product for two, where it is less.  Few rows are
// bound by HBM: 64 requests of 1,000 to 8,191 keys, 8 heads of 128, bf16, 603 MB,
// take 118 us (5.1 TB/s, what the card copies at, reads and writes together) and 7
// for the join, 4 heads of 256 119 us a call; 24 streams of up to 40,000 tokens that
// see a window of 4,095 and their first four, fp16, 202 MB, 46 us (4.4 TB/s; 38 where
// the last-level cache has them from the call before) and 7.  One request of 191
// keys, 15 heads on 5 of 64, fp32, takes 6 us, a chain of six records over four
// waves.  Three prompts of up to 4,096 tokens, 347 GFLOP, take 13 us for opening and
// 365 (950 TFLOP/s, in a row of 200 calls; a large library product reaches 1,239):
// from there on the records are 16 bits wide, as MXFP4's.
#include "hb_attn_ways.h"

namespace hb {

AttnWay WayOfAttention8(const AttnArgs& a) { return WayOf<Fp8>(a); }
hipError_t LaunchAttention8(const AttnArgs& a, Workspace& ws, hipStream_t stream) {
  return Launch<Fp8>(a, ws, stream);
}

}  // namespace hb
