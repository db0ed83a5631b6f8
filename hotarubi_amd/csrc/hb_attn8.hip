// Attention over the paged 8-bit cache: the MXFP4 cache's kernels on records of
// E4M3 codes.
#include "hb_attn_ways.h"

namespace hb {

AttnWay WayOfAttention8(const AttnArgs& a) { return WayOf<Fp8>(a); }
hipError_t LaunchAttention8(const AttnArgs& a, Workspace& ws, hipStream_t stream) {
  return Launch<Fp8>(a, ws, stream);
}

}  // namespace hb
