// The 8-bit cache's layout, scales and visible keys (hb_kv.h) for the tests, on
// the host.
#include "../hotarubi_amd/csrc/hb_kv.h"

extern "C" {

void kv8h_offsets(uint32_t dim, uint32_t t, uint32_t col, uint32_t* out) {
  out[0] = hb::Kv8KCode(dim, t, col);
  out[1] = hb::Kv8VCode(dim, t, col);
  out[2] = hb::Kv8Scale(dim, 0);
  out[3] = hb::Kv8Scale(dim, 1);
  out[4] = hb::Kv8RecordBytes(dim);
}

uint32_t kv8h_scale(uint32_t bits) { return hb::Kv8ScaleOf(bits); }

int32_t kv8h_lead(int32_t prefix, uint32_t sinks, int32_t pos, int32_t total) {
  return hb::KvLead(prefix, sinks, pos, total);
}

uint32_t kv8h_walk(int32_t pos0, int32_t pos1, int32_t total, int32_t prefix, uint32_t window,
                   uint32_t sinks, uint32_t* records, uint32_t room) {
  const hb::KvWalk w =
      hb::KvRecords(pos0, pos1, total, hb::KvLead(prefix, sinks, pos1, total), window);
  for (uint32_t i = 0; i < w.count && i < room; ++i) records[i] = hb::KvWalkRecord(w, i);
  return w.count;
}
}
