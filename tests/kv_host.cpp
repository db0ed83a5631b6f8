// The paged cache's layout and bounds (hb_kv.h) for the tests, on the host.
#include "../hotarubi_amd/csrc/hb_kv.h"

extern "C" {

void kvh_offsets(uint32_t dim, uint32_t t, uint32_t col, uint32_t* out) {
  out[0] = hb::KvKCode(dim, t, col);
  out[1] = hb::KvVCode(dim, t, col);
  out[2] = hb::KvKScale(dim, t, col);
  out[3] = hb::KvVScale(dim, t, col);
}

int kvh_slot(int32_t slot, uint32_t pages, uint32_t heads, uint32_t groups, uint64_t* record,
             uint32_t* t) {
  return hb::KvSlot(slot, pages, heads, groups, record, t);
}

int kvh_record(const int32_t* row, uint32_t columns, uint32_t i, uint32_t head, uint32_t pages,
               uint32_t heads, uint32_t groups, uint64_t* record) {
  return hb::KvRecord(row, columns, i, head, pages, heads, groups, record);
}

void kvh_request(int32_t cu0, int32_t cu1, int32_t kv_len, int32_t prefix, uint32_t tokens,
                 uint32_t max_new, uint64_t max_keys, int64_t* out) {
  const hb::KvSpan s = hb::KvRequest(cu0, cu1, kv_len, prefix, tokens, max_new, max_keys);
  out[0] = s.first;
  out[1] = s.rows;
  out[2] = s.count;
  out[3] = s.total;
  out[4] = s.prefix;
}

uint32_t kvh_walk(int32_t pos0, int32_t pos1, int32_t total, int32_t prefix, uint32_t window,
                  uint32_t* records, uint32_t room) {
  const hb::KvWalk w = hb::KvRecords(pos0, pos1, total, prefix, window);
  for (uint32_t i = 0; i < w.count && i < room; ++i) records[i] = hb::KvWalkRecord(w, i);
  return w.count;
}
}
