// The paged cache's index arithmetic (metalium-rs_amd/csrc/paged.hpp) as a
// host library for test_paged_index.py.
#include "../metalium-rs_amd/csrc/paged.hpp"

extern "C" {
int pos_of(int64_t r, int64_t first, int64_t end, int64_t len, int64_t cap, int64_t *pos) {
  const mi::PagedPos p = mi::paged_pos(r, first, end, len, cap);
  *pos = p.pos;
  return p.state;
}
int64_t row_of(int64_t p, int64_t j, int64_t o, int64_t kv_heads, int64_t page) {
  return mi::paged_row(p, j, o, kv_heads, page);
}
uint32_t quotient(uint32_t n, uint32_t d) { return mi::page_of(n, mi::page_div(d)); }
int64_t limit_of(int64_t sum, int64_t target, int64_t least, int64_t unit) {
  return mi::chunk_limit(sum, 1.0 / static_cast<double>(target), least, unit);
}
int32_t count_of(int32_t len, int64_t limit) { return mi::chunk_count(len, limit); }
int32_t chunk_len_of(int32_t len, int32_t n, int32_t unit) { return mi::chunk_len(len, n, unit); }
int cut_of(int64_t seqs, int64_t cap, int64_t parts, int64_t *shape) {
  const mi::PagedCut c = mi::paged_cut(seqs, cap, parts);
  shape[0] = c.target;
  shape[1] = c.least;
  shape[2] = c.chunks;
  shape[3] = c.slots;
  shape[4] = mi::PA_CHUNKS;
  shape[5] = mi::PA_UNIT;
  return c.cut;
}
int64_t len_of(int64_t len, int64_t cap) { return mi::paged_len(len, cap); }
}
