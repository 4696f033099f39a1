// The index arithmetic of the paged KV cache: where a new row's position
// lies, and which page row holds it.  Plain functions of whole numbers, so a
// host program can compile and check them without a device.
#pragma once

#include <cstdint>

#ifdef __HIP__
#define MI_HD __host__ __device__ __forceinline__
#else
#define MI_HD inline
#endif

namespace mi {

// A new row of an append: its position in its sequence, or why it has none.
enum PagedState : int { PAGED_OK = 0, PAGED_IDLE = 1, PAGED_BAD = 2 };
struct PagedPos {
  int state;
  int64_t pos;
};

// Row r of the new rows [first, end) of a sequence of `len` positions, the
// new ones counted.  Idle: no sequence (a row behind the last one's) or a
// length of 0.  Bad: the row lies outside its sequence's rows (bounds that
// do not ascend from 0), the new rows are more than the length, or the length
// is beyond `cap` positions (what the table names) -- whatever the values,
// an OK position is in [0, cap).
MI_HD PagedPos paged_pos(int64_t r, int64_t first, int64_t end, int64_t len, int64_t cap) {
  if (len == 0) return PagedPos{PAGED_IDLE, 0};
  if (r < first || r >= end || len < end - first || len > cap) return PagedPos{PAGED_BAD, 0};
  return PagedPos{PAGED_OK, len - (end - first) + (r - first)};
}

// The pool row of offset o of page p for kv head j.
MI_HD int64_t paged_row(int64_t p, int64_t j, int64_t o, int64_t kv_heads, int64_t page) {
  return (p * kv_heads + j) * page + o;
}

// A sequence's length as the attention reads it: one outside [0, cap] is 0.
MI_HD int64_t paged_len(int64_t len, int64_t cap) { return len < 0 || len > cap ? 0 : len; }

}  // namespace mi
