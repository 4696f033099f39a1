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

// n / d for 0 <= n < 2^31 without a division: q = (mulhi(n, m) + n) >> s with
// 2^s the power of two at or above d and m = floor(2^32 (2^s - d) / d) + 1
// (mulhi(n, m) < n < 2^31, so the sum holds in 32 bits).
struct PageDiv {
  uint32_t m, s;
};
inline PageDiv page_div(uint32_t d) {
  uint32_t s = 0;
  while ((uint64_t(1) << s) < d) ++s;
  return PageDiv{static_cast<uint32_t>(((uint64_t(1) << 32) * ((uint64_t(1) << s) - d)) / d + 1), s};
}
MI_HD uint32_t page_of(uint32_t n, PageDiv d) {
  return (static_cast<uint32_t>((static_cast<uint64_t>(n) * d.m) >> 32) + n) >> d.s;
}

// How the attention cuts the sequences: chunks of at most C positions, C the
// least multiple of `unit` at which all sequences together make about
// `target` chunks, so every chunk is nearly the same work whatever the
// lengths; a sequence's chunks are of one length, an idle one has one (empty).
// sum: the lengths' sum; per_chunk: 1 / target, target >= 1.  C is above sum /
// target (to the rounding of a double), so all chunks together are at most
// target and one a sequence, and those of cut sequences, which hold more than
// C positions each, at most 2 target.  least: what C is not below (a sequence
// of up to n least positions makes n chunks at most).
MI_HD int64_t chunk_limit(int64_t sum, double per_chunk, int64_t least, int64_t unit) {
  const int64_t c = static_cast<int64_t>(static_cast<double>(sum) * per_chunk);
  return ((c > least - 1 ? c : least - 1) / unit + 1) * unit;
}
MI_HD int32_t chunk_count(int32_t len, int64_t limit) {
  if (len <= limit) return 1;
  const uint32_t c = static_cast<uint32_t>(limit);
  return static_cast<int32_t>((static_cast<uint32_t>(len) + c - 1) / c);
}
// The positions of each of a sequence's n chunks (the last may be shorter or
// empty), a multiple of `unit`.
MI_HD int32_t chunk_len(int32_t len, int32_t n, int32_t unit) {
  if (n == 1) return len;
  const uint32_t units = (static_cast<uint32_t>(len) + unit - 1) / unit;
  return static_cast<int32_t>((units + n - 1) / n) * unit;
}

}  // namespace mi
