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

constexpr int64_t PA_BLOCKS = 512;   // blocks that run at once: two a CU
constexpr int64_t PA_CHUNKS = 2048;  // chunks of one sequence at most: the join's weights in LDS
// Chunk lengths are multiples of it.  80 sequences of up to 4074 (12 heads on
// 1 of 128, F32): 37.9 us at 64, 41.7 at 128, 49.3 at 256; 180 of up to 500 (40 on 8 of
// 128, BF16) 65.1, 60.0 and 59.9.
constexpr int PA_UNIT = 128;
// Positions up to which no sequence is cut, twice as many where the sequences
// alone are a quarter of a round of blocks: no join, and no ends of chunks that do
// not fit the blocks.  Heads 32 on 8 of 128, BF16: 64 sequences of 500 24.1
// us whole, 34.1 cut; 8 of 256 6.6 and 9.3; 1 of 1000 12.8 and 9.4, 8 of 1000 14.3
// and 12.4, 16 of 1000 15.0 and 18.8, 64 of 1000 44.1 and 51.5; 64 of up to 2000
// 58.2 and 51.6.
constexpr int64_t PA_WHOLE = 512;
// Sequences up to which a wavefront forms the cut itself (with a launch before
// it, 100 of up to 250, 9 heads on 3 of 64: 7.4 us, 10.7; 250 of up to 1000 26.1,
// 28.6; 200 of up to 1000, 32 on 8 of 128, 91.1, 90.2).
constexpr int64_t PA_SELF = 256;

// The launch's shape for sequences of up to cap positions, `parts` blocks a
// chunk.
struct PagedCut {
  bool cut;        // at all
  int64_t target;  // chunks the lengths are cut for
  int64_t least;   // positions a chunk at least
  int64_t chunks;  // of all sequences at most
  int64_t slots;   // of cut sequences at most
};
inline PagedCut paged_cut(int64_t seqs, int64_t cap, int64_t parts) {
  PagedCut r;
  // Chunks for as many rounds of blocks as hold one a sequence twice: a cut
  // leaves half a chunk a sequence more than the target on average.
  // Where the sequences alone are many rounds only the longest are cut (700 of
  // up to 300, 32 heads on 8 of 128: 175 us, 248 without this rule).
  const int64_t round = PA_BLOCKS / parts > 1 ? PA_BLOCKS / parts : 1;
  const int64_t rounds = (2 * seqs + round - 1) / round;
  r.target = rounds * round - seqs / 2;
  if (rounds > 8) r.target = seqs / 2 > 6 * round ? seqs / 2 : 6 * round;
  r.cut = cap > (seqs * parts >= PA_BLOCKS / 4 ? 2 : 1) * PA_WHOLE;
  if (!r.cut) {
    r.least = cap;
    r.chunks = seqs;
    r.slots = 0;
    return r;
  }
  r.least = (cap + PA_CHUNKS - 1) / PA_CHUNKS;
  // A sequence makes one chunk and at most one more a unit; all of them
  // together at most the target's beside one each.
  const int64_t most = (cap + PA_UNIT - 1) / PA_UNIT;
  r.chunks = r.target + seqs + 1;
  if (most < r.chunks / seqs) r.chunks = most * seqs;
  r.slots = 2 * r.target + 2;
  return r;
}

}  // namespace mi
