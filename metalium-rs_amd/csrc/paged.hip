// A KV cache in pages: the append with its rotation and the attention of one
// new token per sequence over it.
//
// Reference: the KV cache of crates/tt-models/src/llama.rs:403-446 (RoPE on q
// and k, the slice_assign of the new rows) and Engine::attention_rows
// (crates/burn-tt/src/server.rs:255-265) on a cache of one slot of max_ctx
// rows a sequence, all sequences at one position.  Here a sequence's positions
// lie in pages of a shared pool that its row of a page table names, and every
// sequence has a length of its own, read on the device.
#include <cfloat>
#include <type_traits>

#include "common.hpp"
#include "paged.hpp"
#include "wave.hpp"

namespace mi {
namespace {

// The cache's geometry, checked against its buffers.
struct PagedCache {
  void *k, *v;
  int elem;
  int64_t pages, page, kv_heads, D;
  const int32_t *table, *lens;
  int64_t seqs, per;  // the table: [seqs, per]
  int64_t cap() const { return per * page; }
};

int paged_cache(Ctx *ctx, const char *what, mi_id k_pages, mi_id v_pages, mi_id table, mi_id lens, int64_t heads,
                int64_t kv_heads, int64_t page, PagedCache *c) {
  MI_BUF(ctx, kb, k_pages);
  MI_BUF(ctx, vb, v_pages);
  MI_BUF(ctx, tb, table);
  MI_BUF(ctx, lb, lens);
  if (kb->elem != vb->elem || !elem_float(kb->elem) || kb->tiles || vb->tiles)
    return fail(ctx, MI_E_ARG, "%s takes two F32 or two BF16 page pools (%s, %s)", what, elem_name(kb->elem),
                elem_name(vb->elem));
  if (heads < 1 || kv_heads < 1 || heads % kv_heads || page < 1)
    return fail(ctx, MI_E_ARG, "%s: heads %lld, kv heads %lld, pages of %lld", what, (long long)heads,
                (long long)kv_heads, (long long)page);
  const int64_t D = kb->cols;
  if (D != 16 && D != 32 && D != 64 && D != 128)
    return fail(ctx, MI_E_UNSUPPORTED, "%s: head width %lld (16, 32, 64 or 128)", what, (long long)D);
  if (page > INT32_MAX || kv_heads > INT32_MAX / page || kb->rows < 1 || kb->rows % (kv_heads * page) ||
      vb->rows != kb->rows || vb->cols != D)
    return fail(ctx, MI_E_ARG, "%s: pools [%lld, %lld] and [%lld, %lld], want both [pages * %lld * %lld, d]", what,
                (long long)kb->rows, (long long)kb->cols, (long long)vb->rows, (long long)vb->cols,
                (long long)kv_heads, (long long)page);
  if (tb->elem != MI_I32 || lb->elem != MI_I32 || tb->cols < 1 || lb->numel() != tb->rows)
    return fail(ctx, MI_E_ARG, "%s: table %s [%lld, %lld] and lengths %s [%lld, %lld], want I32 [sequences, pages] and I32 of one a sequence",
                what, elem_name(tb->elem), (long long)tb->rows, (long long)tb->cols, elem_name(lb->elem),
                (long long)lb->rows, (long long)lb->cols);
  if (kb->rows > INT32_MAX)
    return fail(ctx, MI_E_UNSUPPORTED, "%s: pools of %lld rows (at most 2^31 - 1)", what, (long long)kb->rows);
  if (tb->cols > INT32_MAX / page)
    return fail(ctx, MI_E_UNSUPPORTED, "%s: a table row of %lld pages of %lld positions (at most 2^31 - 1)", what,
                (long long)tb->cols, (long long)page);
  c->k = kb->ptr;
  c->v = vb->ptr;
  c->elem = kb->elem;
  c->page = page;
  c->kv_heads = kv_heads;
  c->D = D;
  c->pages = kb->rows / (kv_heads * page);
  c->table = static_cast<const int32_t *>(tb->ptr);
  c->lens = static_cast<const int32_t *>(lb->ptr);
  c->seqs = tb->rows;
  c->per = tb->cols;
  return MI_OK;
}

// ------------------------------------------------------------------ append

struct AppendArgs {
  const void *qkv;
  const float *cosp, *sinp;
  int64_t positions;  // rows of the rotary tables
  const int32_t *table, *lens, *starts;
  int64_t rows, seqs, per, pages, page;
  PageDiv div, per_row;  // by the page, by a row's items
  int heads, kv_heads, items, block_rows;
  void *k, *v, *q;
  uint32_t *flags;
};

// Eight elements a thread: for a q or k head four of the first half and their
// partners of the second, for a v head eight in a row.  A row's items are one
// or more blocks, or the items of `block_rows` rows share one.  rope: x cos +
// rotate(x) sin, two roundings, as mi_rope.  Bound by HBM for prompts and by
// latency for a decode step, so what does not depend on the position -- the
// row itself -- is asked for before the position is known, and the page and
// the angles in one go.  3639 rows of 15 heads of 64, F32 (29 MB): 7.3 us, 4.0
// TB/s; 32 rows of 48 heads of 128 into BF16 pools: 3.0 us, as a launch and
// two dependent reads take.
template <typename TI, typename TC, typename TO>
__global__ void __launch_bounds__(256) append_kernel(AppendArgs a, int D) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * a.block_rows;
  const int sub = a.block_rows > 1 ? static_cast<int>(page_of(static_cast<uint32_t>(tid), a.per_row)) : 0;
  const int item = static_cast<int>(blockIdx.y) * 256 + tid - sub * a.items;
  const int64_t r = r0 + sub;
  const bool live = sub < a.block_rows && r < a.rows && item < a.items;
  const int per_head = D / 8, half = D / 2;
  const int head = item / per_head, quad = item - head * per_head;
  const bool turn = head < a.heads + a.kv_heads;
  const int c0 = turn ? 4 * quad : 8 * quad, c1 = turn ? c0 + half : c0 + 4;
  float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
  if (live) {
    const TI *x = static_cast<const TI *>(a.qkv) + (r * (a.heads + 2 * a.kv_heads) + head) * D;
    lo = f32x4_get(x + c0);
    hi = f32x4_get(x + c1);
  }
  // The sequence of a row: behind those whose rows end at or before it,
  // counted 64 bounds at a time, so a lookup is a few independent loads and
  // not a chain of a binary search's.
  int64_t seq = r, first = r, end = r + 1, len = 0;
  if (a.starts) {
    seq = a.seqs;
    int64_t passed = 0;  // the block's rows whose sequence lies behind this batch
    for (int64_t s0 = 0; s0 < a.seqs && passed < a.block_rows; s0 += 64) {
      const bool in = s0 + lane < a.seqs;
      const int32_t from = in ? a.starts[s0 + lane] : 0, to = in ? a.starts[s0 + lane + 1] : INT32_MAX;
      const int32_t n = in ? a.lens[s0 + lane] : 0;
      for (int o = static_cast<int>(passed); o < a.block_rows; ++o) {
        const int at = __popcll(__ballot(to <= r0 + o));
        if (s0 + at >= a.seqs || at == 64) break;  // rows ascend: the later ones too
        ++passed;
        if (sub == o) {
          seq = s0 + at;
          first = __builtin_amdgcn_readlane(from, at);
          end = __builtin_amdgcn_readlane(to, at);
          len = __builtin_amdgcn_readlane(n, at);
        }
      }
    }
  } else if (live) {
    len = a.lens[r];
  }
  if (!live) return;
  PagedPos p{PAGED_IDLE, 0};
  if (seq < a.seqs) p = paged_pos(r, first, end, len, a.per * a.page);
  if (p.state == PAGED_OK && p.pos >= a.positions) p.state = PAGED_BAD;
  int64_t nth = 0, pg = 0;
  float4 cl = lo, ch = lo, sl = lo, sh = lo;
  if (p.state == PAGED_OK) {  // the page and the angles in one go
    nth = page_of(static_cast<uint32_t>(p.pos), a.div);
    pg = a.table[seq * a.per + nth];
    if (turn) {
      const float *cr = a.cosp + p.pos * D, *sr = a.sinp + p.pos * D;
      cl = f32x4_get(cr + c0);
      ch = f32x4_get(cr + c1);
      sl = f32x4_get(sr + c0);
      sh = f32x4_get(sr + c1);
    }
    if (pg < 0 || pg >= a.pages) p.state = PAGED_BAD;
  }
  if (p.state == PAGED_BAD && item == 0) atomicOr(a.flags, FLAG_INDEX_RANGE);
  TO *q = static_cast<TO *>(a.q) + (r * a.heads + head) * D;
  if (p.state != PAGED_OK) {
    if (head < a.heads) {
      f32x4_put(q + c0, make_float4(0.f, 0.f, 0.f, 0.f));
      f32x4_put(q + c1, make_float4(0.f, 0.f, 0.f, 0.f));
    }
    return;
  }
  if (turn) {
    const float4 l = lo, h = hi;
    lo = make_float4(l.x * cl.x + h.x * sl.x, l.y * cl.y + h.y * sl.y, l.z * cl.z + h.z * sl.z, l.w * cl.w + h.w * sl.w);
    hi = make_float4(h.x * ch.x + l.x * sh.x, h.y * ch.y + l.y * sh.y, h.z * ch.z + l.z * sh.z, h.w * ch.w + l.w * sh.w);
  }
  if (head < a.heads) {
    f32x4_put(q + c0, lo);
    f32x4_put(q + c1, hi);
    return;
  }
  const int64_t j = turn ? head - a.heads : head - a.heads - a.kv_heads;
  TC *dst = static_cast<TC *>(turn ? a.k : a.v) + paged_row(pg, j, p.pos - nth * a.page, a.kv_heads, a.page) * D;
  f32x4_put(dst + c0, lo);
  f32x4_put(dst + c1, hi);
}

template <typename TI, typename TC>
void append_launch(Ctx *ctx, const AppendArgs &a, int64_t D, int out_elem) {
  const dim3 grid(static_cast<unsigned>((a.rows + a.block_rows - 1) / a.block_rows), grid_for(a.items, 256));
  if (out_elem == MI_BF16)
    append_kernel<TI, TC, uint16_t><<<grid, 256, 0, ctx->stream>>>(a, static_cast<int>(D));
  else
    append_kernel<TI, TC, float><<<grid, 256, 0, ctx->stream>>>(a, static_cast<int>(D));
}

// --------------------------------------------------------------- attention
// One new token a sequence: softmax(scale q K^T) V over the sequence's pages.
// Every byte of K and V is read once for a kv head's G query heads, so the
// operator is bound by HBM; the products are small (4 G D operations a
// position) and run on the matrix cores, which read their operands as the
// cache holds them:
//   S^T = K Q^T, 16 positions x 16 heads: a lane's 16 bytes of a key row are
//     its operand (a row of K = D contraction steps);
//   O^T = V^T P^T, 16 columns x 16 heads: P^T is S^T's own result layout (lane
//     (head h, group g) holds positions 4 g .. 4 g + 3 of head h), and V^T's
//     operand, four positions of one column, is a 4 x 4 transpose within the
//     lane's own registers.
// So nothing passes through LDS between the two products.  BF16 pools: the
// F32 queries (scaled, in base 2) and the weights go as three BF16 parts each
// (24 bits, small parts first), K and V as they are -- F32 sums of exact
// products.  F32 pools: the F32 matrix cores.
//
// The sequences are cut into chunks of nearly equal length (paged.hpp), a
// block each: lengths are known on the device only, so every wavefront forms
// the cut from them itself (or, for many sequences, reads what a launch before
// it formed), and the grid is its upper bound.  A block's four
// wavefronts take steps of POS positions in turn, each with running maximum
// and sum, and join in LDS; a chunk of a cut sequence leaves its maximum, sum
// and sums of values to a second launch that joins them.
//
// Measured: one sequence of 100001 positions, 32 heads over 8 of 128, BF16
// pools (410 MB): 65 us, 6.3 TB/s (a plain streaming read reaches 7.0), and 4.5
// for the join; 64 sequences of up to 4000: 83 us, 5.7 TB/s, the blocks'
// unequal ends beside it.  One of 577 positions, 9 heads over 3 of 64, F32: 5.6
// and 2.8 us, a chain of launch, lengths, table, keys and join, each about 1 us.

typedef __bf16 pa_bf16x8 __attribute__((ext_vector_type(8)));
typedef float pa_f32x4 __attribute__((ext_vector_type(4)));

constexpr int PA_WAVES = 4;
constexpr int PA_HEADS = 16;       // query heads a block: the matrix cores' tile

// Positions a wavefront takes a step: 8 KiB of keys at most.  80 sequences of
// up to 4074, F32 keys of 128: 41.7 us at 16, 53.8 at 32; 32 of up to 2000, BF16
// of 64: 12.0 at 32, 12.6 at 64.
template <int D, typename TC>
constexpr int pa_pos() { return D * sizeof(TC) > 256 ? 16 : 32; }

struct AttendArgs {
  const void *q, *k, *v;
  const int32_t *table, *lens;
  int64_t seqs, per, pages, page;
  PageDiv div, by_parts, by_tiles;  // by the page, by the kv heads' tiles, by a kv head's
  int heads, kv_heads, group, tiles, live;  // heads a kv head, their tiles of 16, heads a tile at most
  int out16;
  int32_t least;     // positions a chunk at least
  double per_chunk;  // 1 / the chunks the lengths are cut for
  int64_t slots;     // partials there is room for, a kv head tile
  int2 *cuts;        // a sequence's chunks and the slot of its first partial
  int4 *plan;        // the chunks, where they were formed by a launch of their own
  int64_t chunks;    // their bound
  float scale;     // times log2(e)
  float *part;
  void *out;
  uint32_t *flags;
};

// Floats of one chunk's partial: `live` maxima, `live` sums, room up to a
// multiple of 4, then each head's D sums.
__host__ __device__ constexpr int64_t pa_acc0(int64_t live) { return (2 * live + 3) / 4 * 4; }
__host__ __device__ constexpr int64_t pa_stride(int64_t live, int64_t D) { return pa_acc0(live) + live * D; }

// Inclusive sums over the wavefront's lanes.
__device__ __forceinline__ int32_t wave_scan(int32_t v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ int32_t lane_value(int32_t v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// A chunk of the cut: its sequence (-1 past the last chunk), its number of n,
// the sequence's length, and the slot of the sequence's first partial.
// Bad: the length was out of range.
struct Chunk {
  int32_t seq, c, n, len, slot, bad;
};

// Chunk g of up to 64 * N sequences, N neighbours a lane.
template <int N>
__device__ __forceinline__ Chunk pa_chunk(const AttendArgs &a, int32_t g, int lane) {
  const int seqs = static_cast<int>(a.seqs), s0 = lane * N;
  int32_t raw[N], len[N], n[N], low = 0, high = 0, all = 0, cuts = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) raw[i] = a.lens[s0 + i < seqs ? s0 + i : seqs - 1];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    len[i] = s0 + i < seqs ? static_cast<int32_t>(paged_len(raw[i], a.per * a.page)) : 0;
    low += len[i] & 0xffff;
    high += len[i] >> 16;
  }
  // The sum in halves of 16 bits, whose sums over the lanes hold in 32.
  const int64_t sum = lane_value(wave_scan(low), 63) + (static_cast<int64_t>(lane_value(wave_scan(high), 63)) << 16);
  const int64_t limit = chunk_limit(sum, a.per_chunk, a.least, PA_UNIT);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    n[i] = s0 + i < seqs ? chunk_count(len[i], limit) : 0;
    all += n[i];
    cuts += n[i] > 1 ? n[i] : 0;
  }
  const int32_t in = wave_scan(all), cut_in = wave_scan(cuts);
  if (g >= lane_value(in, 63)) return Chunk{-1, 0, 0, 0, 0, 0};
  const int at = __builtin_amdgcn_readfirstlane(__popcll(__ballot(in <= g)));
  Chunk r;
  r.c = g - lane_value(in - all, at);
  r.slot = lane_value(cut_in - cuts, at);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int32_t mine = lane_value(n[i], at);
    r.seq = at * N + i;
    r.n = mine;
    r.len = lane_value(len[i], at);
    r.bad = lane_value(raw[i], at) != r.len;
    if (i + 1 == N || r.c < mine) break;
    r.c -= mine;
    r.slot += mine > 1 ? mine : 0;
  }
  return r;
}

// The chunks of more sequences, in a launch of one block before the
// attention's: the lengths' sum, then 1024 sequences a turn, their chunk counts
// summed over the block, and each chunk's sequence found in those sums.  Where
// every wavefront formed them from all lengths, 1000 sequences of up to 500 (9
// heads on 3 of 64) took 100 us; with it 60 (cut) and 47 (whole), 5 of them its own.
__global__ void __launch_bounds__(1024) attend_plan_kernel(AttendArgs a) {
  __shared__ int64_t sums[16];
  __shared__ int32_t wsum[16][2], ends[1024], counts[1024], lens[1024], slots[1024];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t cap = a.per * a.page;
  int64_t sum = 0;
  bool bad = false;
  for (int64_t s = tid; s < a.seqs; s += 1024) {
    const int64_t raw = a.lens[s], len = paged_len(raw, cap);
    bad |= raw != len;
    sum += len;
  }
  if (bad) atomicOr(a.flags, FLAG_INDEX_RANGE);
  for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  sum = 0;
  for (int w = 0; w < 16; ++w) sum += sums[w];
  const int64_t limit = chunk_limit(sum, a.per_chunk, a.least, PA_UNIT);
  int64_t before = 0;
  int32_t slot = 0;
  for (int64_t s0 = 0; s0 < a.seqs; s0 += 1024) {
    const int64_t s = s0 + tid;
    const int32_t len = s < a.seqs ? static_cast<int32_t>(paged_len(a.lens[s], cap)) : 0;
    const int32_t n = s < a.seqs ? chunk_count(len, limit) : 0, cut = n > 1 ? n : 0;
    int32_t in = wave_scan(n), cuts = wave_scan(cut);
    if (lane == 63) {
      wsum[wave][0] = in;
      wsum[wave][1] = cuts;
    }
    __syncthreads();
    int32_t all = 0, all_cuts = 0;
    for (int w = 0; w < 16; ++w) {
      in += w < wave ? wsum[w][0] : 0;
      cuts += w < wave ? wsum[w][1] : 0;
      all += wsum[w][0];
      all_cuts += wsum[w][1];
    }
    ends[tid] = in;
    counts[tid] = n;
    lens[tid] = len;
    slots[tid] = slot + cuts - cut;
    if (a.cuts && s < a.seqs) a.cuts[s] = make_int2(n, slot + cuts - cut);
    __syncthreads();
    for (int32_t g = tid; g < all; g += 1024) {
      int at = 0;  // the first whose end lies behind g
      for (int step = 512; step >= 1; step >>= 1) at += ends[at + step - 1] <= g ? step : 0;
      if (before + g < a.chunks)  // always: the count's bound
        a.plan[before + g] = make_int4(static_cast<int>(s0) + at, (g - (ends[at] - counts[at])) | counts[at] << 16, lens[at], slots[at]);
    }
    before += all;
    slot += all_cuts;
    __syncthreads();
  }
  for (int64_t g = before + tid; g < a.chunks; g += 1024) a.plan[g] = make_int4(-1, 0, 0, 0);
}

// Three BF16 parts of two F32 values, packed (a in the low halves): each the
// rounding of what the ones before leave.
__device__ __forceinline__ void split3(float a, float b, uint32_t &h, uint32_t &m, uint32_t &l) {
  h = bf16x2_bits(a, b);
  a -= __uint_as_float(h << 16);
  b -= __uint_as_float(h & 0xffff0000u);
  m = bf16x2_bits(a, b);
  l = bf16x2_bits(a - __uint_as_float(m << 16), b - __uint_as_float(m & 0xffff0000u));
}

__device__ __forceinline__ pa_f32x4 pa_mfma(uint4 a, uint4 b, pa_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pa_bf16x8, a), __builtin_bit_cast(pa_bf16x8, b), c,
                                                 0, 0, 0);
}

// The maximum over the four lanes of one head (l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float head_max(float v) {
  float x, y;
  swap16_pair(v, x, y);
  v = max_nan(x, y);
  swap32_pair(v, x, y);
  return max_nan(x, y);
}

// One wavefront's part of a chunk on BF16 pools.
template <int D>
struct WaveBf16 {
  static constexpr int POS = pa_pos<D, uint16_t>();
  static constexpr int TILES = POS / 16, KS = D < 32 ? 1 : D / 32, CP = D / 16;  // key steps; columns a lane
  uint4 q[3][KS];
  uint4 k[TILES][KS];
  uint32_t v[TILES][4][CP < 2 ? 1 : CP / 2];
  pa_f32x4 acc[CP];

  __device__ __forceinline__ void query(const float *qs, int lane) {  // LDS [16][D + 4]
    const int h = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      uint32_t w[3][4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = 32 * t + 8 * g + 2 * e;
        const float2 x = c < D ? *reinterpret_cast<const float2 *>(qs + h * (D + 4) + c) : make_float2(0.f, 0.f);
        split3(x.x, x.y, w[0][e], w[1][e], w[2][e]);
      }
#pragma unroll
      for (int p = 0; p < 3; ++p) q[p][t] = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
    }
  }
  template <bool NT>
  __device__ __forceinline__ void load_k(const uint16_t *K, const int32_t *rows, int lane) {
    const int g = lane >> 4;
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      const uint16_t *p = K + static_cast<int64_t>(rows[16 * t + (lane & 15)]) * D + (D < 32 ? 8 * (g & 1) : 8 * g);
#pragma unroll
      for (int s = 0; s < KS; ++s) k[t][s] = ldu4<NT>(p + 32 * s);
    }
  }
  template <bool NT>
  __device__ __forceinline__ void load_v(const uint16_t *V, const int32_t *rows, int lane) {
    const int n = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      const int4 r4 = *reinterpret_cast<const int4 *>(rows + 16 * t + 4 * g);
      const int32_t r[4] = {r4.x, r4.y, r4.z, r4.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint16_t *p = V + static_cast<int64_t>(r[j]) * D + CP * n;
        if constexpr (CP == 8) {
          const uint4 x = ldu4<NT>(p);
          v[t][j][0] = x.x; v[t][j][1] = x.y; v[t][j][2] = x.z; v[t][j][3] = x.w;
        } else if constexpr (CP == 4) {
          const uint2 x = *reinterpret_cast<const uint2 *>(p);
          v[t][j][0] = x.x; v[t][j][1] = x.y;
        } else if constexpr (CP == 2) {
          v[t][j][0] = *reinterpret_cast<const uint32_t *>(p);
        } else {
          v[t][j][0] = *p;
        }
      }
    }
  }
  // Scores of tile t, positions 4 g + i of head lane & 15.  D = 16: the
  // upper half of the contraction meets zeros of q.
  __device__ __forceinline__ pa_f32x4 scores(int t) const {
    pa_f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 2; p >= 0; --p)
#pragma unroll
      for (int u = 0; u < KS; ++u) s = pa_mfma(k[t][u], q[p][u], s);
    return s;
  }
  // acc += V^T P^T over all tiles, two at a time: contraction step 8 g + j is
  // position 4 g + j % 4 of tile j / 4 of the pair, for both operands.
  __device__ __forceinline__ void values(const pa_f32x4 (&p)[TILES]) {
    static_assert(TILES % 2 == 0, "tiles in pairs");
#pragma unroll
    for (int t = 0; t < TILES; t += 2) {
      uint32_t w[3][4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        split3(p[t + e / 2][2 * (e & 1)], p[t + e / 2][2 * (e & 1) + 1], w[0][e], w[1][e], w[2][e]);
#pragma unroll
      for (int c = 0; c < CP; ++c) {
        const uint32_t sel = c & 1 ? 0x07060302u : 0x05040100u;
        const int d = c >> 1;
        const uint4 x = make_uint4(__builtin_amdgcn_perm(v[t][1][d], v[t][0][d], sel),
                                   __builtin_amdgcn_perm(v[t][3][d], v[t][2][d], sel),
                                   __builtin_amdgcn_perm(v[t + 1][1][d], v[t + 1][0][d], sel),
                                   __builtin_amdgcn_perm(v[t + 1][3][d], v[t + 1][2][d], sel));
#pragma unroll
        for (int q_ = 2; q_ >= 0; --q_) acc[c] = pa_mfma(x, make_uint4(w[q_][0], w[q_][1], w[q_][2], w[q_][3]), acc[c]);
      }
    }
  }
};

// The same on F32 pools: 16 x 16 x 4 steps of the F32 matrix cores, whose
// operand is one value a lane (row or column lane & 15, step lane >> 4).
template <int D>
struct WaveF32 {
  static constexpr int POS = pa_pos<D, float>();
  static constexpr int TILES = POS / 16, KQ = D / 16, CP = D / 16;
  float4 q[KQ];
  float4 k[TILES][KQ];
  float v[TILES][4][CP];
  pa_f32x4 acc[CP];

  __device__ __forceinline__ void query(const float *qs, int lane) {
#pragma unroll
    for (int u = 0; u < KQ; ++u) q[u] = *reinterpret_cast<const float4 *>(qs + (lane & 15) * (D + 4) + 16 * u + 4 * (lane >> 4));
  }
  template <bool NT>
  __device__ __forceinline__ void load_k(const float *K, const int32_t *rows, int lane) {
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      const float *p = K + static_cast<int64_t>(rows[16 * t + (lane & 15)]) * D + 4 * (lane >> 4);
#pragma unroll
      for (int u = 0; u < KQ; ++u) k[t][u] = ld4<NT>(p + 16 * u);
    }
  }
  template <bool NT>
  __device__ __forceinline__ void load_v(const float *V, const int32_t *rows, int lane) {
    const int n = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      const int4 r4 = *reinterpret_cast<const int4 *>(rows + 16 * t + 4 * g);
      const int32_t r[4] = {r4.x, r4.y, r4.z, r4.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float *p = V + static_cast<int64_t>(r[j]) * D + CP * n;
        if constexpr (CP >= 4) {
#pragma unroll
          for (int c = 0; c < CP; c += 4) {
            const float4 x = ld4<NT>(p + c);
            v[t][j][c] = x.x; v[t][j][c + 1] = x.y; v[t][j][c + 2] = x.z; v[t][j][c + 3] = x.w;
          }
        } else if constexpr (CP == 2) {
          const float2 x = *reinterpret_cast<const float2 *>(p);
          v[t][j][0] = x.x; v[t][j][1] = x.y;
        } else {
          v[t][j][0] = *p;
        }
      }
    }
  }
  __device__ __forceinline__ pa_f32x4 scores(int t) const {
    pa_f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < KQ; ++u) {
      s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][u].x, q[u].x, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][u].y, q[u].y, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][u].z, q[u].z, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][u].w, q[u].w, s, 0, 0, 0);
    }
    return s;
  }
  __device__ __forceinline__ void values(const pa_f32x4 (&p)[TILES]) {
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < CP; ++c) acc[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[t][j][c], p[t][j], acc[c], 0, 0, 0);
  }
};

template <int D, typename TC>
struct WaveOf { using type = WaveF32<D>; };
template <int D>
struct WaveOf<D, uint16_t> { using type = WaveBf16<D>; };

template <int D, typename TQ, typename TC, bool STREAM>
__global__ void __launch_bounds__(PA_WAVES * 64, D == 128 ? 2 : 3) attend_kernel(AttendArgs a) {
  using W = typename WaveOf<D, TC>::type;
  constexpr int POS = W::POS, TILES = W::TILES, CP = W::CP, QS = D + 4;
  // The scaled queries, then (once read) the wavefronts' results.
  __shared__ __align__(16) float sm[PA_WAVES * PA_HEADS * QS];
  __shared__ float stat[PA_WAVES][2][PA_HEADS];
  __shared__ __align__(16) int32_t rowbuf[PA_WAVES][2][POS];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int parts = a.kv_heads * a.tiles;
  const int g = static_cast<int>(page_of(blockIdx.x, a.by_parts)), jt = static_cast<int>(blockIdx.x) - g * parts;
  const int j = static_cast<int>(page_of(static_cast<uint32_t>(jt), a.by_tiles)), h0 = (jt - j * a.tiles) * PA_HEADS;
  Chunk ch;
  if (a.plan) {
    const int4 c = a.plan[g];
    ch = Chunk{__builtin_amdgcn_readfirstlane(c.x), __builtin_amdgcn_readfirstlane(c.y & 0xffff),
               __builtin_amdgcn_readfirstlane(c.y >> 16), __builtin_amdgcn_readfirstlane(c.z),
               __builtin_amdgcn_readfirstlane(c.w), 0};
  } else {
    ch = a.seqs <= 64 ? pa_chunk<1>(a, g, lane) : pa_chunk<PA_SELF / 64>(a, g, lane);
  }
  if (ch.seq < 0) return;
  const int nh = a.group - h0 < PA_HEADS ? a.group - h0 : PA_HEADS;  // heads of this tile
  const int32_t clen = chunk_len(ch.len, ch.n, PA_UNIT);
  const int64_t from = static_cast<int64_t>(ch.c) * clen;
  const int32_t lo = from < ch.len ? static_cast<int32_t>(from) : ch.len;
  const int32_t hi = ch.len - lo < clen ? ch.len : lo + clen;
  const int64_t q0 = (static_cast<int64_t>(ch.seq) * a.heads + static_cast<int64_t>(j) * a.group + h0) * D;

  W w;
#pragma unroll
  for (int c = 0; c < CP; ++c) w.acc[c] = pa_f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -FLT_MAX, l = 0.0f;
  bool bad = ch.bad;
  if (lo < hi) {
    const TC *K = static_cast<const TC *>(a.k), *V = static_cast<const TC *>(a.v);
    const int32_t *trow = a.table + ch.seq * a.per;
    const int32_t stride = static_cast<int32_t>(a.kv_heads * a.page), jrow = static_cast<int32_t>(j * a.page);
    const int32_t pages = static_cast<int32_t>(a.pages), page = static_cast<int32_t>(a.page);
    const int32_t steps = (hi - lo + POS - 1) / POS;
    int32_t (*rows)[POS] = rowbuf[wave];
    // The pool rows of a step's positions, those past the chunk's end the
    // last one's again (their scores are dropped below): page ids a step
    // ahead, so their latency is off the loop.  No load here is under a
    // condition -- past the last step the last row comes again -- for one
    // that may or may not be in flight makes every later wait a wait for all.
    auto position = [&](int32_t i) {  // without a sign: past the end it may pass 2^31
      const uint32_t p = static_cast<uint32_t>(lo) + static_cast<uint32_t>(i) * POS + (lane & (POS - 1));
      return p < static_cast<uint32_t>(hi) ? p : static_cast<uint32_t>(hi) - 1;
    };
    auto page_id = [&](int32_t i) { return trow[page_of(position(i), a.div)]; };
    auto put_rows = [&](int32_t i, int32_t id, int b) {
      const uint32_t p = position(i);
      const bool out = id < 0 || id >= pages;
      bad |= out;
      id = out ? 0 : id;
      if (lane < POS)
        rows[b][lane] = id * stride + jrow + static_cast<int32_t>(p - page_of(p, a.div) * static_cast<uint32_t>(page));
      __builtin_amdgcn_wave_barrier();  // read below by this wavefront, whose LDS accesses run in order
    };
    // The first step's page ids and the queries are asked for together, and
    // the first keys before the queries are waited for; the loop asks for a
    // step's values at its start and for the next step's keys once its own
    // are used.
    int32_t i = wave;
    int b = 0;
    const int32_t id0 = page_id(i);
    // STREAM: large pools go past the caches (one sequence of 100001 positions
    // 72 us, 79 without), unless a neighbouring row of the table begins with
    // the same page, whose block then reads the same keys (64 rows of one
    // sequence of 20000: 358 us through the caches, 535 past them).
    int32_t own = 0, prev = 1, next = 1;
    if constexpr (STREAM) {
      own = trow[0];
      if (ch.seq > 0) prev = trow[-a.per];
      if (ch.seq + 1 < a.seqs) next = trow[a.per];
    }
    constexpr int QN = (PA_HEADS * D / 4 + PA_WAVES * 64 - 1) / (PA_WAVES * 64);
    float4 qv[QN];
#pragma unroll
    for (int u = 0; u < QN; ++u) {
      const int e = 4 * (tid + u * PA_WAVES * 64);
      qv[u] = f32x4_get(static_cast<const TQ *>(a.q) + q0 + (e < nh * D ? e : 0));
    }
    int32_t id = page_id(i + PA_WAVES);
    put_rows(i, id0, 0);
    bool nt = false;
    if constexpr (STREAM) {
      const bool first = ch.seq == 0, last = ch.seq + 1 == a.seqs;
      nt = !__builtin_amdgcn_readfirstlane((!first && own == prev) || (!last && own == next));
    }
    if (STREAM && nt) w.template load_k<true>(K, rows[0], lane);
    else w.template load_k<false>(K, rows[0], lane);
    // Scaled, heads past the tile's as zeros.
#pragma unroll
    for (int u = 0; u < QN; ++u) {
      const int e = 4 * (tid + u * PA_WAVES * 64);
      const float f = e < nh * D ? a.scale : 0.0f;
      float4 x = make_float4(qv[u].x * f, qv[u].y * f, qv[u].z * f, qv[u].w * f);
      if (e >= nh * D) x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (e < PA_HEADS * D) *reinterpret_cast<float4 *>(sm + e / D * QS + e % D) = x;
    }
    __syncthreads();
    w.query(sm, lane);
    auto run = [&](auto stream) {
      constexpr bool NT = decltype(stream)::value;
      for (; i < steps; i += PA_WAVES, b ^= 1) {
        w.template load_v<NT>(V, rows[b], lane);
        put_rows(i + PA_WAVES, id, b ^ 1);
        id = page_id(i + 2 * PA_WAVES);
        pa_f32x4 s[TILES];
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < TILES; ++t) s[t] = w.scores(t);
        w.template load_k<NT>(K, rows[b ^ 1], lane);
        const int32_t left = hi - lo - i * POS;  // positions from this step's first
        if (left < POS) {
#pragma unroll
          for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (16 * t + 4 * (lane >> 4) + e >= left) s[t][e] = -INFINITY;
        }
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx = max_nan(mx, s[t][e]);
        const float mn = max_nan(m, head_max(mx));
        const float r = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= r;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[t][e] = __builtin_amdgcn_exp2f(s[t][e] - mn);
            l += s[t][e];
          }
#pragma unroll
        for (int c = 0; c < CP; ++c) w.acc[c] *= r;
        w.values(s);
      }
    };
    if (STREAM && nt) run(std::integral_constant<bool, STREAM>{});
    else run(std::false_type{});
    __syncthreads();  // the queries are read
  }
  if (__any(bad) && lane == 0) atomicOr(a.flags, FLAG_INDEX_RANGE);
  if (tid == 0 && ch.c == 0 && jt == 0 && a.cuts && !a.plan) a.cuts[ch.seq] = make_int2(ch.n, ch.slot);
  l = fold_columns<16>(l);

  // The wavefronts' results through LDS: head h's D sums at [wave][h][QS].
  {
    const int h = lane & 15, gq = lane >> 4;
    if (lane < PA_HEADS) {
      stat[wave][0][lane] = m;
      stat[wave][1][lane] = l;
    }
    float *dst = sm + (wave * PA_HEADS + h) * QS;
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int c = 0; c < CP; ++c) dst[CP * (4 * gq + e) + c] = w.acc[c][e];
  }
  __syncthreads();
  float *part = nullptr;
  if (ch.n > 1) {
    const int64_t slot = ch.slot + ch.c;
    if (slot >= a.slots) return;  // never: the cut's bound
    part = a.part + (slot * parts + jt) * pa_stride(a.live, D);
  }
  for (int e = 4 * tid; e < nh * D; e += 4 * PA_WAVES * 64) {
    const int h = e / D, c = e % D;
    float mw[PA_WAVES], lw[PA_WAVES];
    float4 x[PA_WAVES];
#pragma unroll
    for (int y = 0; y < PA_WAVES; ++y) {
      mw[y] = stat[y][0][h];
      lw[y] = stat[y][1][h];
      x[y] = *reinterpret_cast<const float4 *>(sm + (y * PA_HEADS + h) * QS + c);
    }
    float M = mw[0], den = 0.0f;
#pragma unroll
    for (int y = 1; y < PA_WAVES; ++y) M = max_nan(M, mw[y]);
    float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int y = 0; y < PA_WAVES; ++y) {
      const float wt = __builtin_amdgcn_exp2f(mw[y] - M);
      den += wt * lw[y];
      t.x += wt * x[y].x;
      t.y += wt * x[y].y;
      t.z += wt * x[y].z;
      t.w += wt * x[y].w;
    }
    if (part) {
      if (c == 0) {
        part[h] = M;
        part[a.live + h] = den;
      }
      *reinterpret_cast<float4 *>(part + pa_acc0(a.live) + e) = t;
    } else {
      den = isnan(den) ? den : (den > FLT_MIN ? den : FLT_MIN);
      t = make_float4(t.x / den, t.y / den, t.z / den, t.w / den);
      if (a.out16) f32x4_put(static_cast<uint16_t *>(a.out) + q0 + e, t);
      else f32x4_put(static_cast<float *>(a.out) + q0 + e, t);
    }
  }
}

// Joins the chunks of a cut sequence, a block a (sequence, query head): the
// chunks' weights 2^(m_c - M) in LDS, then D / 4 lanes a group, the groups
// taking the chunks in turn, and the groups' sums added in order.  A thread
// asks for its first chunks' values together with the statistics.
template <int D>
__global__ void __launch_bounds__(256) attend_join_kernel(AttendArgs a) {
  constexpr int LP = D / 4, NG = 256 / LP, PRE = 8;
  extern __shared__ float wts[];  // a chunk each
  __shared__ float red[4];
  __shared__ float4 sums[256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t s = blockIdx.x / a.heads;
  const int h = static_cast<int>(blockIdx.x % a.heads);
  const int2 cut = a.cuts[s];
  const int n = cut.x;
  if (n < 2 || cut.y + n > a.slots) return;
  const int j = h / a.group, hg = h % a.group, jt = j * a.tiles + hg / PA_HEADS, ht = hg % PA_HEADS;
  const int64_t parts = a.kv_heads * a.tiles, ps = pa_stride(a.live, D);
  const float *p = a.part + (static_cast<int64_t>(cut.y) * parts + jt) * ps;
  const int64_t step = parts * ps;
  const int grp = tid / LP, c4 = 4 * (tid % LP);
  const float *pv = p + pa_acc0(a.live) + ht * D + c4;
  const int c0 = tid < n ? tid : n - 1;
  const float m0 = p[c0 * step + ht], l0 = p[c0 * step + a.live + ht];
  float4 x[PRE];
#pragma unroll
  for (int i = 0; i < PRE; ++i) {
    const int c = grp + i * NG;
    x[i] = *reinterpret_cast<const float4 *>(pv + (c < n ? c : n - 1) * step);
  }
  float M = m0;
  for (int c = tid + 256; c < n; c += 256) M = max_nan(M, p[c * step + ht]);
  M = fold_max<64>(M);
  if (lane == 0) red[wave] = M;
  __syncthreads();
  M = max_nan(max_nan(red[0], red[1]), max_nan(red[2], red[3]));
  __syncthreads();
  float den = 0.0f;
  if (tid < n) {
    const float wt = __builtin_amdgcn_exp2f(m0 - M);
    wts[tid] = wt;
    den = wt * l0;
  }
  for (int c = tid + 256; c < n; c += 256) {
    const float wt = __builtin_amdgcn_exp2f(p[c * step + ht] - M);
    wts[c] = wt;
    den += wt * p[c * step + a.live + ht];
  }
  den = fold_sum<64>(den);
  if (lane == 0) red[wave] = den;
  __syncthreads();
  den = (red[0] + red[1]) + (red[2] + red[3]);
  den = isnan(den) ? den : (den > FLT_MIN ? den : FLT_MIN);
  float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float wt, float4 y) {
    t.x += wt * y.x;
    t.y += wt * y.y;
    t.z += wt * y.z;
    t.w += wt * y.w;
  };
#pragma unroll
  for (int i = 0; i < PRE; ++i)
    if (grp + i * NG < n) add(wts[grp + i * NG], x[i]);
#pragma unroll 8
  for (int c = grp + PRE * NG; c < n; c += NG) add(wts[c], *reinterpret_cast<const float4 *>(pv + c * step));
  sums[tid] = t;
  __syncthreads();
  if (tid < LP) {
    t = sums[tid];
#pragma unroll
    for (int y = 1; y < NG; ++y) {
      const float4 o = sums[y * LP + tid];
      t.x += o.x;
      t.y += o.y;
      t.z += o.z;
      t.w += o.w;
    }
    t = make_float4(t.x / den, t.y / den, t.z / den, t.w / den);
    const int64_t at = (s * a.heads + h) * D + 4 * tid;
    if (a.out16) f32x4_put(static_cast<uint16_t *>(a.out) + at, t);
    else f32x4_put(static_cast<float *>(a.out) + at, t);
  }
}

template <int D, bool STREAM>
void attend_types(Ctx *ctx, const AttendArgs &a, unsigned grid, bool q16, bool kv16) {
  constexpr int THR = PA_WAVES * 64;
  if (q16 && kv16) attend_kernel<D, uint16_t, uint16_t, STREAM><<<grid, THR, 0, ctx->stream>>>(a);
  else if (q16) attend_kernel<D, uint16_t, float, STREAM><<<grid, THR, 0, ctx->stream>>>(a);
  else if (kv16) attend_kernel<D, float, uint16_t, STREAM><<<grid, THR, 0, ctx->stream>>>(a);
  else attend_kernel<D, float, float, STREAM><<<grid, THR, 0, ctx->stream>>>(a);
}

template <int D>
int attend_launch(Ctx *ctx, AttendArgs a, bool q16, bool kv16) {
  const int64_t parts = static_cast<int64_t>(a.kv_heads) * a.tiles;
  const PagedCut shape = paged_cut(a.seqs, a.per * a.page, parts);
  const int64_t chunks = shape.chunks;
  const bool cut = shape.cut, planned = a.seqs > PA_SELF;
  a.least = static_cast<int32_t>(shape.least);
  a.per_chunk = 1.0 / static_cast<double>(shape.target);
  a.chunks = chunks;
  a.slots = shape.slots;
  if (chunks * parts > kGridThreads / 256 || (cut && a.seqs * a.heads > kGridThreads / 256))
    return fail(ctx, MI_E_UNSUPPORTED, "paged_attention: grid too large");
  const size_t cuts = cut ? (static_cast<size_t>(a.seqs) * sizeof(int2) + 255) / 256 * 256 : 0,
               plan = planned ? (static_cast<size_t>(chunks) * sizeof(int4) + 255) / 256 * 256 : 0,
               part = static_cast<size_t>(a.slots * parts * pa_stride(a.live, D)) * sizeof(float);
  if (cuts + plan + part > 0) {
    char *p = static_cast<char *>(scratch(ctx, cuts + plan + part));
    if (!p) return fail(ctx, MI_E_OOM, "paged_attention scratch");
    a.cuts = cut ? reinterpret_cast<int2 *>(p) : nullptr;
    a.plan = planned ? reinterpret_cast<int4 *>(p + cuts) : nullptr;
    a.part = reinterpret_cast<float *>(p + cuts + plan);
  }
  if (planned) {
    attend_plan_kernel<<<1, 1024, 0, ctx->stream>>>(a);
    if (int s = check_launch(ctx, "paged_attention plan")) return s;
  }
  const unsigned grid = static_cast<unsigned>(chunks * parts);
  // Keys are read once, but once a tile where a kv head has more heads.
  const int64_t bytes = 2 * a.pages * a.page * a.kv_heads * D * (kv16 ? 2 : 4);
  if (a.tiles == 1 && bytes >= kStreamBytes) attend_types<D, true>(ctx, a, grid, q16, kv16);
  else attend_types<D, false>(ctx, a, grid, q16, kv16);
  if (int s = check_launch(ctx, "paged_attention")) return s;
  if (!cut) return MI_OK;
  attend_join_kernel<D><<<static_cast<unsigned>(a.seqs * a.heads), 256,
                          (a.slots < PA_CHUNKS ? a.slots : PA_CHUNKS) * sizeof(float), ctx->stream>>>(a);
  return check_launch(ctx, "paged_attention join");
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int mi_qkv_rope_paged(mi_ctx *ctx, mi_id qkv, mi_id cos_table, mi_id sin_table, mi_id table, mi_id lens,
                                 mi_id starts, int64_t heads, int64_t kv_heads, int64_t page, mi_id k_pages,
                                 mi_id v_pages, int out_elem, mi_id *q_out) {
  MI_ENTER(ctx);
  if (!q_out) return fail(ctx, MI_E_ARG, "null out pointer");
  DeviceGuard on(ctx);
  MI_BUF(ctx, xb, qkv);
  MI_BUF(ctx, cb, cos_table);
  MI_BUF(ctx, sb, sin_table);
  PagedCache c;
  if (int s = paged_cache(ctx, "qkv_rope_paged", k_pages, v_pages, table, lens, heads, kv_heads, page, &c)) return s;
  if (k_pages == v_pages) return fail(ctx, MI_E_ARG, "qkv_rope_paged: one buffer given as both page pools");
  if (!elem_float(xb->elem) || xb->tiles || cb->elem != MI_F32 || sb->elem != MI_F32 || !elem_float(out_elem))
    return fail(ctx, MI_E_ARG, "qkv_rope_paged takes F32 or BF16 rows and results and F32 tables");
  if (heads > (INT32_MAX / c.D - 2 * kv_heads) || kv_heads > INT32_MAX / (4 * c.D))
    return fail(ctx, MI_E_UNSUPPORTED, "qkv_rope_paged: %lld heads", (long long)heads);
  const int64_t R = xb->rows, W = (heads + 2 * kv_heads) * c.D;
  if (xb->cols != W)
    return fail(ctx, MI_E_ARG, "qkv_rope_paged: rows of %lld, want (heads + 2 kv_heads) * %lld = %lld",
                (long long)xb->cols, (long long)c.D, (long long)W);
  if (cb->cols != c.D || sb->cols != c.D || cb->rows != sb->rows)
    return fail(ctx, MI_E_ARG, "qkv_rope_paged: rope tables [%lld, %lld] and [%lld, %lld] for heads of %lld",
                (long long)cb->rows, (long long)cb->cols, (long long)sb->rows, (long long)sb->cols, (long long)c.D);
  const int32_t *sp = nullptr;
  if (starts) {
    MI_BUF(ctx, stb, starts);
    if (stb->elem != MI_I32 || stb->numel() != c.seqs + 1)
      return fail(ctx, MI_E_ARG, "qkv_rope_paged: starts %s [%lld, %lld], want I32 of %lld", elem_name(stb->elem),
                  (long long)stb->rows, (long long)stb->cols, (long long)(c.seqs + 1));
    sp = static_cast<const int32_t *>(stb->ptr);
  } else if (R != c.seqs) {
    return fail(ctx, MI_E_ARG, "qkv_rope_paged: %lld rows for %lld sequences (one each without starts)", (long long)R,
                (long long)c.seqs);
  }
  if (R > kGridThreads / 256 || (W / 8 + 255) / 256 > 65535)
    return fail(ctx, MI_E_UNSUPPORTED, "qkv_rope_paged: grid too large");
  mi_id id;
  Buffer *ob;
  int s = new_buffer(ctx, R, heads * c.D, out_elem, &id, &ob);
  if (s) return s;
  if (R > 0) {
    AppendArgs a;
    a.qkv = xb->ptr;
    a.cosp = static_cast<const float *>(cb->ptr);
    a.sinp = static_cast<const float *>(sb->ptr);
    a.positions = cb->rows;
    a.table = c.table;
    a.lens = c.lens;
    a.starts = sp;
    a.rows = R;
    a.seqs = c.seqs;
    a.per = c.per;
    a.pages = c.pages;
    a.page = page;
    a.div = page_div(static_cast<uint32_t>(page));
    a.heads = static_cast<int>(heads);
    a.kv_heads = static_cast<int>(kv_heads);
    a.items = static_cast<int>(W / 8);
    a.per_row = page_div(static_cast<uint32_t>(a.items));
    a.block_rows = a.items < 256 ? 256 / a.items : 1;
    a.k = c.k;
    a.v = c.v;
    a.q = ob->ptr;
    a.flags = flags(ctx);
    if (xb->elem == MI_BF16) {
      if (c.elem == MI_BF16) append_launch<uint16_t, uint16_t>(ctx, a, c.D, out_elem);
      else append_launch<uint16_t, float>(ctx, a, c.D, out_elem);
    } else {
      if (c.elem == MI_BF16) append_launch<float, uint16_t>(ctx, a, c.D, out_elem);
      else append_launch<float, float>(ctx, a, c.D, out_elem);
    }
    s = check_launch(ctx, "qkv_rope_paged");
    if (s) { mi_free(ctx, id); return s; }
  }
  *q_out = id;
  return MI_OK;
}

extern "C" int mi_paged_attention(mi_ctx *ctx, mi_id q, mi_id k_pages, mi_id v_pages, mi_id table, mi_id lens,
                                  int64_t heads, int64_t kv_heads, int64_t page, float scale, int out_elem,
                                  mi_id *out) {
  MI_ENTER(ctx);
  if (!out) return fail(ctx, MI_E_ARG, "null out pointer");
  DeviceGuard on(ctx);
  MI_BUF(ctx, qb, q);
  PagedCache c;
  if (int s = paged_cache(ctx, "paged_attention", k_pages, v_pages, table, lens, heads, kv_heads, page, &c)) return s;
  if (!elem_float(qb->elem) || qb->tiles || !elem_float(out_elem))
    return fail(ctx, MI_E_ARG, "paged_attention takes F32 or BF16 queries and results");
  if (heads > INT32_MAX / c.D || qb->rows != c.seqs || qb->cols != heads * c.D)
    return fail(ctx, MI_E_ARG, "paged_attention: q is [%lld, %lld], want [%lld, %lld * %lld]", (long long)qb->rows,
                (long long)qb->cols, (long long)c.seqs, (long long)heads, (long long)c.D);
  mi_id id;
  Buffer *ob;
  int s = new_buffer(ctx, c.seqs, heads * c.D, out_elem, &id, &ob);
  if (s) return s;
  if (c.seqs > 0) {
    AttendArgs a{};
    a.q = qb->ptr;
    a.k = c.k;
    a.v = c.v;
    a.table = c.table;
    a.lens = c.lens;
    a.seqs = c.seqs;
    a.per = c.per;
    a.pages = c.pages;
    a.page = page;
    a.div = page_div(static_cast<uint32_t>(page));
    a.heads = static_cast<int>(heads);
    a.kv_heads = static_cast<int>(kv_heads);
    a.group = a.heads / a.kv_heads;
    a.tiles = (a.group + PA_HEADS - 1) / PA_HEADS;
    a.live = a.group < PA_HEADS ? a.group : PA_HEADS;
    a.by_parts = page_div(static_cast<uint32_t>(a.kv_heads * a.tiles));
    a.by_tiles = page_div(static_cast<uint32_t>(a.tiles));
    a.out16 = out_elem == MI_BF16;
    a.scale = scale * 1.4426950408889634f;
    a.out = ob->ptr;
    a.flags = flags(ctx);
    const bool q16 = qb->elem == MI_BF16, kv16 = c.elem == MI_BF16;
    switch (c.D) {
      case 16: s = attend_launch<16>(ctx, a, q16, kv16); break;
      case 32: s = attend_launch<32>(ctx, a, q16, kv16); break;
      case 64: s = attend_launch<64>(ctx, a, q16, kv16); break;
      default: s = attend_launch<128>(ctx, a, q16, kv16); break;
    }
    if (s) { mi_free(ctx, id); return s; }
  }
  *out = id;
  return MI_OK;
}
