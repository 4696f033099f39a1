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
  int heads, kv_heads;
  void *k, *v, *q;
  uint32_t *flags;
};

// The sequence of row r: the last one whose rows start at or before it --
// counted over the bounds a wavefront at a time, so a lookup is one or a few
// independent loads and not a chain of a binary search's.
__device__ __forceinline__ int64_t append_seq(const AppendArgs &a, int64_t r) {
  int64_t n = 0;
  const int lane = threadIdx.x & 63;
  for (int64_t s0 = 1; s0 <= a.seqs; s0 += 64) {
    const bool in = s0 + lane <= a.seqs && a.starts[s0 + lane] <= r;
    n += __popcll(__ballot(in));
  }
  return n;
}

// One new row a block column, eight elements a thread: for a q or k head four
// of the first half and their partners of the second, for a v head eight in a
// row.  rope: x cos + rotate(x) sin, two roundings, as mi_rope.
template <typename TI, typename TC, typename TO>
__global__ void __launch_bounds__(256) append_kernel(AppendArgs a, int D) {
  const int64_t r = blockIdx.x;
  const int per_head = D / 8, items = (a.heads + 2 * a.kv_heads) * per_head;
  const int item = blockIdx.y * 256 + threadIdx.x;
  int64_t seq = r, first = r, end = r + 1;
  PagedPos p{PAGED_IDLE, 0};
  if (a.starts) {
    seq = append_seq(a, r);
    if (seq < a.seqs) {
      first = a.starts[seq];
      end = a.starts[seq + 1];
    }
  }
  if (seq < a.seqs) p = paged_pos(r, first, end, a.lens[seq], a.per * a.page);
  int64_t pg = 0;
  if (p.state == PAGED_OK) {
    pg = a.table[seq * a.per + p.pos / a.page];
    if (pg < 0 || pg >= a.pages || p.pos >= a.positions) p.state = PAGED_BAD;
  }
  if (p.state == PAGED_BAD && item == 0) atomicOr(a.flags, FLAG_INDEX_RANGE);
  if (item >= items) return;
  const int head = item / per_head, quad = item - head * per_head, half = D / 2;
  const bool turn = head < a.heads + a.kv_heads;
  const int c0 = turn ? 4 * quad : 8 * quad, c1 = turn ? c0 + half : c0 + 4;
  TO *q = static_cast<TO *>(a.q) + (r * a.heads + head) * D;
  if (p.state != PAGED_OK) {
    if (head < a.heads) {
      f32x4_put(q + c0, make_float4(0.f, 0.f, 0.f, 0.f));
      f32x4_put(q + c1, make_float4(0.f, 0.f, 0.f, 0.f));
    }
    return;
  }
  const TI *x = static_cast<const TI *>(a.qkv) + (r * (a.heads + 2 * a.kv_heads) + head) * D;
  float4 lo = f32x4_get(x + c0), hi = f32x4_get(x + c1);
  if (turn) {
    const float *cr = a.cosp + p.pos * D, *sr = a.sinp + p.pos * D;
    const float4 cl = f32x4_get(cr + c0), ch = f32x4_get(cr + c1), sl = f32x4_get(sr + c0), sh = f32x4_get(sr + c1);
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
  TC *dst = static_cast<TC *>(turn ? a.k : a.v) + paged_row(pg, j, p.pos % a.page, a.kv_heads, a.page) * D;
  f32x4_put(dst + c0, lo);
  f32x4_put(dst + c1, hi);
}

template <typename TI, typename TC>
void append_launch(Ctx *ctx, const AppendArgs &a, int64_t D, int out_elem) {
  const int64_t items = (a.heads + 2 * static_cast<int64_t>(a.kv_heads)) * (D / 8);
  const dim3 grid(static_cast<unsigned>(a.rows), grid_for(items, 256));
  if (out_elem == MI_BF16)
    append_kernel<TI, TC, uint16_t><<<grid, 256, 0, ctx->stream>>>(a, static_cast<int>(D));
  else
    append_kernel<TI, TC, float><<<grid, 256, 0, ctx->stream>>>(a, static_cast<int>(D));
}

// --------------------------------------------------------------- attention

struct AttendArgs {
  const void *q, *k, *v;
  const int32_t *table, *lens;
  int64_t seqs, per, pages, page;
  int heads, kv_heads;
  float scale;
  void *out;
  uint32_t *flags;
};

// One wavefront a (sequence, query head), 64 positions a step: a lane forms
// the score of its position, the running maximum and sum rescale what was
// gathered, and the value rows are added with a lane a column.
template <int D, typename TQ, typename TC, typename TO>
__global__ void __launch_bounds__(64) attend_kernel(AttendArgs a) {
  __shared__ float qs[D];
  const int64_t s = blockIdx.x / a.heads, h = blockIdx.x % a.heads;
  const int lane = threadIdx.x;
  const int64_t j = h / (a.heads / a.kv_heads), cap = a.per * a.page;
  const TQ *q = static_cast<const TQ *>(a.q) + (s * a.heads + h) * D;
  for (int c = 4 * lane; c < D; c += 256) *reinterpret_cast<float4 *>(qs + c) = f32x4_get(q + c);
  __syncthreads();
  const int64_t raw = a.lens[s], len = paged_len(raw, cap);
  if (raw != len && lane == 0) atomicOr(a.flags, FLAG_INDEX_RANGE);
  const TC *K = static_cast<const TC *>(a.k), *V = static_cast<const TC *>(a.v);
  constexpr int CPL = (D + 63) / 64;
  float m = -FLT_MAX, l = 0.0f, acc[CPL] = {};
  for (int64_t p0 = 0; p0 < len; p0 += 64) {
    const int64_t p = p0 + lane < len ? p0 + lane : len - 1;
    int64_t pg = a.table[s * a.per + p / a.page];
    if (pg < 0 || pg >= a.pages) {
      atomicOr(a.flags, FLAG_INDEX_RANGE);
      pg = 0;
    }
    const int64_t row = paged_row(pg, j, p % a.page, a.kv_heads, a.page);
    float sc = 0.0f;
    for (int c = 0; c < D; c += 4) {
      const float4 kv = f32x4_get(K + row * D + c), qv = *reinterpret_cast<const float4 *>(qs + c);
      sc += (qv.x * kv.x + qv.y * kv.y) + (qv.z * kv.z + qv.w * kv.w);
    }
    sc = p0 + lane < len ? sc * a.scale : -INFINITY;
    const float mn = max_nan(m, fold_max<64>(sc));
    const float w = expf(m - mn), e = p0 + lane < len ? expf(sc - mn) : 0.0f;
    l = l * w + fold_sum<64>(e);
    m = mn;
    for (int i = 0; i < CPL; ++i) acc[i] *= w;
    const int n = static_cast<int>(len - p0 < 64 ? len - p0 : 64);
    for (int t = 0; t < n; ++t) {
      const float pt = __shfl(e, t, 64);
      const int64_t rt = __shfl(row, t, 64);
      for (int i = 0; i < CPL; ++i) {
        const int c = i * 64 + lane;
        if (c < D) {
          float x;
          if constexpr (sizeof(TC) == 2) x = bf16_bits_to_f32(V[rt * D + c]);
          else x = V[rt * D + c];
          acc[i] += pt * x;
        }
      }
    }
  }
  const float den = isnan(l) ? l : (l > FLT_MIN ? l : FLT_MIN);
  TO *o = static_cast<TO *>(a.out) + (s * a.heads + h) * D;
  for (int i = 0; i < CPL; ++i)
    if (i * 64 + lane < D) f32_put(o + i * 64 + lane, acc[i] / den);
}

template <int D, typename TQ, typename TC>
void attend_launch(Ctx *ctx, const AttendArgs &a, int out_elem) {
  const unsigned grid = static_cast<unsigned>(a.seqs * a.heads);
  if (out_elem == MI_BF16) attend_kernel<D, TQ, TC, uint16_t><<<grid, 64, 0, ctx->stream>>>(a);
  else attend_kernel<D, TQ, TC, float><<<grid, 64, 0, ctx->stream>>>(a);
}
template <int D>
void attend_types(Ctx *ctx, const AttendArgs &a, int q_elem, int cache_elem, int out_elem) {
  if (q_elem == MI_BF16) {
    if (cache_elem == MI_BF16) attend_launch<D, uint16_t, uint16_t>(ctx, a, out_elem);
    else attend_launch<D, uint16_t, float>(ctx, a, out_elem);
  } else {
    if (cache_elem == MI_BF16) attend_launch<D, float, uint16_t>(ctx, a, out_elem);
    else attend_launch<D, float, float>(ctx, a, out_elem);
  }
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
  if (R > INT32_MAX || (W / 8 + 255) / 256 > 65535)
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
    a.heads = static_cast<int>(heads);
    a.kv_heads = static_cast<int>(kv_heads);
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
  if (c.seqs * heads > INT32_MAX) return fail(ctx, MI_E_UNSUPPORTED, "paged_attention: grid too large");
  mi_id id;
  Buffer *ob;
  int s = new_buffer(ctx, c.seqs, heads * c.D, out_elem, &id, &ob);
  if (s) return s;
  if (c.seqs > 0) {
    AttendArgs a;
    a.q = qb->ptr;
    a.k = c.k;
    a.v = c.v;
    a.table = c.table;
    a.lens = c.lens;
    a.seqs = c.seqs;
    a.per = c.per;
    a.pages = c.pages;
    a.page = page;
    a.heads = static_cast<int>(heads);
    a.kv_heads = static_cast<int>(kv_heads);
    a.scale = scale;
    a.out = ob->ptr;
    a.flags = flags(ctx);
    switch (c.D) {
      case 16: attend_types<16>(ctx, a, qb->elem, c.elem, out_elem); break;
      case 32: attend_types<32>(ctx, a, qb->elem, c.elem, out_elem); break;
      case 64: attend_types<64>(ctx, a, qb->elem, c.elem, out_elem); break;
      default: attend_types<128>(ctx, a, qb->elem, c.elem, out_elem); break;
    }
    s = check_launch(ctx, "paged_attention");
    if (s) { mi_free(ctx, id); return s; }
  }
  *out = id;
  return MI_OK;
}
