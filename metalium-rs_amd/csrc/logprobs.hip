// Log probabilities of given tokens over rows of logits, with each row's
// entropy and its likeliest tokens, and the gradient of the first two.
//
// Reference: the log_softmax composition and the gather of a target's value
// (crates/burn-tt/src/ops.rs:5133-5166, 1001; mi_log_softmax_ce here), and the
// greedy pick of the generation loop (crates/tt-models/src/generate.rs:
// 176-183), of which the alternatives are the ordered form.
//
// With z = scale x, m = max z, S = sum e^(z - m) and T = sum (z - m) e^(z - m):
// lse = m + ln S, logp = z_target - lse, entropy = ln S - T / S (both terms
// are at least 0, so nothing cancels).
#include <cmath>

#include "common.hpp"
#include "wave.hpp"

namespace mi {
namespace {

__device__ __forceinline__ float logit(const float *p) { return *p; }
__device__ __forceinline__ float logit(const uint16_t *p) { return bf16_bits_to_f32(*p); }

struct LogprobArgs {
  const void *x;
  int64_t rows, cols;
  const int32_t *targets;
  float scale;
  int top;
  float *logp, *lse, *entropy, *top_logp;
  int32_t *top_ids;
  uint32_t *flags;
};

// Whether (v, i) comes behind the pick `p` in the order of alternatives.
__device__ __forceinline__ bool behind(float v, int32_t i, ArgBest p) {
  const ArgBest b = better(ArgBest{v, i}, p);
  return b.i == p.i && i != p.i;
}

template <typename T>
__global__ void __launch_bounds__(256) logprobs_kernel(LogprobArgs a) {
  __shared__ float red[4][2];
  __shared__ ArgBest bests[4];
  const int64_t r = blockIdx.x;
  const T *x = static_cast<const T *>(a.x) + r * a.cols;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  float m = -INFINITY;
  for (int64_t c = tid; c < a.cols; c += 256) m = max_nan(m, logit(x + c) * a.scale);
  m = fold_max<64>(m);
  if (lane == 0) red[wave][0] = m;
  __syncthreads();
  m = max_nan(max_nan(red[0][0], red[1][0]), max_nan(red[2][0], red[3][0]));
  __syncthreads();
  float s = 0.0f, t = 0.0f;
  for (int64_t c = tid; c < a.cols; c += 256) {
    const float d = logit(x + c) * a.scale - m, e = expf(d);
    s += e;
    t += e == 0.0f ? 0.0f : d * e;
  }
  s = fold_sum<64>(s);
  t = fold_sum<64>(t);
  if (lane == 0) { red[wave][0] = s; red[wave][1] = t; }
  __syncthreads();
  s = (red[0][0] + red[1][0]) + (red[2][0] + red[3][0]);
  t = (red[0][1] + red[1][1]) + (red[2][1] + red[3][1]);
  const bool none = m == -INFINITY;  // every logit is -inf
  const float lse = none ? -INFINITY : m + logf(s);
  if (tid == 0) {
    if (a.lse) a.lse[r] = lse;
    if (a.entropy) a.entropy[r] = none ? 0.0f : logf(s) - t / s;
    if (a.logp) {
      const int32_t g = a.targets[r];
      const bool ok = g >= 0 && g < a.cols;
      if (!ok) atomicOr(a.flags, FLAG_INDEX_RANGE);
      a.logp[r] = !ok ? 0.0f : none ? -INFINITY : logit(x + g) * a.scale - lse;
    }
  }
  ArgBest last{0.0f, -1};
  for (int k = 0; k < a.top; ++k) {
    ArgBest b{0.0f, -1};
    for (int64_t c = tid; c < a.cols; c += 256) {
      const float v = logit(x + c);
      const int32_t i = static_cast<int32_t>(c);
      if (k > 0 && !behind(v, i, last)) continue;
      b = b.i < 0 ? ArgBest{v, i} : better(b, ArgBest{v, i});
    }
    for (int o = 32; o >= 1; o >>= 1) {
      const ArgBest n{__shfl_xor(b.v, o, 64), __shfl_xor(b.i, o, 64)};
      b = n.i < 0 ? b : b.i < 0 ? n : better(b, n);
    }
    __syncthreads();
    if (lane == 0) bests[wave] = b;
    __syncthreads();
    last = bests[0];
    for (int w = 1; w < 4; ++w) last = bests[w].i < 0 ? last : last.i < 0 ? bests[w] : better(last, bests[w]);
    if (tid == 0) {
      a.top_logp[r * a.top + k] = none ? -INFINITY : last.v * a.scale - lse;
      a.top_ids[r * a.top + k] = last.i;
    }
  }
}

struct LogprobGradArgs {
  const void *x;
  int64_t rows, cols;
  const int32_t *targets;
  const float *lse, *entropy, *d_logp, *d_entropy;
  float scale;
  void *out;
  uint32_t *flags;
};

// dx_j = scale (g ([j = target] - p_j) - h p_j (z_j - lse + H)).
template <typename T, typename TO>
__global__ void __launch_bounds__(256) logprobs_backward_kernel(LogprobGradArgs a) {
  const int64_t r = blockIdx.x;
  const T *x = static_cast<const T *>(a.x) + r * a.cols;
  TO *o = static_cast<TO *>(a.out) + r * a.cols;
  const float lse = a.lse[r], h = a.d_entropy ? a.d_entropy[r] : 0.0f, H = a.d_entropy ? a.entropy[r] : 0.0f;
  float g = a.d_logp ? a.d_logp[r] : 0.0f;
  int32_t target = -1;
  if (a.d_logp) {
    target = a.targets[r];
    if (target < 0 || target >= a.cols) {
      if (threadIdx.x == 0) atomicOr(a.flags, FLAG_INDEX_RANGE);
      target = -1;
      g = 0.0f;
    }
  }
  for (int64_t c = threadIdx.x; c < a.cols; c += 256) {
    const float l = lse == -INFINITY ? -INFINITY : logit(x + c) * a.scale - lse, p = expf(l);
    const float w = p == 0.0f ? 0.0f : p * (g + h * (l + H));
    f32_put(o + c, ((c == target ? g : 0.0f) - w) * a.scale);
  }
}

int logits_check(Ctx *ctx, const char *what, const Buffer *xb, float scale) {
  if (!elem_float(xb->elem) || xb->tiles)
    return fail(ctx, MI_E_ARG, "%s takes F32 or BF16 logits in rows (%s)", what, elem_name(xb->elem));
  if (xb->cols < 1 || xb->cols > INT32_MAX || xb->rows > INT32_MAX)
    return fail(ctx, MI_E_ARG, "%s of [%lld, %lld]", what, (long long)xb->rows, (long long)xb->cols);
  if (!(scale > 0.0f) || std::isinf(scale))
    return fail(ctx, MI_E_ARG, "%s: scale %g (positive and finite)", what, static_cast<double>(scale));
  return MI_OK;
}

// One value a row of `elem`.
int column_check(Ctx *ctx, const char *what, const char *name, const Buffer *b, int elem, int64_t rows) {
  if (b->elem != elem || b->numel() != rows)
    return fail(ctx, MI_E_ARG, "%s: %s are %s [%lld, %lld], want %s of %lld", what, name, elem_name(b->elem),
                (long long)b->rows, (long long)b->cols, elem_name(elem), (long long)rows);
  return MI_OK;
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int mi_token_logprobs(mi_ctx *ctx, mi_id logits, mi_id targets, float scale, int64_t top, mi_id *logp,
                                 mi_id *lse, mi_id *entropy, mi_id *top_logp, mi_id *top_ids) {
  MI_ENTER(ctx);
  DeviceGuard on(ctx);
  MI_BUF(ctx, xb, logits);
  if (int s = logits_check(ctx, "token_logprobs", xb, scale)) return s;
  const int64_t R = xb->rows, C = xb->cols;
  if ((logp != nullptr) != (targets != 0))
    return fail(ctx, MI_E_ARG, "token_logprobs: targets and the place of their log probabilities go together");
  if (top < 0 || top > MI_TOP_MAX || top > C)
    return fail(ctx, MI_E_ARG, "token_logprobs: the top %lld of %lld (at most %d)", (long long)top, (long long)C,
                (int)MI_TOP_MAX);
  if ((top > 0) != (top_logp != nullptr) || (top > 0) != (top_ids != nullptr))
    return fail(ctx, MI_E_ARG, "token_logprobs: top %lld and the places of the alternatives go together",
                (long long)top);
  if (!logp && !lse && !entropy && top == 0) return fail(ctx, MI_E_ARG, "token_logprobs: no result asked for");
  LogprobArgs a{};
  if (targets) {
    MI_BUF(ctx, tb, targets);
    if (int s = column_check(ctx, "token_logprobs", "targets", tb, MI_I32, R)) return s;
    a.targets = static_cast<const int32_t *>(tb->ptr);
  }
  a.x = xb->ptr;
  a.rows = R;
  a.cols = C;
  a.scale = scale;
  a.top = static_cast<int>(top);
  a.flags = flags(ctx);
  mi_id ids[5] = {};
  mi_id *places[5] = {logp, lse, entropy, top_logp, top_ids};
  void *ptrs[5] = {};
  int s = MI_OK;
  for (int i = 0; i < 5 && !s; ++i) {
    if (!places[i]) continue;
    Buffer *b;
    s = new_buffer(ctx, R, i < 3 ? 1 : top, i == 4 ? MI_I32 : MI_F32, &ids[i], &b);
    if (!s) ptrs[i] = b->ptr;
  }
  if (!s && R > 0) {
    a.logp = static_cast<float *>(ptrs[0]);
    a.lse = static_cast<float *>(ptrs[1]);
    a.entropy = static_cast<float *>(ptrs[2]);
    a.top_logp = static_cast<float *>(ptrs[3]);
    a.top_ids = static_cast<int32_t *>(ptrs[4]);
    const unsigned grid = static_cast<unsigned>(R);
    if (xb->elem == MI_BF16) logprobs_kernel<uint16_t><<<grid, 256, 0, ctx->stream>>>(a);
    else logprobs_kernel<float><<<grid, 256, 0, ctx->stream>>>(a);
    s = check_launch(ctx, "token_logprobs");
  }
  if (s) {
    for (mi_id id : ids)
      if (id) mi_free(ctx, id);
    return s;
  }
  for (int i = 0; i < 5; ++i)
    if (places[i]) *places[i] = ids[i];
  return MI_OK;
}

extern "C" int mi_token_logprobs_backward(mi_ctx *ctx, mi_id logits, mi_id targets, mi_id lse, mi_id entropy,
                                          mi_id d_logp, mi_id d_entropy, float scale, int out_elem, mi_id *dlogits) {
  MI_ENTER(ctx);
  if (!dlogits) return fail(ctx, MI_E_ARG, "null out pointer");
  DeviceGuard on(ctx);
  MI_BUF(ctx, xb, logits);
  MI_BUF(ctx, lb, lse);
  if (int s = logits_check(ctx, "token_logprobs_backward", xb, scale)) return s;
  if (!elem_float(out_elem)) return fail(ctx, MI_E_ARG, "token_logprobs_backward result kind %d", out_elem);
  const int64_t R = xb->rows, C = xb->cols;
  if ((targets != 0) != (d_logp != 0) || (entropy != 0) != (d_entropy != 0) || (!d_logp && !d_entropy))
    return fail(ctx, MI_E_ARG, "token_logprobs_backward: targets with the gradients of their log probabilities, "
                               "entropies with theirs, and one of the two");
  if (int s = column_check(ctx, "token_logprobs_backward", "lse", lb, MI_F32, R)) return s;
  LogprobGradArgs a{};
  a.lse = static_cast<const float *>(lb->ptr);
  if (d_logp) {
    MI_BUF(ctx, tb, targets);
    MI_BUF(ctx, gb, d_logp);
    if (int s = column_check(ctx, "token_logprobs_backward", "targets", tb, MI_I32, R)) return s;
    if (int s = column_check(ctx, "token_logprobs_backward", "d_logp", gb, MI_F32, R)) return s;
    a.targets = static_cast<const int32_t *>(tb->ptr);
    a.d_logp = static_cast<const float *>(gb->ptr);
  }
  if (d_entropy) {
    MI_BUF(ctx, eb, entropy);
    MI_BUF(ctx, hb, d_entropy);
    if (int s = column_check(ctx, "token_logprobs_backward", "entropies", eb, MI_F32, R)) return s;
    if (int s = column_check(ctx, "token_logprobs_backward", "d_entropy", hb, MI_F32, R)) return s;
    a.entropy = static_cast<const float *>(eb->ptr);
    a.d_entropy = static_cast<const float *>(hb->ptr);
  }
  a.x = xb->ptr;
  a.rows = R;
  a.cols = C;
  a.scale = scale;
  a.flags = flags(ctx);
  mi_id id;
  Buffer *ob;
  int s = new_buffer(ctx, R, C, out_elem, &id, &ob);
  if (s) return s;
  a.out = ob->ptr;
  if (R > 0) {
    const unsigned grid = static_cast<unsigned>(R);
    const bool x16 = xb->elem == MI_BF16, o16 = out_elem == MI_BF16;
    if (x16 && o16) logprobs_backward_kernel<uint16_t, uint16_t><<<grid, 256, 0, ctx->stream>>>(a);
    else if (x16) logprobs_backward_kernel<uint16_t, float><<<grid, 256, 0, ctx->stream>>>(a);
    else if (o16) logprobs_backward_kernel<float, uint16_t><<<grid, 256, 0, ctx->stream>>>(a);
    else logprobs_backward_kernel<float, float><<<grid, 256, 0, ctx->stream>>>(a);
    s = check_launch(ctx, "token_logprobs_backward");
    if (s) { mi_free(ctx, id); return s; }
  }
  *dlogits = id;
  return MI_OK;
}
