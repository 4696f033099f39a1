// Log probabilities of given tokens over rows of logits, with each row's
// entropy and its likeliest tokens, and the gradient of the first two.
//
// Reference: the log_softmax composition and the gather of a target's value
// (crates/burn-tt/src/ops.rs:5133-5166, 1001; mi_log_softmax_ce here), and the
// greedy pick of the generation loop (crates/tt-models/src/generate.rs:
// 176-183), of which the alternatives are the ordered form.
//
// With m = max x, c = scale log2(e), d = (x - m) c, S = sum 2^d and
// T = sum d 2^d: lse = scale m + ln S, logp = ln 2 (d_target - log2 S),
// entropy = ln 2 (log2 S - T / S), both terms at least 0.  The difference to
// the maximum comes first, so a large common offset costs nothing and a row of
// the type's lowest value does not overflow.
#include <cfloat>
#include <cmath>

#include "common.hpp"
#include "wave.hpp"

namespace mi {
namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int LP_CAND = 1024;         // candidates for the alternatives a block holds
constexpr int64_t LP_TILE = 512 * 24;  // 16-byte chunks a block takes at most
constexpr int LP_SLICES = 64;         // slices of a row at most: a wavefront's lanes rank them
constexpr int64_t LP_BLOCKS = 512;     // blocks that run at once: two a CU
constexpr int64_t LP_WHOLE = 65536;    // columns up to which a row is one slice however few the rows

// 16 bytes of a row: 4 F32 or 8 BF16 logits.
template <typename T>
struct Chunk16;
template <>
struct Chunk16<float> {
  static constexpr int E = 4;
  template <bool NT>
  static __device__ __forceinline__ uint4 load(const float *p) { return ldu4<NT>(p); }
  static __device__ __forceinline__ float get(const uint4 &v, int e) {
    return __uint_as_float(e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w);
  }
};
template <>
struct Chunk16<uint16_t> {
  static constexpr int E = 8;
  template <bool NT>
  static __device__ __forceinline__ uint4 load(const uint16_t *p) { return ldu4<NT>(p); }
  static __device__ __forceinline__ float get(const uint4 &v, int e) {
    const uint32_t w = e < 2 ? v.x : e < 4 ? v.y : e < 6 ? v.z : v.w;
    return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
  }
};

__device__ __forceinline__ float logit(const float *p) { return *p; }
__device__ __forceinline__ float logit(const uint16_t *p) { return bf16_bits_to_f32(*p); }

struct LogprobArgs {
  const void *x;
  int64_t rows, cols;
  const int32_t *targets;
  float scale;
  int top, slices;
  int64_t slice;  // 16-byte chunks a slice
  // Slices' statistics [rows][slices][4] and alternatives [rows][slices][top].
  float *stats;
  uint64_t *lists;
  float *logp, *lse, *entropy, *top_logp;
  int32_t *top_ids;
  uint32_t *flags;
};

// A logit and its column as one whole number that grows in the order of
// alternatives (argmax's rule): the larger value first, 0 and -0 alike, a NaN
// above every number, the lower column among equals.  0 stands for none.
__device__ __forceinline__ uint64_t key_of(float v, int64_t col) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  const uint32_t o = isnan(v) ? 0xffffffffu : b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
  return static_cast<uint64_t>(o) << 32 | (0xffffffffu - static_cast<uint32_t>(col));
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t o = static_cast<uint32_t>(k >> 32);
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);  // 0xffffffff: a NaN
}
__device__ __forceinline__ int32_t key_column(uint64_t k) {
  return static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(k));
}
__device__ __forceinline__ uint64_t lane_key(uint64_t k, int lane) {
  return static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(k >> 32), lane))) << 32 |
         static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(k), lane));
}
// How many of the n keys are above k (keys padded with a 0 to an even number,
// two a 16-byte read).
__device__ __forceinline__ int rank_of(const uint64_t *keys, int n, uint64_t k) {
  const ulonglong2 *p = reinterpret_cast<const ulonglong2 *>(keys);
  int rank = 0;
#pragma unroll 8
  for (int o = 0; o < (n + 1) / 2; ++o) {
    const ulonglong2 w = p[o];
    rank += (w.x > k ? 1 : 0) + (w.y > k ? 1 : 0);
  }
  return rank;
}

// S and T of a maximum m moved to a maximum to >= m.
__device__ __forceinline__ void rescale(float m, float to, float c, float &S, float &T) {
  const float d = fmaxf((m - to) * c, -1e4f), r = __builtin_amdgcn_exp2f(d);
  T = r * __builtin_fmaf(d, S, T);
  S *= r;
}
// What distances are measured from: the largest logit, or a finite value where
// all are -inf, so that those distances are -inf and not NaN.
__device__ __forceinline__ float origin(float m) { return fmaxf(m, -FLT_MAX); }

// A row's results from its statistics over all columns.
template <typename T>
__device__ __forceinline__ void put_stats(const LogprobArgs &a, int64_t r, float m, float S, float Tm) {
  const bool none = S == 0.0f;  // every logit is -inf
  const float ls = __builtin_log2f(S);
  if (a.lse) a.lse[r] = none ? -INFINITY : __builtin_fmaf(LN2, ls, m * a.scale);
  if (a.entropy) a.entropy[r] = none ? 0.0f : LN2 * (ls - Tm / S);
  if (a.logp) {
    const int32_t g = a.targets[r];
    const bool ok = g >= 0 && g < a.cols;
    if (!ok) atomicOr(a.flags, FLAG_INDEX_RANGE);
    const float x = logit(static_cast<const T *>(a.x) + r * a.cols + (ok ? g : 0));
    a.logp[r] = !ok ? 0.0f : none ? -INFINITY : LN2 * ((x - m) * (a.scale * LOG2E) - ls);
  }
}
__device__ __forceinline__ void put_top(const LogprobArgs &a, int64_t at, uint64_t key, float m, float S) {
  a.top_logp[at] = S == 0.0f ? -INFINITY : LN2 * ((key_value(key) - m) * (a.scale * LOG2E) - __builtin_log2f(S));
  a.top_ids[at] = key_column(key);
}

// One slice of a row a block, held in registers: THR threads x NL chunks of 16
// bytes, all asked for at once and read once (bound by HBM: about ten
// operations a logit, two of the four bytes' time of an F32 one).  A thread
// keeps the sums of its own columns under its own running maximum and joins
// them with the others' at the end.
//
// Alternatives: the k-th largest of 64 groups' maxima (THR / 64 threads each)
// is a bound that at least k columns reach; the few columns that do, of the
// order of k, are gathered in LDS and ranked against each other.  More columns
// equal to the bound than there is room for (a constant row) are taken in
// order from the row's start; a row with a NaN or +inf, and one whose columns
// above the bound are too many, is searched k times.
//
// Measured: 2001 x 49152 F32, top 5: 63 us, 6.2 TB/s (without alternatives 60);
// 64 x 49152 BF16, top 20: 9.7 us, 4.8 of it the sums (a block a CU, bound by
// their operations), the rest five dependent steps of 0.3 to 2 us; 1 x 49152
// F32, top 5: 8.3 us.
template <typename T, int THR, int NL, bool TOP, bool NT>
__global__ void __launch_bounds__(THR, THR == 512 ? 4 : 1) logprobs_kernel(LogprobArgs a) {
  using C = Chunk16<T>;
  constexpr int E = C::E, NW = THR / 64;
  constexpr int STEP = NL < 4 ? NL : NL > 16 ? 2 : 4;  // chunks under one maximum
  // Few chunks and their maxima are kept in registers until the bound is
  // known; of more the maxima wait in LDS and a chunk that reaches the bound is
  // read again, which leaves registers for more blocks a CU (4096 x 32000 BF16,
  // top 5: 62.5 us, 70.7 with 8 chunks kept; 8192 x 8192 F32: 62.0, and
  // 58.8 with its 4 kept).
  constexpr bool KEEP = NL <= 4;
  __shared__ float red[NW][3];
  __shared__ float groups[64];
  __shared__ int ranks[NW][64];
  __shared__ __align__(16) uint64_t cand[TOP ? LP_CAND : 2];
  __shared__ int count;
  __shared__ uint64_t bests[NW];
  __shared__ float maxima[TOP && !KEEP ? NL : 1][THR];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t r = blockIdx.x / a.slices;
  const int sl = static_cast<int>(blockIdx.x % a.slices);
  // The row from the 16-byte boundary at or before it: column c is element
  // c + skip there.
  const int64_t flat = r * a.cols;
  const int skip = static_cast<int>(flat & (E - 1));
  const T *x = static_cast<const T *>(a.x) + (flat - skip);
  const int64_t end = a.cols + skip, chunks = (end + E - 1) / E;
  const int64_t c0 = sl * a.slice, c1 = c0 + a.slice < chunks ? c0 + a.slice : chunks;
  const float c = a.scale * LOG2E;
  if (TOP && tid == 0) count = 0;

  // The slice's chunks from its first, n of them; its columns are elements
  // lo .. hi - 1 counted from there.
  const T *base = x + c0 * E;
  const int n16 = static_cast<int>(c1 - c0);
  const int lo = c0 == 0 ? skip : 0, hi = c1 == chunks ? static_cast<int>(end - c0 * E) : n16 * E;
  uint4 v[NL];
#pragma unroll
  for (int u = 0; u < NL; ++u) {
    const int q = u * THR + tid;
    v[u] = C::template load<NT>(base + static_cast<uint32_t>((q < n16 ? q : n16 - 1) * E));
  }
  auto mine = [&](int u, int e) {
    const int i = (u * THR + tid) * E + e;
    return i >= lo && i < hi;
  };
  // A chunk's logits; what lies outside the slice counts as -inf.
  auto logits = [&](int u, float (&w)[E]) {
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] = C::get(v[u], e);
    if ((u == 0 && lo > 0) || (u + 1) * THR * E > hi) {
#pragma unroll
      for (int e = 0; e < E; ++e) w[e] = mine(u, e) ? w[e] : -INFINITY;
    }
  };

  float mx = -INFINITY, m = -FLT_MAX, S = 0.0f, Tm = 0.0f;
  float cm[KEEP ? NL : 1];
#pragma unroll
  for (int u0 = 0; u0 < NL; u0 += STEP) {
    float xs[STEP][E];
    float tm = -INFINITY;
#pragma unroll
    for (int u = 0; u < STEP; ++u) {
      logits(u0 + u, xs[u]);
      float um = xs[u][0];
#pragma unroll
      for (int e = 1; e < E; ++e) um = fmaxf(um, xs[u][e]);
      tm = fmaxf(tm, um);
      if constexpr (KEEP) cm[u0 + u] = um;
      else if constexpr (TOP) maxima[u0 + u][tid] = um;
    }
    if (tm > mx) {
      mx = tm;
      rescale(m, origin(mx), c, S, Tm);
      m = origin(mx);
    }
#pragma unroll
    for (int u = 0; u < STEP; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float d = (xs[u][e] - m) * c, w = __builtin_amdgcn_exp2f(d);
        S += w;
        Tm = __builtin_fmaf(fmaxf(d, -1e4f), w, Tm);  // 2^-inf = 0 adds nothing
      }
  }

  // The block's maximum, then its sums.
  float M = fold_max<64>(mx);
  if (lane == 0) red[wave][0] = M;
  if (TOP) {
    const float gm = fold_max<NW>(mx);
    if ((lane & (NW - 1)) == 0) groups[tid / NW] = gm;
  }
  __syncthreads();
  M = red[0][0];
#pragma unroll
  for (int w = 1; w < NW; ++w) M = fmaxf(M, red[w][0]);
  M = origin(M);
  rescale(m, M, c, S, Tm);
  S = fold_sum<64>(S);
  Tm = fold_sum<64>(Tm);
  if (lane == 0) {
    red[wave][1] = S;
    red[wave][2] = Tm;
  }
  __syncthreads();
  S = red[0][1];
  Tm = red[0][2];
#pragma unroll
  for (int w = 1; w < NW; ++w) {
    S += red[w][1];
    Tm += red[w][2];
  }
  // How many of the groups' maxima are above each (equal ones in the groups'
  // order), a wavefront counting over its share of them.
  float gv = 0.0f;
  if constexpr (TOP) {
    gv = groups[lane];
    int rank = 0;
#pragma unroll
    for (int o = 0; o < 64 / NW; ++o) {
      const int at = wave * (64 / NW) + o;
      const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(gv), at));
      rank += w > gv || (w == gv && at < lane) ? 1 : 0;
    }
    ranks[wave][lane] = rank;
  }
  if (tid == 0) {
    if (a.slices == 1) {
      put_stats<T>(a, r, M, S, Tm);
    } else {
      float *st = a.stats + (r * a.slices + sl) * 4;
      st[0] = M;
      st[1] = S;
      st[2] = Tm;
    }
  }
  if constexpr (!TOP) return;

  __syncthreads();
  const int k = a.top;
  uint64_t *list = a.slices > 1 ? a.lists + (r * a.slices + sl) * k : nullptr;
  auto put = [&](int at, uint64_t key) {
    if (list) list[at] = key;
    else put_top(a, r * k + at, key, M, S);
  };
  const int64_t e0 = c0 * E > skip ? c0 * E - skip : 0;  // the slice's columns [e0, e1)
  const int64_t e1 = c1 * E - skip < a.cols ? c1 * E - skip : a.cols;
  const T *row = x + skip;
  bool search = isnan(S);
  int n = 0;
  float bound = -INFINITY;
  if (!search) {
    int rank = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) rank += ranks[w][lane];
    const uint64_t kth = __ballot(rank == k - 1);
    bound = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(gv), __ffsll(static_cast<unsigned long long>(kth)) - 1));
    // Each thread's chunks whose largest logit reaches the bound, one a turn: a
    // thread seldom has two, so this is one or two turns of a short loop
    // (unrolled over the chunks it took 1.4 us a chunk, most of it for
    // instructions fetched to be run once), in each room for its few hits, in
    // any order (with ballots for the columns' places 64 x 49152 BF16, top 20, took
    // 10.8 us, so 9.9).
    const int col0 = static_cast<int>(c0 * E - skip);
    uint32_t todo = 0;
    if (mx >= bound) {
#pragma unroll
      for (int u = 0; u < NL; ++u) todo |= ((KEEP ? cm[KEEP ? u : 0] : maxima[KEEP ? 0 : u][tid]) >= bound ? 1u : 0u) << u;
    }
#pragma nounroll
    while (todo) {
      const int u = __ffs(todo) - 1;
      uint4 w;
      if constexpr (KEEP) {
        w = v[0];
#pragma unroll
        for (int o = 1; o < NL; ++o) {
          w.x = u == o ? v[o].x : w.x;
          w.y = u == o ? v[o].y : w.y;
          w.z = u == o ? v[o].z : w.z;
          w.w = u == o ? v[o].w : w.w;
        }
      } else {
        const int q = u * THR + tid;
        w = C::template load<false>(base + static_cast<uint32_t>((q < n16 ? q : n16 - 1) * E));
      }
      uint32_t hits = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) hits |= (C::get(w, e) >= bound && mine(u, e) ? 1u : 0u) << e;
      int at = hits ? atomicAdd(&count, __popc(hits)) : 0;
      if (at >= LP_CAND) break;  // more than there is room for
#pragma nounroll
      for (; hits && at < LP_CAND; hits &= hits - 1, ++at) {
        const int e = __ffs(hits) - 1;
        cand[at] = key_of(C::get(w, e), col0 + (u * THR + tid) * E + e);
      }
      todo &= todo - 1;
    }
    __syncthreads();
    n = count;
    if (n > LP_CAND) {
      // More than there is room for.  The columns above the bound alone (where
      // all are equal there is none), then the first ones equal to it.
      __syncthreads();
      if (tid == 0) count = 0;
      __syncthreads();
      for (int64_t b = e0 + tid; b < e1; b += THR) {
        const float w = logit(row + b);
        if (w > bound) {
          const int at = atomicAdd(&count, 1);
          if (at < LP_CAND) cand[at] = key_of(w, b);
        }
      }
      __syncthreads();
      n = count;
      search = n > LP_CAND - k;
      const int want = n + k;
      for (int64_t b = e0; b < e1 && n < want && !search; b += THR) {
        const bool eq = b + tid < e1 && logit(row + b + tid) == bound;
        const uint64_t bal = __ballot(eq);
        if (lane == 0) red[wave][0] = static_cast<float>(__popcll(bal));
        __syncthreads();
        int at = n + __popcll(bal & ((uint64_t(1) << lane) - 1)), all = 0;
        for (int w = 0; w < NW; ++w) {
          const int cw = static_cast<int>(red[w][0]);
          if (w < wave) at += cw;
          all += cw;
        }
        if (eq && at < LP_CAND) cand[at] = key_of(bound, b + tid);
        n += all;
        __syncthreads();
      }
      if (n > LP_CAND) n = LP_CAND;
    }
  }
  if (search) {
    uint64_t last = 0;
    for (int t = 0; t < k; ++t) {
      uint64_t b = 0;
      for (int64_t q = e0 + tid; q < e1; q += THR) {
        const uint64_t w = key_of(logit(row + q), q);
        if ((w < last || t == 0) && w > b) b = w;
      }
      for (int o = 32; o >= 1; o >>= 1) {
        const uint64_t w = __shfl_xor(static_cast<unsigned long long>(b), o, 64);
        if (w > b) b = w;
      }
      if (lane == 0) bests[wave] = b;
      __syncthreads();
      last = bests[0];
      for (int w = 1; w < NW; ++w)
        if (bests[w] > last) last = bests[w];
      __syncthreads();
      if (tid == 0) put(t, last);  // 0 behind a slice's last column
    }
    return;
  }
  if (tid == 0 && (n & 1)) cand[n] = 0;  // n odd: there is room
  __syncthreads();
  for (int i = tid; i < n; i += THR) {
    const int rank = rank_of(cand, n, cand[i]);
    if (rank < k) put(rank, cand[i]);
  }
  for (int i = n + tid; i < k; i += THR) put(i, 0);
}

// Joins the slices of a row.
template <typename T>
__global__ void __launch_bounds__(256) logprobs_join_kernel(LogprobArgs a) {
  constexpr int PER = LP_SLICES * MI_TOP_MAX / 256;
  __shared__ __align__(16) uint64_t cand[LP_SLICES * MI_TOP_MAX];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t r = blockIdx.x;
  const int ns = a.slices, k = a.top, all = ns * k;
  const float *st = a.stats + r * ns * 4;
  const uint64_t *lists = a.lists + r * all;
  uint64_t mine[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) mine[i] = tid + 256 * i < all ? lists[tid + 256 * i] : 0;
  // The lists are in order, so where L of them have a q-th key at or above
  // some key, and L q >= k, the first k are at or above it too: the L-th
  // largest of the q-th keys bounds what has to be ranked.
  const int q = k ? (k + ns - 1) / ns : 1, L = (k + q - 1) / q;
  const uint64_t nth = lane < ns && k ? lists[lane * k + q - 1] : 0;
  const float m = lane < ns ? st[lane * 4] : -FLT_MAX;
  float S = lane < ns ? st[lane * 4 + 1] : 0.0f, Tm = lane < ns ? st[lane * 4 + 2] : 0.0f;
  const float M = fold_max<64>(m);
  rescale(m, M, a.scale * LOG2E, S, Tm);
  S = fold_sum<64>(S);
  Tm = fold_sum<64>(Tm);
  if (tid == 0) {
    put_stats<T>(a, r, M, S, Tm);
    count = 0;
  }
  if (k == 0) return;
  int above = 0;
  for (int o = 0; o < ns; ++o) above += lane_key(nth, o) > nth ? 1 : 0;
  const uint64_t at = __ballot(lane < ns && above == L - 1);
  const uint64_t bound = at ? lane_key(nth, __ffsll(static_cast<unsigned long long>(at)) - 1) : 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (mine[i] > 0 && mine[i] >= bound) cand[atomicAdd(&count, 1)] = mine[i];
  __syncthreads();
  const int n = count;
  if (tid == 0 && (n & 1)) cand[n] = 0;
  __syncthreads();
  for (int i = tid; i < n; i += 256) {
    const int rank = rank_of(cand, n, cand[i]);
    if (rank < k) put_top(a, r * k + rank, cand[i], M, S);
  }
}

template <typename T, int THR, int NL>
void logprobs_launch(Ctx *ctx, const LogprobArgs &a, bool nt) {
  const unsigned grid = static_cast<unsigned>(a.rows * a.slices);
  if (a.top > 0) {
    if (nt) logprobs_kernel<T, THR, NL, true, true><<<grid, THR, 0, ctx->stream>>>(a);
    else logprobs_kernel<T, THR, NL, true, false><<<grid, THR, 0, ctx->stream>>>(a);
  } else {
    if (nt) logprobs_kernel<T, THR, NL, false, true><<<grid, THR, 0, ctx->stream>>>(a);
    else logprobs_kernel<T, THR, NL, false, false><<<grid, THR, 0, ctx->stream>>>(a);
  }
}

template <typename T>
int logprobs_run(Ctx *ctx, LogprobArgs a) {
  constexpr int64_t E = Chunk16<T>::E;
  // A row is one slice where a block's registers hold it: its results need no
  // second launch (128 x 49152 BF16, top 20: 13.3 us, 14.9 in 4 slices; 1 x
  // 49152 F32: 9.6 us, 10.9 in 48).  Wider rows, and few rows of over LP_WHOLE
  // columns, are cut until the CUs have two blocks each (8 x 128256 BF16: 11.5
  // us in 63 slices, 19.2 in 2); many wide rows in the number of slices, up to
  // four times the least, whose last round of blocks is fullest.
  const int64_t chunks = a.cols % E ? (a.cols + 2 * (E - 1)) / E : a.cols / E;  // of a row that starts anywhere
  const int64_t least = (chunks + LP_TILE - 1) / LP_TILE, most = chunks / 256;
  const int64_t want = (LP_BLOCKS + a.rows - 1) / a.rows;
  int64_t ns = least;
  if (least > 1 || (a.cols > LP_WHOLE && 2 * a.rows < LP_BLOCKS)) {
    if (ns < want) ns = want < most ? want : most;
    if (want <= 4 * least) {
      auto rounds = [&](int64_t n) { return static_cast<double>((a.rows * n + LP_BLOCKS - 1) / LP_BLOCKS) / static_cast<double>(n); };
      ns = least;
      for (int64_t n = least + 1; n <= 4 * least; ++n)
        if (rounds(n) < 0.95 * rounds(ns)) ns = n;
    }
  }
  if (ns > LP_SLICES) ns = LP_SLICES;
  a.slice = (chunks + ns - 1) / ns;
  // Every slice holds a column of every row: the shortest row's chunks.
  const int64_t shortest = (a.cols + E - 1) / E;
  ns = (shortest + a.slice - 1) / a.slice;
  if (ns * a.slice < chunks) a.slice = (chunks + ns - 1) / ns;
  if (a.slice > LP_TILE || a.rows * ns > kGridThreads / 512)
    return fail(ctx, MI_E_UNSUPPORTED, "token_logprobs of [%lld, %lld]", (long long)a.rows, (long long)a.cols);
  a.slices = static_cast<int>(ns);
  if (ns > 1) {
    const size_t cells = static_cast<size_t>(a.rows * ns);
    char *p = static_cast<char *>(scratch(ctx, cells * (16 + sizeof(uint64_t) * a.top)));
    if (!p) return fail(ctx, MI_E_OOM, "token_logprobs scratch");
    a.stats = reinterpret_cast<float *>(p);
    a.lists = reinterpret_cast<uint64_t *>(p + cells * 16);
  }
  const bool nt = a.rows * a.cols * static_cast<int64_t>(sizeof(T)) >= kStreamBytes;
  if (a.slice <= 256) logprobs_launch<T, 256, 1>(ctx, a, nt);
  else if (a.slice <= 512) logprobs_launch<T, 256, 2>(ctx, a, nt);
  else if (a.slice <= 1024) logprobs_launch<T, 256, 4>(ctx, a, nt);
  else if (a.slice <= 2048) logprobs_launch<T, 512, 4>(ctx, a, nt);
  else if (a.slice <= 4096) logprobs_launch<T, 512, 8>(ctx, a, nt);
  else if (a.slice <= 6144) logprobs_launch<T, 512, 12>(ctx, a, nt);
  else if (a.slice <= 8192) logprobs_launch<T, 512, 16>(ctx, a, nt);
  else logprobs_launch<T, 512, 24>(ctx, a, nt);
  if (int s = check_launch(ctx, "token_logprobs")) return s;
  if (ns == 1) return MI_OK;
  logprobs_join_kernel<T><<<static_cast<unsigned>(a.rows), 256, 0, ctx->stream>>>(a);
  return check_launch(ctx, "token_logprobs join");
}

struct LogprobGradArgs {
  const void *x;
  int64_t rows, cols;
  const int32_t *targets;
  const float *lse, *entropy, *d_logp, *d_entropy;
  float scale;
  void *out;
  int blocks;    // a row
  int64_t row0;  // the launch's first
  uint32_t *flags;
};

// e^l for a finite l from the hardware's 2^y, y = l log2(e) rounded: what the
// rounding and the constant's own leave out (log2(e) = LOG2E + LOG2E_LO) goes
// into a factor 1 + r, so the error does not grow with |l| (without it 2.2 |l|
// 2^-24 of the value).
__device__ __forceinline__ float exp_full(float l) {
  constexpr float LOG2E_LO = 1.925963033500e-8f;
  const float y = l * LOG2E, p = __builtin_amdgcn_exp2f(y);
  return __builtin_fmaf(p, LN2 * __builtin_fmaf(l, LOG2E_LO, __builtin_fmaf(l, LOG2E, -y)), p);
}

// E consecutive logits widened, and values stored, as 16 bytes of the wider
// side (8 of a BF16 one beside F32).
template <int E, bool NT>
__device__ __forceinline__ void load_logits(const float *p, float (&v)[E]) {
  const uint4 w = ldu4<NT>(p);
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = Chunk16<float>::get(w, e);
}
template <int E, bool NT>
__device__ __forceinline__ void load_logits(const uint16_t *p, float (&v)[E]) {
  uint4 w;
  if constexpr (E == 8) {
    w = ldu4<NT>(p);
  } else {
    const uint2 h = *reinterpret_cast<const uint2 *>(p);
    w = make_uint4(h.x, h.y, 0, 0);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = Chunk16<uint16_t>::get(w, e);
}
template <int E, bool NT>
__device__ __forceinline__ void store_grads(float *p, const float (&v)[E]) {
  st4<NT>(p, make_float4(v[0], v[1], v[2], v[3]));
}
template <int E, bool NT>
__device__ __forceinline__ void store_grads(uint16_t *p, const float (&v)[E]) {
  if constexpr (E == 8)
    stu4<NT>(p, make_uint4(bf16x2_bits(v[0], v[1]), bf16x2_bits(v[2], v[3]), bf16x2_bits(v[4], v[5]), bf16x2_bits(v[6], v[7])));
  else
    *reinterpret_cast<uint2 *>(p) = make_uint2(bf16x2_bits(v[0], v[1]), bf16x2_bits(v[2], v[3]));
}

// dx_j = scale (g ([j = target] - p_j) - h p_j (z_j - lse + H)), a chunk of E
// elements a thread, from a boundary of both sides at or before the row: one
// read and one write of each byte, bound by HBM.  2048 x 8192 F32 (134 MB): 21.7
// us, 6.2 TB/s; 1001 x 40001 BF16 (160 MB): 30.5 us, 5.2 TB/s; a large copy
// reaches 5.0.
template <typename T, typename TO, bool NT>
__global__ void __launch_bounds__(256) logprobs_backward_kernel(LogprobGradArgs a) {
  constexpr int E = sizeof(T) == 2 && sizeof(TO) == 2 ? 8 : 4;
  const int64_t r = a.row0 + blockIdx.x / a.blocks;
  const int64_t flat = r * a.cols;
  const int skip = static_cast<int>(flat & (E - 1));
  const T *x = static_cast<const T *>(a.x) + (flat - skip);
  TO *o = static_cast<TO *>(a.out) + (flat - skip);
  const int64_t end = a.cols + skip, chunks = (end + E - 1) / E;
  const int64_t q = static_cast<int64_t>(blockIdx.x % a.blocks) * 256 + threadIdx.x;
  float v[E];
  load_logits<E, NT>(x + (q < chunks ? q : chunks - 1) * E, v);
  const float lse = a.lse[r], h = a.d_entropy ? a.d_entropy[r] : 0.0f, H = a.d_entropy ? a.entropy[r] : 0.0f;
  float g = a.d_logp ? a.d_logp[r] : 0.0f;
  int64_t target = -1;
  if (a.d_logp) {
    target = a.targets[r];
    if (target < 0 || target >= a.cols) {
      if (q == 0) atomicOr(a.flags, FLAG_INDEX_RANGE);
      target = -1;
      g = 0.0f;
    } else {
      target += skip;
    }
  }
  // dx_j = scale g [j = target] + p_j (b l_j + c); an empty row has no p.
  const bool none = lse == -INFINITY;
  const float b = none ? 0.0f : -h * a.scale, c = none ? 0.0f : __builtin_fmaf(-g, a.scale, b * H);
  float out[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    // Where the probability is 0 a finite distance, so that 0 it stays; a
    // NaN passes.
    float l = none ? -1e4f : __builtin_fmaf(v[e], a.scale, -lse);
    l = l < -1e4f ? -1e4f : l;
    out[e] = exp_full(l) * __builtin_fmaf(b, l, c);
  }
  const int64_t t = target - q * E;
  if (t >= 0 && t < E) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e == t) out[e] = __builtin_fmaf(g, a.scale, out[e]);
  }
  if (q * E >= skip && q * E + E <= end) {
    store_grads<E, NT>(o + q * E, out);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (q * E + e >= skip && q * E + e < end) f32_put(o + q * E + e, out[e]);
  }
}

template <typename T, typename TO>
void logprobs_backward_launch(Ctx *ctx, LogprobGradArgs a) {
  constexpr int64_t E = sizeof(T) == 2 && sizeof(TO) == 2 ? 8 : 4;
  const bool nt = a.rows * a.cols * static_cast<int64_t>(sizeof(T) + sizeof(TO)) >= kStreamBytes;
  const int64_t chunks = (a.cols + 2 * (E - 1)) / E;
  // Four a thread: 8.7 us where one takes 7.2 (512 x 8192 F32), 8.8 and 8.1
  // (256 x 32000 BF16), 25.3 and 23.3 (2048 x 8192 F32), 32.5 and 33.7 (1001 x
  // 40001 BF16).
  a.blocks = static_cast<int>((chunks + 255) / 256);
  // All rows in one launch, but for more blocks than one can have.
  const int64_t span = std::max<int64_t>(kGridThreads / 256 / a.blocks, 1);
  for (a.row0 = 0; a.row0 < a.rows; a.row0 += span) {
    const unsigned grid = static_cast<unsigned>(std::min(span, a.rows - a.row0) * a.blocks);
    if (nt) logprobs_backward_kernel<T, TO, true><<<grid, 256, 0, ctx->stream>>>(a);
    else logprobs_backward_kernel<T, TO, false><<<grid, 256, 0, ctx->stream>>>(a);
  }
}

int logits_check(Ctx *ctx, const char *what, const Buffer *xb, float scale) {
  if (!elem_float(xb->elem) || xb->tiles)
    return fail(ctx, MI_E_ARG, "%s takes F32 or BF16 logits in rows (%s)", what, elem_name(xb->elem));
  if (xb->cols < 1 || xb->cols >= INT32_MAX || xb->rows > INT32_MAX)
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
    s = xb->elem == MI_BF16 ? logprobs_run<uint16_t>(ctx, a) : logprobs_run<float>(ctx, a);
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
    const bool x16 = xb->elem == MI_BF16, o16 = out_elem == MI_BF16;
    if (x16 && o16) logprobs_backward_launch<uint16_t, uint16_t>(ctx, a);
    else if (x16) logprobs_backward_launch<uint16_t, float>(ctx, a);
    else if (o16) logprobs_backward_launch<float, uint16_t>(ctx, a);
    else logprobs_backward_launch<float, float>(ctx, a);
    s = check_launch(ctx, "token_logprobs_backward");
    if (s) { mi_free(ctx, id); return s; }
  }
  *dlogits = id;
  return MI_OK;
}
