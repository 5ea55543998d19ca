// Vocabulary operators on stored logits: log probabilities of given tokens
// with entropy and top alternatives, their gradient, and the divergence from
// a teacher's top logits with its gradient.
//
// A row of V logits is read once from HBM in 16-byte vectors. Each thread
// keeps a running (m, s, u): the maximum, s = sum 2^y and u = sum y 2^y with
// y = (x - m) c log2(e); then logsumexp = m c + ln s and the entropy is
// ln s - ln2 u / s, so one pass gives both. (x - m) is formed before the
// scaling: x c would overflow for masks of the type's lowest value. y is
// clamped at kYMin so that a masked element (-inf, or far below the maximum)
// adds 0 to u instead of 0 * inf; the clamp and the sums keep NaN.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "internal.h"

namespace ig {

namespace cg = cooperative_groups;

constexpr int kVocThreads = 256;
constexpr int kVocWarps = kVocThreads / 32;
constexpr int kVocUnroll = 4;     // 16-byte vectors in flight per thread
constexpr int kTopMax = 32;       // alternatives per row
constexpr int kTopCap = 128;      // a warp's candidate buffer
constexpr int kTeacherMax = kVocThreads;  // teacher entries per row: one thread each
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kYMin = -1.0e4f;  // 2^kYMin = 0
#define IG_INF __int_as_float(0x7f800000)

__device__ __forceinline__ float ex2(float y) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
  return r;
}
// max(a, b), NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// ---- element types --------------------------------------------------------------

template <int DT>
struct VElem;
template <>
struct VElem<IG_DT_F32> {
  using T = float;
  static constexpr int kN = 4;  // per 16-byte vector
  __device__ __forceinline__ static void unpack(const uint4 &v, float *x) {
    x[0] = __uint_as_float(v.x);
    x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z);
    x[3] = __uint_as_float(v.w);
  }
  __device__ __forceinline__ static uint4 pack(const float *x) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
  __device__ __forceinline__ static float get(T v) { return v; }
  __device__ __forceinline__ static T put(float v) { return v; }
};
template <>
struct VElem<IG_DT_BF16> {
  using T = __nv_bfloat16;
  static constexpr int kN = 8;
  __device__ __forceinline__ static void unpack(const uint4 &v, float *x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  __device__ __forceinline__ static uint4 pack(const float *x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ static float get(T v) { return __bfloat162float(v); }
  __device__ __forceinline__ static T put(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct VElem<IG_DT_F16> {
  using T = __half;
  static constexpr int kN = 8;
  __device__ __forceinline__ static void unpack(const uint4 &v, float *x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  __device__ __forceinline__ static uint4 pack(const float *x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ static float get(T v) { return __half2float(v); }
  __device__ __forceinline__ static T put(float v) { return __float2half_rn(v); }
};

// A row seen as 16-byte vectors from the boundary at or before its start:
// vector v holds the columns [v kN - mis, v kN - mis + kN); the first and
// the last may be partial (an odd row stride moves every row's boundary).
template <int DT>
struct RowVecs {
  using E = VElem<DT>;
  using T = typename E::T;
  const T *row;
  int mis, V;
  int nv;
  __device__ __forceinline__ RowVecs(const T *p, int V_) : row(p), V(V_) {
    mis = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
    nv = (mis + V + E::kN - 1) / E::kN;
  }
  __device__ __forceinline__ int col(int v) const { return v * E::kN - mis; }
  __device__ __forceinline__ bool whole(int v) const { return col(v) >= 0 && col(v) + E::kN <= V; }
  __device__ __forceinline__ void load_edge(int v, float *x) const {
#pragma unroll
    for (int i = 0; i < E::kN; i++) {
      const int c = col(v) + i;
      x[i] = c >= 0 && c < V ? E::get(row[c]) : -IG_INF;
    }
  }
};

// ---- running statistics -----------------------------------------------------------

struct VStat {
  float m, s, u;
};

template <bool U>
__device__ __forceinline__ void vstat_shift(VStat &a, float m, float c2) {
  const float mb = m == -IG_INF ? 0.0f : m;
  const float d = fmaxf((a.m - mb) * c2, kYMin);
  const float f = ex2(d);
  if constexpr (U) a.u = (a.u + a.s * d) * f;
  a.s *= f;
  a.m = m;
}

template <bool U>
__device__ __forceinline__ void vstat_merge(VStat &a, VStat b, float c2) {
  const float m = fmaxf(a.m, b.m);
  vstat_shift<U>(a, m, c2);
  vstat_shift<U>(b, m, c2);
  a.s += b.s;
  if constexpr (U) a.u += b.u;
}

// The N values x (N even) with maximum mx.
template <bool U, int N>
__device__ __forceinline__ void vstat_add(VStat &a, const float (&x)[N], float mx, float c2) {
  const float m = fmaxf(a.m, mx);
  if (m > a.m) vstat_shift<U>(a, m, c2);
  const float mb = m == -IG_INF ? 0.0f : m;
  const float2 nm = make_float2(-mb, -mb), cc = make_float2(c2, c2);
  float2 s = make_float2(0.0f, 0.0f), u = s;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    float2 y = __fmul2_rn(__fadd2_rn(make_float2(x[i], x[i + 1]), nm), cc);
    if constexpr (U) {
      y.x = max_nan(y.x, kYMin);
      y.y = max_nan(y.y, kYMin);
    }
    const float2 e = make_float2(ex2(y.x), ex2(y.y));
    s = __fadd2_rn(s, e);
    if constexpr (U) u = __ffma2_rn(e, y, u);
  }
  a.s += s.x + s.y;
  if constexpr (U) a.u += u.x + u.y;
}

template <bool U>
__device__ __forceinline__ VStat vstat_warp(VStat a, float c2) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    VStat b;
    b.m = __shfl_xor_sync(~0u, a.m, o);
    b.s = __shfl_xor_sync(~0u, a.s, o);
    b.u = U ? __shfl_xor_sync(~0u, a.u, o) : 0.0f;
    // Both lanes add in the same order (the lower lane's first), so all lanes hold the same bits.
    if (threadIdx.x & o) {
      const VStat t = a;
      a = b;
      b = t;
    }
    vstat_merge<U>(a, b, c2);
  }
  return a;
}

// ---- top alternatives ---------------------------------------------------------------

// (value, column) order: larger value first, then the lower column.
__device__ __forceinline__ bool top_before(float va, int ca, float vb, int cb) {
  return va > vb || (va == vb && ca < cb);
}
__device__ __forceinline__ int ordered_bits(float v) {
  const int b = __float_as_int(v);
  return b >= 0 ? b : b ^ 0x7FFFFFFF;
}
__device__ __forceinline__ float from_ordered(int b) { return __int_as_float(b >= 0 ? b : b ^ 0x7FFFFFFF); }

struct TopWarp {
  float *val;  // [kTopCap] candidates of this warp (shared memory)
  int *col;
  int *cta_tau;  // ordered bits of the best K-th value any warp has (shared)
  int n, K;      // n, tau, ctau: the same in all lanes
  float tau;     // a candidate has to come before (tau, ctau)
  int ctau;
  bool started;
};

// Keeps the K first candidates, sorted: each entry's rank is the number of
// entries before it (columns are distinct, so ranks are).
__device__ __noinline__ void top_compact(TopWarp &t) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
  float v[kTopCap / 32];
  int c[kTopCap / 32], r[kTopCap / 32];
#pragma unroll
  for (int k = 0; k < kTopCap / 32; k++) {
    const int i = k * 32 + lane;
    v[k] = i < t.n ? t.val[i] : -IG_INF;
    c[k] = i < t.n ? t.col[i] : 0x7FFFFFFF;
    r[k] = i < t.n ? 0 : kTopCap;
  }
  for (int j = 0; j < t.n; j++) {
    const float vj = t.val[j];
    const int cj = t.col[j];
#pragma unroll
    for (int k = 0; k < kTopCap / 32; k++) r[k] += top_before(vj, cj, v[k], c[k]);
  }
  __syncwarp();
#pragma unroll
  for (int k = 0; k < kTopCap / 32; k++)
    if (r[k] < t.K) {
      t.val[r[k]] = v[k];
      t.col[r[k]] = c[k];
    }
  __syncwarp();
  if (t.n >= t.K) {
    t.n = t.K;
    t.tau = t.val[t.K - 1];
    t.ctau = t.col[t.K - 1];
    if (lane == 0) atomicMax(t.cta_tau, ordered_bits(t.tau));
  }
}

// The K-th largest of the lanes' maxima is at most the K-th largest value:
// a first bound, so that the first values do not all become candidates.
__device__ __noinline__ void top_start(TopWarp &t, float mx) {
  const int lane = threadIdx.x & 31;
  int r = 0;
  for (int j = 0; j < 32; j++) {
    const float o = __shfl_sync(~0u, mx, j);
    r += top_before(o, j, mx, lane);
  }
  const float kth = __shfl_sync(~0u, mx, __ffs(__ballot_sync(~0u, r == t.K - 1)) - 1);
  if (kth > t.tau) {
    t.tau = kth;
    t.ctau = 0x7FFFFFFF;
  }
  t.started = true;
}

// Offers N values; value i of a lane is column col(i). mx: their maximum.
template <int N, typename ColFn>
__device__ __forceinline__ void top_offer(TopWarp &t, const float (&x)[N], float mx, ColFn col) {
  const float shared = from_ordered(*(volatile int *)t.cta_tau);
  if (shared > t.tau) {
    t.tau = shared;
    t.ctau = 0x7FFFFFFF;
  }
  if (!__any_sync(~0u, mx >= t.tau && mx > -IG_INF)) return;
  if (!t.started) {
    // NaN maxima cannot arise (fmaxf), but a lane may hold -inf only.
    top_start(t, mx);
  }
#pragma unroll
  for (int i = 0; i < N; i++) {
    bool p = x[i] > t.tau || (x[i] == t.tau && col(i) < t.ctau);
    unsigned b = __ballot_sync(~0u, p);
    if (b) {
      if (t.n + __popc(b) > kTopCap) {
        top_compact(t);
        p = x[i] > t.tau || (x[i] == t.tau && col(i) < t.ctau);
        b = __ballot_sync(~0u, p);
      }
      if (p) {
        const int at = t.n + __popc(b & ((1u << (threadIdx.x & 31)) - 1));
        t.val[at] = x[i];
        t.col[at] = col(i);
      }
      t.n += __popc(b);
    }
  }
}

// ---- forward ------------------------------------------------------------------------

struct LogprobArgs {
  const void *x;
  int64_t ld, rows;
  int V, T, K;
  float c;
  const int32_t *ids;
  float *logprobs, *lse, *entropy;
  int32_t *top_ids;
  float *top_logprobs;
};

// Row results from its statistics and, for top_k, its sorted candidates.
__device__ __forceinline__ void row_lse(const VStat &a, float c, float &log_s, float &lse, float &entropy) {
  const bool empty = a.s == 0.0f;
  log_s = logf(a.s);
  lse = empty ? -IG_INF : fmaf(a.m, c, log_s);
  entropy = empty ? 0.0f : log_s - kLn2 * (a.u / a.s);
  if (entropy < 0.0f) entropy = 0.0f;
}
// Log probability of a logit x in a row with statistics (m, log s).
__device__ __forceinline__ float row_logprob(float x, const VStat &a, float c, float log_s) {
  if (a.s == 0.0f) return -IG_INF;
  const float v = (x - a.m) * c - log_s;
  return v > 0.0f ? 0.0f : v;
}

// Merges `lists` sorted lists (list l: cnt[l] entries at val/col + l * stride)
// of one CTA into the first K, written to out_val/out_col; returns through
// *out_n. All threads call it; lists * K <= kVocThreads entries take part.
__device__ __forceinline__ void top_merge(const float *val, const int *col, const int *cnt, int lists, int stride, int K,
                                          float *out_val, int *out_col, int *out_n) {
  int total = 0;
  for (int l = 0; l < lists; l++) total += cnt[l];
  for (int i = threadIdx.x; i < lists * K; i += kVocThreads) {
    const int l = i / K, k = i % K;
    if (k >= cnt[l]) continue;
    const float v = val[l * stride + k];
    const int c = col[l * stride + k];
    int r = 0;
    for (int j = 0; j < lists; j++) {
      if (j == l) {
        r += k;
        continue;
      }
      // Entries of list j before (v, c): its lists are sorted.
      int lo = 0, hi = cnt[j];
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (top_before(val[j * stride + mid], col[j * stride + mid], v, c))
          lo = mid + 1;
        else
          hi = mid;
      }
      r += lo;
    }
    if (r < K) {
      out_val[r] = v;
      out_col[r] = c;
    }
  }
  if (threadIdx.x == 0) *out_n = total < K ? total : K;
}

template <int DT, bool TOP>
__global__ void __launch_bounds__(kVocThreads, 4) token_logprobs_kernel(const LogprobArgs a) {
  using E = VElem<DT>;
  using T = typename E::T;
  constexpr int kN = E::kN, kX = kN * kVocUnroll;
  __shared__ VStat s_warp[kVocWarps];
  __shared__ VStat s_cta;
  __shared__ float s_val[TOP ? kVocWarps * kTopCap : 1];
  __shared__ int s_col[TOP ? kVocWarps * kTopCap : 1];
  __shared__ float s_oval[TOP ? 8 * kTopMax : 1];  // this CTA's list, and on rank 0 all the cluster's
  __shared__ int s_ocol[TOP ? 8 * kTopMax : 1];
  __shared__ int s_cnt[8], s_on, s_tau;
  __shared__ float s_fval[TOP ? kTopMax : 1];
  __shared__ int s_fcol[TOP ? kTopMax : 1];

  cg::cluster_group cl = cg::this_cluster();
  const int cs = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int64_t row = blockIdx.x / cs;
  const RowVecs<DT> rv(static_cast<const T *>(a.x) + row * a.ld, a.V);
  const int v0 = (int)((int64_t)rv.nv * rank / cs), v1 = (int)((int64_t)rv.nv * (rank + 1) / cs);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float c2 = a.c * kLog2e;

  VStat st{-IG_INF, 0.0f, 0.0f};
  TopWarp tw;
  if constexpr (TOP) {
    tw.val = s_val + warp * kTopCap;
    tw.col = s_col + warp * kTopCap;
    tw.cta_tau = &s_tau;
    tw.n = 0;
    tw.K = a.K;
    tw.tau = -IG_INF;
    tw.ctau = INT32_MIN;  // no -inf is a candidate
    tw.started = false;
    if (threadIdx.x == 0) s_tau = ordered_bits(-IG_INF);
    __syncthreads();
  }
  for (int b = v0; b < v1; b += kVocUnroll * kVocThreads) {
    float x[kX];
    uint4 raw[kVocUnroll];
#pragma unroll
    for (int j = 0; j < kVocUnroll; j++) {
      const int v = b + j * kVocThreads + (int)threadIdx.x;
      if (v < v1 && rv.whole(v)) raw[j] = *reinterpret_cast<const uint4 *>(rv.row + rv.col(v));
    }
#pragma unroll
    for (int j = 0; j < kVocUnroll; j++) {
      const int v = b + j * kVocThreads + (int)threadIdx.x;
      if (v < v1 && rv.whole(v)) {
        E::unpack(raw[j], x + j * kN);
      } else if (v < v1) {
        rv.load_edge(v, x + j * kN);
      } else {
#pragma unroll
        for (int i = 0; i < kN; i++) x[j * kN + i] = -IG_INF;
      }
    }
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < kX; i++) mx = fmaxf(mx, x[i]);
    mx = fmaxf(mx, -IG_INF);  // a chunk of NaN only
    vstat_add<true>(st, x, mx, c2);
    if constexpr (TOP)
      top_offer(tw, x, mx,
                [&](int i) { return rv.col(b + (i / kN) * kVocThreads + (int)threadIdx.x) + i % kN; });
  }
  st = vstat_warp<true>(st, c2);
  if (lane == 0) s_warp[warp] = st;
  if constexpr (TOP) {
    top_compact(tw);
    if (lane == 0) s_cnt[warp] = tw.n;
  }
  __syncthreads();
  st = s_warp[0];
  for (int w = 1; w < kVocWarps; w++) vstat_merge<true>(st, s_warp[w], c2);
  if constexpr (TOP) top_merge(s_val, s_col, s_cnt, kVocWarps, kTopCap, a.K, s_oval, s_ocol, &s_on);
  if (cs > 1) {
    if (threadIdx.x == 0) s_cta = st;
    cl.sync();
    if (rank == 0) {
      for (int r = 1; r < cs; r++) vstat_merge<true>(st, *cl.map_shared_rank(&s_cta, r), c2);
      if constexpr (TOP) {
        if ((int)threadIdx.x < cs) s_cnt[threadIdx.x] = *cl.map_shared_rank(&s_on, threadIdx.x);
        for (int i = threadIdx.x; i < (cs - 1) * a.K; i += kVocThreads) {
          const int r = 1 + i / a.K, k = i % a.K;
          s_oval[r * kTopMax + k] = cl.map_shared_rank(s_oval, r)[k];
          s_ocol[r * kTopMax + k] = cl.map_shared_rank(s_ocol, r)[k];
        }
      }
    }
    cl.sync();
    if (rank != 0) return;
  } else if constexpr (TOP) {
    __syncthreads();
    if (threadIdx.x == 0) s_cnt[0] = s_on;
    __syncthreads();
  }
  float log_s, lse, entropy;
  row_lse(st, a.c, log_s, lse, entropy);
  if (threadIdx.x == 0) {
    if (a.lse) a.lse[row] = lse;
    if (a.entropy) a.entropy[row] = entropy;
  }
  for (int t = threadIdx.x; t < a.T; t += kVocThreads) {
    const int id = a.ids[row * a.T + t];
    float v = 0.0f;
    if (id >= a.V) {
      v = __int_as_float(0x7FC00000);
      set_device_error(kDevBadId);
    } else if (id >= 0) {
      v = row_logprob(E::get(rv.row[id]), st, a.c, log_s);
    }
    a.logprobs[row * a.T + t] = v;
  }
  if constexpr (TOP) {
    top_merge(s_oval, s_ocol, s_cnt, cs, kTopMax, a.K, s_fval, s_fcol, &s_on);
    __syncthreads();
    const bool nan = st.s != st.s;
    for (int k = threadIdx.x; k < a.K; k += kVocThreads) {
      const bool have = k < s_on && !nan;
      a.top_ids[row * a.K + k] = have ? s_fcol[k] : -1;
      a.top_logprobs[row * a.K + k] =
          have ? row_logprob(s_fval[k], st, a.c, log_s) : (nan ? __int_as_float(0x7FC00000) : -IG_INF);
    }
  }
}

// ---- gradient of the log probabilities and the entropy ----------------------------------

struct LogprobGradArgs {
  const void *x;
  int64_t ld, rows;
  int V, T, segs;
  float c;
  const int32_t *ids;
  const float *lse, *entropy, *dlogprobs, *dentropy;
  void *dx;
  int64_t ldd;
};

// The row's gradient outside its given tokens is p (A + B t), t = z - lse:
//   A = -c (sum of the tokens' gradients + gH H), B = -c gH.
struct RowCoef {
  float A, B, lse;
};
__device__ __forceinline__ float dense_grad(float x, float c, const RowCoef &k) {
  const float t = max_nan(fmaf(x, c, -k.lse), kYMin);
  return ex2(t * kLog2e) * fmaf(k.B, t, k.A);
}
// The gradient a given token adds in its own column: c times the sum over the
// row's entries with the same id, in order.
__device__ __forceinline__ float token_grad(const int32_t *ids, const float *g, int T, int id, float c) {
  float s = 0.0f;
  for (int t = 0; t < T; t++)
    if (ids[t] == id) s += g[t];
  return s * c;
}
// Sum over the row's given tokens (ids in the vocabulary), one warp, in a fixed order.
__device__ __forceinline__ float given_grad_sum(const int32_t *ids, const float *g, int T, int V, bool &bad) {
  float s = 0.0f;
  bad = false;
  for (int t = threadIdx.x & 31; t < T; t += 32) {
    const int id = ids[t];
    if (id >= V) bad = true;
    if (id >= 0 && id < V) s += g[t];
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  return s;
}
__device__ __forceinline__ RowCoef row_coef(float lse, float H, float G, float gh, float c) {
  RowCoef k;
  k.B = -c * gh;
  k.A = -c * fmaf(gh, H, G);
  k.lse = lse;
  if (lse == -IG_INF) {  // no distribution: p = 0 everywhere
    k.A = k.B = 0.0f;
    k.lse = IG_INF;
  }
  return k;
}

// Writes the kN results of vector v of a row: as one 16-byte store where the
// output row has the input's alignment, else by element.
template <int DT>
__device__ __forceinline__ void store_vec(typename VElem<DT>::T *drow, const RowVecs<DT> &rv, int v, bool same,
                                          const float *d) {
  using E = VElem<DT>;
  if (same && rv.whole(v)) {
    __stcs(reinterpret_cast<uint4 *>(drow + rv.col(v)), E::pack(d));
  } else {
#pragma unroll
    for (int i = 0; i < E::kN; i++) {
      const int c = rv.col(v) + i;
      if (c >= 0 && c < rv.V) drow[c] = E::put(d[i]);
    }
  }
}

template <int DT>
__global__ void __launch_bounds__(kVocThreads, 4) token_logprobs_grad_kernel(const LogprobGradArgs a) {
  using E = VElem<DT>;
  using T = typename E::T;
  constexpr int kN = E::kN;
  __shared__ float s_G;
  const int64_t row = blockIdx.x / a.segs;
  const int seg = (int)(blockIdx.x - row * a.segs);
  const RowVecs<DT> rv(static_cast<const T *>(a.x) + row * a.ld, a.V);
  T *drow = static_cast<T *>(a.dx) + row * a.ldd;
  const bool same = (reinterpret_cast<uintptr_t>(drow) & 15) == (reinterpret_cast<uintptr_t>(rv.row) & 15);
  const int v0 = (int)((int64_t)rv.nv * seg / a.segs), v1 = (int)((int64_t)rv.nv * (seg + 1) / a.segs);
  const int32_t *ids = a.ids + row * a.T;
  const float *g = a.dlogprobs + row * a.T;
  if (threadIdx.x < 32) {
    bool bad;
    const float s = a.dlogprobs ? given_grad_sum(ids, g, a.T, a.V, bad) : 0.0f;
    if (a.dlogprobs && bad) set_device_error(kDevBadId);
    if (threadIdx.x == 0) s_G = s;
  }
  const float lse = a.lse[row];
  const float gh = a.dentropy ? a.dentropy[row] : 0.0f, H = a.dentropy ? a.entropy[row] : 0.0f;
  __syncthreads();
  const RowCoef k = row_coef(lse, H, s_G, gh, a.c);
  const int cfirst = max(rv.col(v0), 0), clast = min(rv.col(v1), a.V);
  // The given tokens' logits are read before any store: dx may be x.
  float xt = 0.0f;
  int tid_id = -1;
  if ((int)threadIdx.x < a.T && a.dlogprobs) {
    tid_id = ids[threadIdx.x];
    if (tid_id < cfirst || tid_id >= clast) tid_id = -1;
    if (tid_id >= 0) xt = E::get(rv.row[tid_id]);
  }
  __syncthreads();
  for (int b = v0; b < v1; b += kVocUnroll * kVocThreads) {
    uint4 raw[kVocUnroll];
#pragma unroll
    for (int j = 0; j < kVocUnroll; j++) {
      const int v = b + j * kVocThreads + (int)threadIdx.x;
      if (v < v1 && rv.whole(v)) raw[j] = __ldcs(reinterpret_cast<const uint4 *>(rv.row + rv.col(v)));
    }
#pragma unroll
    for (int j = 0; j < kVocUnroll; j++) {
      const int v = b + j * kVocThreads + (int)threadIdx.x;
      if (v >= v1) continue;
      float x[kN], d[kN];
      if (rv.whole(v))
        E::unpack(raw[j], x);
      else
        rv.load_edge(v, x);
#pragma unroll
      for (int i = 0; i < kN; i++) d[i] = dense_grad(x[i], a.c, k);
      store_vec<DT>(drow, rv, v, same, d);
    }
  }
  if (a.T == 0 || !a.dlogprobs) return;
  __syncthreads();
  if (tid_id >= 0 && lse != -IG_INF) drow[tid_id] = E::put(dense_grad(xt, a.c, k) + token_grad(ids, g, a.T, tid_id, a.c));
}

// ---- divergence from a teacher's top logits ----------------------------------------------

struct DistillArgs {
  const void *x;
  int64_t ld, rows;
  int V, K;
  float c;
  const int32_t *tids;
  const float *tlogits, *weights;
  float *loss;
  void *dx;
  int64_t ldd;
};

__device__ __forceinline__ float block_sum(float v, float *s8) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s8[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.0f;
#pragma unroll
  for (int w = 0; w < kVocWarps; w++) t += s8[w];
  return t;
}
__device__ __forceinline__ float block_max(float v, float *s8) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(~0u, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s8[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = s8[0];
#pragma unroll
  for (int w = 1; w < kVocWarps; w++) t = max_nan(t, s8[w]);
  return t;
}

// One cluster per row. With TAIL the mass outside the list is summed on its
// own (1 - the list's mass would lose it to cancellation): a bit per vector
// in shared memory says whether the vector holds listed columns, and those
// vectors (at most K) compare their columns with the list. The second pass
// writes the gradient while the row is still in L2.
template <int DT, bool TAIL>
__global__ void __launch_bounds__(kVocThreads, 4) distill_topk_kernel(const DistillArgs a) {
  using E = VElem<DT>;
  using T = typename E::T;
  constexpr int kN = E::kN, kX = kN * kVocUnroll;
  extern __shared__ uint32_t s_bits[];
  __shared__ VStat s_warp[kVocWarps];
  __shared__ VStat s_cta;
  __shared__ float s8[kVocWarps];
  __shared__ int s_ids[kTeacherMax];
  __shared__ float s_q[kTeacherMax];
  cg::cluster_group cl = cg::this_cluster();
  const int cs = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int64_t row = blockIdx.x / cs;
  const RowVecs<DT> rv(static_cast<const T *>(a.x) + row * a.ld, a.V);
  const int v0 = (int)((int64_t)rv.nv * rank / cs), v1 = (int)((int64_t)rv.nv * (rank + 1) / cs);
  const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const float c2 = a.c * kLog2e;
  const float w = a.weights ? a.weights[row] : 1.0f;
  T *drow = a.dx ? static_cast<T *>(a.dx) + row * a.ldd : nullptr;
  const bool same = (reinterpret_cast<uintptr_t>(drow) & 15) == (reinterpret_cast<uintptr_t>(rv.row) & 15);

  // The teacher's list: thread k holds entry k.
  int id = -1;
  float q = 0.0f, xk = -IG_INF;
  bool once = false;  // the first entry with its id
  if (tid < a.K) {
    id = a.tids[row * a.K + tid];
    if (id >= a.V) {
      set_device_error(kDevBadId);
      id = -1;
    }
    if (id < 0) id = -1;
    s_ids[tid] = id;
    if (id >= 0) xk = E::get(rv.row[id]);
  }
  const int any = __syncthreads_or(id >= 0);
  const bool skip = !any || w == 0.0f;  // uniform over the cluster
  const int cfirst = max(rv.col(v0), 0), clast = min(rv.col(v1), a.V);
  VStat st{-IG_INF, 0.0f, 0.0f};
  float q_rest = 0.0f;
  if (!skip) {
    if (id >= 0) {
      once = true;
      for (int k = 0; k < tid; k++)
        if (s_ids[k] == id) once = false;
    }
    const float t = id >= 0 ? a.tlogits[row * a.K + tid] : -IG_INF;
    if constexpr (TAIL) {
      q = id >= 0 ? expf(t) : 0.0f;
      const float q_list = block_sum(q, s8);
      q_rest = q_list == q_list ? fmaxf(1.0f - q_list, 0.0f) : q_list;
      const int nw = (v1 - v0 + 31) / 32;
      for (int i = tid; i < nw; i += kVocThreads) s_bits[i] = 0;
      __syncthreads();
      if (id >= cfirst && id < clast) {
        const int v = (id + rv.mis) / kN - v0;
        atomicOr(&s_bits[v >> 5], 1u << (v & 31));
      }
      __syncthreads();
    } else {
      const float top = block_max(t, s8);
      q = id >= 0 && top != -IG_INF ? expf((t - top) * a.c) : 0.0f;
      const float sum = block_sum(q, s8);
      if (sum > 0.0f || sum != sum) q /= sum;
    }
    for (int b = v0; b < v1; b += kVocUnroll * kVocThreads) {
      float x[kX];
      uint4 raw[kVocUnroll];
#pragma unroll
      for (int j = 0; j < kVocUnroll; j++) {
        const int v = b + j * kVocThreads + tid;
        if (v < v1 && rv.whole(v)) raw[j] = *reinterpret_cast<const uint4 *>(rv.row + rv.col(v));
      }
#pragma unroll
      for (int j = 0; j < kVocUnroll; j++) {
        const int v = b + j * kVocThreads + tid;
        if (v < v1 && rv.whole(v)) {
          E::unpack(raw[j], x + j * kN);
        } else if (v < v1) {
          rv.load_edge(v, x + j * kN);
        } else {
#pragma unroll
          for (int i = 0; i < kN; i++) x[j * kN + i] = -IG_INF;
        }
        if constexpr (TAIL) {
          if (v < v1 && (s_bits[(v - v0) >> 5] >> ((v - v0) & 31) & 1u)) {
            for (int k = 0; k < a.K; k++) {
              const int at = s_ids[k] - rv.col(v);
#pragma unroll
              for (int i = 0; i < kN; i++)
                if (at == i) x[j * kN + i] = -IG_INF;
            }
          }
        }
      }
      float mx = x[0];
#pragma unroll
      for (int i = 1; i < kX; i++) mx = fmaxf(mx, x[i]);
      mx = fmaxf(mx, -IG_INF);
      vstat_add<false>(st, x, mx, c2);
    }
    st = vstat_warp<false>(st, c2);
    if (lane == 0) s_warp[warp] = st;
    __syncthreads();
    st = s_warp[0];
    for (int i = 1; i < kVocWarps; i++) vstat_merge<false>(st, s_warp[i], c2);
  }
  if (cs > 1) {
    if (tid == 0) s_cta = st;
    cl.sync();
    st = *cl.map_shared_rank(&s_cta, 0);
    for (int r = 1; r < cs; r++) vstat_merge<false>(st, *cl.map_shared_rank(&s_cta, r), c2);
    cl.sync();  // every CTA has read the others' statistics (and the list's logits) before any stores or exits
  }
  // Dense gradient: coef 2^((x - mb) c2 - l2); a listed column: listed p - w c q.
  float coef = 0.0f, listed = 0.0f, pk = 0.0f;
  float mb = 0.0f, l2 = 0.0f;
  if (!skip) {
    VStat all = st;
    if constexpr (TAIL) {
      const float mk = block_max(once ? fmaxf(xk, -IG_INF) : -IG_INF, s8);
      const float mb = mk == -IG_INF ? 0.0f : mk;
      const float sk = block_sum(once ? ex2((xk - mb) * c2) : 0.0f, s8);
      vstat_merge<false>(all, VStat{mk, sk, 0.0f}, c2);
    }
    const float log_s = logf(all.s);
    const float logp = all.s == 0.0f ? -IG_INF : (xk - all.m) * a.c - log_s;
    const float q_list = block_sum(q, s8);
    float loss = block_sum(q > 0.0f || q != q ? q * (logf(q) - logp) : 0.0f, s8);
    float mass = q_list + q_rest, rest = 0.0f;
    bool far = false;
    if constexpr (TAIL) {
      if (st.s == 0.0f) {
        // Nothing outside the list: what is left of 1 is rounding.
        mass = q_list;
      } else if (q_rest > 0.0f || q_rest != q_rest) {
        const float logr = (st.m - all.m) * a.c + logf(st.s) - log_s;
        loss += q_rest * (logf(q_rest) - logr);
        // A tail of less than e^-60: p and q_rest / p_rest would leave the
        // float range. Its columns then take q_rest times their share of the
        // tail alone (p itself adds less than e^-60 / q_rest of that).
        far = logr < -60.0f;
        rest = q_rest * ex2(-logr * kLog2e);
      }
    }
    if (all.s != all.s) loss = all.s;
    if (rank == 0 && tid == 0) a.loss[row] = loss * w;
    listed = w * a.c * mass;
    pk = ex2((xk - (all.s == 0.0f ? 0.0f : all.m)) * c2 - log_s * kLog2e);
    coef = far ? -w * a.c * q_rest : w * a.c * (mass - rest);
    mb = far ? st.m : all.m;
    l2 = (far ? logf(st.s) : log_s) * kLog2e;
    st = all;
  } else if (rank == 0 && tid == 0) {
    a.loss[row] = 0.0f;
  }
  if (!drow) return;
  const bool zero = skip || st.s == 0.0f;
  for (int b = v0; b < v1; b += kVocUnroll * kVocThreads) {
    uint4 raw[kVocUnroll];
#pragma unroll
    for (int j = 0; j < kVocUnroll; j++) {
      const int v = b + j * kVocThreads + tid;
      if (!zero && v < v1 && rv.whole(v)) raw[j] = __ldcs(reinterpret_cast<const uint4 *>(rv.row + rv.col(v)));
    }
#pragma unroll
    for (int j = 0; j < kVocUnroll; j++) {
      const int v = b + j * kVocThreads + tid;
      if (v >= v1) continue;
      float x[kN], d[kN];
      if (zero) {
#pragma unroll
        for (int i = 0; i < kN; i++) d[i] = 0.0f;
      } else {
        if (rv.whole(v))
          E::unpack(raw[j], x);
        else
          rv.load_edge(v, x);
#pragma unroll
        for (int i = 0; i < kN; i++) d[i] = coef * ex2(fmaf(x[i] - mb, c2, -l2));
      }
      store_vec<DT>(drow, rv, v, same, d);
    }
  }
  if (zero) return;
  if (tid < a.K) s_q[tid] = q;
  __syncthreads();
  // The listed columns of this CTA's part; q of equal ids adds up.
  if (once && id >= cfirst && id < clast) {
    float sq = 0.0f;
    for (int k = tid; k < a.K; k++)
      if (s_ids[k] == id) sq += s_q[k];
    drow[id] = E::put(listed * pk - w * a.c * sq);
  }
}

// ---- launches --------------------------------------------------------------------------

// CTAs per row (a cluster): more than one while the rows alone do not give
// every SM several CTAs and a part keeps at least one round of vectors.
static int row_parts(int64_t rows, int V, int per_vec) {
  const int64_t nv = (V + per_vec - 1) / per_vec;
  int cs = 1;
  while (cs < 8 && rows * cs < 4 * 4 * num_sms() && nv / (2 * cs) >= kVocThreads) cs *= 2;
  return cs;
}

template <typename Args>
static cudaError_t launch_rows(void (*kern)(Args), const Args &a, int64_t rows, int cs, size_t smem, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * cs));
  cfg.blockDim = dim3(kVocThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  if (cs > 1) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cs;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, kern, a);
}

template <int DT>
static cudaError_t run_token_logprobs(const LogprobArgs &a, cudaStream_t st) {
  const int cs = row_parts(a.rows, a.V, VElem<DT>::kN);
  return a.K > 0 ? launch_rows(token_logprobs_kernel<DT, true>, a, a.rows, cs, 0, st)
                 : launch_rows(token_logprobs_kernel<DT, false>, a, a.rows, cs, 0, st);
}

template <int DT>
static cudaError_t run_token_logprobs_grad(LogprobGradArgs a, cudaStream_t st) {
  const int64_t nv = (a.V + VElem<DT>::kN - 1) / VElem<DT>::kN;
  const int64_t round = kVocUnroll * kVocThreads;
  a.segs = (int)((nv + round - 1) / round);
  return launch_rows(token_logprobs_grad_kernel<DT>, a, a.rows * a.segs, 1, 0, st);
}

template <int DT>
static cudaError_t run_distill(const DistillArgs &a, bool tail, cudaStream_t st) {
  const int cs = row_parts(a.rows, a.V, VElem<DT>::kN);
  if (!tail) return launch_rows(distill_topk_kernel<DT, false>, a, a.rows, cs, 0, st);
  const int64_t nv = a.V / VElem<DT>::kN + 2;
  const size_t smem = ((nv / cs + 1 + 31) / 32 + 1) * 4;
  static SmemOptIn attr;
  const cudaError_t e = attr.ensure((const void *)distill_topk_kernel<DT, true>, (int)smem);
  if (e != cudaSuccess) return e;
  return launch_rows(distill_topk_kernel<DT, true>, a, a.rows, cs, smem, st);
}

}  // namespace ig
