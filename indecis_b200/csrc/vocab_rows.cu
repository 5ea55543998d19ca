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
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "internal.h"

namespace ig {

constexpr int kVocThreads = 256;  // most threads per CTA (NT below: 32 to 256)
constexpr int kVocWarps = kVocThreads / 32;
constexpr int kVocUnroll = 4;     // 16-byte vectors of a thread per round
constexpr int kTopMax = 32;       // alternatives per row
constexpr int kIdsMax = 256;      // given tokens or teacher entries per row
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kYMin = -1.0e4f;  // 2^kYMin = 0
constexpr float kFltMax = 3.402823466e38f;
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

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// ---- element types --------------------------------------------------------------

// unpack/pack: a 16-byte vector as floats; kNegInf: -inf in every element;
// hmax: element-wise maximum (NaN ignored) of two words; top: the largest of a
// word's elements as a float.
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
  static constexpr uint32_t kNegInf = 0xFF800000u;
  __device__ __forceinline__ static uint32_t hmax(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
  __device__ __forceinline__ static float top(uint32_t a) { return fmaxf(__uint_as_float(a), -IG_INF); }
  __device__ __forceinline__ static uint32_t bits(T v) { return __float_as_uint(v); }
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
  static constexpr uint32_t kNegInf = 0xFF80FF80u;
  __device__ __forceinline__ static uint32_t hmax(uint32_t a, uint32_t b) {
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162 *>(&a), *reinterpret_cast<__nv_bfloat162 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&m);
  }
  __device__ __forceinline__ static float top(uint32_t a) {
    return fmaxf(fmaxf(__uint_as_float(a << 16), __uint_as_float(a & 0xFFFF0000u)), -IG_INF);
  }
  __device__ __forceinline__ static uint32_t bits(T v) { return __bfloat16_as_ushort(v); }
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
  static constexpr uint32_t kNegInf = 0xFC00FC00u;
  __device__ __forceinline__ static uint32_t hmax(uint32_t a, uint32_t b) {
    const __half2 m = __hmax2(*reinterpret_cast<__half2 *>(&a), *reinterpret_cast<__half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&m);
  }
  __device__ __forceinline__ static float top(uint32_t a) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&a));
    return fmaxf(fmaxf(f.x, f.y), -IG_INF);
  }
  __device__ __forceinline__ static uint32_t bits(T v) { return __half_as_ushort(v); }
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
  // A partial vector, -inf outside the row.
  __device__ __forceinline__ uint4 edge(int v) const {
    constexpr int kPer = E::kN / 4;  // elements per word
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      w[i] = E::kNegInf;
#pragma unroll
      for (int j = 0; j < kPer; j++) {
        const int c = col(v) + i * kPer + j;
        if (c >= 0 && c < V) {
          const uint32_t keep = kPer == 1 ? 0u : 0xFFFFu << (16 * (1 - j));
          w[i] = (w[i] & keep) | (E::bits(row[c]) << (16 * j));
        }
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ uint4 load(int v) const {
    return whole(v) ? *reinterpret_cast<const uint4 *>(row + col(v)) : edge(v);
  }
};

// A CTA's part of a row, vectors [v0, v1): the whole ones lie end to end from
// `base` (n of them, the first is vector w0); the row's partial first and last
// vector, if they fall into the part, are read on their own, so that the loops
// over the whole ones test nothing but their end.
template <int DT>
struct RowPart {
  const uint4 *base;
  int v0, v1, w0, n;
  bool first, last;
  __device__ __forceinline__ RowPart(const RowVecs<DT> &rv, uint32_t part, uint32_t parts) {
    const uint32_t per = ((uint32_t)rv.nv + parts - 1) / parts;
    v0 = min(part * per, (uint32_t)rv.nv);
    v1 = min(v0 + per, (uint32_t)rv.nv);
    first = v0 < v1 && !rv.whole(v0);
    last = v1 - v0 > (first ? 1 : 0) && !rv.whole(v1 - 1);
    w0 = v0 + (first ? 1 : 0);
    n = v1 - w0 - (last ? 1 : 0);
    base = reinterpret_cast<const uint4 *>(rv.row + rv.col(w0));
  }
};
// The threads of NT that take the partial vectors.
constexpr int kFirstThread = 0;
constexpr int last_thread(int NT) { return NT > 32 ? 32 : 16; }

// A thread's own vectors i NT of a part, read kAheadRounds rounds of
// kVocUnroll ahead through slots in shared memory that no other thread
// touches: asynchronous 16-byte copies need no registers while they are on
// their way and, since each thread waits for its own, no barrier. Twelve
// vectors a thread keep up to 192 KB per SM in flight. Against four in
// registers: 104 us and 113 for 1024 x 262144 bf16 log probabilities, 157 and
// 172 for the distillation of 4096 x 50021 bf16 (two rounds there: the byte
// masks of the tail need the room, 213 us against 236 for 1024 x 262144
// float16).
constexpr int kAheadRounds = 3;
template <int NT, int ROUNDS = kAheadRounds>
struct Ahead {
  static constexpr int kRound = kVocUnroll * NT;
  static constexpr int kBytes = ROUNDS * kRound * 16;
  uint4 *slots;  // this thread's: [ROUNDS][kVocUnroll], NT apart
  const uint4 *src;
  int mine;  // vector i is there while i < mine (i in steps of NT)
  __device__ __forceinline__ Ahead(void *smem, const uint4 *src_, int mine_)
      : slots(static_cast<uint4 *>(smem) + threadIdx.x), src(src_), mine(mine_) {}
  __device__ __forceinline__ void ask(int b, int stage) {
#pragma unroll
    for (int j = 0; j < kVocUnroll; j++)
      if (b + j * NT < mine) cp_async16(slots + (stage * kVocUnroll + j) * NT, src + b + j * NT);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  __device__ __forceinline__ void start() {
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) ask(r * kRound, r);
  }
  // f(b, raw) for every round b of the thread's vectors, in order; raw[j] is
  // there while b + j NT < mine.
  template <typename F>
  __device__ __forceinline__ void each(F f) {
    int stage = 0;
    for (int b = 0; b < mine; b += kRound) {
      asm volatile("cp.async.wait_group %0;" ::"n"(ROUNDS - 1) : "memory");
      uint4 raw[kVocUnroll];
#pragma unroll
      for (int j = 0; j < kVocUnroll; j++) raw[j] = slots[(stage * kVocUnroll + j) * NT];
      ask(b + ROUNDS * kRound, stage);
      stage = stage + 1 == ROUNDS ? 0 : stage + 1;
      f(b, raw);
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

// One pair of values.
template <bool U>
__device__ __forceinline__ void vstat_pair(float2 x, float2 nm, float2 cc, float2 &s, float2 &u) {
  float2 y = __fmul2_rn(__fadd2_rn(x, nm), cc);
  if constexpr (U) {
    y.x = max_nan(y.x, kYMin);
    y.y = max_nan(y.y, kYMin);
  }
  const float2 e = make_float2(ex2(y.x), ex2(y.y));
  s = __fadd2_rn(s, e);
  if constexpr (U) u = __ffma2_rn(e, y, u);
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
  for (int i = 0; i < N; i += 2) vstat_pair<U>(make_float2(x[i], x[i + 1]), nm, cc, s, u);
  a.s += s.x + s.y;
  if constexpr (U) a.u += u.x + u.y;
}

// R vectors: the maximum on the packed words, then vector by vector.
template <int DT, bool U, int R>
__device__ __forceinline__ void vstat_add_raw(VStat &a, const uint4 (&raw)[R], float c2) {
  using E = VElem<DT>;
  uint32_t w = E::hmax(E::hmax(raw[0].x, raw[0].y), E::hmax(raw[0].z, raw[0].w));
#pragma unroll
  for (int j = 1; j < R; j++)
    w = E::hmax(w, E::hmax(E::hmax(raw[j].x, raw[j].y), E::hmax(raw[j].z, raw[j].w)));
  const float m = fmaxf(a.m, E::top(w));
  if (m > a.m) vstat_shift<U>(a, m, c2);
  const float mb = m == -IG_INF ? 0.0f : m;
  const float2 nm = make_float2(-mb, -mb), cc = make_float2(c2, c2);
  float2 s = make_float2(0.0f, 0.0f), u = s;
#pragma unroll
  for (int j = 0; j < R; j++) {
    float x[E::kN];
    E::unpack(raw[j], x);
#pragma unroll
    for (int i = 0; i < E::kN; i += 2) vstat_pair<U>(make_float2(x[i], x[i + 1]), nm, cc, s, u);
  }
  a.s += s.x + s.y;
  if constexpr (U) a.u += u.x + u.y;
}

__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// The warp's statistics, in all lanes.
template <bool U>
__device__ __forceinline__ VStat vstat_warp(VStat a, float c2) {
  vstat_shift<U>(a, warp_max(a.m), c2);
  a.s = warp_sum(a.s);
  if constexpr (U) a.u = warp_sum(a.u);
  return a;
}

// n statistics in shared memory, joined in order: one maximum, then
// independent terms.
template <bool U>
__device__ __forceinline__ VStat vstat_join(const VStat *p, int n, float c2) {
  VStat a{p[0].m, 0.0f, 0.0f};
  for (int i = 1; i < n; i++) a.m = fmaxf(a.m, p[i].m);
  for (int i = 0; i < n; i++) {
    VStat b = p[i];
    vstat_shift<U>(b, a.m, c2);
    a.s += b.s;
    if constexpr (U) a.u += b.u;
  }
  return a;
}

// Clusters: a CTA hands its statistics to others by asynchronous stores that
// count on the receiver's barrier. The barriers are set up before the loops
// over the row; cluster_ready() makes sure, before the first store to another
// CTA, that it has started and set up its own.
__device__ __forceinline__ void cluster_announce() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_ready() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// ---- top alternatives ---------------------------------------------------------------

// (value, column) order: larger value first, then the lower column.
__device__ __forceinline__ bool top_before(float va, int ca, float vb, int cb) {
  return va > vb || (va == vb && ca < cb);
}
// The K first (value, column) of a CTA's part of a row, after the statistics'
// pass has left each thread its own maximum: the K-th largest of the threads'
// maxima is a lower bound of the K-th largest value (K threads hold a value at
// least as large), and only the vectors of threads that reach it (K, or a few
// more) are read again, from L2. The bound is found bit by bit on the ordered
// bits of the maxima, one counting barrier per bit. What reaches it is
// collected and ranked. With too many equal values for the buffer (a row of
// few distinct values) the K are found one by one instead.
template <int NT>
struct TopShared {
  static constexpr int kCap = NT < 128 ? 256 : 2 * NT;  // candidates a CTA collects
  int kept[NT];
  float val[kCap];
  int col[kCap];
  int nkept, n;
  float wv[NT / 32];
  int wc[NT / 32];
};
// Unsigned integers in the order of the floats (no NaN); -0 and +0 are one.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = v == 0.0f ? 0u : __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_order_key(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

template <int DT, int NT>
__device__ __noinline__ void top_one_by_one(const RowVecs<DT> rv, int v0, int v1, int K, TopShared<NT> &t, float *out_val,
                                            int *out_col, int *out_n) {
  using E = VElem<DT>;
  float lv = IG_INF;
  int lc = -1, n = 0;
  for (; n < K; n++) {
    float bv = -IG_INF;
    int bc = 0x7FFFFFFF;
    for (int v = v0 + (int)threadIdx.x; v < v1; v += NT) {
      float x[E::kN];
      E::unpack(rv.load(v), x);
#pragma unroll
      for (int i = 0; i < E::kN; i++) {
        const int c = rv.col(v) + i;
        if (x[i] > -IG_INF && top_before(lv, lc, x[i], c) && top_before(x[i], c, bv, bc)) {
          bv = x[i];
          bc = c;
        }
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const float ov = __shfl_xor_sync(~0u, bv, o);
      const int oc = __shfl_xor_sync(~0u, bc, o);
      if (top_before(ov, oc, bv, bc)) {
        bv = ov;
        bc = oc;
      }
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
      t.wv[threadIdx.x >> 5] = bv;
      t.wc[threadIdx.x >> 5] = bc;
    }
    __syncthreads();
    for (int w = 0; w < NT / 32; w++)
      if (top_before(t.wv[w], t.wc[w], bv, bc)) {
        bv = t.wv[w];
        bc = t.wc[w];
      }
    if (bc == 0x7FFFFFFF) break;
    if (threadIdx.x == 0) {
      out_val[n] = bv;
      out_col[n] = bc;
    }
    lv = bv;
    lc = bc;
  }
  if (threadIdx.x == 0) *out_n = n;
}

template <int DT, int NT>
__device__ __forceinline__ void top_scan(const uint4 &raw, int col, float tau, TopShared<NT> &t) {
  using E = VElem<DT>;
  if (E::top(E::hmax(E::hmax(raw.x, raw.y), E::hmax(raw.z, raw.w))) < tau) return;
  float x[E::kN];
  E::unpack(raw, x);
#pragma unroll
  for (int i = 0; i < E::kN; i++)
    if (x[i] >= tau && x[i] > -IG_INF) {
      const int at = atomicAdd(&t.n, 1);
      if (at < TopShared<NT>::kCap) {
        t.val[at] = x[i];
        t.col[at] = col + i;
      }
    }
}

// tmax: the thread's maximum over the part's whole vectors threadIdx.x + i
// NT (and a partial one, which is read again in any case).
template <int DT, int NT>
__device__ __forceinline__ void top_select(const RowVecs<DT> &rv, const RowPart<DT> &rp, float tmax, int K, TopShared<NT> &t,
                                           float *out_val, int *out_col, int *out_n) {
  const int tid = (int)threadIdx.x;
  if (tid == 0) t.nkept = t.n = 0;
  const uint32_t key = order_key(tmax);
  uint32_t bound = 0;
  // Bits that tell widened values apart: sign, 8 of exponent and the type's mantissa.
  constexpr int kBits = DT == IG_DT_BF16 ? 16 : DT == IG_DT_F16 ? 19 : 32;
  for (int bit = 31; bit >= 32 - kBits; bit--) {
    const uint32_t next = bound | (1u << bit);
    const int n = __syncthreads_count(key >= next);
    if (n >= K) {
      bound = next;
      if (n <= K + 2) break;
    }
  }
  __syncthreads();  // nkept and n are set whatever the number of barriers above
  const float tau = bound <= order_key(-IG_INF) ? -IG_INF : from_order_key(bound);
  if (key >= bound && tmax > -IG_INF) t.kept[atomicAdd(&t.nkept, 1)] = tid;
  __syncthreads();
  const int rounds = (rp.n + NT - 1) / NT;
  const int items = t.nkept * rounds;
  constexpr int kAhead = 4;  // loads in flight per thread
  for (int it = tid; it < items; it += kAhead * NT) {
    uint4 raw[kAhead];
    int at[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      const int k = it + j * NT, b = k / rounds;
      at[j] = k < items ? (k - b * rounds) * NT + t.kept[b] : rp.n;
      if (at[j] < rp.n) raw[j] = rp.base[at[j]];
    }
#pragma unroll
    for (int j = 0; j < kAhead; j++)
      if (at[j] < rp.n) top_scan<DT, NT>(raw[j], rv.col(rp.w0 + at[j]), tau, t);
  }
  if (tid == kFirstThread && rp.first) top_scan<DT, NT>(rv.edge(rp.v0), rv.col(rp.v0), tau, t);
  if (tid == last_thread(NT) && rp.last) top_scan<DT, NT>(rv.edge(rp.v1 - 1), rv.col(rp.v1 - 1), tau, t);
  __syncthreads();
  const int n = t.n;
  if (n > TopShared<NT>::kCap) {
    top_one_by_one<DT, NT>(rv, rp.v0, rp.v1, K, t, out_val, out_col, out_n);
    return;
  }
  // The order of arrival varies, the ranks do not.
  for (int i = tid; i < n; i += NT) {
    const float v = t.val[i];
    const int c = t.col[i];
    int r = 0;
    for (int j = 0; j < n; j++) r += top_before(t.val[j], t.col[j], v, c);
    if (r < K) {
      out_val[r] = v;
      out_col[r] = c;
    }
  }
  if (tid == 0) *out_n = n < K ? n : K;
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
  int parts;  // CTAs per row (a cluster)
};

// Row results from its statistics and, for top_k, its sorted candidates.
__device__ __forceinline__ void row_lse(const VStat &a, float c, float &log_s, float &lse, float &entropy) {
  const bool empty = a.s == 0.0f;
  log_s = logf(a.s);
  // -inf stands for an empty row alone (NaN is kept).
  lse = empty ? -IG_INF : max_nan(fmaf(a.m, c, log_s), -kFltMax);
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
// into the first K, written to out_val/out_col; their number to *out_n.
template <int NT>
__device__ __forceinline__ void top_merge(const float *val, const int *col, const int *cnt, int lists, int stride, int K,
                                          float *out_val, int *out_col, int *out_n) {
  int total = 0;
  for (int l = 0; l < lists; l++) total += cnt[l];
  for (int i = threadIdx.x; i < lists * K; i += NT) {
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

// A CTA (or a cluster of up to eight) per row: one pass for the statistics,
// the alternatives from the vectors of the best threads, the given tokens'
// logits asked for at the start. 4096 x 50021 float32: 142 us, 5.8 TB/s, 90% of
// the measured copy bandwidth; bf16: 88 us, 4.7 TB/s (73%), where the
// exponentials and their latencies show (half the bytes for each); the 20
// best alternatives add 36 us there (the second read of 8% of the row, the
// bound's barriers and the ranking).
template <int DT, bool TOP, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) token_logprobs_kernel(const LogprobArgs a) {
  using E = VElem<DT>;
  using T = typename E::T;
  __shared__ VStat s_warp[NT / 32];
  __shared__ VStat s_part[8];  // on rank 0, the cluster's statistics
  extern __shared__ uint4 s_ahead[];
  constexpr int kLists = NT == kVocThreads ? 8 : 1;  // smaller CTAs have their row alone
  __shared__ TopShared<NT> s_top[1];
  __shared__ float s_oval[TOP ? kLists * kTopMax : 1];  // this CTA's list, and on rank 0 all the cluster's
  __shared__ int s_ocol[TOP ? kLists * kTopMax : 1];
  __shared__ int s_cnt[8], s_on;
  __shared__ float s_fval[TOP ? kTopMax : 1];
  __shared__ int s_fcol[TOP ? kTopMax : 1];
  __shared__ __align__(8) uint64_t s_bar;

  const int cs = NT == kVocThreads ? a.parts : 1, rank = cs > 1 ? (int)cluster_ctarank() : 0;
  const int64_t row = blockIdx.x / cs;
  const RowVecs<DT> rv(static_cast<const T *>(a.x) + row * a.ld, a.V);
  const RowPart<DT> rp(rv, rank, cs);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float c2 = a.c * kLog2e;
  Ahead<NT> ahead(s_ahead, rp.base + threadIdx.x, rp.n - (int)threadIdx.x);
  ahead.start();
  if (cs > 1) {
    if (threadIdx.x == 0) {
      mbar_init(&s_bar, 1);
      fence_barrier_init();
      // Rank 0 waits for the others' statistics and lists.
      if (rank == 0) mbar_arrive_expect_tx(&s_bar, (uint32_t)(cs - 1) * (12u + 8u * a.K + (TOP ? 4u : 0u)));
    }
    __syncwarp();
    cluster_announce();
  }
  // The given tokens' logits (of the first NT), asked for early.
  int id = -1;
  float xt = 0.0f;
  if (rank == 0 && (int)threadIdx.x < a.T) {
    id = a.ids[row * a.T + threadIdx.x];
    if (id >= 0 && id < a.V) xt = E::get(rv.row[id]);
  }

  VStat st{-IG_INF, 0.0f, 0.0f};
  ahead.each([&](int b, const uint4(&raw)[kVocUnroll]) {
    if (b + (kVocUnroll - 1) * NT < ahead.mine) {
      vstat_add_raw<DT, true>(st, raw, c2);
    } else {
#pragma unroll
      for (int j = 0; j < kVocUnroll; j++)
        if (b + j * NT < ahead.mine) {
          const uint4 one[1] = {raw[j]};
          vstat_add_raw<DT, true>(st, one, c2);
        }
    }
  });
  if (threadIdx.x == kFirstThread && rp.first) {
    const uint4 raw[1] = {rv.edge(rp.v0)};
    vstat_add_raw<DT, true>(st, raw, c2);
  }
  if (threadIdx.x == last_thread(NT) && rp.last) {
    const uint4 raw[1] = {rv.edge(rp.v1 - 1)};
    vstat_add_raw<DT, true>(st, raw, c2);
  }
  const float tmax = st.m;
  st = vstat_warp<true>(st, c2);
  if (lane == 0) s_warp[warp] = st;
  if constexpr (TOP) top_select<DT, NT>(rv, rp, tmax, a.K, s_top[0], s_oval, s_ocol, &s_on);
  __syncthreads();
  st = vstat_join<true>(s_warp, NT / 32, c2);
  if (cs > 1) {
    cluster_ready();
    if (rank != 0) {
      if (threadIdx.x == 0) {
        st_async_f32(&s_part[rank].m, 0, st.m, &s_bar);
        st_async_f32(&s_part[rank].s, 0, st.s, &s_bar);
        st_async_f32(&s_part[rank].u, 0, st.u, &s_bar);
        if constexpr (TOP) st_async_f32(reinterpret_cast<float *>(&s_cnt[rank]), 0, __int_as_float(s_on), &s_bar);
      }
      if constexpr (TOP) {
        if ((int)threadIdx.x < a.K) {  // past the list's end: not read
          st_async_f32(&s_oval[rank * kTopMax + threadIdx.x], 0, s_oval[threadIdx.x], &s_bar);
          st_async_f32(reinterpret_cast<float *>(&s_ocol[rank * kTopMax + threadIdx.x]), 0,
                       __int_as_float(s_ocol[threadIdx.x]), &s_bar);
        }
      }
      return;
    }
    if (threadIdx.x == 0) {
      s_part[0] = st;
      s_cnt[0] = TOP ? s_on : 0;
    }
    mbar_wait_cluster(&s_bar, 0, kDevTimeoutFull);
    __syncthreads();
    st = vstat_join<true>(s_part, cs, c2);
  }
  float log_s, lse, entropy;
  row_lse(st, a.c, log_s, lse, entropy);
  if (threadIdx.x == 0) {
    if (a.lse) a.lse[row] = lse;
    if (a.entropy) a.entropy[row] = entropy;
  }
  for (int k = threadIdx.x; k < a.T; k += NT) {
    if (k >= NT) {
      id = a.ids[row * a.T + k];
      if (id >= 0 && id < a.V) xt = E::get(rv.row[id]);
    }
    float v = 0.0f;
    if (id >= a.V) {
      v = __int_as_float(0x7FC00000);
      set_device_error(kDevBadId);
    } else if (id >= 0) {
      v = row_logprob(xt, st, a.c, log_s);
    }
    a.logprobs[row * a.T + k] = v;
  }
  if constexpr (TOP) {
    const float *fval = s_oval;
    const int *fcol = s_ocol;
    if (cs > 1) {
      top_merge<NT>(s_oval, s_ocol, s_cnt, cs, kTopMax, a.K, s_fval, s_fcol, &s_on);
      __syncthreads();
      fval = s_fval;
      fcol = s_fcol;
    }
    const bool nan = st.s != st.s;
    for (int k = threadIdx.x; k < a.K; k += NT) {
      const bool have = k < s_on && !nan;
      a.top_ids[row * a.K + k] = have ? fcol[k] : -1;
      a.top_logprobs[row * a.K + k] =
          have ? row_logprob(fval[k], st, a.c, log_s) : (nan ? __int_as_float(0x7FC00000) : -IG_INF);
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

// The row's gradient outside its given tokens is p (A + B t) with
// t = log p = x c - l, l the row's logsumexp, in one multiply-add:
//   A = -c (sum of the tokens' gradients + gH H), B = -c gH.
struct RowCoef {
  float A, B, l;
};
constexpr float kTMin = -1.0e4f;  // e^kTMin = 0
// A log probability; HOLD: at or below 0, where l may be one that float32 does
// not resolve. NaN is kept.
template <bool HOLD>
__device__ __forceinline__ float log_prob(float t) {
  t = max_nan(t, kTMin);
  return HOLD ? min_nan(t, 0.0f) : t;
}
// From t = log_prob(..).
__device__ __forceinline__ float dense_grad(float t, const RowCoef &k) { return ex2(t * kLog2e) * fmaf(k.B, t, k.A); }
template <bool HOLD>
__device__ __forceinline__ float2 dense_grad2(float2 x, float c, const RowCoef &k) {
  float2 t = __ffma2_rn(x, make_float2(c, c), make_float2(-k.l, -k.l));
  t.x = log_prob<HOLD>(t.x);
  t.y = log_prob<HOLD>(t.y);
  const float2 y = __fmul2_rn(t, make_float2(kLog2e, kLog2e));
  return __fmul2_rn(make_float2(ex2(y.x), ex2(y.y)), __ffma2_rn(make_float2(k.B, k.B), t, make_float2(k.A, k.A)));
}
// The gradient a given token adds in its own column: c times the sum over the
// row's entries with the same id, in order.
__device__ __forceinline__ float token_grad(const int32_t *ids, const float *g, int T, int id, float c) {
  float s = 0.0f;
  for (int t = 0; t < T; t++)
    if (ids[t] == id) s += g[t];
  return s * c;
}
// Sum over the row's given tokens (ids in the vocabulary), one warp, in a fixed
// order; size: of the absolute values, per lane. Entries that are not given
// count for neither.
__device__ __forceinline__ float given_grad_sum(const int32_t *ids, const float *g, int T, int V, bool &bad, float &size) {
  float s = 0.0f;
  bad = false;
  size = 0.0f;
  for (int t = threadIdx.x & 31; t < T; t += 32) {
    const int id = ids[t];
    if (id >= V) bad = true;
    if (id >= 0 && id < V) {
      s += g[t];
      size += fabsf(g[t]);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  return s;
}
__device__ __forceinline__ RowCoef row_coef(float l, float H, float G, float gh, float c) {
  if (l == -IG_INF) return RowCoef{0.0f, 0.0f, IG_INF};  // no distribution
  return RowCoef{-c * fmaf(gh, H, G), -c * gh, l};
}

// Writes the kN results of a whole vector: as one 16-byte store where the
// output row has the input's alignment, else by element.
template <int DT>
__device__ __forceinline__ void store_whole(typename VElem<DT>::T *dst, bool same, const float *d) {
  using E = VElem<DT>;
  if (same) {
    __stcs(reinterpret_cast<uint4 *>(dst), E::pack(d));
  } else {
#pragma unroll
    for (int i = 0; i < E::kN; i++) dst[i] = E::put(d[i]);
  }
}
template <int DT>
__device__ __forceinline__ void store_edge(typename VElem<DT>::T *drow, const RowVecs<DT> &rv, int v, const float *d) {
  using E = VElem<DT>;
#pragma unroll
  for (int i = 0; i < E::kN; i++) {
    const int c = rv.col(v) + i;
    if (c >= 0 && c < rv.V) drow[c] = E::put(d[i]);
  }
}

// The given tokens' columns of a part, [cfirst, clast): their logits, read
// before any store (dx may be x), and after the part their gradients.
template <int DT, int NT>
__device__ __forceinline__ void given_logits(const typename VElem<DT>::T *row, const int32_t *ids, int T, int cfirst,
                                             int clast, float *s_xt) {
  for (int i = threadIdx.x; i < T; i += NT) {
    const int id = ids[i];
    if (id >= cfirst && id < clast) s_xt[i] = VElem<DT>::get(row[id]);
  }
}
// m: what l is counted from.
template <int DT, int NT>
__device__ __forceinline__ void given_grads(typename VElem<DT>::T *drow, const int32_t *ids, const float *g, int T, int cfirst,
                                            int clast, const float *s_xt, float m, float c, const RowCoef &k) {
  for (int i = threadIdx.x; i < T; i += NT) {
    const int id = ids[i];
    if (id >= cfirst && id < clast)
      drow[id] = VElem<DT>::put(dense_grad(log_prob<false>(fmaf(s_xt[i] - m, c, -k.l)), k) + token_grad(ids, g, T, id, c));
  }
}

// The largest |lse| that the gradient is formed from: float32 holds it to
// |lse| 2^-24, 6e-5 at most, which is the relative error of p. Past it (a row
// wholly masked by a finite value, logits at a large offset, a very low
// temperature) one CTA takes the whole row and its maximum and sum again, as
// the forward has them: 111 us where 2047 x 50021 bf16 takes 70 from lse, 368
// and 259 for 4096 x 50021 float32, 72 and 10 for 16 x 262144. (The row's CTAs
// as a cluster take 19 us for the last, but the launch as clusters costs the
// ordinary rows: 103 and 49 us for 16384 x 4096 bf16.)
constexpr float kLseMost = 1024.0f;

template <int DT, int NT>
__device__ __noinline__ void grad_whole_row(const LogprobGradArgs &a, int64_t row, float G, float H, float gh, void *slots,
                                            float *s_xt, VStat *s_warp) {
  using E = VElem<DT>;
  using T = typename E::T;
  constexpr int kN = E::kN;
  const int tid = (int)threadIdx.x;
  const RowVecs<DT> rv(static_cast<const T *>(a.x) + row * a.ld, a.V);
  const RowPart<DT> rp(rv, 0, 1);
  T *drow = static_cast<T *>(a.dx) + row * a.ldd;
  const bool same = (reinterpret_cast<uintptr_t>(drow) & 15) == (reinterpret_cast<uintptr_t>(rv.row) & 15);
  const float c2 = a.c * kLog2e;
  Ahead<NT> ahead(slots, rp.base + tid, rp.n - tid);
  ahead.start();
  uint4 edge;
  const bool has_edge = (tid == kFirstThread && rp.first) || (tid == last_thread(NT) && rp.last);
  const int edge_v = tid == kFirstThread ? rp.v0 : rp.v1 - 1;
  if (has_edge) edge = rv.edge(edge_v);
  const int32_t *ids = a.ids + row * a.T;
  if (a.dlogprobs) given_logits<DT, NT>(rv.row, ids, a.T, 0, a.V, s_xt);
  VStat st{-IG_INF, 0.0f, 0.0f};
  ahead.each([&](int b, const uint4(&raw)[kVocUnroll]) {
#pragma unroll
    for (int j = 0; j < kVocUnroll; j++)
      if (b + j * NT < ahead.mine) {
        const uint4 one[1] = {raw[j]};
        vstat_add_raw<DT, false>(st, one, c2);
      }
  });
  if (has_edge) {
    const uint4 one[1] = {edge};
    vstat_add_raw<DT, false>(st, one, c2);
  }
  ahead.start();
  st = vstat_warp<false>(st, c2);
  if ((tid & 31) == 0) s_warp[tid >> 5] = st;
  __syncthreads();
  st = vstat_join<false>(s_warp, NT / 32, c2);
  const float m = st.s == 0.0f ? 0.0f : st.m;
  const RowCoef k = row_coef(st.s == 0.0f ? -IG_INF : logf(st.s), H, G, gh, a.c);
  auto grad = [&](const uint4 &v, float *d) {
    float x[kN];
    E::unpack(v, x);
#pragma unroll
    for (int i = 0; i < kN; i += 2) {
      const float2 r = dense_grad2<false>(make_float2(x[i] - m, x[i + 1] - m), a.c, k);
      d[i] = r.x;
      d[i + 1] = r.y;
    }
  };
  T *dp = drow + rv.col(rp.w0) + (int64_t)tid * kN;
  ahead.each([&](int b, const uint4(&raw)[kVocUnroll]) {
#pragma unroll
    for (int j = 0; j < kVocUnroll; j++) {
      if (b + j * NT >= ahead.mine) break;
      float d[kN];
      grad(raw[j], d);
      store_whole<DT>(dp + (int64_t)(b + j * NT) * kN, same, d);
    }
  });
  if (has_edge) {
    float d[kN];
    grad(edge, d);
    store_edge<DT>(drow, rv, edge_v, d);
  }
  if (!a.dlogprobs || st.s == 0.0f) return;
  __syncthreads();
  given_grads<DT, NT>(drow, ids, a.dlogprobs + row * a.T, a.T, 0, a.V, s_xt, m, a.c, k);
}

// A CTA per part of a row, element by element from the row's saved lse and
// entropy: bound by the bytes (each read once, written once). 2047 x 50021
// bf16: 73 us, 5.6 TB/s, 87% of the measured copy bandwidth.
template <int DT, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) token_logprobs_grad_kernel(const __grid_constant__ LogprobGradArgs a) {
  using E = VElem<DT>;
  using T = typename E::T;
  constexpr int kN = E::kN;
  __shared__ float s_G, s_xt[kIdsMax];
  __shared__ VStat s_warp[NT / 32];
  const int64_t row = blockIdx.x / a.segs;
  const int seg = (int)(blockIdx.x - row * a.segs);
  const RowVecs<DT> rv(static_cast<const T *>(a.x) + row * a.ld, a.V);
  T *drow = static_cast<T *>(a.dx) + row * a.ldd;
  const bool same = (reinterpret_cast<uintptr_t>(drow) & 15) == (reinterpret_cast<uintptr_t>(rv.row) & 15);
  const RowPart<DT> rp(rv, seg, a.segs);
  const int32_t *ids = a.ids + row * a.T;
  const float *g = a.dlogprobs + row * a.T;
  extern __shared__ uint4 s_ahead[];
  Ahead<NT> ahead(s_ahead, rp.base + threadIdx.x, rp.n - (int)threadIdx.x);
  ahead.start();  // before the row's scalars
  uint4 edge;
  if (threadIdx.x == kFirstThread && rp.first) edge = rv.edge(rp.v0);
  if (threadIdx.x == last_thread(NT) && rp.last) edge = rv.edge(rp.v1 - 1);
  const float lse = a.lse[row];
  const float gh = a.dentropy ? a.dentropy[row] : 0.0f, H = a.dentropy ? a.entropy[row] : 0.0f;
  if (threadIdx.x < 32) {
    bool bad;
    float size;
    const float s = a.dlogprobs ? given_grad_sum(ids, g, a.T, a.V, bad, size) : 0.0f;
    if (a.dlogprobs && bad) set_device_error(kDevBadId);
    if (threadIdx.x == 0) s_G = s;
  }
  const int cfirst = max(rv.col(rp.v0), 0), clast = min(rv.col(rp.v1), a.V);
  if (a.dlogprobs) given_logits<DT, NT>(rv.row, ids, a.T, cfirst, clast, s_xt);
  __syncthreads();
  if (fabsf(lse) > kLseMost && lse != -IG_INF) {
    cp_async_wait_all();
    if (seg == 0) grad_whole_row<DT, NT>(a, row, s_G, H, gh, s_ahead, s_xt, s_warp);
    return;
  }
  const RowCoef k = row_coef(lse, H, s_G, gh, a.c);
  auto grad = [&](const uint4 &v, float *d) {
    float x[kN];
    E::unpack(v, x);
#pragma unroll
    for (int i = 0; i < kN; i += 2) {
      const float2 r = dense_grad2<false>(make_float2(x[i], x[i + 1]), a.c, k);
      d[i] = r.x;
      d[i + 1] = r.y;
    }
  };
  T *dp = drow + rv.col(rp.w0) + (int64_t)threadIdx.x * kN;
  ahead.each([&](int b, const uint4(&raw)[kVocUnroll]) {
#pragma unroll
    for (int j = 0; j < kVocUnroll; j++) {
      if (b + j * NT >= ahead.mine) break;
      float d[kN];
      grad(raw[j], d);
      store_whole<DT>(dp + (int64_t)(b + j * NT) * kN, same, d);
    }
  });
  if ((threadIdx.x == kFirstThread && rp.first) || (threadIdx.x == last_thread(NT) && rp.last)) {
    float d[kN];
    grad(edge, d);
    store_edge<DT>(drow, rv, threadIdx.x == kFirstThread ? rp.v0 : rp.v1 - 1, d);
  }
  if (a.T == 0 || !a.dlogprobs || k.l == IG_INF) return;
  __syncthreads();
  given_grads<DT, NT>(drow, ids, g, a.T, cfirst, clast, s_xt, 0.0f, a.c, k);
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
  int parts;  // CTAs per row (a cluster)
};

// Less than this left of 1 by the list is the rounding of its sum (3e-7 at
// most over lists of up to 256 that hold everything): no outcome. Against
// columns that are masked by a finite value it would count with their whole
// depth (2e30 nats for the lowest value, 2e-3 for -1e4 at temperature 0.3).
constexpr float kRestLeast = 4.76837158e-7f;  // 2^-21

// A CTA or a cluster per row, in two passes over it: the statistics, then the
// gradient while the row is still in L2 (the row is fetched from DRAM once).
// 4096 x 50021 bf16: 157 us, 5.2 TB/s of its 820 MB, 81% of the measured copy
// bandwidth; 1024 x 262144 float16 with the tail: 213 us, 5.0 TB/s. Holding the
// row's part in shared memory between the passes, by bulk copies, took 207 us
// for the former: the copies' wait and the clusters that make room cost more
// than the second read. The teacher's list is worked on by one warp. With TAIL
// the mass outside the list is summed on its own (1 - the list's mass would
// lose it to cancellation): a byte per vector in shared memory marks its
// listed columns.
template <int DT, bool TAIL, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) distill_topk_kernel(const DistillArgs a) {
  using E = VElem<DT>;
  using T = typename E::T;
  constexpr int kN = E::kN;
  extern __shared__ uint4 s_dyn[];
  __shared__ VStat s_warp[NT / 32];
  __shared__ VStat s_part[8];  // every CTA's statistics
  __shared__ VStat s_list;     // with TAIL: the listed columns'
  __shared__ float s_mass[2];  // the sum of q, what is left of 1
  __shared__ int s_ids[kIdsMax], s_once[kIdsMax];
  __shared__ float s_q[kIdsMax], s_xk[kIdsMax];
  __shared__ __align__(8) uint64_t s_bar;
  const int cs = NT == kVocThreads ? a.parts : 1, rank = cs > 1 ? (int)cluster_ctarank() : 0;
  const int64_t row = blockIdx.x / cs;
  const RowVecs<DT> rv(static_cast<const T *>(a.x) + row * a.ld, a.V);
  const RowPart<DT> rp(rv, rank, cs);
  const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const float c2 = a.c * kLog2e;
  uint8_t *s_mask = reinterpret_cast<uint8_t *>(s_dyn) + Ahead<NT, 2>::kBytes;  // of vector v0 + i
  if (tid == 0 && cs > 1) {
    mbar_init(&s_bar, 1);
    fence_barrier_init();
    mbar_arrive_expect_tx(&s_bar, (uint32_t)(cs - 1) * 8u);
  }
  __syncwarp();
  if (cs > 1) cluster_announce();
  Ahead<NT, 2> ahead(s_dyn, rp.base + tid, rp.n - tid);
  ahead.start();
  uint4 edge;
  const bool has_edge = (tid == kFirstThread && rp.first) || (tid == last_thread(NT) && rp.last);
  const int edge_v = tid == kFirstThread ? rp.v0 : rp.v1 - 1;
  if (has_edge) edge = rv.edge(edge_v);

  const float w = a.weights ? a.weights[row] : 1.0f;
  T *drow = a.dx ? static_cast<T *>(a.dx) + row * a.ldd : nullptr;
  const bool same = (reinterpret_cast<uintptr_t>(drow) & 15) == (reinterpret_cast<uintptr_t>(rv.row) & 15);

  // The teacher's list is the first warp's: the ids now, the values and their
  // logits asked for before the row's pass and worked on after its share of it.
  bool some = false;
  if (warp == 0) {
    for (int k = lane; k < a.K; k += 32) {
      int id = a.tids[row * a.K + k];
      if (id >= a.V) set_device_error(kDevBadId);
      if (id < 0 || id >= a.V) id = -1;
      some |= id >= 0;
      s_ids[k] = id;
    }
  }
  if constexpr (TAIL) {
    const int nw = (rp.v1 - rp.v0 + 3) / 4;
    for (int i = tid; i < nw; i += NT) reinterpret_cast<uint32_t *>(s_mask)[i] = 0;
  }
  const int any = __syncthreads_or(some);
  const bool skip = !any || w == 0.0f;  // uniform over the cluster
  const int cfirst = max(rv.col(rp.v0), 0), clast = min(rv.col(rp.v1), a.V);
  VStat st{-IG_INF, 0.0f, 0.0f};
  if (!skip) {
    constexpr int kHeld = 2;  // entries per lane in registers
    float held_t[kHeld], held_x[kHeld];
    auto entry = [&](int k, float &t, float &x) {
      const int id = s_ids[k];
      t = id >= 0 ? a.tlogits[row * a.K + k] : -IG_INF;
      x = id >= 0 ? E::get(rv.row[id]) : -IG_INF;
    };
    if (warp == 0) {
#pragma unroll
      for (int j = 0; j < kHeld; j++)
        if (lane + 32 * j < a.K) entry(lane + 32 * j, held_t[j], held_x[j]);
    }
    if constexpr (TAIL) {
      for (int k = tid; k < a.K; k += NT) {
        const int id = s_ids[k];
        int once = id >= 0;  // the first entry with its id
        for (int j = 0; j < k; j++)
          if (s_ids[j] == id) once = 0;
        s_once[k] = once;
        if (id >= cfirst && id < clast) {
          const int at = id + rv.mis - rp.v0 * kN, i = at / kN;
          atomicOr(reinterpret_cast<uint32_t *>(s_mask) + (i >> 2), 1u << ((i & 3) * 8 + at % kN));
        }
      }
      __syncthreads();
    }
    // A vector as the statistics see it: the listed columns are left out of the tail's.
    auto unlisted = [&](uint4 raw, int v) {
      if constexpr (TAIL) {
        const uint32_t m = s_mask[v - rp.v0];
        if (m) {
          float x[kN];
          E::unpack(raw, x);
#pragma unroll
          for (int e = 0; e < kN; e++)
            if (m >> e & 1u) x[e] = -IG_INF;
          raw = E::pack(x);
        }
      }
      return raw;
    };
    ahead.each([&](int b, const uint4(&raw)[kVocUnroll]) {
      const int v = rp.w0 + b + tid;
      if (b + (kVocUnroll - 1) * NT < ahead.mine) {
        uint4 cur[kVocUnroll];
#pragma unroll
        for (int j = 0; j < kVocUnroll; j++) cur[j] = unlisted(raw[j], v + j * NT);
        vstat_add_raw<DT, false>(st, cur, c2);
      } else {
#pragma unroll
        for (int j = 0; j < kVocUnroll; j++)
          if (b + j * NT < ahead.mine) {
            const uint4 one[1] = {unlisted(raw[j], v + j * NT)};
            vstat_add_raw<DT, false>(st, one, c2);
          }
      }
    });
    if (has_edge) {
      const uint4 raw[1] = {unlisted(edge, edge_v)};
      vstat_add_raw<DT, false>(st, raw, c2);
    }
    if (drow) ahead.start();  // the second pass's first vectors
    st = vstat_warp<false>(st, c2);
    if (lane == 0) s_warp[warp] = st;
    if (warp == 0) {
      // s_q: q over the list; s_mass: its sum, and what it leaves of 1.
      float q_sum = 0.0f, q_rest = 0.0f, top = -IG_INF;
      VStat l{-IG_INF, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < kIdsMax / 32; j++) {
        const int k = lane + 32 * j;
        if (k >= a.K) break;
        float t, x;
        if (j < kHeld) {
          t = held_t[j < kHeld ? j : 0];
          x = held_x[j < kHeld ? j : 0];
        } else {
          entry(k, t, x);
        }
        s_xk[k] = x;
        if constexpr (TAIL) {
          const float q = expf(t);  // 0 for a missing entry
          s_q[k] = q;
          q_sum += q;
          // A listed +inf or NaN: no distribution, s is NaN from here on.
          const float one = x == -IG_INF ? 0.0f : (x < IG_INF ? 1.0f : __int_as_float(0x7FC00000));
          if (s_once[k]) vstat_merge<false>(l, VStat{fmaxf(x, -IG_INF), one, 0.0f}, c2);
        } else {
          s_q[k] = t;
          top = max_nan(top, t);
        }
      }
      if constexpr (TAIL) {
        q_sum = warp_sum(q_sum);
        q_rest = q_sum < 1.0f - kRestLeast ? 1.0f - q_sum : (q_sum == q_sum ? 0.0f : q_sum);
        l = vstat_warp<false>(l, c2);
        if (lane == 0) s_list = l;
      } else {
        const float nan = top != top ? top : 0.0f;
        top = warp_max(top);
        for (int k = lane; k < a.K; k += 32) {
          const float e = top == -IG_INF ? 0.0f : expf((s_q[k] - top) * a.c);
          s_q[k] = e;
          q_sum += e;
        }
        q_sum = warp_sum(q_sum + nan);
        const float inv = q_sum > 0.0f || q_sum != q_sum ? 1.0f / q_sum : 0.0f;
        for (int k = lane; k < a.K; k += 32) s_q[k] *= inv;
        q_sum = q_sum > 0.0f ? 1.0f : q_sum;
      }
      if (lane == 0) {
        s_mass[0] = q_sum;
        s_mass[1] = q_rest;
      }
    }
    __syncthreads();
    st = vstat_join<false>(s_warp, NT / 32, c2);
  }
  if (cs > 1) {
    // Every CTA hands its statistics to every other one. (Each has its list's
    // logits in s_xk by then, so the others may overwrite the row: dx may be x.)
    cluster_ready();
    if (tid < cs) {
      if (tid == rank) {
        s_part[rank] = st;
      } else {
        st_async_f32(&s_part[rank].m, tid, st.m, &s_bar);
        st_async_f32(&s_part[rank].s, tid, st.s, &s_bar);
      }
    }
    mbar_wait_cluster(&s_bar, 0, kDevTimeoutFull);
    __syncthreads();
    st = vstat_join<false>(s_part, cs, c2);
  }
  // Dense gradient: coef 2^((x - mb) c2 - l2); a listed column: listed p - w c q.
  float coef = 0.0f, listed = 0.0f;
  float mb = 0.0f, l2 = 0.0f;
  float row_m = 0.0f, row_l2 = 0.0f;  // p = 2^((x - row_m) c2 - row_l2)
  bool zero = true;
  if (!skip) {
    VStat all = st;
    const float q_sum = s_mass[0], q_rest = s_mass[1];
    if constexpr (TAIL) vstat_merge<false>(all, s_list, c2);
    const float log_s = logf(all.s);
    float mass = q_sum + q_rest, rest = 0.0f, tail_loss = 0.0f;
    bool far = false;
    if constexpr (TAIL) {
      if (st.s == 0.0f) {
        // Nothing outside the list: what is left of 1 is rounding.
        mass = q_sum;
      } else if (q_rest > 0.0f || q_rest != q_rest) {
        const float logr = (st.m - all.m) * a.c + logf(st.s) - log_s;
        tail_loss = q_rest * (logf(q_rest) - logr);
        // A tail of less than e^-60: p and q_rest / p_rest would leave the
        // float range. Its columns then take q_rest times their share of the
        // tail alone (p itself adds less than e^-60 / q_rest of that).
        far = logr < -60.0f;
        rest = q_rest * ex2(-logr * kLog2e);
      }
    }
    if (rank == 0 && warp == 0) {
      float loss = 0.0f;
      for (int k = lane; k < a.K; k += 32) {
        const float q = s_q[k];
        if (q > 0.0f || q != q) loss += q * (logf(q) - (all.s == 0.0f ? -IG_INF : (s_xk[k] - all.m) * a.c - log_s));
      }
      loss = warp_sum(loss) + tail_loss;
      if (all.s != all.s) loss = all.s;
      if (lane == 0) a.loss[row] = loss * w;
    }
    zero = all.s == 0.0f;
    listed = w * a.c * mass;
    row_m = zero ? 0.0f : all.m;
    row_l2 = log_s * kLog2e;
    coef = far ? -w * a.c * q_rest : w * a.c * (mass - rest);
    mb = far ? st.m : all.m;
    l2 = far ? logf(st.s) * kLog2e : row_l2;
  } else if (rank == 0 && tid == 0) {
    a.loss[row] = 0.0f;
  }
  if (!drow) {
    cp_async_wait_all();
    return;
  }
  if (cs == 1) __syncthreads();  // the list's logits are read before any store: dx may be x
  const float2 nm = make_float2(-mb, -mb), cc = make_float2(c2, c2), nl = make_float2(-l2, -l2);
  auto grad = [&](const uint4 &v, float *d) {
    float x[kN];
    E::unpack(v, x);
#pragma unroll
    for (int e = 0; e < kN; e += 2) {
      const float2 y = __ffma2_rn(__fadd2_rn(make_float2(x[e], x[e + 1]), nm), cc, nl);
      const float2 r = __fmul2_rn(make_float2(ex2(y.x), ex2(y.y)), make_float2(coef, coef));
      d[e] = r.x;
      d[e + 1] = r.y;
    }
  };
  T *dp = drow + rv.col(rp.w0) + (int64_t)tid * kN;
  if (zero) {
    cp_async_wait_all();
    float d[kN] = {};
    for (int i = 0; i < ahead.mine; i += NT) store_whole<DT>(dp + (int64_t)i * kN, same, d);
    if (has_edge) store_edge<DT>(drow, rv, edge_v, d);
  } else {
    ahead.each([&](int b, const uint4(&raw)[kVocUnroll]) {
#pragma unroll
      for (int j = 0; j < kVocUnroll; j++) {
        if (b + j * NT >= ahead.mine) break;
        float d[kN];
        grad(raw[j], d);
        store_whole<DT>(dp + (int64_t)(b + j * NT) * kN, same, d);
      }
    });
    if (has_edge) {
      float d[kN];
      grad(edge, d);
      store_edge<DT>(drow, rv, edge_v, d);
    }
  }
  if (zero) return;
  __syncthreads();
  // The listed columns of this CTA's part; q of equal ids adds up (each of
  // their threads stores the same value).
  for (int i = tid; i < a.K; i += NT) {
    const int id = s_ids[i];
    if (id < cfirst || id >= clast) continue;
    float q = 0.0f;
    for (int k = 0; k < a.K; k++)
      if (s_ids[k] == id) q += s_q[k];
    drow[id] = E::put(listed * ex2((s_xk[i] - row_m) * c2 - row_l2) - w * a.c * q);
  }
}

// ---- launches --------------------------------------------------------------------------

// Threads per CTA and CTAs per row (a cluster).
struct RowShape {
  int threads, parts;
};
// again: the row's vectors are read a second time, so the rows on the way have
// to stay near L2 (126 MB): 1024 x 262144 float32 with 20 alternatives takes
// 282 us with 310 MB of rows on the way, 227 with 78; 4096 x 50021 float32
// 188 with 118 MB and 223 with 59, where the clusters only cost.
static RowShape row_shape(int64_t rows, int64_t nv, bool again) {
  RowShape r{kVocThreads, 1};
  // Many short rows: small CTAs, so that an SM has more rows on the way (a
  // row's start and end cost as much as 16 vectors per thread), while the
  // rows' threads fill the GPU.
  while (r.threads > 32 && nv <= 8 * r.threads && rows * (r.threads / 2) >= num_sms() * 1024) r.threads /= 2;
  // Few rows: several CTAs each, of a round of vectors at least.
  while (r.threads == kVocThreads && r.parts < 8 && rows * r.parts < 2 * 4 * num_sms() &&
         nv / (2 * r.parts) >= kVocThreads)
    r.parts *= 2;
  while (again && r.threads == kVocThreads && r.parts < 8 && nv * 16 * (4 * num_sms() / r.parts) > (140ll << 20))
    r.parts *= 2;
  return r;
}

// The tail's marks, a byte per vector of a CTA's part: at most this many, with
// which two CTAs of 256 threads share an SM beside their slots. With a gradient
// the rule above leaves less in any case; for the loss alone the marks of a
// whole row of 2^20 float32 columns are more than an SM has. Loss of 1184 rows,
// one CTA each and by this rule: 450000 float32 columns (112 KB of marks) 386
// and 332 us, 600000 (150 KB) 502 and 430; below it the clusters only cost
// (262144 bf16 columns, 32 KB: 104 us, and 126 in two parts).
constexpr int64_t kMarkBytes = 74 << 10;

template <typename Args>
static cudaError_t launch_rows(void (*kern)(Args), const Args &a, int64_t ctas, int threads, int cs, size_t smem,
                               cudaStream_t st, SmemOptIn &attr) {
  const cudaError_t e = attr.ensure((const void *)kern, (int)smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  if (cs > 1) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cs;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, kern, a);
}

#define IG_BY_THREADS(n, CALL) \
  ((n) == 256 ? CALL(256) : (n) == 128 ? CALL(128) : (n) == 64 ? CALL(64) : CALL(32))

template <int DT, bool TOP, int NT>
static cudaError_t launch_logprobs(const LogprobArgs &a, int64_t ctas, cudaStream_t st) {
  static SmemOptIn attr;
  return launch_rows(token_logprobs_kernel<DT, TOP, NT>, a, ctas, NT, a.parts, Ahead<NT>::kBytes, st, attr);
}

template <int DT>
static cudaError_t run_token_logprobs(LogprobArgs a, cudaStream_t st) {
  const RowShape r = row_shape(a.rows, a.V / VElem<DT>::kN, a.K > 0);
  a.parts = r.parts;
  const int64_t ctas = a.rows * r.parts;
#define IG_CALL(NT) (a.K > 0 ? launch_logprobs<DT, true, NT>(a, ctas, st) : launch_logprobs<DT, false, NT>(a, ctas, st))
  return IG_BY_THREADS(r.threads, IG_CALL);
#undef IG_CALL
}

template <int DT, int NT>
static cudaError_t launch_grad(const LogprobGradArgs &a, int64_t ctas, cudaStream_t st) {
  static SmemOptIn attr;
  return launch_rows(token_logprobs_grad_kernel<DT, NT>, a, ctas, NT, 1, Ahead<NT>::kBytes, st, attr);
}

template <int DT>
static cudaError_t run_token_logprobs_grad(LogprobGradArgs a, cudaStream_t st) {
  const int64_t nv = (a.V + VElem<DT>::kN - 1) / VElem<DT>::kN + 1;  // a row off the boundary spans one more
  const int nt = row_shape(a.rows, a.V / VElem<DT>::kN, false).threads;
  const int64_t rounds = (nv + kVocUnroll * nt - 1) / (kVocUnroll * nt);
  // Several rounds per CTA (a CTA's start costs about as much as a round)
  // while there are CTAs enough to fill the GPU four times.
  int64_t per = rounds;
  while (per > 1 && a.rows * ((rounds + per - 1) / per) * nt < 4 * 1024 * num_sms()) per = (per + 1) / 2;
  a.segs = (int)((rounds + per - 1) / per);
  const int64_t ctas = a.rows * a.segs;
  if (ctas > INT32_MAX) return cudaErrorInvalidConfiguration;
#define IG_CALL(NT) launch_grad<DT, NT>(a, ctas, st)
  return IG_BY_THREADS(nt, IG_CALL);
#undef IG_CALL
}

template <int DT, bool TAIL, int NT>
static cudaError_t launch_distill(const DistillArgs &a, size_t smem, cudaStream_t st) {
  static SmemOptIn attr;
  return launch_rows(distill_topk_kernel<DT, TAIL, NT>, a, a.rows * a.parts, NT, a.parts, Ahead<NT, 2>::kBytes + smem, st,
                     attr);
}

template <int DT>
static cudaError_t run_distill(DistillArgs a, bool tail, cudaStream_t st) {
  const int64_t nv = a.V / VElem<DT>::kN + 2;
  RowShape r = row_shape(a.rows, a.V / VElem<DT>::kN, a.dx != nullptr);
  while (tail && r.threads == kVocThreads && r.parts < 8 && nv / r.parts > kMarkBytes) r.parts *= 2;
  a.parts = r.parts;
  const size_t smem = tail ? ((nv / r.parts + 1) / 4 + 1) * 4 : 0;
#define IG_CALL(NT) (tail ? launch_distill<DT, true, NT>(a, smem, st) : launch_distill<DT, false, NT>(a, smem, st))
  return IG_BY_THREADS(r.threads, IG_CALL);
#undef IG_CALL
}

}  // namespace ig
