// Layer norm of rows of float32, bfloat16 or float16 and its backward pass.
//
//   y = (x - mean) rstd w + b,   rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   dx = rstd (g - mean(g) - xh mean(g xh)),  g = dy w,  xh = (x - mean) rstd
//   dw = sum over rows dy xh,    db = sum over rows dy
//
// Both are bound by memory: a row is read once into registers, its statistics
// are formed there (the variance from the centred values, so that rows far from
// zero keep their digits), and it is written once. Statistics and sums are
// float32; results are rounded once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "internal.h"
#include "train.h"

namespace ig {

template <int DT>
constexpr int ln_size() {
  return DT == IG_DT_F32 ? 4 : 2;
}

// V neighbouring elements of type DT as one load or store.
template <int DT, int V>
struct LnPack {
  static constexpr int kBytes = V * ln_size<DT>();
  using T = std::conditional_t<
      kBytes == 16, uint4,
      std::conditional_t<kBytes == 8, uint2, std::conditional_t<kBytes == 4, uint32_t, uint16_t>>>;
  static_assert(kBytes == 16 || kBytes == 8 || kBytes == 4 || kBytes == 2, "one access");
  union {
    T t;
    uint32_t w[kBytes >= 4 ? kBytes / 4 : 1];
  };
  __device__ __forceinline__ LnPack() {}
  __device__ __forceinline__ void load(const void *row, int i) {
    t = *reinterpret_cast<const T *>(static_cast<const uint8_t *>(row) + (int64_t)i * ln_size<DT>());
  }
  __device__ __forceinline__ void store(void *row, int i) const {
    *reinterpret_cast<T *>(static_cast<uint8_t *>(row) + (int64_t)i * ln_size<DT>()) = t;
  }
  __device__ __forceinline__ void get(float *v) const {
    if constexpr (DT == IG_DT_F32) {
#pragma unroll
      for (int k = 0; k < V; k++) v[k] = __uint_as_float(w[k]);
    } else if constexpr (V == 1) {
      v[0] = DT == IG_DT_BF16 ? __uint_as_float((uint32_t)t << 16) : __half2float(__ushort_as_half((unsigned short)t));
    } else {
#pragma unroll
      for (int k = 0; k < V / 2; k++) {
        if constexpr (DT == IG_DT_BF16) {
          v[2 * k] = __uint_as_float(w[k] << 16);
          v[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[k]));
          v[2 * k] = f.x;
          v[2 * k + 1] = f.y;
        }
      }
    }
  }
  __device__ __forceinline__ void set(const float *v) {
    if constexpr (DT == IG_DT_F32) {
#pragma unroll
      for (int k = 0; k < V; k++) w[k] = __float_as_uint(v[k]);
    } else if constexpr (V == 1) {
      t = DT == IG_DT_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v[0])) : __half_as_ushort(__float2half_rn(v[0]));
    } else {
#pragma unroll
      for (int k = 0; k < V / 2; k++) {
        if constexpr (DT == IG_DT_BF16) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
          w[k] = *reinterpret_cast<const uint32_t *>(&h);
        } else {
          const __half2 h = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
          w[k] = *reinterpret_cast<const uint32_t *>(&h);
        }
      }
    }
  }
};

// V elements of the weight or bias (any of the three types); `none` where there is no such vector.
template <int V>
__device__ __forceinline__ void ln_weight(const void *p, int dtype, int i, float none, float *v) {
  if (!p) {
#pragma unroll
    for (int k = 0; k < V; k++) v[k] = none;
  } else if (dtype == IG_DT_F32) {
    constexpr int V4 = V < 4 ? V : 4;
#pragma unroll
    for (int k = 0; k < V; k += V4) {
      LnPack<IG_DT_F32, V4> q;
      q.load(p, i + k);
      q.get(v + k);
    }
  } else if (dtype == IG_DT_BF16) {
    LnPack<IG_DT_BF16, V> q;
    q.load(p, i);
    q.get(v);
  } else {
    LnPack<IG_DT_F16, V> q;
    q.load(p, i);
    q.get(v);
  }
}

__device__ __forceinline__ float ln_warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}
// Sum over the T threads of a row: of a warp, or of the whole CTA.
template <int T>
__device__ __forceinline__ float ln_sum(float v, float *s) {
  v = ln_warp_sum(v);
  if constexpr (T == 32) return v;
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < T / 32 ? s[threadIdx.x & 31] : 0.0f;
  return ln_warp_sum(v);
}

__device__ __forceinline__ float2 ln_both(float v) { return make_float2(v, v); }
// V elements (V even, or one beside a 0) as pairs, for half the instructions.
template <int V>
struct LnPairs {
  static constexpr int H = (V + 1) / 2;
  float2 p[H];
  template <typename P>
  __device__ __forceinline__ void get(const P &q) {
    float v[2 * H];
    v[2 * H - 1] = 0.0f;
    q.get(v);
#pragma unroll
    for (int h = 0; h < H; h++) p[h] = make_float2(v[2 * h], v[2 * h + 1]);
  }
  template <typename P>
  __device__ __forceinline__ void put(P &q) const {
    float v[2 * H];
#pragma unroll
    for (int h = 0; h < H; h++) v[2 * h] = p[h].x, v[2 * h + 1] = p[h].y;
    q.set(v);
  }
  __device__ __forceinline__ void weight(const void *w, int dtype, int i, float none) {
    float v[2 * H];
    v[2 * H - 1] = 0.0f;
    ln_weight<V>(w, dtype, i, none, v);
#pragma unroll
    for (int h = 0; h < H; h++) p[h] = make_float2(v[2 * h], v[2 * h + 1]);
  }
};

// NV sums over the warp at once (NV a power of two up to 32): after log2(NV)
// exchanges each lane holds one of them, the index in the lane's upper bits.
template <int NV>
__device__ __forceinline__ float ln_warp_sums(float *v, int lane) {
  int o = 16;
#pragma unroll
  for (int m = NV / 2; m; m >>= 1, o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < m; i++) {
      const float send = up ? v[i] : v[i + m], keep = up ? v[i + m] : v[i];
      v[i] = keep + __shfl_xor_sync(~0u, send, o);
    }
  }
  float r = v[0];
  for (; o; o >>= 1) r += __shfl_xor_sync(~0u, r, o);
  return r;
}
// The sums of R rows over the T threads of each, R > 1 for a warp only.
template <int T, int R>
__device__ __forceinline__ void ln_sums(float (&v)[R], float *s) {
  if constexpr (R == 1) {
    v[0] = ln_sum<T>(v[0], s);
  } else {
    static_assert(T == 32, "several rows to a warp");
    const float one = ln_warp_sums<R>(v, threadIdx.x & 31);
#pragma unroll
    for (int r = 0; r < R; r++) v[r] = __shfl_sync(~0u, one, r * (32 / R));
  }
}

// T threads a row, KV elements of it each: a warp for rows of up to 1024, so
// that no barrier is needed; four warps to a CTA then, R rows of each in flight
// before the first is worked on. Rows past the last are the last again, unused.
template <int TX, int TY, int V, int T, int KV, int R>
__global__ void __launch_bounds__(T < 128 ? 128 : T) ln_fwd_kernel(const LnArgs a) {
  constexpr int K = KV / V, H = LnPairs<V>::H;
  __shared__ float s_sum[2][32];
  dep_wait();
  dep_trigger();
  const int t = T == 32 ? (int)(threadIdx.x & 31) : (int)threadIdx.x;
  const int64_t row0 = T == 32 ? ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 5)) * R : (int64_t)blockIdx.x;
  if (row0 >= a.rows) return;
  const int left = a.rows - row0 < R ? (int)(a.rows - row0) : R;
  LnPack<TX, V> in[R][K];
#pragma unroll
  for (int r = 0; r < R; r++) {
    const uint8_t *x = static_cast<const uint8_t *>(a.x) + (row0 + (r < left ? r : left - 1)) * a.ldx * ln_size<TX>();
#pragma unroll
    for (int k = 0; k < K; k++)
      if ((k * T + t) * V < a.n) in[r][k].load(x, (k * T + t) * V);
  }
  const float inv_n = 1.0f / (float)a.n;
  float mean[R], rstd[R];
#pragma unroll
  for (int r = 0; r < R; r++) {
    float2 s = ln_both(0.0f);
#pragma unroll
    for (int k = 0; k < K; k++) {
      if ((k * T + t) * V < a.n) {
        LnPairs<V> v;
        v.get(in[r][k]);
#pragma unroll
        for (int h = 0; h < H; h++) s = __fadd2_rn(s, v.p[h]);
      }
    }
    mean[r] = s.x + s.y;
  }
  ln_sums<T, R>(mean, s_sum[0]);
#pragma unroll
  for (int r = 0; r < R; r++) {
    mean[r] *= inv_n;
    float2 q = ln_both(0.0f);
#pragma unroll
    for (int k = 0; k < K; k++) {
      if ((k * T + t) * V < a.n) {
        LnPairs<V> v;
        v.get(in[r][k]);
#pragma unroll
        for (int h = 0; h < H; h++) {
          float2 d = __fadd2_rn(v.p[h], ln_both(-mean[r]));
          if (V == 1) d.y = 0.0f;
          q = __ffma2_rn(d, d, q);
        }
      }
    }
    rstd[r] = q.x + q.y;
  }
  ln_sums<T, R>(rstd, s_sum[1]);
#pragma unroll
  for (int r = 0; r < R; r++) {
    rstd[r] = rsqrtf(fmaf(rstd[r], inv_n, a.eps));
    if (t == 0 && r < left) {
      if (a.mean) a.mean[row0 + r] = mean[r];
      if (a.rstd) a.rstd[row0 + r] = rstd[r];
    }
  }
  uint8_t *y = static_cast<uint8_t *>(a.y) + row0 * a.ldy * ln_size<TY>();
#pragma unroll
  for (int k = 0; k < K; k++) {
    const int i = (k * T + t) * V;
    if (i < a.n) {
      LnPairs<V> w, b;
      w.weight(a.w, a.wdt, i, 1.0f);
      b.weight(a.b, a.wdt, i, 0.0f);
#pragma unroll
      for (int r = 0; r < R; r++) {
        if (r < left) {
          LnPairs<V> v;
          v.get(in[r][k]);
#pragma unroll
          for (int h = 0; h < H; h++)
            v.p[h] = __ffma2_rn(__fmul2_rn(__fadd2_rn(v.p[h], ln_both(-mean[r])), ln_both(rstd[r])), w.p[h], b.p[h]);
          LnPack<TY, V> out;
          v.put(out);
          out.store(y + r * a.ldy * ln_size<TY>(), i);
        }
      }
    }
  }
}

// Rows longer than the registers of a CTA: three reads, the later two from L2.
template <int TX, int TY>
__global__ void __launch_bounds__(1024) ln_fwd_long_kernel(const LnArgs a) {
  __shared__ float s_sum[2][32];
  dep_wait();
  dep_trigger();
  const int64_t row = blockIdx.x;
  const uint8_t *x = static_cast<const uint8_t *>(a.x) + row * a.ldx * ln_size<TX>();
  uint8_t *y = static_cast<uint8_t *>(a.y) + row * a.ldy * ln_size<TY>();
  auto at = [&](int i) {
    LnPack<TX, 1> p;
    float v;
    p.load(x, i);
    p.get(&v);
    return v;
  };
  float s = 0.0f, q = 0.0f;
  for (int i = threadIdx.x; i < a.n; i += 1024) s += at(i);
  const float inv_n = 1.0f / (float)a.n, mean = ln_sum<1024>(s, s_sum[0]) * inv_n;
  for (int i = threadIdx.x; i < a.n; i += 1024) {
    const float d = at(i) - mean;
    q = fmaf(d, d, q);
  }
  const float rstd = rsqrtf(fmaf(ln_sum<1024>(q, s_sum[1]), inv_n, a.eps));
  if (threadIdx.x == 0) {
    if (a.mean) a.mean[row] = mean;
    if (a.rstd) a.rstd[row] = rstd;
  }
  for (int i = threadIdx.x; i < a.n; i += 1024) {
    float w, b, o;
    ln_weight<1>(a.w, a.wdt, i, 1.0f, &w);
    ln_weight<1>(a.b, a.wdt, i, 0.0f, &b);
    o = fmaf((at(i) - mean) * rstd, w, b);
    LnPack<TY, 1> out;
    out.set(&o);
    out.store(y, i);
  }
}

// Copies rows on 16-byte boundaries into shared memory, counted on `bar`.
__device__ __forceinline__ void ln_bulk(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
constexpr int kLnRingMost = 8;    // rows of a group on their way
constexpr int kLnGroupsMost = 20; // rows side by side in a CTA

// A row takes T threads with KV elements each (a warp up to 1024, so that the
// exchange of the row's two sums costs 1 instruction in 8), and every thread
// holds the sums of dw and db for its own columns over all rows that come its
// way (persistent CTAs). BULK: the next a.ring rows of every group are on their
// way into shared memory, by one copy each of x and dy. Without, for rows off
// 16-byte boundaries: one row ahead in registers.
// 16384 x 768 bf16: 21 us; 25 with 96 threads a row and 8 elements each, 37 with
// the rows copied 16 bytes a thread (cp.async).
template <int TX, int TY, int V, int KV, int MAXT, bool BULK>
__global__ void __launch_bounds__(MAXT) ln_bwd_kernel(const LnGradArgs a) {
  constexpr int K = KV / V, H = KV / 2;
  using PX = LnPack<TX, V>;
  using PD = LnPack<TY, V>;
  __shared__ float2 s_part[2][32];
  __shared__ uint64_t s_bar[BULK ? kLnGroupsMost * kLnRingMost : 1];
  extern __shared__ __align__(16) uint8_t ln_dyn[];
  if constexpr (BULK) {
    for (int i = threadIdx.x; i < a.G * a.ring; i += blockDim.x) mbar_init(&s_bar[i], 1);
    fence_barrier_init();
    __syncthreads();
  }
  dep_wait();
  const int T = a.T, g = (int)threadIdx.x / T, t = (int)threadIdx.x - g * T, lane = threadIdx.x & 31;
  const int warps = T / 32, warp0 = g * warps, warp = (int)threadIdx.x >> 5;
  const float inv_n = 1.0f / (float)a.n;
  float2 w[H], dw[H], db[H];  // pairs of the thread's elements
  auto pairs = [](const float (&v)[KV], float2 (&p)[H]) {
#pragma unroll
    for (int h = 0; h < H; h++) p[h] = make_float2(v[2 * h], v[2 * h + 1]);
  };
  // Whether piece k lies in the row: all but the last two do, for the KV that the row's length asks for.
  auto on = [&](int k) { return (k * T + t) * V < a.n; };
  const int64_t step = (int64_t)gridDim.x * a.G, first = (int64_t)blockIdx.x * a.G + g;
  const int64_t sx = a.ldx * ln_size<TX>(), sd = a.lddy * ln_size<TY>(), so = a.lddx * ln_size<TX>();
  const uint8_t *px = static_cast<const uint8_t *>(a.x) + first * sx + t * V * ln_size<TX>(),
                *pd = static_cast<const uint8_t *>(a.dy) + first * sd + t * V * ln_size<TY>();
  uint8_t *po = static_cast<uint8_t *>(a.dx) + first * so + t * V * ln_size<TX>();
  const int kx = T * V * ln_size<TX>(), kd = T * V * ln_size<TY>();  // from one of a thread's pieces to the next
  [[maybe_unused]] PX rx[BULK ? 1 : K];
  [[maybe_unused]] PD rd[BULK ? 1 : K];
  // A group's rows on their way: x, then dy.
  const uint32_t bx = a.n * ln_size<TX>(), bd = a.n * ln_size<TY>();
  uint8_t *const ring = ln_dyn + (size_t)g * a.ring * (bx + bd);
  uint64_t *const bars = s_bar + (BULK ? g * a.ring : 0);
  int64_t asked = first;  // the row that px and pd stand at
  auto ask = [&]([[maybe_unused]] int stage) {
    if constexpr (BULK) {
      if (t == 0 && asked < a.rows) {
        uint8_t *to = ring + stage * (bx + bd);
        mbar_arrive_expect_tx(&bars[stage], bx + bd);
        ln_bulk(to, px, bx, &bars[stage]);
        ln_bulk(to + bx, pd, bd, &bars[stage]);
      }
    } else if (asked < a.rows) {
#pragma unroll
      for (int k = 0; k < K; k++) {
        if (on(k)) {
          rx[k].load(px + k * kx, 0);
          rd[k].load(pd + k * kd, 0);
        }
      }
    }
    asked += step;
    px += step * sx;
    pd += step * sd;
  };
  if constexpr (BULK) {
    for (int i = 0; i < a.ring; i++) ask(i);
  } else {
    ask(0);
  }
  {
    float v[KV];
#pragma unroll
    for (int k = 0; k < K; k++) {
      if (on(k)) {
        ln_weight<V>(a.w, a.wdt, (k * T + t) * V, 1.0f, v + k * V);
      } else {
#pragma unroll
        for (int j = 0; j < V; j++) v[k * V + j] = 0.0f;
      }
    }
    pairs(v, w);
  }
#pragma unroll
  for (int h = 0; h < H; h++) dw[h] = db[h] = ln_both(0.0f);

  float mean = 0.0f, rstd = 0.0f;
  if (first < a.rows) mean = a.mean[first], rstd = a.rstd[first];
  int par = 0;
  [[maybe_unused]] int stage = 0;
  [[maybe_unused]] uint32_t phase = 0;
  bool ok = true;
  for (int64_t row = first; row < a.rows; row += step, par ^= 1) {
    if constexpr (BULK) ok = ok && mbar_wait(&bars[stage], phase, kDevTimeoutFull);
    float2 xh[H], gw[H], s1 = ln_both(0.0f), s2 = s1;
    {
      float xs[KV], ds[KV];
#pragma unroll
      for (int k = 0; k < K; k++) {
        if (on(k)) {
          if constexpr (BULK) {
            const uint8_t *from = ring + stage * (bx + bd);
            PX x;
            PD d;
            x.load(from, (k * T + t) * V);
            d.load(from + bx, (k * T + t) * V);
            x.get(xs + k * V);
            d.get(ds + k * V);
          } else {
            rx[k].get(xs + k * V);
            rd[k].get(ds + k * V);
          }
        } else {
#pragma unroll
          for (int j = 0; j < V; j++) xs[k * V + j] = ds[k * V + j] = 0.0f;
        }
      }
      pairs(xs, xh);
      pairs(ds, gw);
    }
    const float scale = rstd;
#pragma unroll
    for (int h = 0; h < H; h++) {
      const float2 d = gw[h];
      xh[h] = __fmul2_rn(__fadd2_rn(xh[h], ln_both(-mean)), ln_both(scale));
      gw[h] = __fmul2_rn(d, w[h]);
      s1 = __fadd2_rn(s1, gw[h]);
      s2 = __ffma2_rn(gw[h], xh[h], s2);
      dw[h] = __ffma2_rn(d, xh[h], dw[h]);
      db[h] = __fadd2_rn(db[h], d);
    }
    if constexpr (!BULK) ask(0);
    if (row + step < a.rows) mean = a.mean[row + step], rstd = a.rstd[row + step];
    float v[2] = {s1.x + s1.y, s2.x + s2.y};
    float one = ln_warp_sums<2>(v, lane);  // the first in lanes 0 to 15, the second in 16 to 31
    float c1 = __shfl_sync(~0u, one, 0), c2 = __shfl_sync(~0u, one, 16);
    if (warps > 1) {
      if (lane == 0) s_part[par][warp] = make_float2(c1, c2);
      named_barrier_sync(1 + g, T);
      // The other parity is written next: nobody is two barriers ahead.
      const float2 q = lane < warps ? s_part[par][warp0 + lane] : make_float2(0.0f, 0.0f);
      v[0] = q.x, v[1] = q.y;
      one = ln_warp_sums<2>(v, lane);
      c1 = __shfl_sync(~0u, one, 0), c2 = __shfl_sync(~0u, one, 16);
    }
    // Every thread of the group has read its elements: by the exchange, or by the barrier.
    if constexpr (BULK) {
      if (ok) ask(stage);
      if (++stage == a.ring) stage = 0, phase ^= 1;
    }
    c1 *= -inv_n;
    c2 *= -inv_n;
    {
      float o[KV];
#pragma unroll
      for (int h = 0; h < H; h++) {
        const float2 d = __fmul2_rn(__ffma2_rn(xh[h], ln_both(c2), __fadd2_rn(gw[h], ln_both(c1))), ln_both(scale));
        o[2 * h] = d.x;
        o[2 * h + 1] = d.y;
      }
#pragma unroll
      for (int k = 0; k < K; k++) {
        if (on(k)) {
          PX q;
          q.set(o + k * V);
          q.store(po + k * kx, 0);
        }
      }
    }
    po += step * so;
  }
  if constexpr (BULK) {
    // A wait was given up (and the rows after it were not waited for, so that the barriers above stay in step): what was
    // asked for may still be on its way into this CTA's memory.
    if (!ok && t == 0)
      for (int i = 0; i < a.ring; i++) mbar_wait(&bars[i], phase, kDevTimeoutFull);
  }
  dep_trigger();
  if (!a.part) return;
  // The groups' sums, side by side in the memory that the rows came through, are added in their order.
  float *s_cols = reinterpret_cast<float *>(ln_dyn);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; k++) {
    if (on(k)) {
      float *to = s_cols + (size_t)g * 2 * a.n + (k * T + t) * V;
#pragma unroll
      for (int j = 0; j < V; j += V < 4 ? 1 : 4) {
        const int h = (k * V + j) / 2;
        if constexpr (V >= 4) {
          *reinterpret_cast<float4 *>(to + j) = make_float4(dw[h].x, dw[h].y, dw[h + 1].x, dw[h + 1].y);
          *reinterpret_cast<float4 *>(to + a.n + j) = make_float4(db[h].x, db[h].y, db[h + 1].x, db[h + 1].y);
        } else {
          to[0] = k & 1 ? dw[h].y : dw[h].x;
          to[a.n] = k & 1 ? db[h].y : db[h].x;
        }
      }
    }
  }
  __syncthreads();
  float *part = a.part + (int64_t)blockIdx.x * 2 * a.n;
  for (int c = threadIdx.x; c < 2 * a.n; c += blockDim.x) {
    float v = s_cols[c];
    for (int i = 1; i < a.G; i++) v += s_cols[(size_t)i * 2 * a.n + c];
    part[c] = v;
  }
}

// Rows longer than the registers of a CTA: x and dy are read twice (the second
// time from L2), and the CTA's sums for dw and db stay in its part of the
// workspace.
template <int TX, int TY>
__global__ void __launch_bounds__(1024) ln_bwd_long_kernel(const LnGradArgs a) {
  __shared__ float s_sum[2][2][32];
  dep_wait();
  const float inv_n = 1.0f / (float)a.n;
  int par = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, par ^= 1) {
    const uint8_t *px = static_cast<const uint8_t *>(a.x) + row * a.ldx * ln_size<TX>();
    const uint8_t *pd = static_cast<const uint8_t *>(a.dy) + row * a.lddy * ln_size<TY>();
    uint8_t *out = static_cast<uint8_t *>(a.dx) + row * a.lddx * ln_size<TX>();
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    auto at = [&](int i, float &xh, float &d, float &w) {
      LnPack<TX, 1> p;
      LnPack<TY, 1> q;
      float x;
      p.load(px, i);
      q.load(pd, i);
      p.get(&x);
      q.get(&d);
      xh = (x - mean) * rstd;
      ln_weight<1>(a.w, a.wdt, i, 1.0f, &w);
    };
    for (int i = threadIdx.x; i < a.n; i += 1024) {
      float xh, d, w;
      at(i, xh, d, w);
      s1 = fmaf(d, w, s1);
      s2 = fmaf(d * w, xh, s2);
    }
    const float c1 = ln_sum<1024>(s1, s_sum[par][0]) * inv_n, c2 = ln_sum<1024>(s2, s_sum[par][1]) * inv_n;
    for (int i = threadIdx.x; i < a.n; i += 1024) {
      float xh, d, w;
      at(i, xh, d, w);
      const float o = rstd * (fmaf(d, w, -c1) - xh * c2);
      LnPack<TX, 1> q;
      q.set(&o);
      q.store(out, i);
      if (a.part) {
        float *p = a.part + (int64_t)blockIdx.x * 2 * a.n + i;
        const bool first = row == blockIdx.x;
        p[0] = fmaf(d, xh, first ? 0.0f : p[0]);
        p[a.n] = d + (first ? 0.0f : p[a.n]);
      }
    }
  }
}

// dw and db: the CTAs' sums, 32 columns to a CTA, each of its warps every 32nd
// part; then the warps' sums in their order.
__global__ void __launch_bounds__(1024) ln_sum_kernel(const float *part, int parts, int n, void *dw, void *db, int dtype) {
  __shared__ float s[2][32][33];
  dep_wait();
  dep_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float x = 0.0f, y = 0.0f;
  if (c < n) {
#pragma unroll 4
    for (int p = warp; p < parts; p += 32) {
      x += part[(int64_t)p * 2 * n + c];
      y += part[(int64_t)p * 2 * n + n + c];
    }
  }
  s[0][warp][lane] = x;
  s[1][warp][lane] = y;
  __syncthreads();
  if (warp < 2) {
    float v = 0.0f;
#pragma unroll
    for (int k = 0; k < 32; k++) v += s[warp][k][lane];
    void *out = warp ? db : dw;
    if (out && c < n) {
      if (dtype == IG_DT_F32)
        static_cast<float *>(out)[c] = v;
      else if (dtype == IG_DT_BF16)
        static_cast<__nv_bfloat16 *>(out)[c] = __float2bfloat16_rn(v);
      else
        static_cast<__half *>(out)[c] = __float2half_rn(v);
    }
  }
}

// ---- launches ----------------------------------------------------------------------------

// Whether V elements at a time fall on the boundaries of one access.
static bool ln_on(const void *p, int64_t ld, int64_t rows, int bytes, int es) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && (rows <= 1 || ld * es % bytes == 0);
}
static bool ln_weight_on(const void *p, int dtype, int V) {
  const int bytes = dtype == IG_DT_F32 ? 16 : 2 * V;
  return reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

constexpr int kLnLong = 16384;  // longer rows are read more than once

template <int TX, int TY, int V, int KV, int R>
static cudaError_t ln_fwd_warps(const LnArgs &a, cudaStream_t st) {
  // Several rows to a warp once every SM has its warps (16 an SM).
  if (a.rows >= (int64_t)16 * R * device_sms())
    return launch_dep(ln_fwd_kernel<TX, TY, V, 32, KV, R>, dim3((unsigned)((a.rows + 4 * R - 1) / (4 * R))), dim3(128), 0, st, a);
  return launch_dep(ln_fwd_kernel<TX, TY, V, 32, KV, 1>, dim3((unsigned)((a.rows + 3) / 4)), dim3(128), 0, st, a);
}
template <int TX, int TY, int V>
static cudaError_t ln_fwd(const LnArgs &a, cudaStream_t st) {
  const dim3 rows((unsigned)a.rows);
  if (a.n <= 256) return ln_fwd_warps<TX, TY, V, 8, 4>(a, st);
  if (a.n <= 512) return ln_fwd_warps<TX, TY, V, 16, V == 8 ? 4 : 2>(a, st);
  if (a.n <= 768) return ln_fwd_warps<TX, TY, V, 24, 2>(a, st);
  if (a.n <= 1024) return ln_fwd_warps<TX, TY, V, 32, 2>(a, st);
  if (a.n <= 2048) return launch_dep(ln_fwd_kernel<TX, TY, V, 128, 16, 1>, rows, dim3(128), 0, st, a);
  if (a.n <= 4096) return launch_dep(ln_fwd_kernel<TX, TY, V, 128, 32, 1>, rows, dim3(128), 0, st, a);
  if (a.n <= 8192) return launch_dep(ln_fwd_kernel<TX, TY, V, 512, 16, 1>, rows, dim3(512), 0, st, a);
  return launch_dep(ln_fwd_kernel<TX, TY, V, 512, 32, 1>, rows, dim3(512), 0, st, a);
}

template <int TX, int TY>
static cudaError_t run_layer_norm(const LnArgs &a, cudaStream_t st) {
  constexpr int V = TX == IG_DT_F32 ? 4 : 8;
  if (a.n > kLnLong) return launch_dep(ln_fwd_long_kernel<TX, TY>, dim3((unsigned)a.rows), dim3(1024), 0, st, a);
  const bool wide = a.n % V == 0 && ln_on(a.x, a.ldx, a.rows, V * ln_size<TX>(), ln_size<TX>()) &&
                    ln_on(a.y, a.ldy, a.rows, V * ln_size<TY>(), ln_size<TY>()) && ln_weight_on(a.w, a.wdt, V) &&
                    ln_weight_on(a.b, a.wdt, V);
  return wide ? ln_fwd<TX, TY, V>(a, st) : ln_fwd<TX, TY, 1>(a, st);
}

// The backward pass's shape: elements a thread holds, threads a row (whole
// warps), rows side by side in a CTA, and CTAs.
constexpr int kLnGradLong = 8192;  // longer rows are read twice there
struct LnPlan {
  int KV, T, G;
  int64_t ctas;
};
// Threads of a CTA that have the registers for KV elements each (sums, weights and two values of each).
static constexpr int ln_most_threads(int KV) { return KV == 8 ? 640 : KV == 16 ? 512 : KV == 24 ? 384 : 256; }
static LnPlan ln_plan(int64_t rows, int n, bool wide) {
  LnPlan p{};
  if (n > kLnGradLong) {
    p.ctas = rows < device_sms() ? rows : device_sms();
    return p;
  }
  p.KV = !wide || n <= 256 ? 8 : n <= 512 ? 16 : n <= 768 ? 24 : 32;
  p.T = ((n + p.KV - 1) / p.KV + 31) / 32 * 32;
  p.G = std::max(1, std::min(ln_most_threads(p.KV) / p.T, p.T == 32 ? kLnGroupsMost : 15));  // a named barrier each
  const int64_t want = (rows + p.G - 1) / p.G, most = device_sms();
  p.ctas = want < most ? want : most;
  return p;
}

template <int TX, int TY, int V, int KV, int MAXT>
static cudaError_t ln_bwd_launch(LnGradArgs a, const LnPlan &p, cudaStream_t st) {
  const size_t round = (size_t)p.G * a.n * (ln_size<TX>() + ln_size<TY>());
  a.ring = V == 1 ? 0 : (int)std::max<size_t>(1, std::min<size_t>(kLnRingMost, 200 * 1024 / round));
  const size_t smem = std::max(a.ring * round, a.part ? (size_t)p.G * 2 * a.n * 4 : 0);
  static SmemOptIn attr;
  const auto kernel = ln_bwd_kernel<TX, TY, V, KV, MAXT, V != 1>;
  const cudaError_t e = smem > 32 * 1024 ? attr.ensure((const void *)kernel, (int)smem) : cudaSuccess;
  return e != cudaSuccess ? e : launch_dep(kernel, dim3((unsigned)p.ctas), dim3(p.T * p.G), smem, st, a);
}
template <int TX, int TY, int V>
static cudaError_t ln_bwd(const LnGradArgs &a, const LnPlan &p, cudaStream_t st) {
  if constexpr (V == 1)
    return p.T > ln_most_threads(8) ? ln_bwd_launch<TX, TY, V, 8, 1024>(a, p, st) : ln_bwd_launch<TX, TY, V, 8, ln_most_threads(8)>(a, p, st);
  else
    return p.KV == 8    ? ln_bwd_launch<TX, TY, V, 8, ln_most_threads(8)>(a, p, st)
           : p.KV == 16 ? ln_bwd_launch<TX, TY, V, 16, ln_most_threads(16)>(a, p, st)
           : p.KV == 24 ? ln_bwd_launch<TX, TY, V, 24, ln_most_threads(24)>(a, p, st)
                        : ln_bwd_launch<TX, TY, V, 32, ln_most_threads(32)>(a, p, st);
}

// Whether all rows lie on 16-byte boundaries, and the weight on those of V elements.
template <int TX, int TY, int V>
static bool ln_grad_wide(const LnGradArgs &a) {
  return a.n * ln_size<TX>() % 16 == 0 && a.n * ln_size<TY>() % 16 == 0 && ln_on(a.x, a.ldx, a.rows, 16, ln_size<TX>()) &&
         ln_on(a.dx, a.lddx, a.rows, 16, ln_size<TX>()) && ln_on(a.dy, a.lddy, a.rows, 16, ln_size<TY>()) &&
         ln_weight_on(a.w, a.wdt, V);
}
template <int TX, int TY>
static cudaError_t run_layer_norm_grad(LnGradArgs a, void *dw, void *db, cudaStream_t st) {
  constexpr int V = TX == IG_DT_F32 ? 4 : 8;
  const bool wide = ln_grad_wide<TX, TY, V>(a);
  const LnPlan p = ln_plan(a.rows, a.n, wide);
  a.T = p.T;
  a.G = p.G;
  cudaError_t e;
  if (a.n > kLnGradLong)
    e = launch_dep(ln_bwd_long_kernel<TX, TY>, dim3((unsigned)p.ctas), dim3(1024), 0, st, a);
  else
    e = wide ? ln_bwd<TX, TY, V>(a, p, st) : ln_bwd<TX, TY, 1>(a, p, st);
  if (e != cudaSuccess || !a.part) return e;
  return launch_dep(ln_sum_kernel, dim3((unsigned)((a.n + 31) / 32)), dim3(1024), 0, st, (const float *)a.part, (int)p.ctas, a.n,
                    dw, db, a.wdt);
}

// Types of x and of the result (and its gradient): the same, or float32 in and 16 bits out.
template <typename F>
static cudaError_t ln_types(int tx, int ty, F f) {
  using std::integral_constant;
  constexpr integral_constant<int, IG_DT_F32> f32{};
  constexpr integral_constant<int, IG_DT_BF16> bf16{};
  constexpr integral_constant<int, IG_DT_F16> f16{};
  if (tx == IG_DT_F32) return ty == IG_DT_F32 ? f(f32, f32) : ty == IG_DT_BF16 ? f(f32, bf16) : f(f32, f16);
  return tx == IG_DT_BF16 ? f(bf16, bf16) : f(f16, f16);
}

cudaError_t launch_layer_norm(const LnArgs &a, int tx, int ty, cudaStream_t st) {
  return ln_types(tx, ty, [&](auto x, auto y) { return run_layer_norm<decltype(x)::value, decltype(y)::value>(a, st); });
}

// A CTA an SM at most, whatever the shape.
int64_t layer_norm_workspace(int64_t rows, int n) {
  return std::min<int64_t>(rows, device_sms()) * 2 * n * (int64_t)sizeof(float);
}

cudaError_t launch_layer_norm_grad(const LnGradArgs &a, int tx, int ty, void *dw, void *db, cudaStream_t st) {
  return ln_types(tx, ty, [&](auto x, auto y) {
    return run_layer_norm_grad<decltype(x)::value, decltype(y)::value>(a, dw, db, st);
  });
}

}  // namespace ig
