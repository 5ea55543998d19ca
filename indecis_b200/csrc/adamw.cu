// One AdamW step over many tensors, moments in float32 or in 8 bits.
//
//   t = steps taken + 1,  g = gradient (times grad_scale)
//   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2
//   p = p (1 - lr decay) - lr (m / (1 - b1^t)) / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound by memory: every element of the parameter, gradient and moments is read
// once and written once. The tensors' addresses travel as kernel arguments (up
// to 32,764 bytes), so a step is one small launch that counts it and one that
// does it, whatever the number of tensors up to kAdamwMost, and nothing is
// copied to the device first.
//
// A warp takes 256 elements at a time, as two runs of 32 x 4: 16-byte accesses
// of float32, 8 of 16 bits, 4 of 8 bits, each of them whole lines of the warp.
//
// 8-bit moments: m and r = sqrt(v) as e4m3 (4 exponent, 3 fraction bits) times
// a float32 scale for each 256 elements, the largest of them at 448. The root,
// as its codes then span 2^-17.8 of the block's largest gradient instead of
// 2^-8.9. Rounding to the nearest would leave a moment where it is whenever a
// step changes it by less than half a unit (b2 = 0.999 changes r by 0.05%, a
// unit is 6 to 12%), so a value goes up to the next code where the fraction cut
// off and u reach 1; u = frac(i phi + t psi) fills [0, 1) evenly over the steps
// t (an additive recurrence, Weyl), so the codes follow the value in the mean
// with neither a generator's state nor a seed. In 64 bits, 2000 steps after
// gradients fall to a tenth of what they were: rounded to the nearest r is 3.8
// times what it should be, with random u 1.00 +- 0.31, with this u 0.92 +- 0.08;
// 3500 steps later 9.3, 1.01 +- 0.13 and 0.96 +- 0.04. r > 0 is never stored as 0: with
// eps alone below it a later update would be without measure.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "internal.h"
#include "train.h"

namespace ig {

constexpr int kAdamwBlock = 256;
constexpr int kAdamwFew = 40;     // tensors of the smaller argument list (3 KB)
constexpr int kAdamwMost = 400;   // of the larger one (31 KB)
constexpr int kAdamwWarps = 8;
constexpr int kAdamwRun = 16;     // blocks of 256 that a warp takes from one tensor at most

template <int NT>
struct AdamwList {
  AdamwTensor t[NT];
  uint32_t first[NT + 1];  // runs of blocks before each tensor
  int count, run;          // tensors, blocks of a run (a warp's at a time)
};

// The step is counted before it is made, so that every launch of a step reads the same number.
__global__ void adamw_count_kernel(int32_t *step, const float *skip) {
  dep_wait();
  dep_trigger();
  if (!skip || *skip == 0.0f) *step += 1;
}

// b^t by squaring, in double: 1 - b^t loses nothing that float32 would show.
__device__ __forceinline__ double adamw_pow(double b, int t) {
  double r = 1.0;
  for (; t > 0; t >>= 1, b *= b)
    if (t & 1) r *= b;
  return r;
}

constexpr uint32_t kWeylI = 0x9E3779B9u;                        // 2^32 / the golden ratio
constexpr uint32_t kWeylM = 0xC13FA9A9u, kWeylV = 0x91E10DA5u;  // 2^32 / the plastic number, and its square

template <int TYPE>
constexpr int adamw_size() {
  return TYPE == IG_DT_F32 ? 4 : 2;
}
// Four elements of a type.
template <int TYPE>
__device__ __forceinline__ void adamw_load4(const uint8_t *p, float (&v)[4]) {
  if constexpr (TYPE == IG_DT_F32) {
    const float4 x = *reinterpret_cast<const float4 *>(p);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
  } else {
    const uint2 x = *reinterpret_cast<const uint2 *>(p);
    if constexpr (TYPE == IG_DT_BF16) {
      v[0] = __uint_as_float(x.x << 16), v[1] = __uint_as_float(x.x & 0xFFFF0000u);
      v[2] = __uint_as_float(x.y << 16), v[3] = __uint_as_float(x.y & 0xFFFF0000u);
    } else {
      const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&x.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&x.y));
      v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
    }
  }
}
template <int TYPE>
__device__ __forceinline__ void adamw_store4(uint8_t *p, const float (&v)[4]) {
  if constexpr (TYPE == IG_DT_F32) {
    *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else if constexpr (TYPE == IG_DT_BF16) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
  } else {
    const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
  }
}
// Single elements, for tensors off the boundaries of four and for their ends.
__device__ __forceinline__ float adamw_load1(const void *p, int type, int64_t i) {
  if (type == IG_DT_F32) return static_cast<const float *>(p)[i];
  const uint16_t h = static_cast<const uint16_t *>(p)[i];
  return type == IG_DT_BF16 ? __uint_as_float((uint32_t)h << 16) : __half2float(__ushort_as_half(h));
}
__device__ __forceinline__ void adamw_store1(void *p, int type, int64_t i, float v) {
  if (type == IG_DT_F32)
    static_cast<float *>(p)[i] = v;
  else
    static_cast<uint16_t *>(p)[i] = type == IG_DT_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
// e4m3 codes.
__device__ __forceinline__ void adamw_decode(uint32_t x, float (&v)[4]) {
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(x >> (16 * k)), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
    v[2 * k] = f.x;
    v[2 * k + 1] = f.y;
  }
}
// Values past 448 become it (a value of 448 and its rounding).
__device__ __forceinline__ uint32_t adamw_encode(const float (&v)[4]) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[0], v[1]), __NV_SATFINITE, __NV_E4M3) |
         (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[2], v[3]), __NV_SATFINITE, __NV_E4M3) << 16;
}

__device__ __forceinline__ float adamw_finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.0f;
}
__device__ __forceinline__ float adamw_warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  return v;
}
// 1 / scale, or 0 for a block whose values are all below 448e-32 (stored as 0).
__device__ __forceinline__ float adamw_inverse(float scale) { return scale > 1e-32f ? __frcp_rn(scale) : 0.0f; }

// Products of two elements that are rounded before they are added to anything:
// a packed product and a packed sum are joined into one operation whatever
// rounding they ask for, so the product is itself one, with a -0 that the
// compiler does not know (an argument).
__device__ __forceinline__ float2 adamw_mul(float2 a, float2 b, float zero) { return __ffma2_rn(a, b, make_float2(zero, zero)); }

// Four values x as codes' values x / scale, up where the fraction cut off and u
// (the upper 20 bits of k) reach 1. e4m3 has the leading fraction bits of
// float32, so for its normal values u is added to the 20 bits that are cut;
// below 2^-6, in units of 2^-9, the sum is cut by an addition that rounds down.
// What is not finite becomes NaN. All of it is integer, exact or IEEE
// arithmetic: the codes are a function of x, scale and u alone.
template <bool ROOT>
__device__ __forceinline__ void adamw_codes(float (&x)[4], float inv, uint32_t k) {
  uint32_t y[4], far = 0;
#pragma unroll
  for (int j = 0; j < 4; j += 2) {
    const float2 q = __fmul2_rn(make_float2(x[j], x[j + 1]), make_float2(inv, inv));
    y[j] = __float_as_uint(q.x);
    y[j + 1] = __float_as_uint(q.y);
  }
#pragma unroll
  for (int j = 0; j < 4; j++) far = max(far, 2 * y[j] - 2 * 0x3C800000u);  // |y| from 2^-6
  if (far < 2 * (0x44000000u - 0x3C800000u)) {                              // to 512
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = __uint_as_float((y[j] + (k + j * kWeylI >> 12)) & 0xFFF00000u);
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const uint32_t u = k + j * kWeylI >> 12, a = y[j] & 0x7FFFFFFFu;
    float c = __uint_as_float((a + u) & 0xFFF00000u);
    if (a < 0x3C800000u) {
      const float s = __fadd_rn(__uint_as_float(a), (float)u * 0x1p-29f);
      c = __fadd_rd(s, 16384.0f) - 16384.0f;
    }
    if (ROOT && x[j] > 0.0f) c = fmaxf(c, 0x1p-9f);
    x[j] = fabsf(x[j]) <= 3.402823466e38f ? copysignf(c, x[j]) : __uint_as_float(0x7FC00000u);
  }
}

// Square roots: s = v y of an approximate y = 1 / sqrt(v), and Newton's step on
// v - s^2, which one multiply-add forms exactly, with y for the slope (Markstein,
// 1990). From v = 2^-102 on they are those to the nearest (compared for every
// float), so that codes of a root are those of its definition; below, where v -
// s^2 is rounded, the last place may be another. 0, infinities and NaN make s a
// NaN, and denormal v too: there the approximate root does. 312 million
// parameters in 8 bits: 1,018 us; 995 with the approximate root, off by 2^-23,
// everywhere, which moved one code in 3.2 million and with it the next step;
// 1,125 with the function for the root to the nearest. 200 million: 559 us, 643
// where all roots are 0 (549 and 598 with the approximate root).
__device__ __forceinline__ float2 adamw_root(float2 v) {
  float2 y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(v.x));
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(v.y));
  const float2 s = __fmul2_rn(v, y), d = __ffma2_rn(make_float2(-s.x, -s.y), s, v);
  float2 r = __ffma2_rn(d, __fmul2_rn(y, make_float2(0.5f, 0.5f)), s);
  const float any = r.x + r.y;
  if (any != any) {
    float2 q;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(q.x) : "f"(v.x));
    asm("sqrt.approx.f32 %0, %1;" : "=f"(q.y) : "f"(v.y));
    r = make_float2(r.x == r.x ? r.x : q.x, r.y == r.y ? r.y : q.y);
  }
  return r;
}

// What a step needs beside the tensors.
struct AdamwNow {
  float c1, c2, gs;  // -lr / (1 - b1^t), 1 / sqrt(1 - b2^t), the gradients' factor
  uint32_t wm, wv;   // the sequences' places at step t
};
// Two elements' moments (v as its root for 8 bits) and parameters: every
// product and sum of the moments rounded by itself, as the definition has it.
// decay is -lr times the tensor's. It joins the update before that meets p: 1 -
// lr decay is off by up to 2^-25 in float32, to the same side for every element
// and step (1e-5 times 0.01: 19% more decay, 1e-6 times 0.01: none).
template <bool BITS8>
__device__ __forceinline__ void adamw_two(float2 &p, float2 g, float2 &m, float2 &v, float ms, float vs, float decay, const AdamwArgs &a,
                                          const AdamwNow &n) {
  auto both = [](float x) { return make_float2(x, x); };
  g = __fmul2_rn(g, both(n.gs));
  if constexpr (BITS8) {
    m = __fmul2_rn(m, both(ms));
    v = __fmul2_rn(v, both(vs));
    v = __fmul2_rn(v, v);
  }
  m = __fadd2_rn(adamw_mul(m, both(a.b1), a.zero), adamw_mul(g, both(a.ob1), a.zero));
  v = __fadd2_rn(adamw_mul(v, both(a.b2), a.zero), adamw_mul(__fmul2_rn(g, g), both(a.ob2), a.zero));
  const float2 r = adamw_root(v);
  float2 q;
  const float2 d = __ffma2_rn(r, both(n.c2), both(a.eps));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q.x) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q.y) : "f"(d.y));
  p = __fadd2_rn(p, __ffma2_rn(p, both(decay), __fmul2_rn(__fmul2_rn(m, both(n.c1)), q)));
  if constexpr (BITS8) v = r;
}
template <bool BITS8>
__device__ __forceinline__ void adamw_one(float &p, float g, float &m, float &v, float ms, float vs, float decay, const AdamwArgs &a,
                                          const AdamwNow &n) {
  float2 p2 = make_float2(p, 0.0f), m2 = make_float2(m, 0.0f), v2 = make_float2(v, 0.0f);
  adamw_two<BITS8>(p2, make_float2(g, 0.0f), m2, v2, ms, vs, decay, a, n);
  p = p2.x;
  m = m2.x;
  v = v2.x;
}

// Whole blocks of 256 elements on boundaries of four, `count` of them from
// `block` on: the addresses are formed once and move on by constants (with one
// block at a time they took half of the instructions).
template <bool BITS8, int PT, int GT>
__device__ __forceinline__ void adamw_blocks(const AdamwTensor &t, uint32_t block, int count, int lane, const AdamwArgs &a,
                                             const AdamwNow &n) {
  constexpr int kM = BITS8 ? 1 : 4, kP = adamw_size<PT>(), kG = adamw_size<GT>();
  const int64_t i0 = (int64_t)block * kAdamwBlock + 4 * lane;
  uint8_t *p_at = static_cast<uint8_t *>(t.p) + i0 * kP, *m_at = static_cast<uint8_t *>(t.m) + i0 * kM,
          *v_at = static_cast<uint8_t *>(t.v) + i0 * kM, *c_at = static_cast<uint8_t *>(t.copy) + (t.copy ? i0 * 2 : 0);
  const uint8_t *g_at = static_cast<const uint8_t *>(t.g) + i0 * kG;
  [[maybe_unused]] float *ms_at = t.ms + (BITS8 ? block : 0), *vs_at = t.vs + (BITS8 ? block : 0);
  const float decay = -a.lr * t.decay;
  const bool copy16 = t.ct == IG_DT_BF16;
  uint32_t place = (uint32_t)i0 * kWeylI;
#pragma unroll 1
  for (; count > 0; count--) {
    float p[2][4], g[2][4], m[2][4], v[2][4], ms = 1.0f, vs = 1.0f, top_m = 0.0f, top_r = 0.0f;
    [[maybe_unused]] uint32_t mc[2], vc[2];
#pragma unroll
    for (int q = 0; q < 2; q++) {
      adamw_load4<GT>(g_at + 128 * q * kG, g[q]);
      if constexpr (BITS8) {
        mc[q] = *reinterpret_cast<const uint32_t *>(m_at + 128 * q);
        vc[q] = *reinterpret_cast<const uint32_t *>(v_at + 128 * q);
      } else {
        adamw_load4<IG_DT_F32>(m_at + 512 * q, m[q]);
        adamw_load4<IG_DT_F32>(v_at + 512 * q, v[q]);
      }
      adamw_load4<PT>(p_at + 128 * q * kP, p[q]);
    }
    if constexpr (BITS8) {
      ms = *ms_at;
      vs = *vs_at;
#pragma unroll
      for (int q = 0; q < 2; q++) {
        adamw_decode(mc[q], m[q]);
        adamw_decode(vc[q], v[q]);
      }
    }
#pragma unroll
    for (int q = 0; q < 2; q++) {
#pragma unroll
      for (int k = 0; k < 4; k += 2) {
        float2 p2 = make_float2(p[q][k], p[q][k + 1]), m2 = make_float2(m[q][k], m[q][k + 1]), v2 = make_float2(v[q][k], v[q][k + 1]);
        adamw_two<BITS8>(p2, make_float2(g[q][k], g[q][k + 1]), m2, v2, ms, vs, decay, a, n);
        p[q][k] = p2.x, p[q][k + 1] = p2.y;
        m[q][k] = m2.x, m[q][k + 1] = m2.y;
        v[q][k] = v2.x, v[q][k + 1] = v2.y;
        if constexpr (BITS8) {
          top_m = fmaxf(top_m, fmaxf(fabsf(m2.x), fabsf(m2.y)));
          top_r = fmaxf(top_r, fmaxf(v2.x, v2.y));
        }
      }
      adamw_store4<PT>(p_at + 128 * q * kP, p[q]);
      if (t.copy) {
        if (copy16)
          adamw_store4<IG_DT_BF16>(c_at + 256 * q, p[q]);
        else
          adamw_store4<IG_DT_F16>(c_at + 256 * q, p[q]);
      }
      if constexpr (!BITS8) {
        adamw_store4<IG_DT_F32>(m_at + 512 * q, m[q]);
        adamw_store4<IG_DT_F32>(v_at + 512 * q, v[q]);
      }
    }
    if constexpr (BITS8) {
      top_m = adamw_warp_max(top_m);
      top_r = adamw_warp_max(top_r);
      if (!(top_m <= 3.402823466e38f && top_r <= 3.402823466e38f)) {  // infinities do not count
        top_m = top_r = 0.0f;
#pragma unroll
        for (int q = 0; q < 2; q++) {
#pragma unroll
          for (int k = 0; k < 4; k++) {
            top_m = fmaxf(top_m, adamw_finite_abs(m[q][k]));
            top_r = fmaxf(top_r, adamw_finite_abs(v[q][k]));
          }
        }
        top_m = adamw_warp_max(top_m);
        top_r = adamw_warp_max(top_r);
      }
      ms = __fmul_rn(top_m, 1.0f / 448.0f);
      vs = __fmul_rn(top_r, 1.0f / 448.0f);
      const float im = adamw_inverse(ms), iv = adamw_inverse(vs);
      if (lane == 0) {
        *ms_at = ms;
        *vs_at = vs;
      }
#pragma unroll
      for (int q = 0; q < 2; q++) {
        adamw_codes<false>(m[q], im, place + 128u * q * kWeylI + n.wm);
        adamw_codes<true>(v[q], iv, place + 128u * q * kWeylI + n.wv);
        *reinterpret_cast<uint32_t *>(m_at + 128 * q) = adamw_encode(m[q]);
        *reinterpret_cast<uint32_t *>(v_at + 128 * q) = adamw_encode(v[q]);
      }
      ms_at++;
      vs_at++;
      place += kAdamwBlock * kWeylI;
    }
    p_at += kAdamwBlock * kP;
    g_at += kAdamwBlock * kG;
    m_at += kAdamwBlock * kM;
    v_at += kAdamwBlock * kM;
    c_at += kAdamwBlock * 2;
  }
}

// Any other block: element by element, the same arithmetic.
template <bool BITS8>
__device__ __noinline__ void adamw_ragged(const AdamwTensor &t, uint32_t block, int lane, const AdamwArgs &a, const AdamwNow &n) {
  const int64_t i0 = (int64_t)block * kAdamwBlock + 4 * lane;
  float m[2][4], v[2][4], ms = 1.0f, vs = 1.0f, top_m = 0.0f, top_r = 0.0f;
  if constexpr (BITS8) {
    ms = t.ms[block];
    vs = t.vs[block];
  }
  const float decay = -a.lr * t.decay;
#pragma unroll
  for (int q = 0; q < 2; q++) {
    const int64_t i = i0 + 128 * q;
    if constexpr (BITS8) {
      uint32_t x = 0, y = 0;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        if (i + k < t.n) {
          x |= (uint32_t) static_cast<const uint8_t *>(t.m)[i + k] << (8 * k);
          y |= (uint32_t) static_cast<const uint8_t *>(t.v)[i + k] << (8 * k);
        }
      }
      adamw_decode(x, m[q]);
      adamw_decode(y, v[q]);
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
      if (i + k < t.n) {
        if constexpr (!BITS8) {
          m[q][k] = static_cast<const float *>(t.m)[i + k];
          v[q][k] = static_cast<const float *>(t.v)[i + k];
        }
        float p = adamw_load1(t.p, t.pt, i + k);
        adamw_one<BITS8>(p, adamw_load1(t.g, t.gt, i + k), m[q][k], v[q][k], ms, vs, decay, a, n);
        adamw_store1(t.p, t.pt, i + k, p);
        if (t.copy) adamw_store1(t.copy, t.ct, i + k, p);
        if constexpr (!BITS8) {
          static_cast<float *>(t.m)[i + k] = m[q][k];
          static_cast<float *>(t.v)[i + k] = v[q][k];
        }
      } else {
        m[q][k] = v[q][k] = 0.0f;
      }
      top_m = fmaxf(top_m, adamw_finite_abs(m[q][k]));
      top_r = fmaxf(top_r, adamw_finite_abs(v[q][k]));
    }
  }
  if constexpr (BITS8) {
    ms = __fmul_rn(adamw_warp_max(top_m), 1.0f / 448.0f);
    vs = __fmul_rn(adamw_warp_max(top_r), 1.0f / 448.0f);
    const float im = adamw_inverse(ms), iv = adamw_inverse(vs);
    if (lane == 0) {
      t.ms[block] = ms;
      t.vs[block] = vs;
    }
#pragma unroll
    for (int q = 0; q < 2; q++) {
      const int64_t i = i0 + 128 * q;
      const uint32_t k0 = (uint32_t)i * kWeylI;
      adamw_codes<false>(m[q], im, k0 + n.wm);
      adamw_codes<true>(v[q], iv, k0 + n.wv);
      const uint32_t x = adamw_encode(m[q]), y = adamw_encode(v[q]);
#pragma unroll
      for (int k = 0; k < 4; k++) {
        if (i + k < t.n) {
          static_cast<uint8_t *>(t.m)[i + k] = (uint8_t)(x >> (8 * k));
          static_cast<uint8_t *>(t.v)[i + k] = (uint8_t)(y >> (8 * k));
        }
      }
    }
  }
}

template <int NT, bool BITS8>
__global__ void __launch_bounds__(32 * kAdamwWarps, 3) adamw_kernel(const __grid_constant__ AdamwList<NT> list, const AdamwArgs a) {
  __shared__ float s_inv[2];
  __shared__ int s_step;
  dep_wait();
  dep_trigger();
  if (a.skip && *a.skip != 0.0f) return;
  if (threadIdx.x == 0) {
    const int t = *a.step;
    s_step = t;
    s_inv[0] = (float)(1.0 / (1.0 - adamw_pow(a.db1, t)));
    s_inv[1] = (float)(1.0 / sqrt(1.0 - adamw_pow(a.db2, t)));
  }
  __syncthreads();
  const AdamwNow now{-a.lr * s_inv[0], s_inv[1], a.grad_scale ? *a.grad_scale : 1.0f, (uint32_t)s_step * kWeylM, (uint32_t)s_step * kWeylV};
  const int lane = threadIdx.x & 31;
  const uint32_t runs = list.first[list.count];
  int ti = 0;
  uint32_t next = list.first[1];
  for (uint64_t u = (uint64_t)blockIdx.x * kAdamwWarps + (threadIdx.x >> 5); u < runs; u += (uint64_t)gridDim.x * kAdamwWarps) {
    if (u >= next) {
      int lo = ti + 1, hi = list.count - 1;  // the last tensor that starts at or before u
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (list.first[mid] <= u)
          lo = mid;
        else
          hi = mid - 1;
      }
      ti = lo;
      next = list.first[ti + 1];
    }
    const AdamwTensor &t = list.t[ti];
    const uint32_t block = ((uint32_t)u - list.first[ti]) * list.run;
    const int64_t whole_all = t.wide ? t.n / kAdamwBlock : 0, all = (t.n + kAdamwBlock - 1) / kAdamwBlock;
    const int count = (int)(all - block < list.run ? all - block : list.run);
    const int whole = whole_all <= block ? 0 : (int)(whole_all - block < count ? whole_all - block : count);
    auto go = [&](auto pt) {
      constexpr int PT = decltype(pt)::value;
      if (t.gt == IG_DT_F32)
        adamw_blocks<BITS8, PT, IG_DT_F32>(t, block, whole, lane, a, now);
      else if (t.gt == IG_DT_BF16)
        adamw_blocks<BITS8, PT, IG_DT_BF16>(t, block, whole, lane, a, now);
      else
        adamw_blocks<BITS8, PT, IG_DT_F16>(t, block, whole, lane, a, now);
    };
    if (t.pt == IG_DT_F32)
      go(std::integral_constant<int, IG_DT_F32>());
    else if (t.pt == IG_DT_BF16)
      go(std::integral_constant<int, IG_DT_BF16>());
    else
      go(std::integral_constant<int, IG_DT_F16>());
    for (int i = whole; i < count; i++) adamw_ragged<BITS8>(t, block + i, lane, a, now);
  }
}

template <int NT, bool BITS8>
static cudaError_t launch_adamw_list(const AdamwTensor *t, int count, const AdamwArgs &a, cudaStream_t st) {
  static PerDevice resident;
  const int ctas = resident.get([] {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, adamw_kernel<NT, BITS8>, 32 * kAdamwWarps, 0) != cudaSuccess || n < 1) {
      (void)cudaGetLastError();
      n = 1;
    }
    return n * device_sms();
  });
  AdamwList<NT> list;
  list.count = count;
  int64_t blocks = 0;
  for (int i = 0; i < count; i++) blocks += (t[i].n + kAdamwBlock - 1) / kAdamwBlock;
  // Long runs where every warp has several of them all the same.
  list.run = (int)std::max<int64_t>(1, std::min<int64_t>(kAdamwRun, blocks / ((int64_t)ctas * kAdamwWarps * 4)));
  uint32_t runs = 0;
  for (int i = 0; i < count; i++) {
    list.t[i] = t[i];
    list.first[i] = runs;
    runs += (uint32_t)(((t[i].n + kAdamwBlock - 1) / kAdamwBlock + list.run - 1) / list.run);
  }
  list.first[count] = runs;
  const int64_t want = ((int64_t)runs + kAdamwWarps - 1) / kAdamwWarps;
  return launch_dep(adamw_kernel<NT, BITS8>, dim3((unsigned)(want < ctas ? want : ctas)), dim3(32 * kAdamwWarps), 0, st, list, a);
}

// Tensors of at least one element each; a launch's blocks fit 32 bits.
cudaError_t launch_adamw(const AdamwTensor *t, int count, const AdamwArgs &a, bool bits8, cudaStream_t st) {
  cudaError_t e = launch_dep(adamw_count_kernel, dim3(1), dim3(1), 0, st, a.step, a.skip);
  for (int at = 0; at < count && e == cudaSuccess;) {
    int n = 0;
    uint64_t blocks = 0;
    for (; at + n < count && n < kAdamwMost; n++) {
      blocks += (uint64_t)((t[at + n].n + kAdamwBlock - 1) / kAdamwBlock);
      if (blocks > 0xFFFFFFFFull) break;
    }
    if (n <= kAdamwFew)
      e = bits8 ? launch_adamw_list<kAdamwFew, true>(t + at, n, a, st) : launch_adamw_list<kAdamwFew, false>(t + at, n, a, st);
    else
      e = bits8 ? launch_adamw_list<kAdamwMost, true>(t + at, n, a, st) : launch_adamw_list<kAdamwMost, false>(t + at, n, a, st);
    at += n;
  }
  return e;
}

}  // namespace ig
