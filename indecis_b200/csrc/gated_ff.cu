// The gated feed-forward block on bfloat16 or float16 rows, and its backward pass:
//
//   [a | b] = x Wi^T  (Wi [2I][H], the activated rows first),  h = act(a) b,  y = h Wo^T
//   dh = dy Wo,  da = dh b act'(a),  db = dh act(a)
//   dx = [da | db] Wi,  dWi = [da | db]^T x,  dWo = dy^T h
//
// All products run on the tensor cores (tcgen05 kind::f16, float32 accumulators
// in TMEM) in one persistent kernel with three epilogues. For h a tile holds the
// same columns of a and b, whose weight rows come as two TMA boxes, so that the
// activation and the product meet in the epilogue's registers and neither a nor
// b is stored for answers. [da | db] are made from dh's accumulators the same
// way. The plain products take a list of problems: dx, dWi and dWo are one
// launch whose tiles fill the GPU together, and those with few tiles are split
// over K with float32 partial sums that a second launch adds in order.
//
// h and [da | db] are held in the operands' type, which the tensor cores need:
// the only rounding in between, of the size of the results' own, so that those
// are off by 1.4 times what one rounding gives. For the backward pass a and b
// are kept in float32: in 16 bits their rounding would enter da twice (through
// b and act') and the error would be 2 times. float16 keeps values up to 65504
// in between, and needs the usual loss scale for small gradients.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "internal.h"

namespace ig {

enum FfEpi : int { kFfForward = 0, kFfGrad = 1, kFfProduct = 2 };

// ---- activations, two elements at a time --------------------------------------------------

__device__ __forceinline__ float2 ff_ex2(float2 v) {
  float2 r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(v.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(v.y));
  return r;
}
__device__ __forceinline__ float2 ff_rcp(float2 v) {
  float2 r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(v.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(v.y));
  return r;
}
__device__ __forceinline__ float2 ff_mul(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 ff_fma(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 ff_both(float v) { return make_float2(v, v); }

// act(a), and act'(a) where it is wanted.
template <int ACT, bool GRAD>
__device__ __forceinline__ void ff_act(float2 a, float2 &f, [[maybe_unused]] float2 &df) {
  if constexpr (ACT == IG_ACT_GELU) {
    // a P(a), P the normal distribution. P(-x) = exp(-x^2 / 2) R(x), R a polynomial in t = 1 / (1 + p x), fitted for the
    // smallest largest relative error on [0, 14] (4.2e-6, 4.4e-6 with its float32 roundings; past that exp is 0). The
    // exponent's rounding comes to that, 3 half steps of it or 9e-8 x^2 at most: with an exact exponential P is off by
    // 4.5e-6 up to x = 2, 5.3e-6 up to 6, 7.0e-6 up to 8 and 9.6e-6 up to 13. The exponential is the density's too, so
    // the derivative P + a exp(-a^2 / 2) / sqrt(2 pi) costs two operations.
    const float2 x = make_float2(fabsf(a.x), fabsf(a.y));
    const float2 t = ff_rcp(ff_fma(x, ff_both(0.3075f), ff_both(1.0f)));
    float2 q = ff_fma(t, ff_both(-0.07553954422473907f), ff_both(0.1911918967962265f));
    q = ff_fma(t, q, ff_both(0.005902447737753391f));
    q = ff_fma(t, q, ff_both(0.13693517446517944f));
    q = ff_fma(t, q, ff_both(0.11857893317937851f));
    q = ff_fma(t, q, ff_both(0.12293054908514023f));
    const float2 e = ff_ex2(ff_mul(ff_mul(a, ff_both(-0.72134752044448170f)), a));
    q = ff_mul(ff_mul(q, t), e);
    const float2 p = make_float2(a.x >= 0.0f ? 1.0f - q.x : q.x, a.y >= 0.0f ? 1.0f - q.y : q.y);
    f = ff_mul(a, p);
    if constexpr (GRAD) df = ff_fma(ff_mul(a, ff_both(0.39894228040143268f)), e, p);
  } else if constexpr (ACT == IG_ACT_GELU_TANH) {
    // (1 + tanh u) / 2 = 1 / (1 + exp(-2 u)), u = k (a + c a^3).
    constexpr float k = 0.79788456080286536f, c = 0.044715f, log2e = 1.4426950408889634f;
    const float2 a2 = ff_mul(a, a);
    const float2 s = ff_rcp(__fadd2_rn(ff_ex2(ff_mul(a, ff_fma(a2, ff_both(-2 * k * c * log2e), ff_both(-2 * k * log2e)))), ff_both(1.0f)));
    f = ff_mul(a, s);
    if constexpr (GRAD) {
      // d(2 u), which what is past float32 would make infinite beside a factor of 0: far before that f or rest is 0.
      const float2 u1 = ff_fma(make_float2(fminf(a2.x, 1e30f), fminf(a2.y, 1e30f)), ff_both(6 * k * c), ff_both(2 * k));
      const float2 rest = ff_fma(s, ff_both(-1.0f), ff_both(1.0f));
      df = ff_fma(ff_mul(f, rest), u1, s);
    }
  } else {
    const float2 s = ff_rcp(__fadd2_rn(ff_ex2(ff_mul(a, ff_both(-1.4426950408889634f))), ff_both(1.0f)));
    f = ff_mul(a, s);
    if constexpr (GRAD) df = ff_fma(f, ff_fma(s, ff_both(-1.0f), ff_both(1.0f)), s);
  }
}

// ---- the kernel of h, of [da | db] and of the plain products --------------------------------

// One product: tiles of M x N (N: columns of I for h and [da | db]), K in parts.
struct FfProblem {
  int M, N;
  int kblocks, parts;   // blocks of 64 of K, and how many parts they are cut in
  int units_m, units_n, units;
  int a_mn, b_mn;       // operands whose rows run along M or N instead of K
  int a_rows;           // rows of A's box (one CTA per tile: the rows there are, rounded up to 8; else 128)
  uint32_t idesc;
  void *out;            // 16 bits, row stride ldo
  int64_t ldo;
  bool sectors;         // its rows start at multiples of 32 bytes
  float4 *part;         // parts > 1: [parts][rows / 32][columns / 32][8][32 rows][4 columns]
};
constexpr int kFfProblems = 3;
constexpr int kFfListed = 1024;  // units of several problems that are dealt out by the host
struct FfArgs {
  FfProblem p[kFfProblems];
  int count, units;
  int dtype;
  float4 *z;   // a and b in float32 (NULL: not kept): [rows / 32][columns / 8][a, b][2][32 rows][4 columns]
  int early;   // the next launch may take the SMs that this one leaves free
  int listed;  // the CTAs' (pairs') units are listed; else every gridDim-th
  uint16_t first[160], unit[kFfListed];
};
struct FfMaps {
  CUtensorMap a[kFfProblems], b[kFfProblems];  // kFfForward: b[0] the rows of a, b[1] those of b
};

struct FfUnit {
  int i, m, n, s, k0, k1;
};
__device__ __forceinline__ FfUnit ff_unit(const FfArgs &a, int u) {
  FfUnit r;
  r.i = 0;
  while (u >= a.p[r.i].units) u -= a.p[r.i++].units;
  const FfProblem &p = a.p[r.i];
  r.n = u % p.units_n;
  u /= p.units_n;
  r.m = u % p.units_m;
  r.s = u / p.units_m;
  r.k0 = (int)((int64_t)p.kblocks * r.s / p.parts);
  r.k1 = (int)((int64_t)p.kblocks * (r.s + 1) / p.parts);
  return r;
}
// The units of one CTA (pair), in order.
struct FfWalk {
  int at, end, step;
  __device__ __forceinline__ FfWalk(const FfArgs &a, int me, int all)
      : at(a.listed ? a.first[me] : me), end(a.listed ? a.first[me + 1] : a.units), step(a.listed ? 1 : all) {}
  __device__ __forceinline__ bool next(const FfArgs &a, FfUnit &u) {
    if (at >= end) return false;
    u = ff_unit(a, a.listed ? a.unit[at] : at);
    at += step;
    return true;
  }
};

// BN: accumulator columns of a tile: BN/2 of a and as many of b, or BN of the
// result. An epilogue warp takes 64 of them for 32 rows.
template <int CG, int BN, int EPI>
struct FfShape {
  static constexpr int kGroups = BN / 64;
  static constexpr int kWarps = 4 * kGroups;
  static constexpr int kThreads = 64 + 32 * kWarps;
  static constexpr int kCols = EPI == kFfForward ? BN / 2 : BN;  // columns of the result
  static constexpr int kABytes = 128 * kVBK * 2;
  static constexpr int kBBytes = (BN / CG) * kVBK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  // A warp's memory: 32 rows x 32 columns of 16 bits on their way out; for [da | db]
  // kPieces of a and b on their way in, of kPieceCols columns: all 64 at once where the memory allows it; 16 KB for the
  // large tile leave three stages for the operands (16384 x 768 x 1152: 60 us; one piece of 32 65, four of 8 71).
  static constexpr int kPieces = CG == 1 ? 1 : 2, kPieceCols = CG == 1 ? 64 : 16;
  static constexpr int kStaging = EPI == kFfGrad ? kPieces * kPieceCols * 256 : 2048;
  static constexpr int kExtra = kWarps * kStaging;
  static constexpr int kRaw = (225 * 1024 - kExtra) / kStageBytes;
  static constexpr int kStages = kRaw > 8 ? 8 : kRaw;
  static constexpr int kExtraOff = kStages * kStageBytes;
  static constexpr int kBar = kExtraOff + kExtra;
  static constexpr int kZBar = kBar + 8 * (2 * kStages + 4);
  static constexpr int kTmemSlot = kZBar + 8 * kPieces * kWarps;
  static constexpr int kTotal = kTmemSlot + 16 + 1024;
  static_assert(kStages >= 3 && kTotal <= 227 * 1024, "shared memory");
  static_assert(BN == 64 || BN == 128 || BN == 256, "TMEM columns are a power of two");
};

// 32 rows x 32 columns of 16 bits that lie turned in buf (a row's 16-byte pieces
// exchanged by its number) to rows row0.. and columns col0.. of out: by 16 bytes
// where every row starts on such a boundary and has all of the columns, else the
// lanes take neighbouring columns of a row, two each on 4-byte boundaries, so
// that a store still touches few sectors (16 bytes of a row a lane, stored one
// value at a time, took the three gradients of 3957 x 542 x 142 26 us, now 19).
__device__ __forceinline__ void ff_store_turned(const uint8_t *buf, int lane, int row0, int M, int col0, int cols, uint16_t *out, int64_t ldo) {
  auto piece = [&](int r, int j) { return buf + r * 64 + ((j ^ ((r >> 1) & 3)) << 4); };
  const uintptr_t at = reinterpret_cast<uintptr_t>(out) | (uintptr_t)(ldo * 2);
  if (at % 16 == 0 && col0 + 32 <= cols) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int r = 8 * i + (lane >> 2), j = lane & 3;
      if (row0 + r < M) *reinterpret_cast<uint4 *>(out + (int64_t)(row0 + r) * ldo + col0 + 8 * j) = *reinterpret_cast<const uint4 *>(piece(r, j));
    }
  } else if (at % 4 == 0) {
    const int c = 2 * (lane & 15), col = col0 + c;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const int r = 2 * i + (lane >> 4);
      if (row0 + r >= M || col >= cols) continue;
      const uint32_t v = *reinterpret_cast<const uint32_t *>(piece(r, c >> 3) + (c & 7) * 2);
      uint16_t *dst = out + (int64_t)(row0 + r) * ldo + col;
      if (col + 1 < cols)
        *reinterpret_cast<uint32_t *>(dst) = v;
      else
        *dst = (uint16_t)v;
    }
  } else {
    const int col = col0 + lane;
#pragma unroll 8
    for (int r = 0; r < 32; r++) {
      if (row0 + r < M && col < cols)
        out[(int64_t)(row0 + r) * ldo + col] = *reinterpret_cast<const uint16_t *>(piece(r, lane >> 3) + (lane & 7) * 2);
    }
  }
}

// 32 rows x 32 columns of 16 bits, a lane's row in w, through 2 KB of shared memory.
__device__ __forceinline__ void ff_store_tile(uint8_t *buf, const uint32_t (&w)[16], int lane, int row0, int M, int col0, int cols,
                                              uint16_t *out, int64_t ldo) {
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 4; j++)
    *reinterpret_cast<uint4 *>(buf + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) =
        make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
  __syncwarp();
  ff_store_turned(buf, lane, row0, M, col0, cols, out, ldo);
}

// Sixteen columns of a row on a 32-byte boundary: a whole sector a lane.
__device__ __forceinline__ void ff_store16(uint16_t *dst, const uint32_t *w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
// 32 columns of the lanes' rows: straight from the registers where whole
// sectors can be written (through shared memory, whose ports the operands need,
// the products of 16384 x 768 x 1152 took 33 and 120 us), else turned there.
__device__ __forceinline__ void ff_store_rows(uint8_t *buf, const uint32_t (&w)[16], int lane, int row0, int M, int col0, int cols,
                                              uint16_t *out, int64_t ldo, bool sectors) {
  if (sectors && col0 + 32 <= cols) {
    if (row0 + lane < M) {
      uint16_t *dst = out + (int64_t)(row0 + lane) * ldo + col0;
      ff_store16(dst, w);
      ff_store16(dst + 16, w + 8);
    }
  } else {
    ff_store_tile(buf, w, lane, row0, M, col0, cols, out, ldo);
  }
}
// The same for 16 columns, turned in 1 KB. Four of these lie in one tile's code:
// stored by columns as above, three forms each, they were slower (42 x 163 x 1069:
// 15.6 against 9.4 us).
__device__ __forceinline__ void ff_store_half(uint8_t *buf, const uint32_t (&w)[8], int lane, int row0, int M, int col0, int cols,
                                              uint16_t *out, int64_t ldo, bool sectors) {
  if (sectors && col0 + 16 <= cols) {
    if (row0 + lane < M) ff_store16(out + (int64_t)(row0 + lane) * ldo + col0, w);
    return;
  }
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 2; j++)
    *reinterpret_cast<uint4 *>(buf + lane * 32 + ((j ^ ((lane >> 2) & 1)) << 4)) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int r = i * 16 + (lane >> 1), j = lane & 1, col = col0 + 8 * j;
    if (row0 + r >= M || col >= cols) continue;
    const uint4 v = *reinterpret_cast<const uint4 *>(buf + r * 32 + ((j ^ ((r >> 2) & 1)) << 4));
    uint16_t *dst = out + (int64_t)(row0 + r) * ldo + col;
    if (col + 8 <= cols && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
      *reinterpret_cast<uint4 *>(dst) = v;
    } else {
      const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 8; k++)
        if (col + k < cols) dst[k] = (uint16_t)(x[k >> 1] >> (16 * (k & 1)));
    }
  }
}

template <int CG, int BN, int EPI, int ACT>
__global__ void __launch_bounds__(FfShape<CG, BN, EPI>::kThreads, 1)
    ff_kernel(const __grid_constant__ FfMaps maps, const __grid_constant__ FfArgs a) {
  using S = FfShape<CG, BN, EPI>;
  constexpr int kStages = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + S::kBar);
  uint64_t *empty = full + kStages;
  uint64_t *accf = empty + kStages;
  uint64_t *acce = accf + 2;
  uint64_t *zbar = reinterpret_cast<uint64_t *>(smem + S::kZBar);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + S::kTmemSlot);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CG == 2 ? (int)cluster_ctarank() : 0;
  const int me = blockIdx.x / CG, all = gridDim.x / CG;

  if (warp == 0 && lane == 0) {
    for (int i = 0; i < a.count; i++) {
      prefetch_tensormap(&maps.a[i]);
      prefetch_tensormap(&maps.b[i]);
    }
    if (EPI == kFfForward) prefetch_tensormap(&maps.b[1]);
    for (int s = 0; s < kStages; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(&accf[b], 1);
      mbar_init(&acce[b], CG * S::kWarps);
    }
    for (int e = 0; e < S::kPieces * S::kWarps; e++) mbar_init(&zbar[e], 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    if constexpr (CG == 2)
      tmem_alloc_pair(tmem_slot, 2 * BN);
    else
      tmem_alloc(tmem_slot, 2 * BN);
  }
  tc_fence_before();
  if constexpr (CG == 2)
    cluster_sync_all();
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  dep_wait();
  if (a.early) dep_trigger();
  FfWalk walk(a, me, all);
  FfUnit q;

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      while (ok && walk.next(a, q)) {
        const FfProblem &p = a.p[q.i];
        const bool a_mn = EPI == kFfProduct && p.a_mn, b_mn = EPI == kFfGrad || (EPI == kFfProduct && p.b_mn);
        const CUtensorMap *ma = &maps.a[q.i], *mb = &maps.b[q.i];
        const int m0 = q.m * (CG * 128) + rank * 128, n0 = q.n * S::kCols;
        for (int kb = q.k0; kb < q.k1; kb++, it++) {
          const int s = it % kStages;
          if (!mbar_wait(&empty[s], ((it / kStages) & 1) ^ 1, kDevTimeoutEmpty)) {
            ok = false;
            break;
          }
          uint8_t *sa = smem + s * S::kStageBytes, *sb = sa + S::kABytes;
          if (rank == 0) mbar_arrive_expect_tx(&full[s], CG * (S::kBBytes + p.a_rows * kVBK * 2));
          auto load = [&](const CUtensorMap *map, uint8_t *dst, int c0, int c1) {
            if constexpr (CG == 2)
              tma_load_2d_pair(map, dst, cluster_addr(&full[s], 0), c0, c1);
            else
              tma_load_2d(map, dst, &full[s], c0, c1);
          };
          if (a_mn) {
            load(ma, sa, m0, kb * kVBK);
            load(ma, sa + 8192, m0 + 64, kb * kVBK);
          } else {
            load(ma, sa, kb * kVBK, m0);
          }
          if constexpr (EPI == kFfForward) {
            // a's weight rows, then b's: of a pair, a CTA each.
            if constexpr (CG == 2) {
              load(rank == 0 ? mb : &maps.b[1], sb, kb * kVBK, n0);
            } else {
              load(mb, sb, kb * kVBK, n0);
              load(&maps.b[1], sb + S::kBBytes / 2, kb * kVBK, n0);
            }
          } else if (b_mn) {
#pragma unroll
            for (int i = 0; i < BN / CG / 64; i++) load(mb, sb + i * 8192, n0 + rank * (BN / CG) + i * 64, kb * kVBK);
          } else {
            load(mb, sb, kb * kVBK, n0 + rank * (BN / CG));
          }
        }
      }
      if constexpr (CG == 2) {
        // No commit from the even CTA may still be on its way at exit.
        for (int i = 0; i < kStages && ok; i++, it++)
          if (!mbar_wait(&empty[it % kStages], ((it / kStages) & 1) ^ 1, kDevTimeoutEmpty)) break;
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      int it = 0, tile = 0;
      bool ok = true;
      for (; ok && walk.next(a, q); tile++) {
        const FfProblem &p = a.p[q.i];
        const bool a_mn = EPI == kFfProduct && p.a_mn, b_mn = EPI == kFfGrad || (EPI == kFfProduct && p.b_mn);
        const uint32_t idesc = p.idesc;
        const int b = tile & 1;
        if (!mbar_wait(&acce[b], ((tile >> 1) & 1) ^ 1, kDevTimeoutEmpty)) break;
        tc_fence_after();
        const uint32_t d = tmem + b * BN;
        for (int kb = q.k0; kb < q.k1; kb++, it++) {
          const int s = it % kStages;
          if (!mbar_wait(&full[s], (it / kStages) & 1, kDevTimeoutFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + s * S::kStageBytes), sb = sa + S::kABytes;
          const uint64_t da = a_mn ? smem_desc_mn_sw128(sa) : smem_desc_k_sw128(sa),
                         db = b_mn ? smem_desc_mn_sw128(sb) : smem_desc_k_sw128(sb);
          // 16 of K on: 32 bytes along a row, or 16 rows of 128 bytes (the descriptor counts 16 bytes).
          const uint32_t step_a = a_mn ? 2048 >> 4 : 32 >> 4, step_b = b_mn ? 2048 >> 4 : 32 >> 4;
#pragma unroll
          for (uint32_t kk = 0; kk < kVBK / 16; kk++)
            mma_f16<CG>(d, da + kk * step_a, db + kk * step_b, idesc, (kb > q.k0 || kk > 0) ? 1u : 0u);
          if constexpr (CG == 2) {
            mma_commit_pair(cluster_addr(&empty[s], 0));
            mma_commit_pair(cluster_addr(&empty[s], 1));
          } else {
            mma_commit(&empty[s]);
          }
        }
        if (!ok) break;
        if constexpr (CG == 2) {
          mma_commit_pair(cluster_addr(&accf[b], 0));
          mma_commit_pair(cluster_addr(&accf[b], 1));
        } else {
          mma_commit(&accf[b]);
        }
      }
    }
  } else {
    const int q4 = warp & 3, e = warp - 2, g = e >> 2;  // TMEM lane quarter, group of columns
    uint8_t *buf = smem + S::kExtraOff + e * S::kStaging;
    int tile = 0;
    // kFfGrad: the warp's next pieces of z are on their way while it waits for the accumulators and works on those before.
    [[maybe_unused]] FfWalk ahead = walk;
    [[maybe_unused]] FfUnit zq{};
    [[maybe_unused]] int zi = 64, zgot = 0, zasked = 0;
    [[maybe_unused]] auto ask = [&] {  // for the next piece there is
      if constexpr (EPI == kFfGrad) {
        const int N = a.p[0].N, wide = (N + 31) / 32 * 32;  // columns that z has
        for (;;) {
          if (zi == 64) {
            if (!ahead.next(a, zq)) return;
            zi = 0;
          }
          const int row0 = zq.m * (CG * 128) + rank * 128 + q4 * 32, col0 = zq.n * S::kCols + 64 * g + zi;
          zi += S::kPieceCols;
          if (row0 >= a.p[0].M || col0 >= N) continue;
          const int at = zasked++ % S::kPieces;
          if (lane == 0) {
            uint64_t *bar = &zbar[S::kPieces * e + at];
            const uint32_t bytes = (S::kPieceCols < wide - col0 ? S::kPieceCols : wide - col0) * 256;
            mbar_arrive_expect_tx(bar, bytes);
            bulk_g2s(buf + S::kPieceCols * 256 * at, a.z + ((int64_t)(row0 / 32) * wide + col0) * 16, bytes, bar);
          }
          return;
        }
      }
    };
    for (int i = 0; i < S::kPieces; i++) ask();
    bool ok = true;
    for (; ok && walk.next(a, q); tile++) {
      const FfProblem &p = a.p[q.i];
      const int b = tile & 1, n0 = q.n * S::kCols;
      const int row0 = q.m * (CG * 128) + rank * 128 + q4 * 32;
      uint16_t *out = static_cast<uint16_t *>(p.out);
      if (!mbar_wait(&accf[b], (tile >> 1) & 1, kDevTimeoutAccum)) break;
      tc_fence_after();
      auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (CG == 1 || rank == 0)
            mbar_arrive(&acce[b]);
          else
            mbar_arrive_cluster(cluster_addr(&acce[b], 0));
        }
      };
      if (row0 >= p.M) {
        release();
        continue;
      }
      const uint32_t tb = tmem + b * BN + ((uint32_t)(q4 * 32) << 16);
      if constexpr (EPI == kFfForward) {
        uint32_t ra[32], rb[32];
        __syncwarp();
        tmem_ld_32x32b_x32(tb + 32 * g, ra);
        tmem_ld_32x32b_x32(tb + BN / 2 + 32 * g, rb);
        tmem_ld_wait();
        release();
        const int col0 = n0 + 32 * g;
        if (col0 >= p.N) continue;
        if (a.z) {
          float4 *z = a.z + ((int64_t)(row0 / 32) * ((p.N + 31) / 32) + col0 / 32) * 512 + lane;
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const int at = j / 2 * 128 + j % 2 * 32;
            z[at] = make_float4(__uint_as_float(ra[4 * j]), __uint_as_float(ra[4 * j + 1]), __uint_as_float(ra[4 * j + 2]),
                                __uint_as_float(ra[4 * j + 3]));
            z[at + 64] = make_float4(__uint_as_float(rb[4 * j]), __uint_as_float(rb[4 * j + 1]), __uint_as_float(rb[4 * j + 2]),
                                      __uint_as_float(rb[4 * j + 3]));
          }
        }
        uint32_t w[16];
#pragma unroll
        for (int k = 0; k < 16; k++) {
          float2 f, unused;
          ff_act<ACT, false>(make_float2(__uint_as_float(ra[2 * k]), __uint_as_float(ra[2 * k + 1])), f, unused);
          f = ff_mul(f, make_float2(__uint_as_float(rb[2 * k]), __uint_as_float(rb[2 * k + 1])));
          w[k] = pack16(f.x, f.y, a.dtype);
        }
        ff_store_rows(buf, w, lane, row0, p.M, col0, p.N, out, p.ldo, p.sectors);
      } else {
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const bool last = i + 1 == 2;
          __syncwarp();
          uint32_t r[32];
          tmem_ld_32x32b_x32(tb + 64 * g + 32 * i, r);
          tmem_ld_wait();
          if (last) release();
          const int col0 = n0 + 64 * g + 32 * i;
          if (col0 >= p.N) continue;
          if constexpr (EPI == kFfGrad) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const int at = (32 * i + 16 * h) % S::kPieceCols, col = col0 + 16 * h;  // columns into the piece
              uint8_t *piece = buf + S::kPieceCols * 256 * (zgot % S::kPieces);
              if (col < p.N && ok) {
                if (at == 0) ok = __all_sync(~0u, mbar_wait(&zbar[S::kPieces * e + zgot % S::kPieces], zgot / S::kPieces & 1, kDevTimeoutFull));
                const float4 *z = reinterpret_cast<const float4 *>(piece) + at * 16 + lane;
                uint32_t wa[8], wb[8];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                  const float4 za = z[j / 2 * 128 + j % 2 * 32], zb = z[j / 2 * 128 + 64 + j % 2 * 32];
#pragma unroll
                  for (int k = 0; k < 2; k++) {
                    float2 f, df;
                    ff_act<ACT, true>(k ? make_float2(za.z, za.w) : make_float2(za.x, za.y), f, df);
                    const int d0 = 16 * h + 4 * j + 2 * k;
                    const float2 d = make_float2(__uint_as_float(r[d0]), __uint_as_float(r[d0 + 1]));
                    const float2 da = ff_mul(d, ff_mul(k ? make_float2(zb.z, zb.w) : make_float2(zb.x, zb.y), df));
                    const float2 db = ff_mul(d, f);
                    wa[2 * j + k] = pack16(da.x, da.y, a.dtype);
                    wb[2 * j + k] = pack16(db.x, db.y, a.dtype);
                  }
                }
                // Rows that are not of whole sectors are turned where these columns' a and b were.
                const bool sectors = p.sectors && p.N % 16 == 0;
                uint8_t *turn = piece + at * 256;
                ff_store_half(turn, wa, lane, row0, p.M, col, p.N, out, p.ldo, sectors);
                ff_store_half(turn + 1024, wb, lane, row0, p.M, col, p.N, out + p.N, p.ldo, sectors);
                if (ok && (at + 16 == S::kPieceCols || col + 16 >= p.N)) {  // the piece's last columns
                  zgot++;
                  if (!sectors) fence_proxy_async_smem();
                  __syncwarp();
                  ask();
                }
              }
            }
          } else if (p.parts > 1) {
            float4 *t = p.part + ((((int64_t)q.s * ((p.M + 31) / 32)) + row0 / 32) * ((p.N + 31) / 32) + col0 / 32) * 256 + lane;
#pragma unroll
            for (int j = 0; j < 8; j++)
              t[32 * j] = make_float4(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1]), __uint_as_float(r[4 * j + 2]),
                                      __uint_as_float(r[4 * j + 3]));
          } else {
            uint32_t w[16];
#pragma unroll
            for (int k = 0; k < 16; k++) w[k] = pack16(__uint_as_float(r[2 * k]), __uint_as_float(r[2 * k + 1]), a.dtype);
            ff_store_rows(buf, w, lane, row0, p.M, col0, p.N, out, p.ldo, p.sectors);
          }
        }
      }
    }
    if constexpr (EPI == kFfGrad) {
      // Given up: copies may still be on their way into this CTA's memory.
      for (; zgot < zasked; zgot++) mbar_wait(&zbar[S::kPieces * e + zgot % S::kPieces], zgot / S::kPieces & 1, kDevTimeoutFull);
      __syncwarp();
    }
  }

  tc_fence_before();
  __syncthreads();
  dep_trigger();
  if constexpr (CG == 2) cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CG == 2)
      tmem_dealloc_pair(tmem, 2 * BN);
    else
      tmem_dealloc(tmem, 2 * BN);
  }
}

// The parts of the products that have more than one, added in order: a CTA to a
// piece of 32 rows x 32 columns, its warps eight columns each, with the loads of
// eight parts in flight.
struct FfSum {
  const float4 *part;
  void *out;
  int64_t ldo;
  int M, N, parts;
  int64_t pieces;
};
struct FfSumArgs {
  FfSum s[kFfProblems];
  int count, dtype;
};
__global__ void __launch_bounds__(128) ff_sum_kernel(const FfSumArgs a) {
  __shared__ __align__(16) uint8_t s_buf[2048];
  dep_wait();
  dep_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t t = blockIdx.x;
  int i = 0;
  while (i < a.count && t >= a.s[i].pieces) t -= a.s[i++].pieces;
  if (i == a.count) return;
  const FfSum &s = a.s[i];
  const float4 *src = s.part + t * 256 + 64 * warp + lane;
  float4 v[2] = {src[0], src[32]};
#pragma unroll 8
  for (int p = 1; p < s.parts; p++) {
    src += s.pieces * 256;
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const float4 x = src[32 * j];
      v[j] = make_float4(v[j].x + x.x, v[j].y + x.y, v[j].z + x.z, v[j].w + x.w);
    }
  }
  *reinterpret_cast<uint4 *>(s_buf + lane * 64 + ((warp ^ ((lane >> 1) & 3)) << 4)) =
      make_uint4(pack16(v[0].x, v[0].y, a.dtype), pack16(v[0].z, v[0].w, a.dtype), pack16(v[1].x, v[1].y, a.dtype), pack16(v[1].z, v[1].w, a.dtype));
  __syncthreads();
  const int nb = (s.N + 31) / 32;
  if (warp == 0)
    ff_store_turned(s_buf, lane, (int)(t / nb) * 32, s.M, (int)(t % nb) * 32, s.N, static_cast<uint16_t *>(s.out), s.ldo);
}

// ---- operands whose rows do not start on 16-byte boundaries ------------------------------------

struct FfPack {
  const uint16_t *src[4];
  uint16_t *dst[4];
  int64_t units[4], lds[4], ldd[4];
  int cols[4];
  int count;
};
// Copies them into rows that do, all of them in one launch: a warp to 512
// columns of a row, all of its loads in flight before its stores of 16 bytes.
// Past a row's columns come zeros, as far as its last 16 bytes.
constexpr int kFfPackCols = 512;
__global__ void __launch_bounds__(128) ff_pack_kernel(const FfPack a) {
  dep_wait();
  dep_trigger();
  int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  int i = 0;
  while (i < a.count && unit >= a.units[i]) unit -= a.units[i++];
  if (i == a.count) return;
  const int cols = a.cols[i], across = (cols + kFfPackCols - 1) / kFfPackCols;
  const int64_t row = unit / across;
  const int c0 = (int)(unit - row * across) * kFfPackCols + 8 * (threadIdx.x & 31);
  const uint16_t *s = a.src[i] + row * a.lds[i];
  uint16_t *d = a.dst[i] + row * a.ldd[i];
  uint32_t w[2][4];
  if (((reinterpret_cast<uintptr_t>(a.src[i]) | (uintptr_t)(a.lds[i] * 2)) & 3) == 0) {
#pragma unroll
    for (int q = 0; q < 2; q++) {
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int c = c0 + 256 * q + 2 * k;
        w[q][k] = c + 1 < cols ? *reinterpret_cast<const uint32_t *>(s + c) : c < cols ? s[c] : 0u;
      }
    }
  } else {
#pragma unroll
    for (int q = 0; q < 2; q++) {
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int c = c0 + 256 * q + 2 * k;
        const uint32_t lo = c < cols ? s[c] : 0, hi = c + 1 < cols ? s[c + 1] : 0;
        w[q][k] = lo | hi << 16;
      }
    }
  }
#pragma unroll
  for (int q = 0; q < 2; q++)
    if (c0 + 256 * q < cols) *reinterpret_cast<uint4 *>(d + c0 + 256 * q) = make_uint4(w[q][0], w[q][1], w[q][2], w[q][3]);
}

// ---- few rows -----------------------------------------------------------------------------------

// Dot products of R rows of float32 or 16-bit x with W weight rows (w apart by
// `next`), a warp's lanes VEC neighbouring columns each: 8 on 16-byte
// boundaries, 2 on 4-byte ones, else 1. Rows past `rows` are the last again.
// The loads of four steps are in flight together.
template <int R, int W, bool F32X, int VEC>
__device__ __forceinline__ void ff_dots(const void *x, int64_t ldx, int rows, const uint16_t *w, int64_t next, int n, int dtype, int lane,
                                        float (&s)[W][R]) {
  constexpr int kAhead = VEC == 8 ? (R * W > 2 ? 2 : 4) : 4;
#pragma unroll
  for (int q = 0; q < W; q++) {
#pragma unroll
    for (int r = 0; r < R; r++) s[q][r] = 0.0f;
  }
  const int whole = n / VEC * VEC;
  for (int c0 = VEC * lane; c0 < whole; c0 += 32 * VEC * kAhead) {
    float wf[kAhead][W][VEC], xf[kAhead][R][VEC];
#pragma unroll
    for (int i = 0; i < kAhead; i++) {
      const int c = c0 + 32 * VEC * i;
      const bool there = c < whole;
#pragma unroll
      for (int q = 0; q < W; q++) {
        const uint16_t *at = w + q * next + c;
        if constexpr (VEC == 8) {
          const uint4 v = there ? __ldg(reinterpret_cast<const uint4 *>(at)) : make_uint4(0, 0, 0, 0);
          const uint32_t ws[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const float2 f = widen2(ws[k], dtype);
            wf[i][q][2 * k] = f.x, wf[i][q][2 * k + 1] = f.y;
          }
        } else if constexpr (VEC == 2) {
          const float2 f = widen2(there ? __ldg(reinterpret_cast<const uint32_t *>(at)) : 0u, dtype);
          wf[i][q][0] = f.x, wf[i][q][1] = f.y;
        } else {
          wf[i][q][0] = there ? widen1(*at, dtype) : 0.0f;
        }
      }
#pragma unroll
      for (int r = 0; r < R; r++) {
        const int64_t at = (r < rows ? r : rows - 1) * ldx + c;
        if constexpr (F32X && VEC == 8) {
          const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(x) + at);
          const float4 u = there ? p[0] : make_float4(0, 0, 0, 0), v = there ? p[1] : make_float4(0, 0, 0, 0);
          const float f[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k = 0; k < 8; k++) xf[i][r][k] = f[k];
        } else if constexpr (F32X) {
#pragma unroll
          for (int k = 0; k < VEC; k++) xf[i][r][k] = there ? static_cast<const float *>(x)[at + k] : 0.0f;
        } else if constexpr (VEC == 8) {
          const uint4 v = there ? *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(x) + at) : make_uint4(0, 0, 0, 0);
          const uint32_t xs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const float2 f = widen2(xs[k], dtype);
            xf[i][r][2 * k] = f.x, xf[i][r][2 * k + 1] = f.y;
          }
        } else if constexpr (VEC == 2) {
          const float2 f = widen2(there ? *reinterpret_cast<const uint32_t *>(static_cast<const uint16_t *>(x) + at) : 0u, dtype);
          xf[i][r][0] = f.x, xf[i][r][1] = f.y;
        } else {
          xf[i][r][0] = there ? widen1(static_cast<const uint16_t *>(x)[at], dtype) : 0.0f;
        }
      }
    }
    // Past the row both are 0.
#pragma unroll
    for (int i = 0; i < kAhead; i++) {
#pragma unroll
      for (int q = 0; q < W; q++) {
#pragma unroll
        for (int r = 0; r < R; r++) {
#pragma unroll
          for (int k = 0; k < VEC; k++) s[q][r] = fmaf(xf[i][r][k], wf[i][q][k], s[q][r]);
        }
      }
    }
  }
  if (VEC > 1 && whole + lane < n) {
#pragma unroll
    for (int q = 0; q < W; q++) {
      const float wf = widen1(w[q * next + whole + lane], dtype);
#pragma unroll
      for (int r = 0; r < R; r++) {
        const int64_t at = (r < rows ? r : rows - 1) * ldx + whole + lane;
        s[q][r] = fmaf(F32X ? static_cast<const float *>(x)[at] : widen1(static_cast<const uint16_t *>(x)[at], dtype), wf, s[q][r]);
      }
    }
  }
#pragma unroll
  for (int q = 0; q < W; q++) {
#pragma unroll
    for (int r = 0; r < R; r++) s[q][r] = warp_sum(s[q][r]);
  }
}

struct FfRowsArgs {
  const void *x, *w_in, *w_out;
  int64_t ldx, ldi, ldw;
  int rows, H;
  int64_t I, O;
  int dtype, act;
  float *h;  // [rows][ldh], ldh a multiple of 8
  int64_t ldh;
  void *y;
  int64_t ldy;
};

__device__ __forceinline__ float ff_act1(float a, int act) {
  float2 f, unused;
  if (act == IG_ACT_GELU)
    ff_act<IG_ACT_GELU, false>(ff_both(a), f, unused);
  else if (act == IG_ACT_GELU_TANH)
    ff_act<IG_ACT_GELU_TANH, false>(ff_both(a), f, unused);
  else
    ff_act<IG_ACT_SILU, false>(ff_both(a), f, unused);
  return f.x;
}

// Up to R rows, bound by the weights' read: a warp per column of h (both its
// weight rows), then a warp per column of y. h stays in float32.
template <int R, int VEC>
__global__ void __launch_bounds__(128) ff_rows_in_kernel(const FfRowsArgs a) {
  dep_wait();
  dep_trigger();
  const int lane = threadIdx.x & 31;
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (i >= a.I) return;
  float s[2][R];
  ff_dots<R, 2, false, VEC>(a.x, a.ldx, a.rows, static_cast<const uint16_t *>(a.w_in) + i * a.ldi, a.I * a.ldi, a.H, a.dtype, lane, s);
#pragma unroll
  for (int r = 0; r < R; r++)
    if (lane == r && r < a.rows) a.h[r * a.ldh + i] = ff_act1(s[0][r], a.act) * s[1][r];
}
template <int R, int VEC>
__global__ void __launch_bounds__(128) ff_rows_out_kernel(const FfRowsArgs a) {
  dep_wait();
  dep_trigger();
  const int lane = threadIdx.x & 31;
  const int64_t o = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (o >= a.O) return;
  float s[1][R];
  ff_dots<R, 1, true, VEC>(a.h, a.ldh, a.rows, static_cast<const uint16_t *>(a.w_out) + o * a.ldw, 0, (int)a.I, a.dtype, lane, s);
#pragma unroll
  for (int r = 0; r < R; r++)
    if (lane == r && r < a.rows) store16(a.y, r * a.ldy + o, s[0][r], a.dtype);
}

// ---- plans and launches ---------------------------------------------------------------------------

// One row goes to warps instead of tensor cores, and up to four where rows times
// weights are few: beyond, every weight's products with each row cost more than
// its read. 768 x 1152, 1 to 4 rows: 7.7, 8.1, 10.8 and 12.0 us, on the tensor
// cores 16.6; 1024 x 2048, 2 and 3 rows: 8.5 and 20.6 against 16.8; 4096 x 8192,
// 1 and 2: 47 and 80 against 69.
constexpr int kFfRows = 4;
constexpr int64_t kFfFewProducts = 14 << 20;

// Tiles of 256 x 256 on a CTA pair, or of 128 x 64 on one CTA where those are
// too few to fill the GPU. What a block of 64 of K takes of either, and what a
// tile's start and end add, in microseconds.
struct FfTile {
  int cg, bn;
  double block, tile;
};
constexpr FfTile kFfLarge{2, 256, 0.48, 1.5}, kFfSmall{1, 64, 0.17, 0.8};

struct FfSizes {
  int64_t rows;
  int H, I, O;
  int pack;  // bits: operands to be copied into rows on 16-byte boundaries (x 1, w_in 2, w_out 4, dy 8)
};
static inline int64_t ff_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }
static inline int64_t ff_ld(int64_t cols) { return ff_up(cols, 16); }  // rows of whole sectors

// How a list of products is cut: the tile, and the parts of each one's K.
struct FfCut {
  bool small;
  int parts[kFfProblems];
  size_t off[kFfProblems], bytes;  // of the partial sums
};
struct FfShapeOf {
  int64_t M, N, K;
};
struct FfPlan {
  size_t h_bytes, z_bytes;              // of what is saved: h, then a and b
  size_t off[4], pack_bytes;            // the copied operands
  size_t dz_bytes;
  int64_t ldz;
  FfCut cut;                            // of y; or of dWi, dWo and dx, the longest sums first
};

static int64_t ff_div(int64_t v, int64_t a) { return (v + a - 1) / a; }

// The cut with the smallest estimated time: all blocks of K spread over the
// GPU, but no less than the longest unit takes; partial sums are written and
// read again at 4 TB/s by one more launch.
static FfCut ff_cut(const FfShapeOf *p, int count) {
  FfCut best{};
  double least = 1e300;
  for (int small = 0; small < 2; small++) {
    const FfTile &t = small ? kFfSmall : kFfLarge;
    const int64_t slots = num_sms() / t.cg;
    int64_t most = 1;  // blocks of K in a unit
    for (int i = 0; i < count; i++) most = std::max(most, ff_div(p[i].K, kVBK));
    do {
      FfCut c{};
      c.small = small;
      double total = 0.0, longest = 0.0, units = 0.0;
      for (int i = 0; i < count; i++) {
        const int64_t kb = ff_div(p[i].K, kVBK);
        c.parts[i] = (int)std::min<int64_t>(ff_div(kb, most), 64);
        const double tiles = (double)ff_div(p[i].M, 128 * t.cg) * ff_div(p[i].N, t.bn), len = (double)ff_div(kb, c.parts[i]);
        const double one = len * t.block + t.tile;
        total += tiles * c.parts[i] * one;
        units += tiles * c.parts[i];
        longest = std::max(longest, one);
        if (c.parts[i] > 1) {
          c.off[i] = c.bytes;
          c.bytes += (size_t)c.parts[i] * ff_up(p[i].M, 32) * ff_up(p[i].N, 32) * 4;
        }
      }
      // Equal units fill whole rounds; unequal ones are dealt out within about a short one.
      const double rounds = count == 1 ? std::ceil(units / slots) * longest : std::max(longest, total / slots + 0.3 * total / units);
      const double time = rounds + (c.bytes ? 3.0 + 2.0 * (double)c.bytes / 4e6 : 0.0);
      if (time < least) {
        least = time;
        best = c;
      }
      most = most * 3 / 4;
    } while (most >= 4);
  }
  return best;
}

static size_t ff_h_bytes(int64_t rows, int I) { return align_up((size_t)rows * ff_ld(I) * 2, 256); }
static size_t ff_z_bytes(int64_t rows, int I) { return (size_t)ff_up(rows, 32) * ff_up(I, 32) * 8; }
static FfPlan ff_plan(const FfSizes &s, bool backward) {
  FfPlan p{};
  p.h_bytes = ff_h_bytes(s.rows, s.I);
  p.z_bytes = ff_z_bytes(s.rows, s.I);
  const int64_t rows[4] = {s.rows, 2 * (int64_t)s.I, s.O, s.rows}, cols[4] = {s.H, s.H, s.I, s.O};
  for (int i = 0; i < 4; i++) {
    p.off[i] = p.pack_bytes;
    if (s.pack >> i & 1) p.pack_bytes += align_up((size_t)rows[i] * ff_ld(cols[i]) * 2, 256);
  }
  p.ldz = ff_ld(2 * (int64_t)s.I);
  if (backward) {
    p.dz_bytes = align_up((size_t)s.rows * p.ldz * 2, 256);
    const FfShapeOf n[3] = {{2 * (int64_t)s.I, s.H, s.rows}, {s.O, s.I, s.rows}, {s.rows, s.H, 2 * (int64_t)s.I}};
    p.cut = ff_cut(n, 3);
  } else {
    const FfShapeOf n[1] = {{s.rows, s.O, s.I}};
    p.cut = ff_cut(n, 1);
  }
  return p;
}
static bool ff_few(const FfSizes &s, bool save) {
  return !save && (s.rows == 1 || (s.rows <= kFfRows && s.rows * s.I * (2 * (int64_t)s.H + s.O) <= kFfFewProducts));
}
static size_t ff_bytes(const FfSizes &s, const FfPlan &p, int pass) {
  if (ff_few(s, pass > 0)) return (size_t)s.rows * ff_ld(s.I) * 4;
  return p.pack_bytes + p.cut.bytes + (pass == 0 ? p.h_bytes : pass == 2 ? p.dz_bytes : 0);
}

struct FfMatrix {
  const void *p;
  int64_t ld;
};
static bool ff_on(const FfMatrix &m) { return m.ld % 8 == 0 && (reinterpret_cast<uintptr_t>(m.p) & 15) == 0; }

// Copies the operands whose bits are set into the workspace, and points them there.
static cudaError_t ff_pack(FfMatrix *const (&m)[4], const FfSizes &s, const FfPlan &p, uint8_t *ws, cudaStream_t st) {
  FfPack a{};
  const int64_t rows[4] = {s.rows, 2 * (int64_t)s.I, s.O, s.rows};
  const int cols[4] = {s.H, s.H, s.I, s.O};
  int64_t units = 0;
  for (int i = 0; i < 4; i++) {
    if (!(s.pack >> i & 1)) continue;
    const int k = a.count++;
    a.src[k] = static_cast<const uint16_t *>(m[i]->p);
    a.dst[k] = reinterpret_cast<uint16_t *>(ws + p.off[i]);
    a.units[k] = rows[i] * ff_div(cols[i], kFfPackCols);
    a.lds[k] = m[i]->ld;
    a.ldd[k] = ff_ld(cols[i]);
    a.cols[k] = cols[i];
    *m[i] = FfMatrix{a.dst[k], a.ldd[k]};
    units += a.units[k];
  }
  return a.count ? launch_dep(ff_pack_kernel, dim3((unsigned)ff_div(units, 4)), dim3(128), 0, st, a) : cudaSuccess;
}

template <int CG, int BN, int EPI, int ACT>
static cudaError_t ff_launch(const FfMaps &maps, FfArgs &a, cudaStream_t st) {
  using S = FfShape<CG, BN, EPI>;
  static SmemOptIn attr;
  cudaError_t e = attr.ensure((const void *)ff_kernel<CG, BN, EPI, ACT>, S::kTotal);
  if (e != cudaSuccess) return e;
  int slots = num_sms();
  if constexpr (CG == 2) {
    static PerDevice clusters;
    slots = clusters.get([] {
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = CG;
      at[0].val.clusterDim.y = 1;
      at[0].val.clusterDim.z = 1;
      cfg.gridDim = dim3(CG * (num_sms() / CG));
      cfg.blockDim = dim3(S::kThreads);
      cfg.dynamicSmemBytes = S::kTotal;
      cfg.attrs = at;
      cfg.numAttrs = 1;
      int c = 0;
      if (cudaOccupancyMaxActiveClusters(&c, ff_kernel<CG, BN, EPI, ACT>, &cfg) != cudaSuccess) {
        (void)cudaGetLastError();
        c = 0;
      }
      return c;
    });
  }
  if (slots <= 0) return cudaErrorInvalidConfiguration;
  if (slots > a.units) slots = a.units;
  // A launch that leaves SMs free lets the next one set itself up there at once; one that fills them would have the next
  // one's CTAs parked on its own.
  a.early = CG * slots <= num_sms() / 2;
  // Units of several lengths are dealt out, the longest first, each to whoever has least.
  constexpr int kBins = (int)(sizeof(a.first) / sizeof(a.first[0])) - 1;
  a.listed = a.count > 1 && a.units <= kFfListed && slots <= kBins && a.units > slots;
  if (a.listed) {
    uint16_t owner[kFfListed], n[kBins + 1] = {};
    int load[kBins] = {};
    int u = 0;
    for (int i = 0; i < a.count; i++) {
      const int len = (a.p[i].kblocks + a.p[i].parts - 1) / a.p[i].parts + 3;
      for (int k = 0; k < a.p[i].units; k++, u++) {
        const int b = (int)(std::min_element(load, load + slots) - load);
        owner[u] = (uint16_t)b;
        load[b] += len;
        n[b]++;
      }
    }
    a.first[0] = 0;
    for (int b = 0; b < slots; b++) a.first[b + 1] = (uint16_t)(a.first[b] + n[b]);
    uint16_t at[kBins];
    std::copy(a.first, a.first + slots, at);
    for (u = 0; u < a.units; u++) a.unit[at[owner[u]]++] = (uint16_t)u;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  cfg.gridDim = dim3((unsigned)(CG * slots));
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = S::kTotal;
  cfg.stream = st;
  if (CG > 1) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = CG;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  cfg.attrs = at;
  add_dep_attr(at, cfg.numAttrs);
  return cudaLaunchKernelEx(&cfg, ff_kernel<CG, BN, EPI, ACT>, maps, a);
}

// Adds a product to the list: A and B K-major ([M][K], [N][K]), or with M (N) along their rows ([K][M], [K][N]).
// cols: columns of the result in a tile.
static int ff_add(FfMaps &maps, FfArgs &f, const FfTile &t, const FfMatrix &A, bool a_mn, const FfMatrix &B, bool b_mn, const FfShapeOf &n,
                  int box_b, int cols, int parts, void *out, int64_t ldo, float4 *part) {
  const int i = f.count++;
  FfProblem &p = f.p[i];
  p.M = (int)n.M;
  p.N = (int)n.N;
  p.kblocks = (int)ff_div(n.K, kVBK);
  p.parts = parts;
  p.units_m = (int)ff_div(n.M, 128 * t.cg);
  p.units_n = (int)ff_div(n.N, cols);
  p.units = p.units_m * p.units_n * parts;
  p.a_mn = a_mn;
  p.b_mn = b_mn;
  // Boxes of the rows there are leave the shared memory behind them as it was: rows past M, which nobody reads.
  p.a_rows = t.cg == 1 && !a_mn && n.M < 128 ? (int)ff_up(n.M, 8) : 128;
  p.idesc = idesc_f16(128 * t.cg, t.bn, f.dtype, a_mn, b_mn);
  p.out = out;
  p.ldo = ldo;
  p.sectors = (reinterpret_cast<uintptr_t>(out) & 31) == 0 && ldo % 16 == 0;
  p.part = part;
  f.units += p.units;
  if (a_mn)
    IG_VMAP(&maps.a[i], A.p, n.M, n.K, A.ld, 64, kVBK, f.dtype, false);
  else
    IG_VMAP(&maps.a[i], A.p, n.K, n.M, A.ld, kVBK, p.a_rows, f.dtype, false);
  if (b_mn)
    IG_VMAP(&maps.b[i], B.p, n.N, n.K, B.ld, 64, kVBK, f.dtype, false);
  else
    IG_VMAP(&maps.b[i], B.p, n.K, n.N, B.ld, kVBK, box_b, f.dtype, false);
  return 0;
}

// Whether h's products (grad: dh's) take the small tile: less estimated time, whole rounds of tiles.
static bool ff_inner_small(const FfSizes &s, bool grad) {
  // h's tiles take twice its columns.
  const FfShapeOf cost{s.rows, grad ? s.I : 2 * (int64_t)s.I, grad ? s.O : s.H};
  double time[2];
  for (int small = 0; small < 2; small++) {
    const FfTile &t = small ? kFfSmall : kFfLarge;
    time[small] = (double)ff_div(ff_div(cost.M, 128 * t.cg) * ff_div(cost.N, t.bn), num_sms() / t.cg) *
                  (ff_div(cost.K, kVBK) * t.block + t.tile);
  }
  return time[1] < time[0];
}

// h (and a, b), or [da | db], of the rows.
template <int EPI>
static int ff_inner(const FfMatrix &a, const FfMatrix &w, const FfSizes &s, int dtype, int act, void *out, int64_t ldo, float4 *z,
                    cudaStream_t st) {
  const FfShapeOf n{s.rows, s.I, EPI == kFfForward ? s.H : s.O};
  const bool small = ff_inner_small(s, EPI == kFfGrad);
  const FfTile &t = small ? kFfSmall : kFfLarge;
  FfMaps maps;
  FfArgs f;
  f.count = f.units = 0;
  f.dtype = dtype;
  f.z = z;
  const int cols = EPI == kFfForward ? t.bn / 2 : t.bn;
  IG_TRY(ff_add(maps, f, t, a, false, w, EPI == kFfGrad, n, EPI == kFfForward && !small ? 128 : cols, cols, 1, out, ldo, nullptr));
  if (EPI == kFfForward)
    IG_VMAP(&maps.b[1], static_cast<const uint16_t *>(w.p) + s.I * w.ld, s.H, s.I, w.ld, kVBK, small ? cols : 128, dtype, false);
  auto go = [&](auto act_) {
    constexpr int A = decltype(act_)::value;
    return small ? ff_launch<1, 64, EPI, A>(maps, f, st) : ff_launch<2, 256, EPI, A>(maps, f, st);
  };
  using std::integral_constant;
  IG_CU(act == IG_ACT_GELU        ? go(integral_constant<int, IG_ACT_GELU>())
        : act == IG_ACT_GELU_TANH ? go(integral_constant<int, IG_ACT_GELU_TANH>())
                                  : go(integral_constant<int, IG_ACT_SILU>()));
  return 0;
}

// Runs a list of products, and adds up the parts of those that have more than one.
static int ff_products(const FfMaps &maps, FfArgs &f, bool small, cudaStream_t st) {
  IG_CU(small ? (ff_launch<1, 64, kFfProduct, 0>(maps, f, st)) : (ff_launch<2, 256, kFfProduct, 0>(maps, f, st)));
  FfSumArgs sum{};
  sum.dtype = f.dtype;
  int64_t pieces = 0;
  for (int i = 0; i < f.count; i++) {
    const FfProblem &p = f.p[i];
    if (p.parts == 1) continue;
    const int64_t n = ff_div(p.M, 32) * ff_div(p.N, 32);
    sum.s[sum.count++] = FfSum{p.part, p.out, p.ldo, p.M, p.N, p.parts, n};
    pieces += n;
  }
  if (pieces) IG_CU(launch_dep(ff_sum_kernel, dim3((unsigned)pieces), dim3(128), 0, st, sum));
  return 0;
}

// Columns that one access takes: 8, 2 or 1, by where the rows start.
static int ff_vec(const FfMatrix &m) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(m.p) | (uintptr_t)(m.ld * 2);
  return at % 16 == 0 ? 8 : at % 4 == 0 ? 2 : 1;
}
template <int R>
static cudaError_t ff_rows(const FfRowsArgs &a, int vec_in, int vec_out, cudaStream_t st) {
  const dim3 gi((unsigned)ff_div(a.I, 4)), go((unsigned)ff_div(a.O, 4));
  const cudaError_t e = vec_in == 8   ? launch_dep(ff_rows_in_kernel<R, 8>, gi, dim3(128), 0, st, a)
                        : vec_in == 2 ? launch_dep(ff_rows_in_kernel<R, 2>, gi, dim3(128), 0, st, a)
                                      : launch_dep(ff_rows_in_kernel<R, 1>, gi, dim3(128), 0, st, a);
  if (e != cudaSuccess) return e;
  return vec_out == 8   ? launch_dep(ff_rows_out_kernel<R, 8>, go, dim3(128), 0, st, a)
         : vec_out == 2 ? launch_dep(ff_rows_out_kernel<R, 2>, go, dim3(128), 0, st, a)
                        : launch_dep(ff_rows_out_kernel<R, 1>, go, dim3(128), 0, st, a);
}

static int run_gated_ff(FfMatrix x, FfMatrix wi, FfMatrix wo, const FfSizes &s, const FfPlan &p, int dtype, int act, void *y, int64_t ldy,
                        uint8_t *saved, uint8_t *ws, cudaStream_t st) {
  if (ff_few(s, saved != nullptr)) {
    FfRowsArgs a{x.p, wi.p, wo.p, x.ld, wi.ld, wo.ld, (int)s.rows, s.H, (int64_t)s.I, (int64_t)s.O, dtype, act, reinterpret_cast<float *>(ws), ff_ld(s.I),
                 y, ldy};
    const int in = std::min(ff_vec(x), ff_vec(wi)), out = ff_vec(wo);
    IG_CU(s.rows == 1 ? ff_rows<1>(a, in, out, st) : s.rows == 2 ? ff_rows<2>(a, in, out, st) : ff_rows<kFfRows>(a, in, out, st));
    return 0;
  }
  FfMatrix none{};
  IG_CU(ff_pack({&x, &wi, &wo, &none}, s, p, ws, st));
  ws += p.pack_bytes;
  uint8_t *h = saved;
  if (!saved) {
    h = ws;
    ws += p.h_bytes;
  }
  const int64_t ldh = ff_ld(s.I);
  IG_TRY(ff_inner<kFfForward>(x, wi, s, dtype, act, h, ldh, saved ? reinterpret_cast<float4 *>(saved + p.h_bytes) : nullptr, st));
  const FfTile &t = p.cut.small ? kFfSmall : kFfLarge;
  FfMaps maps;
  FfArgs f;
  f.count = f.units = 0;
  f.dtype = dtype;
  f.z = nullptr;
  IG_TRY(ff_add(maps, f, t, FfMatrix{h, ldh}, false, wo, false, FfShapeOf{s.rows, s.O, s.I}, t.bn / t.cg, t.bn, p.cut.parts[0], y, ldy,
                reinterpret_cast<float4 *>(ws)));
  return ff_products(maps, f, p.cut.small, st);
}

static int run_gated_ff_grad(FfMatrix dy, FfMatrix x, FfMatrix wi, FfMatrix wo, const FfSizes &s, const FfPlan &p, int dtype,
                             int act, const uint8_t *saved, void *dx, int64_t lddx, void *dwi, int64_t lddi, void *dwo, int64_t lddo,
                             uint8_t *ws, cudaStream_t st) {
  IG_CU(ff_pack({&x, &wi, &wo, &dy}, s, p, ws, st));
  uint8_t *dz = ws + p.pack_bytes, *part = dz + p.dz_bytes;
  const FfMatrix h{saved, ff_ld(s.I)}, z{dz, p.ldz};
  if (dx || dwi) {
    IG_TRY(ff_inner<kFfGrad>(dy, wo, s, dtype, act, dz, p.ldz, reinterpret_cast<float4 *>(const_cast<uint8_t *>(saved) + p.h_bytes),
                             st));
  }
  const FfTile &t = p.cut.small ? kFfSmall : kFfLarge;
  FfMaps maps;
  FfArgs f;
  f.count = f.units = 0;
  f.dtype = dtype;
  f.z = nullptr;
  float4 *to[3];
  for (int i = 0; i < 3; i++) to[i] = reinterpret_cast<float4 *>(part + p.cut.off[i]);
  const int *parts = p.cut.parts;
  if (dwi) IG_TRY(ff_add(maps, f, t, z, true, x, true, FfShapeOf{2 * (int64_t)s.I, s.H, s.rows}, 0, t.bn, parts[0], dwi, lddi, to[0]));
  if (dwo) IG_TRY(ff_add(maps, f, t, dy, true, h, true, FfShapeOf{s.O, s.I, s.rows}, 0, t.bn, parts[1], dwo, lddo, to[1]));
  if (dx) IG_TRY(ff_add(maps, f, t, z, false, wi, true, FfShapeOf{s.rows, s.H, 2 * (int64_t)s.I}, 0, t.bn, parts[2], dx, lddx, to[2]));
  return ff_products(maps, f, p.cut.small, st);
}

}  // namespace ig
