// Vocabulary operators from hidden states: logits = hidden . weight^T on the
// tensor cores (tcgen05 kind::f16, bf16 or f16 operands, float32
// accumulators in TMEM) without ever storing them, and the gradients.
//
// One persistent kernel serves the four products:
//   statistics  rows x vocab, K = hidden: the epilogue keeps each row's
//               running (m, s, u) (vocab_rows.cu) in registers over the
//               column tiles of its unit and writes one partial per unit, and
//               for the alternatives the maximum of every 16 columns: the K
//               best columns lie in the K best groups, whose logits the
//               joining kernel computes again (16 K dot products a row);
//   dZ          the same product again (a row's logits cost less to compute
//               than to store and read back), turned into the gradient of the
//               logits, rounded to the operands' type and stored;
//   dhidden     dZ . weight, K = vocab, split over K with float32 partials;
//   dweight     dZ^T . hidden, K = rows.
// The last two read operands whose rows run along M or N instead of K: the
// TMA boxes are then 64 (M or N) x 64 (K) and the matrix descriptors
// MN-major, so nothing is transposed in memory.
//
// 4096 x 65536 x 768 bf16, one call at a time: the forward takes 323 us (1,280
// TFLOP/s) where the library's product alone takes 297 and stores the logits;
// the backward 966 us for its three products (1,280 TFLOP/s). The power limit
// sets the rate of long runs: 1.38 ms for 4096 x 262144 x 768 back to back
// (1,190 TFLOP/s, 85% of the measured sustained rate), 1.21 ms one at a time.
//
// Tiles are 256 x 256 on a CTA pair (cta_group::2: each CTA holds half of
// either operand, 32 KB per 64 of K, where one CTA alone would fetch 48 KB
// per 128 x 256) or 128 x 256 on one CTA for at most 128 rows, which leaves
// every SM its own stream of the weights (one row x 262144 x 768: 69 us, 5.9
// TB/s; 94 with operand boxes of 128 rows instead of the rows there are). Two
// accumulators of 256 TMEM columns let the epilogue of one tile run under the
// next one's products.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "common.cuh"
#include "internal.h"

namespace ig {

enum VEpi : int { kVStats = 0, kVDz = 1, kVOut = 2 };

constexpr int kVBN = 256;   // tile columns
constexpr int kVBK = 64;    // 16-bit elements of K per stage (128 bytes)
// Sixteen epilogue warps, four per scheduler, a quarter of the tile's columns
// each: with eight, 4096 x 65536 x 256 took 184 us forward and 546 us backward,
// with sixteen 170 and 488, and one row's gradients at 262144 x 768 326 and 311;
// where K is 768 or more and the rows are many the products cover either
// (within 1%).
constexpr int kVEpiWarps = 16;
constexpr int kVEpiGroups = kVEpiWarps / 4;      // warps per TMEM lane quarter
constexpr int kVEpiCols = kVBN / kVEpiGroups;    // tile columns of a warp
constexpr int kVGemmThreads = 64 + 32 * kVEpiWarps;

// Row coefficients of dZ (RowCoef with the output scale applied by the reader).
struct VRowCoef {
  float A, B, l, pad;
};

constexpr int kVGroup = 16;  // columns per stored maximum
// The tensor cores' sums are cut off, not rounded: a logit of 10 from 1000
// terms comes out 1e-5 low, and lse by that times the column's probability.
// Against a logit summed with rounding, the log probability of a token that
// takes most of its row (-0.13 in the mean) was off by 6e-5 of itself. For at
// most this many given tokens a row the accumulator's own logit is kept too,
// and the row's lse is corrected by what it is short. More tokens make it less
// likely that one is the likeliest of the row, and a row's look-up grows with
// their number: 4096 x 65536 x 256 takes 150 us without, 155 with one token and
// 162 with eight.
constexpr int kVCaught = 8;
// The lowest of a row's given tokens that is at least `from` and lies in the
// columns of epilogue group g.
__device__ __forceinline__ int next_given(const int32_t *ids, int T, int from, int g) {
  int m = 0x7FFFFFFF;
#pragma unroll
  for (int t = 0; t < kVCaught; t++) {
    const int id = t < T ? ids[t] : -1;
    if (id >= from && id < m && id / kVEpiCols % kVEpiGroups == g) m = id;
  }
  return m;
}

struct VGemmArgs {
  int M, N;
  int kblocks;  // blocks of kVBK of K
  int kparts;   // 2: blocks come in pairs, one of either part of A (`shift` elements apart along its rows) with one of B
  int shift;
  uint32_t idesc;
  int units_m, units_n, units_s;  // units: M tiles x N parts x K parts
  int a_rows;  // rows of A's box (one CTA per tile: the rows there are, rounded up to 8; else 128)
  int n_fastest;                  // unit order: N parts innermost, else M tiles
  float c, c2;  // 1 / temperature, log2(e) / temperature
  // kVStats: [M][units_n * kVEpiGroups] partials; group maxima [M][ldmax] or NULL
  float4 *part;
  float *gmax;
  int64_t ldmax;
  const int32_t *ids;  // [M][T]: their logits go to xid [M][T]; T = 0: none
  int T;
  float *xid;
  // kVDz
  const VRowCoef *coef;
  int split;  // dZ as two 16-bit parts, the second `shift` elements on
  // kVDz, kVOut: dtype of the 16-bit output; bits of dZ's bound (vocab_scale), NULL: unscaled
  int dtype;
  const int *bound;
  // kVOut: out16 (final) or part32 [units_s][M][ldo] (accumulate: added to what is there)
  void *out16;
  int64_t ldo;
  float *part32;
  int accumulate;
};

// float16 has 5 exponent bits: dZ is scaled by a power of two that brings the
// largest bound of the rows to 2^14..2^15, so that probabilities down to
// 2^-28 of it keep all their bits; the products' float32 sums are scaled
// back. bfloat16 has float32's range and needs none.
__device__ __forceinline__ float vocab_scale(const int *bound) {
  if (!bound) return 1.0f;
  const int b = *bound;
  if (b <= 0) return 1.0f;
  const int e = min(max(14 - (((b >> 23) & 255) - 127), -100), 100);
  return __int_as_float((e + 127) << 23);
}

template <int CG, int EPI>
struct VSmem {
  static constexpr int kABytes = 128 * kVBK * 2;
  static constexpr int kBBytes = (kVBN / CG) * kVBK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  // Staging per warp: two buffers for dZ's bulk stores, one to turn rows for the plain 16-bit stores.
  static constexpr int kExtra = EPI == kVDz ? kVEpiWarps * 2 * 2048 : EPI == kVOut ? kVEpiWarps * 2048 : 0;
  static constexpr int kRaw = (224 * 1024 - kExtra) / kStageBytes;
  static constexpr int kStages = kRaw > 6 ? 6 : kRaw;
  static constexpr int kExtraOff = kStages * kStageBytes;
  static constexpr int kBar = kExtraOff + kExtra;
  static constexpr int kTmemSlot = kBar + 8 * (2 * kStages + 4);
  static constexpr int kTotal = kTmemSlot + 16 + 1024;
  static_assert(kStages >= 3, "three stages at least");
  static_assert(kTotal <= 227 * 1024, "shared memory");
};

// MN-major operand, 128-byte swizzle: 64 M (or N) x 8 K atoms of 1024 bytes;
// the next 8 of K 1024 bytes on, the next 64 of M one box (64 K) on.
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFFu) >> 4);
  d |= (uint64_t)((64 * kVBK * 2) >> 4) << 16;  // leading byte offset
  d |= (uint64_t)(1024 >> 4) << 32;             // stride byte offset
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// Instruction descriptor for kind::f16: D float32, A and B both f16 or both bf16.
static uint32_t idesc_f16(int M, int N, int dtype, bool a_mn, bool b_mn) {
  const uint32_t f = dtype == IG_DT_BF16 ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}

template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}

struct VUnit {
  int m, n, s;    // M tile, N part, K part
  int n0, n1;     // column tiles
  int k0, k1;     // K blocks
};
__device__ __forceinline__ VUnit vunit(const VGemmArgs &a, int u, int ntiles) {
  VUnit r;
  if (a.n_fastest) {
    r.n = u % a.units_n;
    u /= a.units_n;
    r.m = u % a.units_m;
    r.s = u / a.units_m;
  } else {
    r.m = u % a.units_m;
    u /= a.units_m;
    r.n = u % a.units_n;
    r.s = u / a.units_n;
  }
  r.n0 = (int)((int64_t)ntiles * r.n / a.units_n);
  r.n1 = (int)((int64_t)ntiles * (r.n + 1) / a.units_n);
  r.k0 = (int)((int64_t)a.kblocks * r.s / a.units_s);
  r.k1 = (int)((int64_t)a.kblocks * (r.s + 1) / a.units_s);
  return r;
}

__device__ __forceinline__ float2 widen2(uint32_t v, int dtype) {
  if (dtype == IG_DT_BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}
__device__ __forceinline__ float widen1(uint16_t v, int dtype) {
  if (dtype == IG_DT_BF16) return __uint_as_float((uint32_t)v << 16);
  return __half2float(*reinterpret_cast<const __half *>(&v));
}

__device__ __forceinline__ uint32_t pack16(float a, float b, int dtype) {
  if (dtype == IG_DT_BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void store16(void *p, int64_t i, float v, int dtype) {
  if (dtype == IG_DT_BF16)
    static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
  else
    static_cast<__half *>(p)[i] = __float2half_rn(v);
}

template <int CG, bool A_MN, bool B_MN, int EPI>
__global__ void __launch_bounds__(kVGemmThreads, 1)
    vocab_gemm_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB,
                      const __grid_constant__ CUtensorMap mapC, const VGemmArgs a) {
  using S = VSmem<CG, EPI>;
  constexpr int kStages = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + S::kBar);
  uint64_t *empty = full + kStages;
  uint64_t *accf = empty + kStages;
  uint64_t *acce = accf + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + S::kTmemSlot);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CG == 2 ? (int)cluster_ctarank() : 0;
  const int first = blockIdx.x / CG, step = gridDim.x / CG;
  const int ntiles = (a.N + kVBN - 1) / kVBN;
  const int units = a.units_m * a.units_n * a.units_s;

  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&mapA);
    prefetch_tensormap(&mapB);
    for (int s = 0; s < kStages; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(&accf[b], 1);
      mbar_init(&acce[b], CG * kVEpiWarps);
    }
    fence_barrier_init();
  }
  if (warp == 1) {
    if constexpr (CG == 2)
      tmem_alloc_pair(tmem_slot, 2 * kVBN);
    else
      tmem_alloc(tmem_slot, 2 * kVBN);
  }
  tc_fence_before();
  if constexpr (CG == 2)
    cluster_sync_all();
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  dep_wait();

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int u = first; u < units && ok; u += step) {
        const VUnit q = vunit(a, u, ntiles);
        const int m0 = q.m * (CG * 128) + rank * 128;
        for (int n = q.n0; n < q.n1 && ok; n++) {
          const int n0 = n * kVBN + rank * (kVBN / CG);
          for (int kb = q.k0; kb < q.k1; kb++, it++) {
            const int s = it % kStages;
            if (!mbar_wait(&empty[s], ((it / kStages) & 1) ^ 1, kDevTimeoutEmpty)) {
              ok = false;
              break;
            }
            uint8_t *sa = smem + s * S::kStageBytes, *sb = sa + S::kABytes;
            if (rank == 0) mbar_arrive_expect_tx(&full[s], CG * (S::kBBytes + a.a_rows * kVBK * 2));
            auto load = [&](const CUtensorMap *map, uint8_t *dst, int c0, int c1) {
              if constexpr (CG == 2)
                tma_load_2d_pair(map, dst, cluster_addr(&full[s], 0), c0, c1);
              else
                tma_load_2d(map, dst, &full[s], c0, c1);
            };
            const int kc = (a.kparts == 2 ? kb >> 1 : kb) * kVBK, as = a.kparts == 2 && (kb & 1) ? a.shift : 0;
            if constexpr (A_MN) {
#pragma unroll
              for (int i = 0; i < 2; i++) load(&mapA, sa + i * 8192, as + m0 + i * 64, kc);
            } else {
              load(&mapA, sa, as + kc, m0);
            }
            if constexpr (B_MN) {
#pragma unroll
              for (int i = 0; i < kVBN / CG / 64; i++) load(&mapB, sb + i * 8192, n0 + i * 64, kc);
            } else {
              load(&mapB, sb, kc, n0);
            }
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
      for (int u = first; u < units && ok; u += step) {
        const VUnit q = vunit(a, u, ntiles);
        for (int n = q.n0; n < q.n1 && ok; n++, tile++) {
          const int b = tile & 1;
          if (!mbar_wait(&acce[b], ((tile >> 1) & 1) ^ 1, kDevTimeoutEmpty)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d = tmem + b * kVBN;
          for (int kb = q.k0; kb < q.k1; kb++, it++) {
            const int s = it % kStages;
            if (!mbar_wait(&full[s], (it / kStages) & 1, kDevTimeoutFull)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t sa = smem_u32(smem + s * S::kStageBytes), sb = sa + S::kABytes;
#pragma unroll
            for (int kk = 0; kk < kVBK / 16; kk++) {
              const uint64_t da = A_MN ? smem_desc_mn_sw128(sa + kk * 2048) : smem_desc_k_sw128(sa + kk * 32);
              const uint64_t db = B_MN ? smem_desc_mn_sw128(sb + kk * 2048) : smem_desc_k_sw128(sb + kk * 32);
              mma_f16<CG>(d, da, db, a.idesc, (kb > q.k0 || kk > 0) ? 1u : 0u);
            }
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
    }
  } else {
    // TMEM lane quarter; columns [kCols g, kCols g + kCols).
    constexpr int kCols = kVEpiCols;
    const int q4 = warp & 3, e = warp - 2, g = e >> 2;
    int tile = 0;
    bool ok = true;
    [[maybe_unused]] int stores = 0;
    for (int u = first; u < units && ok; u += step) {
      const VUnit q = vunit(a, u, ntiles);
      const int row0 = q.m * (CG * 128) + rank * 128 + q4 * 32, row = row0 + lane;
      const bool warp_live = row0 < a.M, live = row < a.M;
      [[maybe_unused]] VStat st{-IG_INF, 0.0f, 0.0f};
      [[maybe_unused]] int next = 0x7FFFFFFF;  // the row's next given column to catch
      if constexpr (EPI == kVStats) {
        if (live && a.T > 0) next = next_given(a.ids + (int64_t)row * a.T, a.T, q.n0 * kVBN, g);
      }
      [[maybe_unused]] RowCoef rc{0.0f, 0.0f, 0.0f};
      [[maybe_unused]] bool hold = false;
      if constexpr (EPI == kVDz) {
        if (live) {
          const VRowCoef v = a.coef[row];
          const float sc = vocab_scale(a.bound);
          rc = RowCoef{v.A * sc, v.B * sc, v.l};
        }
        // One more operation an element, for the warps that need it: 8192 x
        // 50021 x 768 1,677 us with it everywhere, 1,663 so.
        hold = __any_sync(~0u, !(fabsf(rc.l) <= kLseMost));
      }
      [[maybe_unused]] float unscale = 1.0f;
      if constexpr (EPI == kVOut) {
        if (a.out16) unscale = 1.0f / vocab_scale(a.bound);
      }
      for (int n = q.n0; n < q.n1; n++, tile++) {
        const int b = tile & 1;
        if (!mbar_wait(&accf[b], (tile >> 1) & 1, kDevTimeoutAccum)) {
          ok = false;
          break;
        }
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
        if (!warp_live) {
          release();
          continue;
        }
        const uint32_t tb = tmem + b * kVBN + ((uint32_t)(q4 * 32) << 16);
        constexpr int kChunks = kCols / 32;
        [[maybe_unused]] float gm[2 * kChunks];
#pragma unroll
        for (int i = 0; i < kChunks; i++) {
          __syncwarp();  // the branches below are per lane; the TMEM loads take the whole warp
          uint32_t r[32];
          tmem_ld_32x32b_x32(tb + g * kCols + 32 * i, r);
          tmem_ld_wait();
          if (i + 1 == kChunks) release();
          const int col0 = n * kVBN + g * kCols + 32 * i;
          if constexpr (EPI != kVDz) {
            if (col0 >= a.N) {
              if constexpr (EPI == kVStats) gm[2 * i] = gm[2 * i + 1] = -IG_INF;
              continue;
            }
          }
          float x[32];
#pragma unroll
          for (int k = 0; k < 32; k++) x[k] = __uint_as_float(r[k]);
          if constexpr (EPI == kVStats) {
            if (col0 + 32 > a.N) {
#pragma unroll
              for (int k = 0; k < 32; k++)
                if (col0 + k >= a.N) x[k] = -IG_INF;
            }
            while (next < col0 + 32) {  // seldom
              const int32_t *ids = a.ids + (int64_t)row * a.T;
              const int at = next - col0;
              float v = x[0];
#pragma unroll
              for (int k = 1; k < 32; k++) v = at == k ? x[k] : v;
#pragma unroll
              for (int t = 0; t < kVCaught; t++)
                if (t < a.T && ids[t] == next) a.xid[(int64_t)row * a.T + t] = v;
              next = next_given(ids, a.T, next + 1, g);
            }
            float m4[4] = {x[0], x[1], x[16], x[17]};
#pragma unroll
            for (int k = 2; k < 16; k += 2) {
              m4[0] = fmaxf(m4[0], x[k]);
              m4[1] = fmaxf(m4[1], x[k + 1]);
              m4[2] = fmaxf(m4[2], x[k + 16]);
              m4[3] = fmaxf(m4[3], x[k + 17]);
            }
            gm[2 * i] = fmaxf(fmaxf(m4[0], m4[1]), -IG_INF);
            gm[2 * i + 1] = fmaxf(fmaxf(m4[2], m4[3]), -IG_INF);
            vstat_add<true>(st, x, fmaxf(gm[2 * i], gm[2 * i + 1]), a.c2);
          } else if constexpr (EPI == kVDz) {
            float d[32];
            auto dense = [&](auto held) {
#pragma unroll
              for (int k = 0; k < 32; k += 2) {
                const float2 v = dense_grad2<decltype(held)::value>(make_float2(x[k], x[k + 1]), a.c, rc);
                d[k] = v.x;
                d[k + 1] = v.y;
              }
            };
            if (hold)
              dense(std::true_type());
            else
              dense(std::false_type());
            if (col0 + 32 > a.N) {
              // Zero up to the tile's end: dhidden's last block of K reads it.
#pragma unroll
              for (int k = 0; k < 32; k++)
                if (col0 + k >= a.N) d[k] = 0.0f;
            }
            for (int part = 0; part <= a.split; part++) {
              uint8_t *buf = smem + S::kExtraOff + (e * 2 + (stores & 1)) * 2048;
              if (lane == 0) bulk_wait_read<1>();
              __syncwarp();
              uint32_t w[16];
#pragma unroll
              for (int k = 0; k < 16; k++) {
                w[k] = pack16(d[2 * k], d[2 * k + 1], a.dtype);
                if (a.split) {  // what this part leaves of d
                  const float2 v = widen2(w[k], a.dtype);
                  d[2 * k] -= v.x;
                  d[2 * k + 1] -= v.y;
                }
              }
#pragma unroll
              for (int j = 0; j < 4; j++)
                *reinterpret_cast<uint4 *>(buf + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) =
                    make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                tma_store_2d(&mapC, buf, part * a.shift + col0, row0);
                bulk_commit();
              }
              stores++;
            }
          } else {
            if (a.out16) {
              // A thread holds a row's 32 columns; through shared memory four
              // lanes store a row's 64 bytes, whole sectors (a thread storing
              // its own row 16 bytes at a time took 222 us for the 402 MB of
              // one row's dweight, 262144 x 768).
              uint8_t *buf = smem + S::kExtraOff + e * 2048;
              __syncwarp();
#pragma unroll
              for (int j = 0; j < 4; j++)
                *reinterpret_cast<uint4 *>(buf + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) =
                    make_uint4(pack16(x[8 * j] * unscale, x[8 * j + 1] * unscale, a.dtype),
                               pack16(x[8 * j + 2] * unscale, x[8 * j + 3] * unscale, a.dtype),
                               pack16(x[8 * j + 4] * unscale, x[8 * j + 5] * unscale, a.dtype),
                               pack16(x[8 * j + 6] * unscale, x[8 * j + 7] * unscale, a.dtype));
              __syncwarp();
#pragma unroll
              for (int i8 = 0; i8 < 4; i8++) {
                const int r8 = i8 * 8 + (lane >> 2), j = lane & 3, col = col0 + 8 * j;
                if (row0 + r8 >= a.M || col >= a.N) continue;
                const uint4 v = *reinterpret_cast<const uint4 *>(buf + r8 * 64 + ((j ^ ((r8 >> 1) & 3)) << 4));
                uint16_t *dst = static_cast<uint16_t *>(a.out16) + (int64_t)(row0 + r8) * a.ldo + col;
                if (col + 8 <= a.N && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
                  *reinterpret_cast<uint4 *>(dst) = v;
                } else {
                  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                  for (int k = 0; k < 8; k++)
                    if (col + k < a.N) dst[k] = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
                }
              }
            } else if (live) {
              // part32 rows are padded to a multiple of 4 floats.
              float *dst = a.part32 + ((int64_t)q.s * a.M + row) * a.ldo + col0;
#pragma unroll
              for (int k = 0; k < 32; k += 4) {
                if (col0 + k >= a.N) break;
                float4 v = make_float4(x[k], x[k + 1], x[k + 2], x[k + 3]);
                if (a.accumulate) {
                  const float4 o = *reinterpret_cast<const float4 *>(dst + k);
                  v = make_float4(v.x + o.x, v.y + o.y, v.z + o.z, v.w + o.w);
                }
                *reinterpret_cast<float4 *>(dst + k) = v;
              }
            }
          }
        }
        if constexpr (EPI == kVStats) {
          if (a.gmax && live) {
            static_assert(kCols / kVGroup == 4, "one float4 of maxima");
            *reinterpret_cast<float4 *>(a.gmax + (int64_t)row * a.ldmax + n * (kVBN / kVGroup) + g * 4) =
                make_float4(gm[0], gm[1], gm[2], gm[3]);
          }
        }
      }
      if constexpr (EPI == kVStats) {
        if (ok && live) a.part[((int64_t)row * a.units_n + q.n) * kVEpiGroups + g] = make_float4(st.m, st.s, st.u, 0.0f);
      }
    }
    if constexpr (EPI == kVDz) {
      if (lane == 0) bulk_wait_all();
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
      tmem_dealloc_pair(tmem, 2 * kVBN);
    else
      tmem_dealloc(tmem, 2 * kVBN);
  }
}

// ---- joining the partials, the given tokens' and the alternatives' dot products ---------

struct VJoinArgs {
  const uint16_t *h, *w;
  int64_t ldh, ldw;
  int V, H, T, K, parts, dtype;
  float c;
  const int32_t *ids;
  const float4 *part;
  const float *xid;  // the given tokens' logits as accumulated, or NULL
  const float *gmax;
  int64_t ldmax;
  int ngroups;
  float *logprobs, *lse, *entropy;
  int32_t *top_ids;
  float *top_logprobs;
};

// One CTA per row: the statistics of the row's parts, then the dot products of
// the given tokens and of the best groups' columns, eight lanes each (128
// bytes of either operand a step). A logit summed here is float32 in another
// order than the tensor core's: `full` against `cut`, lse is short by
// p c (full - cut) of the column's probability p, which a log probability of
// that column, or of one beside the row's best, takes back.
__device__ __forceinline__ float back(float x, float p, float full, float cut) {
  return p > 0.0f ? fmaf(-p, full - cut, x) : x;
}
template <bool TOP>
__global__ void __launch_bounds__(kVocThreads) vocab_join_kernel(const VJoinArgs a) {
  __shared__ VStat s_warp[kVocWarps];
  __shared__ float s_dot[kIdsMax];
  __shared__ TopShared<kVocThreads> s_top[1];
  __shared__ float s_oval[kTopMax];
  __shared__ int s_ocol[kTopMax];
  __shared__ int s_on, s_left;
  const int64_t row = blockIdx.x;
  const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31, nthreads = (int)blockDim.x;
  const float c2 = a.c * kLog2e;
  if (tid == 0) s_left = 0;
  dep_wait();
  float xid = 0.0f;  // asked for early
  if (a.xid && tid < a.T) xid = a.xid[row * a.T + tid];
  VStat st{-IG_INF, 0.0f, 0.0f};
  for (int p = tid; p < a.parts; p += nthreads) {
    const float4 v = a.part[row * a.parts + p];
    vstat_merge<true>(st, VStat{v.x, v.y, v.z}, c2);
  }
  st = vstat_warp<true>(st, c2);
  if (lane == 0) s_warp[warp] = st;
  if constexpr (TOP) {
    // The best groups of columns.
    const RowVecs<IG_DT_F32> rv(a.gmax + row * a.ldmax, a.ngroups);
    const RowPart<IG_DT_F32> rp(rv, 0, 1);
    uint32_t m = VElem<IG_DT_F32>::kNegInf;
    constexpr int kAhead = 8;
    for (int i = tid; i < rp.n; i += kAhead * kVocThreads) {
      uint4 v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; j++)
        v[j] = rp.base[min(i + j * kVocThreads, i + (rp.n - 1 - i) / kVocThreads * kVocThreads)];  // the last again past the end
#pragma unroll
      for (int j = 0; j < kAhead; j++)
        m = VElem<IG_DT_F32>::hmax(m, VElem<IG_DT_F32>::hmax(VElem<IG_DT_F32>::hmax(v[j].x, v[j].y),
                                                             VElem<IG_DT_F32>::hmax(v[j].z, v[j].w)));
    }
    if (tid == last_thread(kVocThreads) && rp.last)
      for (int i = rv.col(rp.v1 - 1); i < a.ngroups; i++) m = VElem<IG_DT_F32>::hmax(m, __float_as_uint(rv.row[i]));
    top_select<IG_DT_F32, kVocThreads>(rv, rp, __uint_as_float(m), a.K, s_top[0], s_oval, s_ocol, &s_on);
  } else {
    if (tid == 0) s_on = 0;
  }
  __syncthreads();
  st = vstat_join<true>(s_warp, nthreads / 32, c2);
  float log_s, lse, entropy;
  row_lse(st, a.c, log_s, lse, entropy);
  if (tid == 0) {
    if (a.lse) a.lse[row] = lse;
    if (a.entropy) a.entropy[row] = entropy;
  }
  const int cand = s_on * kVGroup, total = a.T + cand;
  const uint16_t *h = a.h + row * a.ldh;
  const int sub = tid & 7;
  [[maybe_unused]] float best = -IG_INF;  // of the alternatives
  for (int d0 = 0; d0 < total; d0 += nthreads / 8) {
    const int d = d0 + (tid >> 3);
    int id = -1;
    if (d < a.T)
      id = a.ids[row * a.T + d];
    else if (d < total)
      id = s_ocol[(d - a.T) / kVGroup] * kVGroup + (d - a.T) % kVGroup;
    float s = 0.0f;
    if (id >= 0 && id < a.V) {
      const uint16_t *w = a.w + (int64_t)id * a.ldw;
      constexpr int kAhead = 6;  // loads in flight of either operand
      const int h8 = a.H & ~7;
      for (int i0 = sub * 8; i0 < h8; i0 += 64 * kAhead) {
        uint4 x[kAhead], y[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
          const int i = i0 + 64 * j;
          x[j] = y[j] = make_uint4(0, 0, 0, 0);
          if (i < h8) {
            x[j] = *reinterpret_cast<const uint4 *>(h + i);
            y[j] = __ldg(reinterpret_cast<const uint4 *>(w + i));
          }
        }
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
          const uint32_t xs[4] = {x[j].x, x[j].y, x[j].z, x[j].w}, ys[4] = {y[j].x, y[j].y, y[j].z, y[j].w};
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const float2 p = widen2(xs[k], a.dtype), q = widen2(ys[k], a.dtype);
            s = fmaf(p.x, q.x, s);
            s = fmaf(p.y, q.y, s);
          }
        }
      }
      const int tail = a.H & ~7;
      if (tail + sub < a.H) s = fmaf(widen1(h[tail + sub], a.dtype), widen1(w[tail + sub], a.dtype), s);
    }
    __syncwarp();
#pragma unroll
    for (int o = 4; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    if (sub == 0) {
      if (d < a.T) {
        s_dot[d] = s;
      } else if (TOP && d < total) {
        // A masked column of a group is no alternative.
        const bool left = id < a.V && s > -IG_INF;
        s_top[0].val[d - a.T] = left ? s : -IG_INF;
        s_top[0].col[d - a.T] = left ? id : 0x7FFFFFFF;
        if (left) {
          atomicAdd(&s_left, 1);
          best = fmaxf(best, s);
        }
      }
    }
  }
  if constexpr (TOP) {
    best = warp_max(best);
    if (lane == 0) s_top[0].wv[warp] = best;
  }
  __syncthreads();
  for (int t = tid; t < a.T; t += nthreads) {
    const int id = a.ids[row * a.T + t];
    float v = 0.0f;
    if (id >= a.V) {
      v = __int_as_float(0x7FC00000);
      set_device_error(kDevBadId);
    } else if (id >= 0) {
      float x = s_dot[t];
      if (a.xid) x = back(x, expf(row_logprob(xid, st, a.c, log_s)), x, xid);
      v = row_logprob(x, st, a.c, log_s);
    }
    a.logprobs[row * a.T + t] = v;
  }
  if constexpr (TOP) {
    const bool nan = st.s != st.s;
    for (int w = 0; w < kVocWarps; w++) best = fmaxf(best, s_top[0].wv[w]);
    for (int i = tid; i < cand && !nan; i += nthreads) {
      const float v = s_top[0].val[i];
      const int c = s_top[0].col[i];
      if (c == 0x7FFFFFFF) continue;
      int r = 0;
      for (int j = 0; j < cand; j++) r += top_before(s_top[0].val[j], s_top[0].col[j], v, c);
      if (r < a.K) {
        a.top_ids[row * a.K + r] = c;
        a.top_logprobs[row * a.K + r] = row_logprob(back(v, 1.0f / st.s, best, st.m), st, a.c, log_s);
      }
    }
    // Past the unmasked columns, or in a row that is no distribution.
    for (int k = (nan ? 0 : s_left) + tid; k < a.K; k += nthreads) {
      a.top_ids[row * a.K + k] = -1;
      a.top_logprobs[row * a.K + k] = nan ? __int_as_float(0x7FC00000) : -IG_INF;
    }
  }
}

// ---- gradient: row coefficients, given tokens, sum of the partials ---------------------

struct VCoefArgs {
  int64_t rows;
  int V, T;
  float c;
  const int32_t *ids;
  const float *lse, *entropy, *dlogprobs, *dentropy;
  VRowCoef *coef;
  int *bound;  // bits of the largest |dZ| bound of any row (positive floats order as their bits); NULL: not needed
};

// One warp per row.
__global__ void vocab_coef_kernel(const VCoefArgs a) {
  dep_trigger();  // dZ's CTAs set themselves up meanwhile
  const int64_t row = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (row >= a.rows) return;
  const int lane = threadIdx.x & 31;
  bool bad = false;
  float G = 0.0f, size = 0.0f;
  if (a.dlogprobs) {
    G = given_grad_sum(a.ids + row * a.T, a.dlogprobs + row * a.T, a.T, a.V, bad, size);
    if (bad) set_device_error(kDevBadId);
    size = warp_sum(size);
  }
  if (lane) return;
  const float gh = a.dentropy ? a.dentropy[row] : 0.0f, H = a.dentropy ? a.entropy[row] : 0.0f;
  const float lse = a.lse[row];
  // An lse at float32's end says nothing of the columns either.
  const RowCoef k = row_coef(lse == -kFltMax ? -IG_INF : lse, H, G, gh, a.c);
  a.coef[row] = VRowCoef{k.A, k.B, k.l, 0.0f};
  // |dZ| <= c (sum |g| (1 + p) + |gH| p (|log p| + H)) <= c (2 sum |g| + |gH| (1 + H)), as p <= 1
  const float b = a.c * (2.0f * size + fabsf(gh) * (1.0f + H));
  if (a.bound && k.l != IG_INF && b > 0.0f && b < 3.0e38f) atomicMax(a.bound, __float_as_int(b));
}

struct VTokenArgs {
  int64_t n;  // rows * T
  int T, v0, v1, dtype;
  float c;
  const int32_t *ids;
  const float *logprobs, *dlogprobs;
  const VRowCoef *coef;
  const int *bound;
  void *dz;
  int64_t ldz;
  int shift;  // of dZ's second part (0: none)
};

// dZ at the given tokens of columns [v0, v1): the dense part from the saved
// log probability plus the tokens' own gradients, rounded once.
__global__ void vocab_token_kernel(const VTokenArgs a) {
  dep_wait();
  dep_trigger();
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= a.n) return;
  const int64_t row = i / a.T;
  const int id = a.ids[i];
  if (id < a.v0 || id >= a.v1) return;
  const VRowCoef v = a.coef[row];
  const RowCoef k{v.A, v.B, v.l};
  if (k.l == IG_INF) return;  // no distribution
  float d = dense_grad(log_prob<true>(a.logprobs[i]), k) + token_grad(a.ids + row * a.T, a.dlogprobs + row * a.T, a.T, id, a.c);
  d *= vocab_scale(a.bound);
  const int64_t at = row * a.ldz + id - a.v0;
  const uint32_t w = pack16(d, 0.0f, a.dtype);
  static_cast<uint16_t *>(a.dz)[at] = (uint16_t)w;
  if (a.shift) store16(a.dz, at + a.shift, d - widen1((uint16_t)w, a.dtype), a.dtype);
}

// dhidden = sum over the K parts, scaled back and rounded. One CTA per row,
// four columns per thread; with many parts four groups of threads
// (threadIdx.y) take every fourth part, and their sums are added in order (37
// parts of 500 x 256: 11.2 us by one group, 7.9 by four; 3 parts of 8192 x
// 768: 20 and 90).
__global__ void __launch_bounds__(1024) vocab_sum_kernel(const float *part, int parts, int64_t rows, int H, int64_t ldp,
                                                         const int *bound, void *out, int64_t ldo, int dtype) {
  extern __shared__ float4 s_sum[];
  dep_wait();
  dep_trigger();
  const int64_t row = blockIdx.x;
  const float unscale = 1.0f / vocab_scale(bound);
  for (int c0 = 0; c0 < H; c0 += 4 * blockDim.x) {
    const int col = c0 + 4 * threadIdx.x;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (col < H) {
#pragma unroll 8
      for (int p = threadIdx.y; p < parts; p += blockDim.y) {
        const float4 v = *reinterpret_cast<const float4 *>(part + ((int64_t)p * rows + row) * ldp + col);
        s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
      }
    }
    s_sum[threadIdx.y * blockDim.x + threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && col < H) {
      for (int g = 1; g < (int)blockDim.y; g++) {
        const float4 v = s_sum[g * blockDim.x + threadIdx.x];
        s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
      }
      const float v[4] = {s.x * unscale, s.y * unscale, s.z * unscale, s.w * unscale};
      uint16_t *dst = static_cast<uint16_t *>(out) + row * ldo + col;
      if (col + 4 <= H && (reinterpret_cast<uintptr_t>(dst) & 7) == 0) {
        *reinterpret_cast<uint2 *>(dst) = make_uint2(pack16(v[0], v[1], dtype), pack16(v[2], v[3], dtype));
      } else {
        for (int k = 0; k < 4 && col + k < H; k++) store16(dst, k, v[k], dtype);
      }
    }
    __syncthreads();
  }
}

// ---- plans and launches ------------------------------------------------------------------

// 16-bit matrix [outer][inner], row stride ld elements.
static int make_map_16(CUtensorMap *map, const void *base, int64_t inner, int64_t outer, int64_t ld, int box_in, int box_out,
                       int dtype, bool swizzle64) {
  auto enc = get_encode_fn();
  if (!enc) return -1;
  cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
  cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  cuuint32_t box[2] = {(cuuint32_t)box_in, (cuuint32_t)box_out};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(map, dtype == IG_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                         const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         swizzle64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -2;
}

// CTA pairs (or CTAs) that can be resident at once.
template <int CG, bool A_MN, bool B_MN, int EPI>
static int vgemm_slots() {
  using S = VSmem<CG, EPI>;
  static SmemOptIn attr;
  if (attr.ensure((const void *)vocab_gemm_kernel<CG, A_MN, B_MN, EPI>, S::kTotal) != cudaSuccess) return 0;
  if (CG == 1) return num_sms();
  static PerDevice clusters;
  return clusters.get([] {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = CG;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(CG * (num_sms() / CG));
    cfg.blockDim = dim3(kVGemmThreads);
    cfg.dynamicSmemBytes = S::kTotal;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int c = 0;
    if (cudaOccupancyMaxActiveClusters(&c, vocab_gemm_kernel<CG, A_MN, B_MN, EPI>, &cfg) != cudaSuccess) {
      (void)cudaGetLastError();
      c = 0;
    }
    return c;
  });
}

template <int CG, bool A_MN, bool B_MN, int EPI>
static cudaError_t launch_vgemm(const CUtensorMap &ma, const CUtensorMap &mb, const CUtensorMap &mc, const VGemmArgs &a,
                                cudaStream_t st) {
  const int slots = vgemm_slots<CG, A_MN, B_MN, EPI>();
  if (slots <= 0) return cudaErrorInvalidConfiguration;
  const int64_t units = (int64_t)a.units_m * a.units_n * a.units_s;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  cfg.gridDim = dim3((unsigned)(CG * (units < slots ? units : slots)));
  cfg.blockDim = dim3(kVGemmThreads);
  cfg.dynamicSmemBytes = VSmem<CG, EPI>::kTotal;
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
  return cudaLaunchKernelEx(&cfg, vocab_gemm_kernel<CG, A_MN, B_MN, EPI>, ma, mb, mc, a);
}

// Parts (of column tiles, or of K blocks) per M tile. With `tiles` pieces to
// cut and `outer` M tiles, a cut in p parts runs ceil(outer p / slots) rounds
// of ceil(tiles / p) pieces plus a fixed overhead (in pieces); the best cuts
// fill whole rounds, so only those are tried.
static int best_parts(int64_t outer, int64_t tiles, int64_t slots, int64_t most, double overhead) {
  if (most > tiles) most = tiles;
  int64_t best = 1;
  double cost = (double)((outer + slots - 1) / slots) * ((double)tiles + overhead);
  for (int64_t rounds = (outer + slots - 1) / slots; rounds <= 64; rounds++) {
    int64_t p = rounds * slots / outer;
    if (p > most) p = most;
    if (p < 1) continue;
    const double c = (double)((outer * p + slots - 1) / slots) * ((double)((tiles + p - 1) / p) + overhead);
    if (c < cost * 0.995) {
      cost = c;
      best = p;
    }
    if (p == most) break;
  }
  return (int)best;
}

constexpr int kVMaxParts = 256;        // column parts per M tile
// At most this many rows: single CTAs (one row x 262144 x 768: 86 us, by pairs
// 113; 128 rows 88 and 92).
constexpr int kVOneCtaRows = 128;
// At most this many rows: dZ in two 16-bit parts, and the gradients as exact as
// their own type. With more rows dZ is held in the operands' type, as a caller
// that stored the logits' gradient for its products would hold it: its rounding
// adds to the gradients' own one of the same size, so they are off by 1.4 times
// what they would be with dZ in 32 bits (0.0024 against 0.0017 in the norm in
// bfloat16, 0.00030 against 0.00021 in float16; at 129 rows up to 1.5 times,
// as few rows do not average). Two parts for all rows would double K in two of
// the three products (256 x 262144 x 768: 385 us in one, 508 in two).
constexpr int kVSplitRows = 128;
constexpr int64_t kVDzBytes = 1ll << 30;  // dZ is formed in column chunks of at most this size

struct VPlan {
  int64_t rows;
  int V, H;
  int cg, a_rows;
  int units_m, units_n;  // statistics
  int64_t ldmax;
  size_t part_bytes, max_bytes, fwd_bytes;
  // backward
  bool split;
  int64_t chunk, ldz, ldp;
  int ks;
  size_t coef_bytes, dz_bytes, bwd_bytes;
};

static VPlan vocab_plan(int64_t rows, int V, int H, int top_k) {
  VPlan p{};
  p.rows = rows;
  p.V = V;
  p.H = H;
  p.cg = rows <= kVOneCtaRows ? 1 : 2;
  p.a_rows = p.cg == 1 ? (int)((rows + 7) / 8 * 8) : 128;
  const int64_t tm = 128 * p.cg, slots = num_sms() / p.cg;
  p.units_m = (int)((rows + tm - 1) / tm);
  const int64_t tiles = ((int64_t)V + kVBN - 1) / kVBN;
  p.units_n = best_parts(p.units_m, tiles, slots, kVMaxParts, 0.25);
  p.part_bytes = align_up((size_t)p.units_n * kVEpiGroups * rows * sizeof(float4), 256);
  p.ldmax = tiles * (kVBN / kVGroup);
  p.max_bytes = top_k > 0 ? (size_t)rows * p.ldmax * 4 : 0;
  p.fwd_bytes = p.part_bytes + p.max_bytes + (size_t)rows * kVCaught * 4;
  // With few rows, a given token's column or two carry most of the gradients,
  // and nothing averages the rounding of dZ: it is kept in two 16-bit parts
  // (16 or more bits), which doubles K where the weights' traffic bounds.
  p.split = rows <= kVSplitRows;
  int64_t chunk = kVDzBytes / (p.split ? 4 : 2) / (rows > 0 ? rows : 1) / kVBN * kVBN;
  if (chunk < kVBN) chunk = kVBN;
  if (chunk > tiles * kVBN) chunk = tiles * kVBN;
  const int64_t nch = (tiles * kVBN + chunk - 1) / chunk;  // chunks of about equal size
  p.chunk = (tiles + nch - 1) / nch * kVBN;
  p.ldz = p.chunk * (p.split ? 2 : 1);
  p.ldp = (H + 3) / 4 * 4;
  const int64_t out_tiles = p.units_m * (((int64_t)H + kVBN - 1) / kVBN);
  p.ks = best_parts(out_tiles, p.ldz / kVBK, slots, 64, 8.0);
  p.coef_bytes = align_up((size_t)rows * sizeof(VRowCoef), 256) + 256;
  p.dz_bytes = align_up((size_t)rows * p.ldz * 2, 256);
  p.bwd_bytes = p.coef_bytes + p.dz_bytes + align_up((size_t)p.ks * rows * p.ldp * 4, 256);
  return p;
}

struct VMatrices {
  const void *h, *w;
  int64_t ldh, ldw;
  int dtype;
};

#define IG_VMAP(...)                                                              \
  do {                                                                            \
    if (make_map_16(__VA_ARGS__)) return fail(IG_ERR_CUDA, "vocab: tensor map"); \
  } while (0)

static int run_vocab_logprobs(const VMatrices &x, const VPlan &p, const LogprobArgs &o, uint8_t *ws, cudaStream_t st) {
  CUtensorMap ma, mb;
  IG_VMAP(&ma, x.h, p.H, p.rows, x.ldh, kVBK, p.a_rows, x.dtype, false);
  IG_VMAP(&mb, x.w, p.H, p.V, x.ldw, kVBK, kVBN / p.cg, x.dtype, false);
  VGemmArgs a{};
  a.M = (int)p.rows;
  a.N = p.V;
  a.a_rows = p.a_rows;
  a.kblocks = (p.H + kVBK - 1) / kVBK;
  a.kparts = 1;
  a.idesc = idesc_f16(128 * p.cg, kVBN, x.dtype, false, false);
  a.units_m = p.units_m;
  a.units_n = p.units_n;
  a.units_s = 1;
  a.c2 = o.c * kLog2e;
  a.part = reinterpret_cast<float4 *>(ws);
  a.gmax = o.K > 0 ? reinterpret_cast<float *>(ws + p.part_bytes) : nullptr;
  a.ldmax = p.ldmax;
  if (o.T <= kVCaught) {
    a.ids = o.ids;
    a.T = o.T;
    a.xid = reinterpret_cast<float *>(ws + p.part_bytes + p.max_bytes);
  }
  IG_CU(p.cg == 1 ? (launch_vgemm<1, false, false, kVStats>(ma, mb, mb, a, st))
                  : (launch_vgemm<2, false, false, kVStats>(ma, mb, mb, a, st)));
  VJoinArgs j{};
  j.h = static_cast<const uint16_t *>(x.h);
  j.w = static_cast<const uint16_t *>(x.w);
  j.ldh = x.ldh;
  j.ldw = x.ldw;
  j.V = p.V;
  j.H = p.H;
  j.T = o.T;
  j.K = o.K;
  j.parts = kVEpiGroups * p.units_n;
  j.dtype = x.dtype;
  j.c = o.c;
  j.ids = o.ids;
  j.part = a.part;
  j.xid = a.xid;
  j.gmax = a.gmax;
  j.ldmax = p.ldmax;
  j.ngroups = (p.V + kVGroup - 1) / kVGroup;
  j.logprobs = o.logprobs;
  j.lse = o.lse;
  j.entropy = o.entropy;
  j.top_ids = o.top_ids;
  j.top_logprobs = o.top_logprobs;
  IG_CU(o.K > 0 ? launch_dep(vocab_join_kernel<true>, dim3((unsigned)p.rows), dim3(kVocThreads), 0, st, j)
                : launch_dep(vocab_join_kernel<false>, dim3((unsigned)p.rows), dim3(64), 0, st, j));
  return 0;
}

struct VocabGradOut {
  const float *logprobs;
  void *dh, *dw;
  int64_t lddh, lddw;
};

static int run_vocab_grad(const VMatrices &x, const VPlan &p, const LogprobGradArgs &g, const VocabGradOut &o, uint8_t *ws,
                          cudaStream_t st) {
  VRowCoef *coef = reinterpret_cast<VRowCoef *>(ws);
  int *bound = x.dtype == IG_DT_F16 ? reinterpret_cast<int *>(ws + p.coef_bytes - 256) : nullptr;
  uint8_t *dz = ws + p.coef_bytes;
  float *p32 = reinterpret_cast<float *>(dz + p.dz_bytes);
  if (bound) IG_CU(cudaMemsetAsync(bound, 0, 4, st));
  const VCoefArgs ca{p.rows, p.V, g.T, g.c, g.ids, g.lse, g.entropy, g.dlogprobs, g.dentropy, coef, bound};
  vocab_coef_kernel<<<(unsigned)((p.rows + 7) / 8), 256, 0, st>>>(ca);
  IG_CU(cudaGetLastError());
  const int tm = 128 * p.cg, shift = p.split ? (int)p.chunk : 0;
  CUtensorMap mh, mw, mz, mzs;
  int done = 0, parts = 1;
  for (int64_t v0 = 0; v0 < p.V; v0 += p.chunk, done++) {
    const int64_t vc = p.V - v0 < p.chunk ? p.V - v0 : p.chunk;
    const bool last = v0 + vc == p.V;
    const uint8_t *wc = static_cast<const uint8_t *>(x.w) + v0 * x.ldw * 2;
    // dZ of the chunk.
    IG_VMAP(&mh, x.h, p.H, p.rows, x.ldh, kVBK, p.a_rows, x.dtype, false);
    IG_VMAP(&mw, wc, p.H, vc, x.ldw, kVBK, kVBN / p.cg, x.dtype, false);
    IG_VMAP(&mzs, dz, p.ldz, p.rows, p.ldz, 32, 32, x.dtype, true);
    VGemmArgs a{};
    a.M = (int)p.rows;
    a.N = (int)vc;
    a.a_rows = p.a_rows;
    a.kblocks = (p.H + kVBK - 1) / kVBK;
    a.kparts = 1;
    a.idesc = idesc_f16(tm, kVBN, x.dtype, false, false);
    a.units_m = p.units_m;
    a.units_n = (int)((vc + kVBN - 1) / kVBN);
    a.units_s = 1;
    a.c = g.c;
    a.coef = coef;
    a.split = p.split;
    a.shift = shift;
    a.bound = bound;
    a.dtype = x.dtype;
    IG_CU(p.cg == 1 ? (launch_vgemm<1, false, false, kVDz>(mh, mw, mzs, a, st))
                    : (launch_vgemm<2, false, false, kVDz>(mh, mw, mzs, a, st)));
    if (g.dlogprobs && g.T > 0) {
      VTokenArgs t{p.rows * g.T, g.T, (int)v0, (int)(v0 + vc), x.dtype, g.c, g.ids, o.logprobs, g.dlogprobs,
                   coef, bound, dz, p.ldz, shift};
      IG_CU(launch_dep(vocab_token_kernel, dim3((unsigned)((t.n + 255) / 256)), dim3(256), 0, st, t));
    }
    IG_VMAP(&mz, dz, p.ldz, p.rows, p.ldz, kVBK, p.a_rows, x.dtype, false);
    if (o.dh) {
      IG_VMAP(&mw, wc, p.H, vc, x.ldw, 64, kVBK, x.dtype, false);
      VGemmArgs b{};
      b.M = (int)p.rows;
      b.N = p.H;
      b.a_rows = p.a_rows;
      b.kparts = p.split ? 2 : 1;
      b.kblocks = (int)((vc + kVBK - 1) / kVBK) * b.kparts;
      b.shift = shift;
      b.idesc = idesc_f16(tm, kVBN, x.dtype, false, true);
      b.units_m = p.units_m;
      b.units_n = (p.H + kVBN - 1) / kVBN;
      b.units_s = b.kblocks < p.ks ? b.kblocks : p.ks;
      b.n_fastest = 1;
      b.dtype = x.dtype;
      b.bound = bound;
      b.part32 = p32;
      b.ldo = p.ldp;
      b.accumulate = done > 0;
      if (done == 0) parts = b.units_s;  // a later, smaller chunk adds into the first of them
      if (done == 0 && last && parts == 1) {
        b.out16 = o.dh;
        b.ldo = o.lddh;
      }
      IG_CU(p.cg == 1 ? (launch_vgemm<1, false, true, kVOut>(mz, mw, mw, b, st))
                      : (launch_vgemm<2, false, true, kVOut>(mz, mw, mw, b, st)));
      if (!b.out16 && last) {
        const int threads = p.H >= 1024 ? 256 : (p.H + 127) / 128 * 32;
        const int groups = parts >= 16 ? 4 : 1;
        IG_CU(launch_dep(vocab_sum_kernel, dim3((unsigned)p.rows), dim3(threads, groups), threads * groups * 16, st,
                         (const float *)p32, parts, p.rows, p.H, p.ldp, (const int *)bound, o.dh, o.lddh, x.dtype));
      }
    }
    if (o.dw) {
      IG_VMAP(&mz, dz, p.ldz, p.rows, p.ldz, 64, kVBK, x.dtype, false);
      IG_VMAP(&mh, x.h, p.H, p.rows, x.ldh, 64, kVBK, x.dtype, false);
      VGemmArgs b{};
      b.M = (int)vc;
      b.N = p.H;
      b.a_rows = 128;  // of M: two boxes of 64
      b.kparts = p.split ? 2 : 1;
      b.kblocks = (int)((p.rows + kVBK - 1) / kVBK) * b.kparts;
      b.shift = shift;
      b.idesc = idesc_f16(256, kVBN, x.dtype, true, true);
      b.units_m = (int)((vc + 255) / 256);
      b.units_n = (p.H + kVBN - 1) / kVBN;
      b.units_s = 1;
      b.n_fastest = 1;
      b.dtype = x.dtype;
      b.bound = bound;
      b.out16 = static_cast<uint8_t *>(o.dw) + v0 * o.lddw * 2;
      b.ldo = o.lddw;
      IG_CU((launch_vgemm<2, true, true, kVOut>(mz, mh, mh, b, st)));
    }
  }
  return 0;
}

}  // namespace ig
