// Vocabulary operators from hidden states: logits = hidden . weight^T on the
// tensor cores (tcgen05 kind::f16, bf16 or f16 operands, float32
// accumulators in TMEM) without ever storing them, and the gradients.
//
// One persistent kernel serves the four products:
//   statistics  rows x vocab, K = hidden: the epilogue keeps each row's
//               running (m, s, u) (vocab_rows.cu) in registers over the
//               column tiles of its unit and writes one partial per unit;
//   dZ          the same product again (a row's logits cost less to compute
//               than to store and read back), turned into the gradient of the
//               logits, rounded to the operands' type and stored;
//   dhidden     dZ . weight, K = vocab, split over K with float32 partials;
//   dweight     dZ^T . hidden, K = rows.
// The last two read operands whose rows run along M or N instead of K: the
// TMA boxes are then 64 (M or N) x 64 (K) and the matrix descriptors
// MN-major, so nothing is transposed in memory.
//
// Tiles are 256 x 256 on a CTA pair (cta_group::2: each CTA holds half of
// either operand, 32 KB per 64 of K, where one CTA alone would fetch 48 KB
// per 128 x 256) or 128 x 256 on one CTA for at most 128 rows, which leaves
// every SM its own stream of the weights. Two accumulators of 256 TMEM
// columns let the epilogue of one tile run under the next one's products.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "internal.h"

namespace ig {

enum VEpi : int { kVStats = 0, kVStatsTop = 1, kVDz = 2, kVOut = 3 };

constexpr int kVBN = 256;   // tile columns
constexpr int kVBK = 64;    // 16-bit elements of K per stage (128 bytes)
constexpr int kVEpiWarps = 8;
constexpr int kVGemmThreads = 64 + 32 * kVEpiWarps;

// Row coefficients of dZ (RowCoef with the output scale applied by the reader).
struct VRowCoef {
  float A, B, lse, pad;
};

struct VGemmArgs {
  int M, N, K;
  uint32_t idesc;
  int units_m, units_n, units_s;  // units: M tiles x N parts x K parts
  int n_fastest;                  // unit order: N parts innermost, else M tiles
  // kVStats, kVStatsTop: [units_n * 2][M] partials
  float c2;
  float4 *part;
  int top_k;
  float *top_val;
  int32_t *top_col;  // [units_n * 2][M][top_k]
  // kVDz
  float c;
  const VRowCoef *coef;
  const float *scale;  // 2^k applied to dZ (power of two), removed from the outputs
  // kVDz, kVOut: dtype of the 16-bit output
  int dtype;
  // kVOut: out16 (final) or part32 [units_s][M][N] (accumulate: added to what is there)
  void *out16;
  int64_t ldo;
  float *part32;
  int accumulate;
};

template <int CG, int EPI>
struct VSmem {
  static constexpr int kABytes = 128 * kVBK * 2;
  static constexpr int kBBytes = (kVBN / CG) * kVBK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kExtra = EPI == kVStatsTop ? 32 * kVEpiWarps * kTopMax * 8 : EPI == kVDz ? kVEpiWarps * 2 * 2048 : 0;
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
template <int EPI>
__device__ __forceinline__ VUnit vunit(const VGemmArgs &a, int u, int ntiles, int kblocks) {
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
  r.k0 = (int)((int64_t)kblocks * r.s / a.units_s);
  r.k1 = (int)((int64_t)kblocks * (r.s + 1) / a.units_s);
  return r;
}

// Inserts (v, col) into a thread's descending list of K (slot k at k *
// stride); columns come in increasing order, so equal values stay behind.
__device__ __noinline__ float list_insert(float *val, int *col, int stride, int K, float v, int c) {
  int k = K - 1;
  while (k > 0 && val[(k - 1) * stride] < v) {
    val[k * stride] = val[(k - 1) * stride];
    col[k * stride] = col[(k - 1) * stride];
    k--;
  }
  val[k * stride] = v;
  col[k * stride] = c;
  return val[(K - 1) * stride];
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
  const int kblocks = (a.K + kVBK - 1) / kVBK;
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
        const VUnit q = vunit<EPI>(a, u, ntiles, kblocks);
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
            if (rank == 0) mbar_arrive_expect_tx(&full[s], CG * S::kStageBytes);
            auto load = [&](const CUtensorMap *map, uint8_t *dst, int c0, int c1) {
              if constexpr (CG == 2)
                tma_load_2d_pair(map, dst, cluster_addr(&full[s], 0), c0, c1);
              else
                tma_load_2d(map, dst, &full[s], c0, c1);
            };
            if constexpr (A_MN) {
#pragma unroll
              for (int i = 0; i < 2; i++) load(&mapA, sa + i * 8192, m0 + i * 64, kb * kVBK);
            } else {
              load(&mapA, sa, kb * kVBK, m0);
            }
            if constexpr (B_MN) {
#pragma unroll
              for (int i = 0; i < kVBN / CG / 64; i++) load(&mapB, sb + i * 8192, n0 + i * 64, kb * kVBK);
            } else {
              load(&mapB, sb, kb * kVBK, n0);
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
        const VUnit q = vunit<EPI>(a, u, ntiles, kblocks);
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
    const int q4 = warp & 3, e = warp - 2, g = e >> 2;  // TMEM lane quarter; column chunks g, g + 2, ...
    int tile = 0;
    bool ok = true;
    [[maybe_unused]] int stores = 0;
    for (int u = first; u < units && ok; u += step) {
      const VUnit q = vunit<EPI>(a, u, ntiles, kblocks);
      const int row0 = q.m * (CG * 128) + rank * 128 + q4 * 32, row = row0 + lane;
      const bool warp_live = row0 < a.M, live = row < a.M;
      [[maybe_unused]] VStat st{-IG_INF, 0.0f, 0.0f};
      [[maybe_unused]] float thr = -IG_INF;
      [[maybe_unused]] float *lval = nullptr;
      [[maybe_unused]] int *lcol = nullptr;
      constexpr int kLs = 32 * kVEpiWarps;  // list slot stride
      if constexpr (EPI == kVStatsTop) {
        lval = reinterpret_cast<float *>(smem + S::kExtraOff) + e * 32 + lane;
        lcol = reinterpret_cast<int *>(lval) + kLs * kTopMax;
        for (int k = 0; k < a.top_k; k++) {
          lval[k * kLs] = -IG_INF;
          lcol[k * kLs] = -1;
        }
      }
      [[maybe_unused]] RowCoef rc{0.0f, 0.0f, IG_INF};
      if constexpr (EPI == kVDz) {
        if (live) {
          const VRowCoef v = a.coef[row];
          const float sc = __ldg(a.scale);
          rc = RowCoef{v.A * sc, v.B * sc, v.lse};
        }
      }
      [[maybe_unused]] float unscale = 1.0f;
      if constexpr (EPI == kVOut) {
        if (a.out16 && a.scale) unscale = 1.0f / __ldg(a.scale);
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
        constexpr int kChunks = kVBN / 64;
        uint32_t r[2][32];
        tmem_ld_32x32b_x32(tb + g * 32, r[0]);
#pragma unroll
        for (int i = 0; i < kChunks; i++) {
          __syncwarp();  // the branches below are per lane; the TMEM loads take the whole warp
          tmem_ld_wait();
          if (i + 1 < kChunks)
            tmem_ld_32x32b_x32(tb + g * 32 + 64 * (i + 1), r[(i + 1) & 1]);
          else
            release();
          const int col0 = n * kVBN + g * 32 + 64 * i;
          if (col0 >= a.N) continue;
          float x[32];
#pragma unroll
          for (int k = 0; k < 32; k++) x[k] = __uint_as_float(r[i & 1][k]);
          if constexpr (EPI == kVStats || EPI == kVStatsTop) {
            if (col0 + 32 > a.N) {
#pragma unroll
              for (int k = 0; k < 32; k++)
                if (col0 + k >= a.N) x[k] = -IG_INF;
            }
            float m4[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
            for (int k = 4; k < 32; k++) m4[k & 3] = fmaxf(m4[k & 3], x[k]);
            const float mx = fmaxf(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])), -IG_INF);
            vstat_add<true>(st, x, mx, a.c2);
            if constexpr (EPI == kVStatsTop) {
              if (live && mx > thr) {
#pragma unroll
                for (int k = 0; k < 32; k++)
                  if (x[k] > thr) thr = list_insert(lval, lcol, kLs, a.top_k, x[k], col0 + k);
              }
            }
          } else if constexpr (EPI == kVDz) {
            uint8_t *buf = smem + S::kExtraOff + (e * 2 + (stores & 1)) * 2048;
            if (lane == 0) bulk_wait_read<1>();
            __syncwarp();
            uint32_t w[16];
#pragma unroll
            for (int k = 0; k < 16; k++)
              w[k] = pack16(dense_grad(x[2 * k], a.c, rc), dense_grad(x[2 * k + 1], a.c, rc), a.dtype);
#pragma unroll
            for (int j = 0; j < 4; j++)
              *reinterpret_cast<uint4 *>(buf + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) =
                  make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&mapC, buf, col0, row0);
              bulk_commit();
            }
            stores++;
          } else {
            if (live && a.out16) {
#pragma unroll
              for (int k = 0; k < 32; k++) x[k] *= unscale;
              const int64_t at = (int64_t)row * a.ldo + col0;
              uint8_t *dst = static_cast<uint8_t *>(a.out16) + at * 2;
              if (col0 + 32 <= a.N && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
#pragma unroll
                for (int j = 0; j < 4; j++)
                  reinterpret_cast<uint4 *>(dst)[j] =
                      make_uint4(pack16(x[8 * j], x[8 * j + 1], a.dtype), pack16(x[8 * j + 2], x[8 * j + 3], a.dtype),
                                 pack16(x[8 * j + 4], x[8 * j + 5], a.dtype), pack16(x[8 * j + 6], x[8 * j + 7], a.dtype));
              } else {
#pragma unroll
                for (int k = 0; k < 32; k++)
                  if (col0 + k < a.N) store16(a.out16, at + k, x[k], a.dtype);
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
      }
      if constexpr (EPI == kVStats || EPI == kVStatsTop) {
        if (ok && live) {
          const int64_t at = (int64_t)(q.n * 2 + g) * a.M + row;
          a.part[at] = make_float4(st.m, st.s, st.u, 0.0f);
          if constexpr (EPI == kVStatsTop) {
            for (int k = 0; k < a.top_k; k++) {
              a.top_val[at * a.top_k + k] = lval[k * kLs];
              a.top_col[at * a.top_k + k] = lcol[k * kLs];
            }
          }
        }
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

// ---- joining the partials, the given tokens' dot products ------------------------------

struct VJoinArgs {
  const uint16_t *h, *w;
  int64_t ldh, ldw;
  int64_t rows;
  int V, H, T, K, parts, dtype;
  float c;
  const int32_t *ids;
  const float4 *part;
  const float *top_val;
  const int32_t *top_col;
  float *logprobs, *lse, *entropy;
  int32_t *top_ids;
  float *top_logprobs;
};

constexpr int kJoinThreads = 128;

__device__ __forceinline__ float2 widen2(uint32_t v, int dtype) {
  if (dtype == IG_DT_BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}
__device__ __forceinline__ float widen1(uint16_t v, int dtype) {
  if (dtype == IG_DT_BF16) return __uint_as_float((uint32_t)v << 16);
  return __half2float(*reinterpret_cast<const __half *>(&v));
}

// One CTA per row.
__global__ void __launch_bounds__(kJoinThreads) vocab_join_kernel(const VJoinArgs a) {
  __shared__ VStat s_warp[kJoinThreads / 32];
  const int64_t row = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float c2 = a.c * kLog2e;
  dep_wait();
  VStat st{-IG_INF, 0.0f, 0.0f};
  for (int p = threadIdx.x; p < a.parts; p += kJoinThreads) {
    const float4 v = a.part[(int64_t)p * a.rows + row];
    vstat_merge<true>(st, VStat{v.x, v.y, v.z}, c2);
  }
  st = vstat_warp<true>(st, c2);
  if (lane == 0) s_warp[warp] = st;
  __syncthreads();
  st = s_warp[0];
  for (int w = 1; w < kJoinThreads / 32; w++) vstat_merge<true>(st, s_warp[w], c2);
  float log_s, lse, entropy;
  row_lse(st, a.c, log_s, lse, entropy);
  if (threadIdx.x == 0) {
    if (a.lse) a.lse[row] = lse;
    if (a.entropy) a.entropy[row] = entropy;
  }
  const uint16_t *h = a.h + row * a.ldh;
  for (int t = warp; t < a.T; t += kJoinThreads / 32) {
    const int id = a.ids[row * a.T + t];
    float v = 0.0f;
    if (id >= 0 && id < a.V) {
      const uint16_t *w = a.w + (int64_t)id * a.ldw;
      float s = 0.0f;
      for (int i = lane * 8; i + 8 <= a.H; i += 256) {
        const uint4 x = *reinterpret_cast<const uint4 *>(h + i), y = __ldg(reinterpret_cast<const uint4 *>(w + i));
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const float2 p = widen2(xs[k], a.dtype), q = widen2(ys[k], a.dtype);
          s = fmaf(p.x, q.x, s);
          s = fmaf(p.y, q.y, s);
        }
      }
      const int tail = a.H & ~7;
      if (tail + lane < a.H) s = fmaf(widen1(h[tail + lane], a.dtype), widen1(w[tail + lane], a.dtype), s);
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
      v = row_logprob(s, st, a.c, log_s);
    } else if (id >= a.V) {
      v = __int_as_float(0x7FC00000);
      if (lane == 0) set_device_error(kDevBadId);
    }
    if (lane == 0) a.logprobs[row * a.T + t] = v;
  }
  if (a.K == 0 || warp != 0) return;
  // The alternatives: every part's list is sorted; lane l walks the lists l,
  // l + 32, ... (at most kHeads of them) and the best head wins.
  constexpr int kHeads = 16;  // 2 * 256 parts
  int head[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; i++) head[i] = 0;
  const bool nan = st.s != st.s;
  for (int k = 0; k < a.K; k++) {
    float bv = -IG_INF;
    int bc = 0x7FFFFFFF, bi = -1;
#pragma unroll
    for (int i = 0; i < kHeads; i++) {
      const int p = lane + 32 * i;
      if (p < a.parts && head[i] < a.K) {
        const int64_t at = ((int64_t)p * a.rows + row) * a.K + head[i];
        const float v = a.top_val[at];
        const int c = a.top_col[at];
        if (c >= 0 && top_before(v, c, bv, bc)) {
          bv = v;
          bc = c;
          bi = i;
        }
      }
    }
    float wv = bv;
    int wc = bc;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const float ov = __shfl_xor_sync(~0u, wv, o);
      const int oc = __shfl_xor_sync(~0u, wc, o);
      if (top_before(ov, oc, wv, wc)) {
        wv = ov;
        wc = oc;
      }
    }
#pragma unroll
    for (int i = 0; i < kHeads; i++)
      if (bi == i && bc == wc && wc != 0x7FFFFFFF) head[i]++;
    if (lane == 0) {
      const bool have = wc != 0x7FFFFFFF && !nan;
      a.top_ids[row * a.K + k] = have ? wc : -1;
      a.top_logprobs[row * a.K + k] =
          have ? row_logprob(wv, st, a.c, log_s) : (nan ? __int_as_float(0x7FC00000) : -IG_INF);
    }
  }
}

// ---- gradient: row coefficients, given tokens, sum of the partials ---------------------

struct VCoefArgs {
  int64_t rows;
  int V, T, dtype;
  float c;
  const int32_t *ids;
  const float *lse, *entropy, *dlogprobs, *dentropy;
  VRowCoef *coef;
  int *bound;  // bits of the largest |dZ| bound of any row (float32 bits of a positive number order as integers)
};

// One warp per row.
__global__ void vocab_coef_kernel(const VCoefArgs a) {
  const int64_t row = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (row >= a.rows) return;
  const int lane = threadIdx.x & 31;
  bool bad = false;
  float G = 0.0f, size = 0.0f;
  if (a.dlogprobs) {
    G = given_grad_sum(a.ids + row * a.T, a.dlogprobs + row * a.T, a.T, a.V, bad);
    if (bad) set_device_error(kDevBadId);
    for (int t = lane; t < a.T; t += 32) size += fabsf(a.dlogprobs[row * a.T + t]);
#pragma unroll
    for (int o = 16; o; o >>= 1) size += __shfl_xor_sync(~0u, size, o);
  }
  if (lane) return;
  const float gh = a.dentropy ? a.dentropy[row] : 0.0f, H = a.dentropy ? a.entropy[row] : 0.0f;
  const float lse = a.lse[row];
  const RowCoef k = row_coef(lse, H, G, gh, a.c);
  a.coef[row] = VRowCoef{k.A, k.B, k.lse, 0.0f};
  // |dZ| <= c (sum |g| (1 + p) + |gH| p (|log p| + H)) <= c (2 sum |g| + |gH| (1 + H))
  const float b = a.c * (2.0f * size + fabsf(gh) * (1.0f + H));
  if (lse != -IG_INF && b > 0.0f && b < 3.0e38f) atomicMax(a.bound, __float_as_int(b));
}

// float16 has 5 exponent bits: dZ is scaled by a power of two that brings the
// largest bound of the rows to 2^14..2^15, so that probabilities down to
// 2^-28 of it keep all their bits; the products' float32 sums are scaled
// back. bfloat16 has float32's range and needs none.
__global__ void vocab_scale_kernel(const int *bound, float *scale, int dtype) {
  float s = 1.0f;
  const int b = *bound;
  if (dtype == IG_DT_F16 && b > 0) {
    int e = ((b >> 23) & 255) - 127;  // bound in [2^e, 2^(e+1))
    e = min(max(14 - e, -100), 100);
    s = __int_as_float((e + 127) << 23);
  }
  *scale = s;
}

struct VTokenArgs {
  int64_t rows, n;  // n = rows * T
  int T, V, v0, v1, dtype;
  float c;
  const int32_t *ids;
  const float *logprobs, *dlogprobs, *lse;
  const VRowCoef *coef;
  const float *scale;
  void *dz;
  int64_t ldz;
};

// dZ at the given tokens of columns [v0, v1): the dense part from the saved
// log probability plus the tokens' own gradients, rounded once.
__global__ void vocab_token_kernel(const VTokenArgs a) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= a.n) return;
  const int64_t row = i / a.T;
  const int id = a.ids[i];
  if (id < a.v0 || id >= a.v1 || a.lse[row] == -IG_INF) return;
  const VRowCoef k = a.coef[row];
  const float t = max_nan(a.logprobs[i], kYMin);
  const float d = ex2(t * kLog2e) * fmaf(k.B, t, k.A) + token_grad(a.ids + row * a.T, a.dlogprobs + row * a.T, a.T, id, a.c);
  store16(a.dz, row * a.ldz + id - a.v0, d * __ldg(a.scale), a.dtype);
}

// dhidden = sum over the K parts, in order, scaled back and rounded.
__global__ void vocab_sum_kernel(const float *part, int parts, int64_t rows, int H, int64_t ldp, const float *scale,
                                 void *out, int64_t ldo, int dtype) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t row = i / H;
  if (row >= rows) return;
  const int col = (int)(i - row * H);
  float s = 0.0f;
  for (int p = 0; p < parts; p++) s += part[((int64_t)p * rows + row) * ldp + col];
  store16(out, row * ldo + col, s * (1.0f / __ldg(scale)), dtype);
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
  cudaLaunchAttribute at[1];
  cfg.gridDim = dim3((unsigned)(CG * (units < slots ? units : slots)));
  cfg.blockDim = dim3(kVGemmThreads);
  cfg.dynamicSmemBytes = VSmem<CG, EPI>::kTotal;
  cfg.stream = st;
  if (CG > 1) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = CG;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, vocab_gemm_kernel<CG, A_MN, B_MN, EPI>, ma, mb, mc, a);
}

// Parts (of column tiles, or of K blocks) per M tile: the fewest that keep the
// rounds of units close to the work's share per slot. With `tiles` pieces to
// cut and `outer` M tiles, a cut in p parts runs ceil(outer p / slots) rounds
// of ceil(tiles / p) pieces.
static int best_parts(int64_t outer, int64_t tiles, int64_t slots, int most, double overhead) {
  int best = 1;
  double cost = 1e300;
  for (int p = 1; p <= most && p <= tiles; p++) {
    const double rounds = (double)((outer * p + slots - 1) / slots);
    const double c = rounds * ((double)((tiles + p - 1) / p) + overhead);
    if (c < cost * 0.995) {
      cost = c;
      best = p;
    }
  }
  return best;
}

constexpr int kVMaxParts = 256;        // column parts per M tile (two partials each)
constexpr int kVOneCtaRows = 128;      // at most this many rows: single CTAs
constexpr int64_t kVDzBytes = 1ll << 30;  // dZ is formed in column chunks of at most this size

struct VPlan {
  int64_t rows;
  int V, H;
  int cg;
  int units_m, units_n;  // statistics
  size_t part_bytes, top_bytes, fwd_bytes;
  // backward
  int64_t chunk, ldz, ldp;
  int ks;
  size_t coef_bytes, dz_bytes, p32_bytes, bwd_bytes;
};

static VPlan vocab_plan(int64_t rows, int V, int H, int top_k) {
  VPlan p{};
  p.rows = rows;
  p.V = V;
  p.H = H;
  p.cg = rows <= kVOneCtaRows ? 1 : 2;
  const int64_t tm = 128 * p.cg, slots = num_sms() / p.cg;
  p.units_m = (int)((rows + tm - 1) / tm);
  const int64_t tiles = ((int64_t)V + kVBN - 1) / kVBN;
  p.units_n = best_parts(p.units_m, tiles, slots, kVMaxParts, 0.25);
  p.part_bytes = align_up((size_t)p.units_n * 2 * rows * sizeof(float4), 256);
  p.top_bytes = align_up((size_t)p.units_n * 2 * rows * top_k * 4, 256);
  p.fwd_bytes = p.part_bytes + 2 * p.top_bytes;
  int64_t chunk = kVDzBytes / 2 / (rows > 0 ? rows : 1) / kVBN * kVBN;
  if (chunk < kVBN) chunk = kVBN;
  const int64_t vpad = tiles * kVBN;
  if (chunk > vpad) chunk = vpad;
  // Chunks of equal size.
  const int64_t nch = (vpad + chunk - 1) / chunk;
  chunk = ((tiles + nch - 1) / nch) * kVBN;
  p.chunk = chunk;
  p.ldz = chunk;
  p.ldp = (H + 3) / 4 * 4;
  const int64_t out_tiles = p.units_m * (((int64_t)H + kVBN - 1) / kVBN);
  p.ks = best_parts(out_tiles, chunk / kVBK, slots, 64, 8.0);
  p.coef_bytes = align_up((size_t)rows * sizeof(VRowCoef), 256) + 256;
  p.dz_bytes = align_up((size_t)rows * p.ldz * 2, 256);
  p.p32_bytes = align_up((size_t)p.ks * rows * p.ldp * 4, 256);
  p.bwd_bytes = p.coef_bytes + p.dz_bytes + p.p32_bytes;
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
  IG_VMAP(&ma, x.h, p.H, p.rows, x.ldh, kVBK, 128, x.dtype, false);
  IG_VMAP(&mb, x.w, p.H, p.V, x.ldw, kVBK, kVBN / p.cg, x.dtype, false);
  VGemmArgs a{};
  a.M = (int)p.rows;
  a.N = p.V;
  a.K = p.H;
  a.idesc = idesc_f16(128 * p.cg, kVBN, x.dtype, false, false);
  a.units_m = p.units_m;
  a.units_n = p.units_n;
  a.units_s = 1;
  a.c2 = o.c * kLog2e;
  a.part = reinterpret_cast<float4 *>(ws);
  a.top_k = o.K;
  a.top_val = reinterpret_cast<float *>(ws + p.part_bytes);
  a.top_col = reinterpret_cast<int32_t *>(ws + p.part_bytes + p.top_bytes);
  if (p.cg == 1) {
    IG_CU(o.K > 0 ? (launch_vgemm<1, false, false, kVStatsTop>(ma, mb, mb, a, st))
                  : (launch_vgemm<1, false, false, kVStats>(ma, mb, mb, a, st)));
  } else {
    IG_CU(o.K > 0 ? (launch_vgemm<2, false, false, kVStatsTop>(ma, mb, mb, a, st))
                  : (launch_vgemm<2, false, false, kVStats>(ma, mb, mb, a, st)));
  }
  VJoinArgs j{};
  j.h = static_cast<const uint16_t *>(x.h);
  j.w = static_cast<const uint16_t *>(x.w);
  j.ldh = x.ldh;
  j.ldw = x.ldw;
  j.rows = p.rows;
  j.V = p.V;
  j.H = p.H;
  j.T = o.T;
  j.K = o.K;
  j.parts = 2 * p.units_n;
  j.dtype = x.dtype;
  j.c = o.c;
  j.ids = o.ids;
  j.part = a.part;
  j.top_val = a.top_val;
  j.top_col = a.top_col;
  j.logprobs = o.logprobs;
  j.lse = o.lse;
  j.entropy = o.entropy;
  j.top_ids = o.top_ids;
  j.top_logprobs = o.top_logprobs;
  IG_CU(launch_dep(vocab_join_kernel, dim3((unsigned)p.rows), dim3(kJoinThreads), 0, st, j));
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
  int *bound = reinterpret_cast<int *>(ws + p.coef_bytes - 256);
  float *scale = reinterpret_cast<float *>(bound + 1);
  uint8_t *dz = ws + p.coef_bytes;
  float *p32 = reinterpret_cast<float *>(dz + p.dz_bytes);
  IG_CU(cudaMemsetAsync(bound, 0, 4, st));
  VCoefArgs ca{p.rows, p.V, g.T, x.dtype, g.c, g.ids, g.lse, g.entropy, g.dlogprobs, g.dentropy, coef, bound};
  vocab_coef_kernel<<<(unsigned)((p.rows + 7) / 8), 256, 0, st>>>(ca);
  vocab_scale_kernel<<<1, 1, 0, st>>>(bound, scale, x.dtype);
  IG_CU(cudaGetLastError());
  const int tm = 128 * p.cg;
  CUtensorMap mh, mw, mz, mzs;
  int chunks = 0;
  for (int64_t v0 = 0; v0 < p.V; v0 += p.chunk) chunks++;
  int done = 0, parts = 1;
  for (int64_t v0 = 0; v0 < p.V; v0 += p.chunk, done++) {
    const int64_t vc = p.V - v0 < p.chunk ? p.V - v0 : p.chunk;
    const uint8_t *wc = static_cast<const uint8_t *>(x.w) + v0 * x.ldw * 2;
    // dZ of the chunk.
    IG_VMAP(&mh, x.h, p.H, p.rows, x.ldh, kVBK, 128, x.dtype, false);
    IG_VMAP(&mw, wc, p.H, vc, x.ldw, kVBK, kVBN / p.cg, x.dtype, false);
    IG_VMAP(&mzs, dz, vc, p.rows, p.ldz, 32, 32, x.dtype, true);
    VGemmArgs a{};
    a.M = (int)p.rows;
    a.N = (int)vc;
    a.K = p.H;
    a.idesc = idesc_f16(tm, kVBN, x.dtype, false, false);
    a.units_m = p.units_m;
    a.units_n = (int)((vc + kVBN - 1) / kVBN);
    a.units_s = 1;
    a.c = g.c;
    a.coef = coef;
    a.scale = scale;
    a.dtype = x.dtype;
    IG_CU(p.cg == 1 ? (launch_vgemm<1, false, false, kVDz>(mh, mw, mzs, a, st))
                    : (launch_vgemm<2, false, false, kVDz>(mh, mw, mzs, a, st)));
    if (g.dlogprobs && g.T > 0) {
      VTokenArgs t{p.rows, p.rows * g.T, g.T, p.V, (int)v0, (int)(v0 + vc), x.dtype, g.c, g.ids, o.logprobs, g.dlogprobs,
                   g.lse, coef, scale, dz, p.ldz};
      vocab_token_kernel<<<(unsigned)((t.n + 255) / 256), 256, 0, st>>>(t);
      IG_CU(cudaGetLastError());
    }
    if (o.dh) {
      IG_VMAP(&mz, dz, vc, p.rows, p.ldz, kVBK, 128, x.dtype, false);
      IG_VMAP(&mw, wc, p.H, vc, x.ldw, 64, kVBK, x.dtype, false);
      VGemmArgs b{};
      b.M = (int)p.rows;
      b.N = p.H;
      b.K = (int)vc;
      b.idesc = idesc_f16(tm, kVBN, x.dtype, false, true);
      b.units_m = p.units_m;
      b.units_n = (p.H + kVBN - 1) / kVBN;
      const int64_t kb = (vc + kVBK - 1) / kVBK;
      b.units_s = (int)(kb < p.ks ? kb : p.ks);
      b.n_fastest = 1;
      b.dtype = x.dtype;
      b.scale = scale;
      b.part32 = p32;
      b.ldo = p.ldp;
      b.accumulate = done > 0;
      if (chunks == 1 && b.units_s == 1) {
        b.out16 = o.dh;
        b.ldo = o.lddh;
      }
      IG_CU(p.cg == 1 ? (launch_vgemm<1, false, true, kVOut>(mz, mw, mw, b, st))
                      : (launch_vgemm<2, false, true, kVOut>(mz, mw, mw, b, st)));
      if (done == 0) parts = b.units_s;  // a later, smaller chunk adds into the first of them
      if (!b.out16 && done == chunks - 1) {
        const int64_t n = p.rows * p.H;
        vocab_sum_kernel<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(p32, parts, p.rows, p.H, p.ldp, scale, o.dh, o.lddh,
                                                                    x.dtype);
        IG_CU(cudaGetLastError());
      }
    }
    if (o.dw) {
      IG_VMAP(&mz, dz, vc, p.rows, p.ldz, 64, kVBK, x.dtype, false);
      IG_VMAP(&mh, x.h, p.H, p.rows, x.ldh, 64, kVBK, x.dtype, false);
      VGemmArgs b{};
      b.M = (int)vc;
      b.N = p.H;
      b.K = (int)p.rows;
      b.idesc = idesc_f16(256, kVBN, x.dtype, true, true);
      b.units_m = (int)((vc + 255) / 256);
      b.units_n = (p.H + kVBN - 1) / kVBN;
      b.units_s = 1;
      b.n_fastest = 1;
      b.dtype = x.dtype;
      b.scale = scale;
      b.out16 = static_cast<uint8_t *>(o.dw) + v0 * o.lddw * 2;
      b.ldo = o.lddw;
      IG_CU((launch_vgemm<2, true, true, kVOut>(mz, mh, mh, b, st)));
    }
  }
  return 0;
}

}  // namespace ig
