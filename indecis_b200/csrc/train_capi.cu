// C entry points of the operators that blocks are trained with (layer_norm.cu, gated_ff.cu, adamw.cu).
#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <new>
#include <string>
#include <utility>
#include <vector>

#include "common.cuh"
#include "internal.h"
#include "train.h"

namespace ig {

// An output beside an operand: the same matrix (in place), or apart from it.
static const char *bad_in_place_of(const RowSpan &in, const RowSpan &out, bool same_type) {
  if (same_type && in.at == out.at && in.stride == out.stride) return nullptr;
  return overlap(in, out) ? "an output may replace an operand of its type and stride, but not overlap one otherwise" : nullptr;
}

// A dense vector of n; a null pointer or no elements: nothing.
static RowSpan vector_span(const void *p, int64_t n, int es) { return RowSpan(n > 0 ? p : nullptr, 1, n, n, es); }
// Outputs against operands and one another.
static const char *bad_shared(std::initializer_list<RowSpan> out, std::initializer_list<RowSpan> in) {
  for (auto o = out.begin(); o != out.end(); ++o) {
    for (const RowSpan &i : in)
      if (overlap(*o, i)) return "outputs and the workspace cannot share memory with an operand or one another";
    for (auto q = out.begin(); q != o; ++q)
      if (overlap(*o, *q)) return "outputs and the workspace cannot share memory with an operand or one another";
  }
  return nullptr;
}

static const char *bad_norm_args(int32_t x_dtype, int32_t y_dtype, int64_t rows, int32_t n, const void *weight,
                                 const void *bias, int32_t weight_dtype, const float *mean, const float *rstd) {
  const int wes = vocab_elem_size(weight_dtype);
  if (!vocab_elem_size(x_dtype) || !vocab_elem_size(y_dtype)) return "dtype must be float32, bfloat16 or float16";
  if (x_dtype != y_dtype && x_dtype != IG_DT_F32) return "the result of 16-bit rows has their type";
  if (rows < 0 || n < 1) return "negative or empty size";
  if (n > (1 << 30) || rows > INT32_MAX) return "too many rows or columns";
  if ((weight || bias) && !wes) return "dtype must be float32, bfloat16 or float16";
  if (wes && ((reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(bias)) % wes))
    return "weight or bias not aligned to its element size";
  if ((reinterpret_cast<uintptr_t>(mean) | reinterpret_cast<uintptr_t>(rstd)) & 3) return "mean or rstd not aligned to 4 bytes";
  return nullptr;
}

static const char *bad_gated_args(int32_t dtype, int64_t rows, int32_t hidden, int32_t inner, int32_t out_size, int32_t act) {
  if (dtype != IG_DT_BF16 && dtype != IG_DT_F16) return "dtype must be bfloat16 or float16";
  if (rows < 0 || hidden < 1 || inner < 1 || out_size < 1) return "negative or empty size";
  if (rows > (1 << 24) || hidden > (1 << 20) || inner > (1 << 20) || out_size > (1 << 20)) return "too many rows or columns";
  if (act < IG_ACT_GELU || act > IG_ACT_SILU) return "unknown activation";
  return nullptr;
}
// A single row has no stride.
static FfMatrix ff_matrix(const void *p, int64_t ld, int64_t rows, int32_t cols) { return FfMatrix{p, rows > 1 ? ld : ff_ld(cols)}; }
static int ff_pack_bits(const FfMatrix &x, const FfMatrix &wi, const FfMatrix &wo, const FfMatrix &dy) {
  return !ff_on(x) | !ff_on(wi) << 1 | !ff_on(wo) << 2 | !ff_on(dy) << 3;
}
static bool bad_workspace(const void *ws, int64_t have, size_t need) {
  return need > 0 && (!ws || have < (int64_t)need || (reinterpret_cast<uintptr_t>(ws) & 255));
}

}  // namespace ig

using namespace ig;

extern "C" {

int ig_layer_norm(const void *x, int32_t x_dtype, int64_t ldx, int64_t rows, int32_t n, const void *weight,
                  const void *bias, int32_t weight_dtype, double eps, void *y, int32_t y_dtype, int64_t ldy, float *mean,
                  float *rstd, void *stream) {
  t_last_error.clear();
  const char *m = bad_norm_args(x_dtype, y_dtype, rows, n, weight, bias, weight_dtype, mean, rstd);
  const int ex = vocab_elem_size(x_dtype), ey = vocab_elem_size(y_dtype);
  if (!m && (!(eps >= 0.0) || !std::isfinite((float)eps))) m = "eps must be finite and not negative";
  if (!m) m = bad_matrix(x, rows, n, ldx, ex);
  if (!m) m = bad_matrix(y, rows, n, ldy, ey);
  if (!m) {
    const RowSpan in(x, rows, n, ldx, ex), out(y, rows, n, ldy, ey), s0 = vector_span(mean, rows, 4), s1 = vector_span(rstd, rows, 4);
    const int ew = vocab_elem_size(weight_dtype);
    m = bad_in_place_of(in, out, ex == ey);
    if (!m) m = bad_shared({out, s0, s1}, {vector_span(weight, n, ew), vector_span(bias, n, ew)});
    if (!m) m = bad_shared({s0, s1}, {in});
  }
  if (m) return fail(IG_ERR_BAD_ARG, std::string("ig_layer_norm: ") + m);
  if (rows == 0) return 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  ProfScope ps("layer_norm", (double)rows * n * (ex + ey), 8.0 * rows * n, 1, st);
  IG_CU(launch_layer_norm(LnArgs{x, ldx, rows, n, weight, bias, weight_dtype, (float)eps, y, ldy, mean, rstd}, x_dtype, y_dtype,
                          st));
  return 0;
}

int64_t ig_layer_norm_workspace(int64_t rows, int32_t n) {
  return rows < 0 || n < 1 || n > (1 << 30) || rows > INT32_MAX ? 0 : layer_norm_workspace(rows, n);
}

int ig_layer_norm_backward(const void *dy, int32_t y_dtype, int64_t lddy, const void *x, int32_t x_dtype, int64_t ldx,
                           int64_t rows, int32_t n, const void *weight, int32_t weight_dtype, const float *mean,
                           const float *rstd, void *dx, int64_t lddx, void *dweight, void *dbias, void *workspace,
                           int64_t workspace_bytes, void *stream) {
  t_last_error.clear();
  const char *m = bad_norm_args(x_dtype, y_dtype, rows, n, weight, nullptr, weight_dtype, mean, rstd);
  const int ex = vocab_elem_size(x_dtype), ey = vocab_elem_size(y_dtype), ew = vocab_elem_size(weight_dtype);
  const bool sums = dweight || dbias;
  if (!m && sums && !ew) m = "dtype must be float32, bfloat16 or float16";
  if (!m && sums && ((reinterpret_cast<uintptr_t>(dweight) | reinterpret_cast<uintptr_t>(dbias)) % ew))
    m = "gradient of weight or bias not aligned to its element size";
  if (!m) m = bad_matrix(dy, rows, n, lddy, ey);
  if (!m) m = bad_matrix(x, rows, n, ldx, ex);
  if (!m) m = bad_matrix(dx, rows, n, lddx, ex);
  if (!m && rows > 0 && (!mean || !rstd)) m = "null argument";
  if (!m) {
    const RowSpan out(dx, rows, n, lddx, ex), in(x, rows, n, ldx, ex), up(dy, rows, n, lddy, ey), sw = vector_span(dweight, n, ew),
        sb = vector_span(dbias, n, ew), ws = vector_span(workspace, sums ? layer_norm_workspace(rows, n) : 0, 1);
    m = bad_in_place_of(in, out, true);
    if (!m) m = bad_in_place_of(up, out, x_dtype == y_dtype);
    if (!m) m = bad_shared({out, sw, sb, ws}, {vector_span(weight, n, ew), vector_span(mean, rows, 4), vector_span(rstd, rows, 4)});
    if (!m) m = bad_shared({sw, sb, ws}, {in, up});
  }
  if (m) return fail(IG_ERR_BAD_ARG, std::string("ig_layer_norm_backward: ") + m);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (rows == 0) {
    if (dweight) IG_CU(cudaMemsetAsync(dweight, 0, (size_t)n * ew, st));
    if (dbias) IG_CU(cudaMemsetAsync(dbias, 0, (size_t)n * ew, st));
    return 0;
  }
  if (sums && (!workspace || workspace_bytes < layer_norm_workspace(rows, n) || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return fail(IG_ERR_BAD_ARG, "ig_layer_norm_backward: workspace missing, too small or not aligned to 16 bytes");
  LnGradArgs a{};
  a.dy = dy;
  a.x = x;
  a.lddy = lddy;
  a.ldx = ldx;
  a.rows = rows;
  a.n = n;
  a.w = weight;
  a.wdt = weight_dtype;
  a.mean = mean;
  a.rstd = rstd;
  a.dx = dx;
  a.lddx = lddx;
  a.part = sums ? static_cast<float *>(workspace) : nullptr;
  ProfScope ps("layer_norm_backward", (double)rows * n * (2 * ex + ey), 14.0 * rows * n, 1 + sums, st);
  IG_CU(launch_layer_norm_grad(a, x_dtype, y_dtype, dweight, dbias, st));
  return 0;
}

int64_t ig_gated_ff_saved(int64_t rows, int32_t inner) {
  if (rows <= 0 || rows > (1 << 24) || inner < 1 || inner > (1 << 20)) return 0;
  return (int64_t)(ff_h_bytes(rows, inner) + ff_z_bytes(rows, inner));
}

int64_t ig_gated_ff_workspace(int64_t rows, int32_t hidden, int32_t inner, int32_t out_size, int32_t unaligned, int32_t pass) {
  if (bad_gated_args(IG_DT_BF16, rows, hidden, inner, out_size, IG_ACT_GELU) || rows == 0 || pass < 0 || pass > 2) return 0;
  const FfSizes s{rows, hidden, inner, out_size, unaligned & 15};
  return (int64_t)ff_bytes(s, ff_plan(s, pass == 2), pass);
}

int ig_check_gated_ff(int64_t rows, int32_t hidden, int32_t inner, int32_t out_size, int32_t pass, int32_t *cut) {
  t_last_error.clear();
  const char *m = bad_gated_args(IG_DT_BF16, rows, hidden, inner, out_size, IG_ACT_GELU);
  if (!m && (rows == 0 || pass < 0 || pass > 2 || !cut)) m = "no rows, no such pass or null argument";
  if (m) return fail(IG_ERR_BAD_ARG, std::string("ig_check_gated_ff: ") + m);
  const FfSizes s{rows, hidden, inner, out_size, 0};
  const FfPlan p = ff_plan(s, pass == 2);
  const bool few = ff_few(s, pass > 0);
  cut[0] = few ? 0 : ff_inner_small(s, pass == 2) ? 1 : 2;
  cut[1] = few ? 0 : p.cut.small ? 1 : 2;
  for (int i = 0; i < kFfProblems; i++) cut[2 + i] = few || (pass < 2 && i > 0) ? 0 : p.cut.parts[i];
  return 0;
}

int ig_gated_ff(const void *x, int64_t ldx, const void *w_in, int64_t ldi, const void *w_out, int64_t ldw, int32_t dtype,
                int64_t rows, int32_t hidden, int32_t inner, int32_t out_size, int32_t activation, void *y, int64_t ldy,
                void *saved, void *workspace, int64_t workspace_bytes, void *stream) {
  t_last_error.clear();
  const char *m = bad_gated_args(dtype, rows, hidden, inner, out_size, activation);
  if (!m) m = bad_matrix(x, rows, hidden, ldx, 2);
  if (!m) m = bad_matrix(w_in, 2 * (int64_t)inner, hidden, ldi, 2);
  if (!m) m = bad_matrix(w_out, out_size, inner, ldw, 2);
  if (!m) m = bad_matrix(y, rows, out_size, ldy, 2);
  if (!m && (reinterpret_cast<uintptr_t>(saved) & 255)) m = "what is saved must start at a multiple of 256 bytes";
  if (m) return fail(IG_ERR_BAD_ARG, std::string("ig_gated_ff: ") + m);
  if (rows == 0) return 0;
  const FfMatrix mx = ff_matrix(x, ldx, rows, hidden), mi = ff_matrix(w_in, ldi, 2, hidden), mo = ff_matrix(w_out, ldw, out_size, inner);
  const FfSizes s{rows, hidden, inner, out_size, ff_pack_bits(mx, mi, mo, FfMatrix{})};
  const FfPlan p = ff_plan(s, false);
  const size_t need = ff_bytes(s, p, saved ? 1 : 0);
  if (bad_workspace(workspace, workspace_bytes, need))
    return fail(IG_ERR_BAD_ARG, "ig_gated_ff: workspace missing, too small or not aligned to 256 bytes");
  m = bad_shared({RowSpan(y, rows, out_size, ldy, 2), vector_span(saved, (int64_t)(p.h_bytes + p.z_bytes), 1), vector_span(workspace, (int64_t)need, 1)},
                 {RowSpan(x, rows, hidden, ldx, 2), RowSpan(w_in, 2 * (int64_t)inner, hidden, ldi, 2), RowSpan(w_out, out_size, inner, ldw, 2)});
  if (m) return fail(IG_ERR_BAD_ARG, std::string("ig_gated_ff: ") + m);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  ProfScope ps("gated_ff", 2.0 * ((double)rows * (hidden + out_size) + (double)inner * (2.0 * hidden + out_size)),
               2.0 * rows * inner * (2.0 * hidden + out_size), 2, st);
  return run_gated_ff(mx, mi, mo, s, p, dtype, activation, y, ldy, static_cast<uint8_t *>(saved), static_cast<uint8_t *>(workspace), st);
}

int ig_gated_ff_backward(const void *dy, int64_t lddy, const void *x, int64_t ldx, const void *w_in, int64_t ldi,
                         const void *w_out, int64_t ldw, int32_t dtype, int64_t rows, int32_t hidden, int32_t inner,
                         int32_t out_size, int32_t activation, const void *saved, void *dx, int64_t lddx, void *dw_in,
                         int64_t lddi, void *dw_out, int64_t lddw, void *workspace, int64_t workspace_bytes, void *stream) {
  t_last_error.clear();
  const int64_t i2 = 2 * (int64_t)inner;
  const char *m = bad_gated_args(dtype, rows, hidden, inner, out_size, activation);
  if (!m) m = bad_matrix(dy, rows, out_size, lddy, 2);
  if (!m) m = bad_matrix(x, rows, hidden, ldx, 2);
  if (!m) m = bad_matrix(w_in, i2, hidden, ldi, 2);
  if (!m) m = bad_matrix(w_out, out_size, inner, ldw, 2);
  if (!m && dx) m = bad_matrix(dx, rows, hidden, lddx, 2);
  if (!m && dw_in) m = bad_matrix(dw_in, i2, hidden, lddi, 2);
  if (!m && dw_out) m = bad_matrix(dw_out, out_size, inner, lddw, 2);
  if (!m && rows > 0 && (!saved || (reinterpret_cast<uintptr_t>(saved) & 255)))
    m = "what the forward saved is missing or does not start at a multiple of 256 bytes";
  if (m) return fail(IG_ERR_BAD_ARG, std::string("ig_gated_ff_backward: ") + m);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (!dx && !dw_in && !dw_out) return 0;
  const RowSpan sdx(dx, rows, hidden, lddx, 2), sdi(dw_in, i2, hidden, lddi, 2), sdo(dw_out, out_size, inner, lddw, 2), sy(dy, rows, out_size, lddy, 2),
      sx(x, rows, hidden, ldx, 2), si(w_in, i2, hidden, ldi, 2), so(w_out, out_size, inner, ldw, 2),
      sv = vector_span(saved, ig_gated_ff_saved(rows, inner), 1);
  if ((m = bad_shared({sdx, sdi, sdo}, {sy, sx, si, so, sv}))) return fail(IG_ERR_BAD_ARG, std::string("ig_gated_ff_backward: ") + m);
  if (rows == 0) {
    if (dw_in) IG_CU(cudaMemset2DAsync(dw_in, (size_t)lddi * 2, 0, (size_t)hidden * 2, i2, st));
    if (dw_out) IG_CU(cudaMemset2DAsync(dw_out, (size_t)lddw * 2, 0, (size_t)inner * 2, out_size, st));
    return 0;
  }
  const FfMatrix md = ff_matrix(dy, lddy, rows, out_size), mx = ff_matrix(x, ldx, rows, hidden), mi = ff_matrix(w_in, ldi, 2, hidden),
                 mo = ff_matrix(w_out, ldw, out_size, inner);
  const FfSizes s{rows, hidden, inner, out_size, ff_pack_bits(mx, mi, mo, md)};
  const FfPlan p = ff_plan(s, true);
  const size_t need = ff_bytes(s, p, 2);
  if (bad_workspace(workspace, workspace_bytes, need))
    return fail(IG_ERR_BAD_ARG, "ig_gated_ff_backward: workspace missing, too small or not aligned to 256 bytes");
  if ((m = bad_shared({vector_span(workspace, (int64_t)need, 1)}, {sdx, sdi, sdo, sy, sx, si, so, sv})))
    return fail(IG_ERR_BAD_ARG, std::string("ig_gated_ff_backward: ") + m);
  const int products = (dx || dw_in) + 2 * (dx != nullptr) + 2 * (dw_in != nullptr) + (dw_out != nullptr);
  ProfScope ps("gated_ff_backward", 4.0 * ((double)rows * (hidden + out_size) + (double)inner * (2.0 * hidden + out_size)),
               2.0 * products * rows * inner * hidden, 4, st);
  return run_gated_ff_grad(md, mx, mi, mo, s, p, dtype, activation, static_cast<const uint8_t *>(saved), dx, lddx, dw_in, lddi, dw_out, lddw,
                           static_cast<uint8_t *>(workspace), st);
}

int ig_adamw_step(const ig_adamw_tensors *tensors, int32_t state_bits, double lr, double beta1, double beta2, double eps,
                  int32_t *step, const float *grad_scale, const float *skip, void *stream) {
  t_last_error.clear();
  const char *m = nullptr;
  const bool bits8 = state_bits == 8;
  if (!tensors || !step || tensors->count < 0 || tensors->count > (1 << 24)) m = "null argument or count out of range";
  if (!m && state_bits != 32 && !bits8) m = "moments are held in 32 or in 8 bits";
  if (!m && tensors->count > 0 &&
      (!tensors->n || !tensors->param || !tensors->grad || !tensors->exp_avg || !tensors->exp_avg_sq || !tensors->param_dtype ||
       !tensors->grad_dtype || !tensors->weight_decay || (bits8 && (!tensors->exp_avg_scale || !tensors->exp_avg_sq_scale)) ||
       (tensors->copy && !tensors->copy_dtype)))
    m = "null argument";
  if (!m && (!(lr >= 0.0) || !std::isfinite((float)lr) || !(beta1 >= 0.0) || !(beta1 < 1.0) || !(beta2 >= 0.0) ||
             !(beta2 < 1.0) || !((float)eps >= 0x1p-126f) || !std::isfinite((float)eps)))
    m = "lr must be finite and not negative, the betas in [0, 1), eps at least 2^-126";
  if (!m && ((reinterpret_cast<uintptr_t>(step) | reinterpret_cast<uintptr_t>(grad_scale) | reinterpret_cast<uintptr_t>(skip)) & 3))
    m = "step, grad_scale or skip not aligned to 4 bytes";
  if (m) return fail(IG_ERR_BAD_ARG, std::string("ig_adamw_step: ") + m);
  double bytes = 0.0;
  try {
    const int64_t count = tensors->count;
    std::vector<AdamwTensor> t;
    std::vector<std::pair<uintptr_t, uintptr_t>> out;  // what is written
    t.reserve(count);
    out.reserve(6 * (size_t)count + 1);
    auto span = [](const void *p, int64_t n) {
      return std::make_pair(reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + (uintptr_t)n);
    };
    out.push_back(span(step, 4));
    for (int64_t i = 0; i < count && !m; i++) {
      AdamwTensor d{};
      d.n = tensors->n[i];
      d.pt = tensors->param_dtype[i];
      d.gt = tensors->grad_dtype[i];
      d.decay = tensors->weight_decay[i];
      d.copy = tensors->copy ? tensors->copy[i] : nullptr;
      d.ct = d.copy ? tensors->copy_dtype[i] : 0;
      const int pe = vocab_elem_size(d.pt), ge = vocab_elem_size(d.gt), se = bits8 ? 1 : 4;
      if (d.n < 0 || d.n > (1ll << 39)) m = "a tensor's size is out of range";
      else if (!pe || !ge) m = "dtype must be float32, bfloat16 or float16";
      else if (d.copy && d.ct != IG_DT_BF16 && d.ct != IG_DT_F16) m = "copies are bfloat16 or float16";
      else if (!std::isfinite(d.decay) || d.decay < 0.0f) m = "weight_decay must be finite and not negative";
      if (m || d.n == 0) continue;
      d.p = tensors->param[i];
      d.g = tensors->grad[i];
      d.m = tensors->exp_avg[i];
      d.v = tensors->exp_avg_sq[i];
      if (bits8) {
        d.ms = tensors->exp_avg_scale[i];
        d.vs = tensors->exp_avg_sq_scale[i];
      }
      if (!d.p || !d.g || !d.m || !d.v || (bits8 && (!d.ms || !d.vs))) {
        m = "null argument";
        continue;
      }
      const uintptr_t p = reinterpret_cast<uintptr_t>(d.p), g = reinterpret_cast<uintptr_t>(d.g), c = reinterpret_cast<uintptr_t>(d.copy),
                      st = reinterpret_cast<uintptr_t>(d.m) | reinterpret_cast<uintptr_t>(d.v),
                      sc = reinterpret_cast<uintptr_t>(d.ms) | reinterpret_cast<uintptr_t>(d.vs);
      if (p % pe || g % ge || (c & 1) || st % se || (sc & 3)) {
        m = "a tensor is not aligned to its element size";
        continue;
      }
      d.wide = p % (4 * pe) == 0 && g % (4 * ge) == 0 && c % 8 == 0 && st % (4 * se) == 0;
      t.push_back(d);
      out.push_back(span(d.p, d.n * pe));
      out.push_back(span(d.m, d.n * se));
      out.push_back(span(d.v, d.n * se));
      if (d.copy) out.push_back(span(d.copy, d.n * 2));
      if (bits8) {
        const int64_t blocks = d.n / 256 + (d.n % 256 != 0);
        out.push_back(span(d.ms, blocks * 4));
        out.push_back(span(d.vs, blocks * 4));
      }
      bytes += (double)d.n * (2 * pe + ge + (d.copy ? 2 : 0) + 4 * se);
    }
    if (!m) {
      std::sort(out.begin(), out.end());
      for (size_t i = 1; i < out.size() && !m; i++)
        if (out[i].first < out[i - 1].second) m = "a parameter, moment, copy or the step shares memory with another";
      // What is read must not be written: the first output that ends after its start begins after its end.
      auto written = [&](const void *p, int64_t n) {
        const auto q = span(p, n);
        const auto it = std::upper_bound(out.begin(), out.end(), q.first, [](uintptr_t v, const auto &o) { return v < o.second; });
        return it != out.end() && it->first < q.second;
      };
      for (size_t i = 0; i < t.size() && !m; i++)
        if (written(t[i].g, t[i].n * vocab_elem_size(t[i].gt))) m = "a gradient shares memory with what is written";
      if (!m && ((grad_scale && written(grad_scale, 4)) || (skip && written(skip, 4))))
        m = "grad_scale or skip shares memory with what is written";
    }
    if (m) return fail(IG_ERR_BAD_ARG, std::string("ig_adamw_step: ") + m);
    const AdamwArgs a{(float)lr, (float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps, beta1, beta2, -0.0f,
                      step, grad_scale, skip};
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    ProfScope ps("adamw_step", bytes, 0.0, 1 + (int)((t.size() + 399) / 400), st);
    IG_CU(launch_adamw(t.data(), (int)t.size(), a, bits8, st));
  } catch (const std::bad_alloc &) {
    return fail(IG_ERR_BAD_ARG, "ig_adamw_step: out of host memory");
  }
  return 0;
}

}  // extern "C"
