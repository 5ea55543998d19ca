// C entry points of the vocabulary operators (vocab_rows.cu, vocab_gemm.cu).
#include <cmath>
#include <string>

#include "common.cuh"
#include "internal.h"

namespace ig {

static int vocab_elem_size(int dtype) {
  return dtype == IG_DT_F32 ? 4 : dtype == IG_DT_BF16 || dtype == IG_DT_F16 ? 2 : 0;
}

// A matrix argument: rows x cols elements of es bytes, row stride ld.
static const char *bad_matrix(const void *p, int64_t rows, int64_t cols, int64_t ld, int es) {
  if (rows > 0 && !p) return "null argument";
  if (ld < cols) return "row stride shorter than the row";
  if (reinterpret_cast<uintptr_t>(p) % es) return "matrix not aligned to its element size";
  return nullptr;
}

// A matrix's rows as intervals of addresses: `width` bytes each, `stride` >= width apart.
struct RowSpan {
  uintptr_t at;
  int64_t rows, stride, width;
  RowSpan(const void *p, int64_t rows_, int64_t cols, int64_t ld, int es)
      : at(reinterpret_cast<uintptr_t>(p)), rows(p ? rows_ : 0), stride(ld * es), width(cols * es) {}
  uintptr_t end() const { return at + (uintptr_t)((rows - 1) * stride + width); }
};
// Whether two matrices share a byte (rows of one may lie between those of the other).
static bool overlap(const RowSpan &p, const RowSpan &q) {
  if (p.rows <= 0 || q.rows <= 0 || p.end() <= q.at || q.end() <= p.at) return false;
  const RowSpan &a = p.at <= q.at ? p : q, &b = p.at <= q.at ? q : p;
  if (a.stride == b.stride) {
    // b's first row starts in a's row k, `r` bytes from its start; all later pairs of rows are alike.
    const int64_t k = (int64_t)((b.at - a.at) / a.stride), r = (int64_t)((b.at - a.at) % a.stride);
    return (k < a.rows && r < a.width) || (k + 1 < a.rows && r + b.width > a.stride);
  }
  uintptr_t x = a.at, y = b.at;
  for (int64_t i = 0, j = 0; i < a.rows && j < b.rows;) {
    if (x + a.width <= y) {
      i++;
      x += a.stride;
    } else if (y + b.width <= x) {
      j++;
      y += b.stride;
    } else {
      return true;
    }
  }
  return false;
}
// Logits' gradient in place of the logits, or apart from them.
static const char *bad_in_place(const void *x, int64_t ld, const void *d, int64_t ldd, int64_t rows, int64_t cols, int es) {
  if (x == d) return ld != ldd ? "in place, both row strides must be the same" : nullptr;
  return overlap(RowSpan(x, rows, cols, ld, es), RowSpan(d, rows, cols, ldd, es))
             ? "the gradient may replace the logits, but not overlap them" : nullptr;
}

static const char *bad_row_args(int64_t rows, int64_t vocab, int32_t nids, const void *ids, const float *io, double t) {
  if (rows < 0 || vocab < 1 || nids < 0) return "negative or empty size";
  if (vocab > (1 << 30) || rows > (int64_t)INT32_MAX / 8) return "too many rows or columns";
  if (nids > IG_VOCAB_IDS_MAX) return "too many given tokens per row";
  if (rows > 0 && nids > 0 && (!ids || !io)) return "null argument";
  if (!(t > 0.0) || !std::isfinite(t) || !std::isfinite((float)(1.0 / t)) || (float)(1.0 / t) <= 0.0f)
    return "temperature must be positive and finite";
  return nullptr;
}

static const char *bad_vocab_args(const void *h, int64_t ldh, const void *w, int64_t ldw, int32_t dtype, int64_t rows,
                                  int32_t vocab, int32_t hidden) {
  if (dtype != IG_DT_BF16 && dtype != IG_DT_F16) return "dtype must be bfloat16 or float16";
  if (hidden < 1 || hidden > (1 << 20)) return "hidden size out of range";
  if (rows > (1 << 24)) return "too many rows";
  const char *m = bad_matrix(h, rows, hidden, ldh, 2);
  if (!m) m = bad_matrix(w, vocab, hidden, ldw, 2);
  if (m) return m;
  if (ldh % 8 || ldw % 8 || ((reinterpret_cast<uintptr_t>(h) | reinterpret_cast<uintptr_t>(w)) & 15))
    return "rows of hidden and weight must start at multiples of 16 bytes (strides multiples of 8)";
  return nullptr;
}

}  // namespace ig

using namespace ig;

extern "C" {

int ig_token_logprobs(const void *logits, int32_t dtype, int64_t ld, int64_t rows, int32_t vocab, double temperature,
                      const int32_t *ids, int32_t nids, float *logprobs, float *lse, float *entropy, int32_t top_k,
                      int32_t *top_ids, float *top_logprobs, void *stream) {
  t_last_error.clear();
  const int es = vocab_elem_size(dtype);
  if (!es) return fail(IG_ERR_BAD_ARG, "ig_token_logprobs: dtype must be float32, bfloat16 or float16");
  if (const char *m = bad_row_args(rows, vocab, nids, ids, logprobs, temperature))
    return fail(IG_ERR_BAD_ARG, std::string("ig_token_logprobs: ") + m);
  if (const char *m = bad_matrix(logits, rows, vocab, ld, es))
    return fail(IG_ERR_BAD_ARG, std::string("ig_token_logprobs: ") + m);
  if (top_k < 0 || top_k > IG_VOCAB_TOP_MAX)
    return fail(IG_ERR_BAD_ARG, "ig_token_logprobs: top_k must be between 0 and 32");
  if (rows > 0 && top_k > 0 && (!top_ids || !top_logprobs)) return fail(IG_ERR_BAD_ARG, "ig_token_logprobs: null argument");
  if (rows == 0) return 0;
  LogprobArgs a{logits, ld, rows, vocab, nids, top_k, (float)(1.0 / temperature), ids, logprobs, lse, entropy, top_ids,
                top_logprobs, 1};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  ProfScope ps("token_logprobs", (double)rows * ((double)vocab * es + 8.0 * (nids + 1 + top_k)), 8.0 * rows * vocab, 1, st);
  IG_CU(dtype == IG_DT_F32    ? run_token_logprobs<IG_DT_F32>(a, st)
        : dtype == IG_DT_BF16 ? run_token_logprobs<IG_DT_BF16>(a, st)
                              : run_token_logprobs<IG_DT_F16>(a, st));
  return 0;
}

int ig_token_logprobs_backward(const void *logits, int32_t dtype, int64_t ld, int64_t rows, int32_t vocab,
                               double temperature, const int32_t *ids, int32_t nids, const float *lse,
                               const float *entropy, const float *dlogprobs, const float *dentropy, void *dlogits,
                               int64_t ldd, void *stream) {
  t_last_error.clear();
  const int es = vocab_elem_size(dtype);
  if (!es) return fail(IG_ERR_BAD_ARG, "ig_token_logprobs_backward: dtype must be float32, bfloat16 or float16");
  if (const char *m = bad_row_args(rows, vocab, nids, ids, dlogprobs, temperature))
    return fail(IG_ERR_BAD_ARG, std::string("ig_token_logprobs_backward: ") + m);
  const char *m = bad_matrix(logits, rows, vocab, ld, es);
  if (!m) m = bad_matrix(dlogits, rows, vocab, ldd, es);
  if (!m && rows > 0 && (!lse || (dentropy && !entropy))) m = "null argument";
  if (!m) m = bad_in_place(logits, ld, dlogits, ldd, rows, vocab, es);
  if (m) return fail(IG_ERR_BAD_ARG, std::string("ig_token_logprobs_backward: ") + m);
  if (rows == 0) return 0;
  LogprobGradArgs a{logits, ld, rows, vocab, nids, 1, (float)(1.0 / temperature), ids, lse, entropy,
                    nids > 0 ? dlogprobs : nullptr, dentropy, dlogits, ldd};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  ProfScope ps("token_logprobs_backward", 2.0 * rows * vocab * es, 8.0 * rows * vocab, 1, st);
  IG_CU(dtype == IG_DT_F32    ? run_token_logprobs_grad<IG_DT_F32>(a, st)
        : dtype == IG_DT_BF16 ? run_token_logprobs_grad<IG_DT_BF16>(a, st)
                              : run_token_logprobs_grad<IG_DT_F16>(a, st));
  return 0;
}

int ig_distill_topk(const void *logits, int32_t dtype, int64_t ld, int64_t rows, int32_t vocab, double temperature,
                    const int32_t *teacher_ids, const float *teacher_logits, int32_t k, int32_t tail,
                    const float *weights, float *loss, void *dlogits, int64_t ldd, void *stream) {
  t_last_error.clear();
  const int es = vocab_elem_size(dtype);
  if (!es) return fail(IG_ERR_BAD_ARG, "ig_distill_topk: dtype must be float32, bfloat16 or float16");
  const char *m = bad_row_args(rows, vocab, k, teacher_ids, teacher_logits, temperature);
  if (!m) m = bad_matrix(logits, rows, vocab, ld, es);
  if (!m && dlogits) m = bad_matrix(dlogits, rows, vocab, ldd, es);
  if (!m && rows > 0 && !loss) m = "null argument";
  if (m) return fail(IG_ERR_BAD_ARG, std::string("ig_distill_topk: ") + m);
  if (tail && vocab > (1 << 20))
    return fail(IG_ERR_UNSUPPORTED, "ig_distill_topk: with the tail, at most 1048576 columns");
  if (dlogits && (m = bad_in_place(logits, ld, dlogits, ldd, rows, vocab, es)))
    return fail(IG_ERR_BAD_ARG, std::string("ig_distill_topk: ") + m);
  if (rows == 0) return 0;
  DistillArgs a{logits, ld, rows, vocab, k, (float)(1.0 / temperature), teacher_ids, teacher_logits, weights, loss,
                dlogits, ldd, 1};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  ProfScope ps("distill_topk", (double)rows * ((dlogits ? 2.0 : 1.0) * vocab * es + 8.0 * k), 10.0 * rows * vocab, 1, st);
  IG_CU(dtype == IG_DT_F32    ? run_distill<IG_DT_F32>(a, tail != 0, st)
        : dtype == IG_DT_BF16 ? run_distill<IG_DT_BF16>(a, tail != 0, st)
                              : run_distill<IG_DT_F16>(a, tail != 0, st));
  return 0;
}

int64_t ig_vocab_workspace(int64_t rows, int32_t vocab, int32_t hidden, int32_t top_k, int32_t backward) {
  if (rows <= 0 || rows > (1 << 24) || vocab < 1 || vocab > (1 << 30) || hidden < 1 || hidden > (1 << 20) || top_k < 0 ||
      top_k > IG_VOCAB_TOP_MAX)
    return 0;
  const VPlan p = vocab_plan(rows, vocab, hidden, backward ? 0 : top_k);
  return (int64_t)(backward ? p.bwd_bytes : p.fwd_bytes);
}

int ig_vocab_logprobs(const void *hidden, int64_t ldh, const void *weight, int64_t ldw, int32_t dtype, int64_t rows,
                      int32_t vocab, int32_t hidden_size, double temperature, const int32_t *ids, int32_t nids,
                      float *logprobs, float *lse, float *entropy, int32_t top_k, int32_t *top_ids, float *top_logprobs,
                      void *workspace, int64_t workspace_bytes, void *stream) {
  t_last_error.clear();
  const char *m = bad_row_args(rows, vocab, nids, ids, logprobs, temperature);
  if (!m) m = bad_vocab_args(hidden, ldh, weight, ldw, dtype, rows, vocab, hidden_size);
  if (!m && (top_k < 0 || top_k > IG_VOCAB_TOP_MAX)) m = "top_k must be between 0 and 32";
  if (!m && rows > 0 && top_k > 0 && (!top_ids || !top_logprobs)) m = "null argument";
  if (m) return fail(IG_ERR_BAD_ARG, std::string("ig_vocab_logprobs: ") + m);
  if (rows == 0) return 0;
  const VPlan p = vocab_plan(rows, vocab, hidden_size, top_k);
  if (!workspace || workspace_bytes < (int64_t)p.fwd_bytes || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return fail(IG_ERR_BAD_ARG, "ig_vocab_logprobs: workspace missing, too small or not aligned to 256 bytes");
  LogprobArgs o{};
  o.rows = rows;
  o.V = vocab;
  o.T = nids;
  o.K = top_k;
  o.c = (float)(1.0 / temperature);
  o.ids = ids;
  o.logprobs = logprobs;
  o.lse = lse;
  o.entropy = entropy;
  o.top_ids = top_ids;
  o.top_logprobs = top_logprobs;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  ProfScope ps("vocab_logprobs", 2.0 * ((double)rows + vocab) * hidden_size, 2.0 * rows * vocab * hidden_size, 2, st);
  return run_vocab_logprobs(VMatrices{hidden, weight, ldh, ldw, dtype}, p, o, static_cast<uint8_t *>(workspace), st);
}

int ig_vocab_logprobs_backward(const void *hidden, int64_t ldh, const void *weight, int64_t ldw, int32_t dtype,
                               int64_t rows, int32_t vocab, int32_t hidden_size, double temperature, const int32_t *ids,
                               int32_t nids, const float *logprobs, const float *lse, const float *entropy,
                               const float *dlogprobs, const float *dentropy, void *dhidden, int64_t lddh, void *dweight,
                               int64_t lddw, void *workspace, int64_t workspace_bytes, void *stream) {
  t_last_error.clear();
  const char *m = bad_row_args(rows, vocab, nids, ids, dlogprobs, temperature);
  if (!m) m = bad_vocab_args(hidden, ldh, weight, ldw, dtype, rows, vocab, hidden_size);
  if (!m && dhidden) m = bad_matrix(dhidden, rows, hidden_size, lddh, 2);
  if (!m && dweight) m = bad_matrix(dweight, vocab, hidden_size, lddw, 2);
  if (!m && rows > 0 && (!lse || (nids > 0 && !logprobs) || (dentropy && !entropy))) m = "null argument";
  if (!m) {
    const RowSpan h(hidden, rows, hidden_size, ldh, 2), w(weight, vocab, hidden_size, ldw, 2),
        dh(dhidden, rows, hidden_size, lddh, 2), dw(dweight, vocab, hidden_size, lddw, 2);
    if (overlap(dh, h) || overlap(dh, w) || overlap(dw, h) || overlap(dw, w) || overlap(dh, dw))
      m = "the gradients cannot overlap the operands or one another";
  }
  if (m) return fail(IG_ERR_BAD_ARG, std::string("ig_vocab_logprobs_backward: ") + m);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (!dhidden && !dweight) return 0;
  if (rows == 0) {
    if (dweight) IG_CU(cudaMemset2DAsync(dweight, (size_t)lddw * 2, 0, (size_t)hidden_size * 2, vocab, st));
    return 0;
  }
  const VPlan p = vocab_plan(rows, vocab, hidden_size, 0);
  if (!workspace || workspace_bytes < (int64_t)p.bwd_bytes || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return fail(IG_ERR_BAD_ARG, "ig_vocab_logprobs_backward: workspace missing, too small or not aligned to 256 bytes");
  LogprobGradArgs g{};
  g.rows = rows;
  g.V = vocab;
  g.T = nids;
  g.c = (float)(1.0 / temperature);
  g.ids = ids;
  g.lse = lse;
  g.entropy = entropy;
  g.dlogprobs = nids > 0 ? dlogprobs : nullptr;
  g.dentropy = dentropy;
  const int products = 1 + (dhidden != nullptr) + (dweight != nullptr);
  ProfScope ps("vocab_logprobs_backward", 4.0 * ((double)rows + vocab) * hidden_size,
               2.0 * products * rows * vocab * hidden_size, 4 + products, st);
  return run_vocab_grad(VMatrices{hidden, weight, ldh, ldw, dtype}, p, g,
                        VocabGradOut{logprobs, dhidden, dweight, lddh, lddw}, static_cast<uint8_t *>(workspace), st);
}

}  // extern "C"
