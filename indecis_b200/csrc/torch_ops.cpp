// The training operators' calls from Python: arguments checked, outputs and
// workspaces allocated and the C entry point called in one step. A call through
// ctypes and torch's Python interface takes 14 to 20 us of the host (layer norm
// 14.5, its backward pass 20), which is longer than the small calls' kernels;
// this takes about half, and for AdamW a tenth (2 us a tensor there). Nothing
// is computed here; the entry points are those of the header.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <cstdint>
#include <string>
#include <vector>

#include "../../include/indecis_b200.h"

namespace {

struct BadValue {
  std::string what;
};
struct Status {  // of an entry point that did not succeed
  int rc;
};

// A size as the entry points take it: one past 31 bits stays too large, and is refused there.
int32_t narrow(int64_t v) { return (int32_t)std::min<int64_t>(v, INT32_MAX); }

int type_of(const at::Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return IG_DT_F32;
    case at::kBFloat16: return IG_DT_BF16;
    case at::kHalf: return IG_DT_F16;
    default: return -1;
  }
}

// A tensor argument; None: an undefined tensor where that is allowed.
const at::Tensor &tensor(PyObject *o, const char *name, bool optional = false) {
  static const at::Tensor none;
  if (optional && o == Py_None) return none;
  if (!THPVariable_Check(o)) throw BadValue{std::string(name) + ": expected a tensor"};
  return THPVariable_Unpack(o);
}

// A CUDA matrix with a unit column stride and rows apart by at least their length.
struct Matrix {
  const at::Tensor *t;
  void *p;
  int64_t rows, cols, ld;
  int type;
};
Matrix matrix(const at::Tensor &t, const char *name) {
  Matrix m{&t, nullptr, 0, 0, 0, type_of(t)};
  if (t.dim() == 2 && t.is_cuda() && m.type >= 0) {
    m.rows = t.size(0);
    m.cols = t.size(1);
    m.ld = m.rows <= 1 ? m.cols : t.stride(0);
    if ((m.cols <= 1 || t.stride(1) == 1) && m.ld >= m.cols) {
      m.p = t.data_ptr();
      return m;
    }
  }
  throw BadValue{std::string(name) +
                 ": expected a CUDA float32, bfloat16 or float16 matrix with a unit column stride, rows apart by at least their "
                 "length"};
}
void like(const Matrix &m, const Matrix &x, const char *name, bool type) {
  if (m.t->device() != x.t->device() || (type && m.type != x.type) || m.rows != x.rows || m.cols != x.cols)
    throw BadValue{std::string(name) + ": expected x's shape" + (type ? ", type" : "") + " and device"};
}

// A contiguous vector of n on x's device.
void *vector(const at::Tensor &t, int64_t n, const Matrix &x, const char *name, int &type) {
  if (!t.defined()) return nullptr;
  const int ty = type_of(t);
  if (ty < 0 || t.dim() != 1 || t.size(0) != n || t.device() != x.t->device() || !t.is_contiguous())
    throw BadValue{std::string(name) + ": expected a contiguous float32, bfloat16 or float16 vector of " + std::to_string(n) +
                   " on x's device"};
  if (type >= 0 && type != ty) throw BadValue{"weight and bias: expected one type"};
  type = ty;
  return t.data_ptr();
}
const float *stats(const at::Tensor &t, const Matrix &x, const char *name) {
  if (t.scalar_type() != at::kFloat || t.dim() != 1 || t.size(0) != x.rows || t.device() != x.t->device() || !t.is_contiguous())
    throw BadValue{std::string(name) + ": expected a contiguous float32 vector of x's rows on its device"};
  return static_cast<const float *>(t.data_ptr());
}

at::Tensor new_matrix(const Matrix &x, int64_t rows, int64_t cols, int type) {
  static const at::ScalarType types[3] = {at::kFloat, at::kBFloat16, at::kHalf};
  return at::empty({rows, cols}, x.t->options().dtype(types[type]).requires_grad(false));
}
at::Tensor new_vector(const Matrix &x, int64_t n, int type) {
  static const at::ScalarType types[3] = {at::kFloat, at::kBFloat16, at::kHalf};
  return at::empty({n}, x.t->options().dtype(types[type]).requires_grad(false));
}
at::Tensor scratch(const Matrix &x, int64_t bytes) {
  return bytes > 0 ? at::empty({bytes}, x.t->options().dtype(at::kByte).requires_grad(false)) : at::Tensor();
}
void *address(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// Autograd notices that what it may have kept is another value now.
void written(const at::Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

struct On {  // x's device current, and its current stream
  c10::cuda::CUDAGuard guard;
  void *stream;
  explicit On(const at::Tensor &x)
      : guard(x.device()), stream(static_cast<void *>(c10::cuda::getCurrentCUDAStream(x.device().index()).stream())) {}
};
void check(int rc) {
  if (rc) throw Status{rc};
}

double number(PyObject *o, const char *name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    throw BadValue{std::string(name) + ": expected a number"};
  }
  return v;
}
int integer(PyObject *o) { return (int)PyLong_AsLong(o); }

PyObject *wrap(const at::Tensor &t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}
template <typename... T>
PyObject *tuple(const T &...t) {
  PyObject *items[] = {wrap(t)...};
  PyObject *r = PyTuple_New(sizeof...(T));
  for (size_t i = 0; i < sizeof...(T); i++) {
    if (!items[i] || !r) {
      for (size_t k = i; k < sizeof...(T); k++) Py_XDECREF(items[k]);
      Py_XDECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i, items[i]);
  }
  return r;
}

// ---- layer norm ----------------------------------------------------------------------------

// (x, weight, bias, eps, type of the result or -1, out or None) -> (y, mean, rstd)
PyObject *layer_norm(PyObject *const *a) {
  const Matrix x = matrix(tensor(a[0], "x"), "x");
  int wt = -1;
  const void *w = vector(tensor(a[1], "weight", true), x.cols, x, "weight", wt),
             *b = vector(tensor(a[2], "bias", true), x.cols, x, "bias", wt);
  const double eps = number(a[3], "eps");
  int type = integer(a[4]);
  at::Tensor y = tensor(a[5], "out", true);
  int64_t ldy = x.cols;
  if (y.defined()) {
    const Matrix o = matrix(y, "out");
    like(o, x, "out", false);
    if (type >= 0 && type != o.type) throw BadValue{"out: expected out_dtype"};
    type = o.type;
    ldy = o.ld;
  } else {
    if (type < 0) type = x.type;
    y = new_matrix(x, x.rows, x.cols, type);
  }
  at::Tensor mean = new_vector(x, x.rows, IG_DT_F32), rstd = new_vector(x, x.rows, IG_DT_F32);
  const On on(*x.t);
  check(ig_layer_norm(x.p, x.type, x.ld, x.rows, narrow(x.cols), w, b, wt < 0 ? IG_DT_F32 : wt, eps, y.data_ptr(), type, ldy,
                      static_cast<float *>(mean.data_ptr()), static_cast<float *>(rstd.data_ptr()), on.stream));
  if (a[5] != Py_None) written(y);
  return tuple(y, mean, rstd);
}

// (dy, x, mean, rstd, weight, need_weight, need_bias, out or None) -> (dx, dweight, dbias)
PyObject *layer_norm_backward(PyObject *const *a) {
  const Matrix dy = matrix(tensor(a[0], "dy"), "dy"), x = matrix(tensor(a[1], "x"), "x");
  like(dy, x, "dy", false);
  const float *mean = stats(tensor(a[2], "mean"), x, "mean"), *rstd = stats(tensor(a[3], "rstd"), x, "rstd");
  int wt = -1;
  const void *w = vector(tensor(a[4], "weight", true), x.cols, x, "weight", wt);
  if (wt < 0) wt = IG_DT_F32;
  const bool need_w = a[5] == Py_True, need_b = a[6] == Py_True;
  at::Tensor dx = tensor(a[7], "out", true);
  int64_t ldo = x.cols;
  if (dx.defined()) {
    const Matrix o = matrix(dx, "out");
    like(o, x, "out", true);
    ldo = o.ld;
  } else {
    dx = new_matrix(x, x.rows, x.cols, x.type);
  }
  at::Tensor dw, db, ws;
  if (need_w) dw = new_vector(x, x.cols, wt);
  if (need_b) db = new_vector(x, x.cols, wt);
  const On on(*x.t);
  const int64_t bytes = need_w || need_b ? ig_layer_norm_workspace(x.rows, narrow(x.cols)) : 0;
  ws = scratch(x, bytes);
  check(ig_layer_norm_backward(dy.p, dy.type, dy.ld, x.p, x.type, x.ld, x.rows, narrow(x.cols), w, wt, mean, rstd, dx.data_ptr(), ldo,
                               address(dw), address(db), address(ws), bytes, on.stream));
  if (a[7] != Py_None) written(dx);
  return tuple(dx, dw, db);
}

// ---- the gated block -------------------------------------------------------------------------

struct Block {
  Matrix x, wi, wo;
  int64_t rows, hidden, inner, out;
  int unaligned, act;
  Block(PyObject *ox, PyObject *oi, PyObject *oo, PyObject *oa)
      : x(matrix(tensor(ox, "x"), "x")), wi(matrix(tensor(oi, "w_in"), "w_in")), wo(matrix(tensor(oo, "w_out"), "w_out")) {
    if (x.type == IG_DT_F32 || wi.type != x.type || wo.type != x.type || wi.t->device() != x.t->device() ||
        wo.t->device() != x.t->device())
      throw BadValue{"x, w_in and w_out: expected all bfloat16 or all float16, on one device"};
    rows = x.rows;
    hidden = x.cols;
    inner = wo.cols;
    out = wo.rows;
    if (wi.rows != 2 * inner || wi.cols != hidden)
      throw BadValue{"w_in: expected [2 * inner, hidden], inner as in w_out [out, inner]"};
    act = integer(oa);
    unaligned = off(x) | off(wi) << 1 | off(wo) << 2;
  }
  static int off(const Matrix &m) { return reinterpret_cast<uintptr_t>(m.p) % 16 != 0 || (m.rows > 1 && m.ld % 8 != 0); }
};

// (x, w_in, w_out, activation, save) -> (y, saved or None)
PyObject *gated_ff(PyObject *const *a) {
  const Block b(a[0], a[1], a[2], a[3]);
  const bool save = a[4] == Py_True;
  at::Tensor y = new_matrix(b.x, b.rows, b.out, b.x.type), saved, ws;
  if (save) saved = at::empty({ig_gated_ff_saved(b.rows, narrow(b.inner))}, b.x.t->options().dtype(at::kByte).requires_grad(false));
  const On on(*b.x.t);
  const int64_t bytes = ig_gated_ff_workspace(b.rows, narrow(b.hidden), narrow(b.inner), narrow(b.out), b.unaligned, save);
  ws = scratch(b.x, bytes);
  check(ig_gated_ff(b.x.p, b.x.ld, b.wi.p, b.wi.ld, b.wo.p, b.wo.ld, b.x.type, b.rows, narrow(b.hidden), narrow(b.inner),
                    narrow(b.out), b.act, y.data_ptr(), b.out, address(saved), address(ws), bytes, on.stream));
  return tuple(y, saved);
}

// (dy, x, w_in, w_out, saved, activation, need_input, need_in, need_out) -> (dx, dw_in, dw_out)
PyObject *gated_ff_backward(PyObject *const *a) {
  const Matrix dy = matrix(tensor(a[0], "dy"), "dy");
  const Block b(a[1], a[2], a[3], a[5]);
  if (dy.rows != b.rows || dy.cols != b.out || dy.type != b.x.type || dy.t->device() != b.x.t->device())
    throw BadValue{"dy: expected [rows, out] of x's type and device"};
  const at::Tensor &saved = tensor(a[4], "saved");
  if (saved.scalar_type() != at::kByte || saved.device() != b.x.t->device() || !saved.is_contiguous() ||
      saved.numel() != ig_gated_ff_saved(b.rows, narrow(b.inner)))
    throw BadValue{"saved: expected what gated_ff saved for operands of these sizes"};
  at::Tensor dx, dwi, dwo, ws;
  if (a[6] == Py_True) dx = new_matrix(b.x, b.rows, b.hidden, b.x.type);
  if (a[7] == Py_True) dwi = new_matrix(b.x, 2 * b.inner, b.hidden, b.x.type);
  if (a[8] == Py_True) dwo = new_matrix(b.x, b.out, b.inner, b.x.type);
  const On on(*b.x.t);
  const int64_t bytes = ig_gated_ff_workspace(b.rows, narrow(b.hidden), narrow(b.inner), narrow(b.out),
                                              b.unaligned | Block::off(dy) << 3, 2);
  ws = scratch(b.x, bytes);
  check(ig_gated_ff_backward(dy.p, dy.ld, b.x.p, b.x.ld, b.wi.p, b.wi.ld, b.wo.p, b.wo.ld, b.x.type, b.rows, narrow(b.hidden),
                             narrow(b.inner), narrow(b.out), b.act, saved.data_ptr(), address(dx), b.hidden, address(dwi), b.hidden,
                             address(dwo), b.inner, address(ws), bytes, on.stream));
  return tuple(dx, dwi, dwo);
}

// ---- AdamW --------------------------------------------------------------------------------------

struct List {  // a list or tuple, held while it is read
  PyObject *seq;
  Py_ssize_t n;
  List(PyObject *o, const char *name) : seq(PySequence_Fast(o, "")) {
    if (!seq) {
      PyErr_Clear();
      throw BadValue{std::string(name) + ": expected a list"};
    }
    n = PySequence_Fast_GET_SIZE(seq);
  }
  List(const List &) = delete;
  ~List() { Py_DECREF(seq); }
  PyObject *operator[](Py_ssize_t i) const { return PySequence_Fast_GET_ITEM(seq, i); }
};

void *dense(PyObject *o, int64_t n, const at::Device &dev, const char *name) {
  const at::Tensor &t = tensor(o, name);
  if (t.numel() != n || t.device() != dev || !t.is_contiguous())
    throw BadValue{std::string(name) + ": expected contiguous tensors of the parameters' sizes, all on their device"};
  return t.data_ptr();
}
void *typed(PyObject *o, int64_t n, const at::Device &dev, const char *name, at::ScalarType type) {
  void *p = dense(o, n, dev, name);
  if (THPVariable_Unpack(o).scalar_type() != type) throw BadValue{std::string(name) + ": expected " + at::toString(type)};
  return p;
}
void *one(PyObject *o, at::ScalarType type, const at::Device &dev, const char *name) {
  if (o == Py_None) return nullptr;
  const at::Tensor &t = tensor(o, name);
  if (t.scalar_type() != type || t.numel() != 1 || t.device() != dev)
    throw BadValue{std::string(name) + ": expected one " + at::toString(type) + " value on the parameters' device"};
  return t.data_ptr();
}

// (params, grads, exp_avg, exp_avg_sq, step, lr, beta1, beta2, eps, weight_decay, copies, grad_scale, skip)
PyObject *adamw_step(PyObject *const *a) {
  const at::Tensor &step = tensor(a[4], "step");
  if (!step.is_cuda() || step.scalar_type() != at::kInt || step.numel() != 1)
    throw BadValue{"step: expected one int32 value on the GPU"};
  const at::Device dev = step.device();
  const List params(a[0], "params"), grads(a[1], "grads"), ms(a[2], "exp_avg"), vs(a[3], "exp_avg_sq");
  const bool one_decay = PyNumber_Check(a[9]) && !PySequence_Check(a[9]), copying = a[10] != Py_None;
  const List decays(one_decay ? a[0] : a[9], "weight_decay"), copies(copying ? a[10] : a[0], "copies");
  const Py_ssize_t n = params.n;
  if (grads.n != n || ms.n != n || vs.n != n || copies.n != n) throw BadValue{"expected lists of one length"};
  if (decays.n != n) throw BadValue{"weight_decay: expected one number, or one for each tensor"};
  std::vector<int64_t> size;
  std::vector<void *> p, m, v, c;
  std::vector<const void *> g;
  std::vector<float *> msc, vsc;
  std::vector<uint8_t> pt, gt, ct;
  std::vector<float> wd;
  size.reserve(n), p.reserve(n), m.reserve(n), v.reserve(n), g.reserve(n), pt.reserve(n), gt.reserve(n), wd.reserve(n);
  Py_ssize_t used = 0;  // the first tensor that takes part says how the moments are held
  while (used < n && grads[used] == Py_None) used++;
  const bool bits8 = used < n && !THPVariable_Check(ms[used]);
  for (Py_ssize_t i = 0; i < n; i++) {
    if (grads[i] == Py_None) continue;  // left out
    const at::Tensor &param = tensor(params[i], "params");
    const int64_t k = param.numel();
    size.push_back(k);
    p.push_back(dense(params[i], k, dev, "params"));
    g.push_back(dense(grads[i], k, dev, "grads"));
    const int tp = type_of(param), tg = type_of(THPVariable_Unpack(grads[i]));
    if (tp < 0 || tg < 0) throw BadValue{"params, grads: expected float32, bfloat16 or float16"};
    pt.push_back((uint8_t)tp);
    gt.push_back((uint8_t)tg);
    if (bits8) {
      const List mc(ms[i], "exp_avg"), vc(vs[i], "exp_avg_sq");
      if (mc.n != 2 || vc.n != 2) throw BadValue{"exp_avg, exp_avg_sq: expected (codes, scales) pairs"};
      const int64_t blocks = (k + 255) / 256;
      m.push_back(typed(mc[0], k, dev, "exp_avg", at::kFloat8_e4m3fn));
      v.push_back(typed(vc[0], k, dev, "exp_avg_sq", at::kFloat8_e4m3fn));
      msc.push_back(static_cast<float *>(typed(mc[1], blocks, dev, "exp_avg scales", at::kFloat)));
      vsc.push_back(static_cast<float *>(typed(vc[1], blocks, dev, "exp_avg_sq scales", at::kFloat)));
    } else {
      m.push_back(typed(ms[i], k, dev, "exp_avg", at::kFloat));
      v.push_back(typed(vs[i], k, dev, "exp_avg_sq", at::kFloat));
    }
    if (copying) {
      c.push_back(dense(copies[i], k, dev, "copies"));
      const int t = type_of(THPVariable_Unpack(copies[i]));
      if (t != IG_DT_BF16 && t != IG_DT_F16) throw BadValue{"copies: expected bfloat16 or float16"};
      ct.push_back((uint8_t)t);
    }
    wd.push_back((float)number(one_decay ? a[9] : decays[i], "weight_decay"));
  }
  ig_adamw_tensors t{};
  t.count = (int64_t)size.size();
  t.n = size.data();
  t.param = p.data();
  t.grad = g.data();
  t.exp_avg = m.data();
  t.exp_avg_sq = v.data();
  t.exp_avg_scale = msc.data();
  t.exp_avg_sq_scale = vsc.data();
  t.copy = copying ? c.data() : nullptr;
  t.param_dtype = pt.data();
  t.grad_dtype = gt.data();
  t.copy_dtype = ct.data();
  t.weight_decay = wd.data();
  const float *gs = static_cast<const float *>(one(a[11], at::kFloat, dev, "grad_scale")),
              *skip = static_cast<const float *>(one(a[12], at::kFloat, dev, "skip"));
  const On on(step);
  check(ig_adamw_step(&t, bits8 ? 8 : 32, number(a[5], "lr"), number(a[6], "beta1"), number(a[7], "beta2"), number(a[8], "eps"),
                      static_cast<int32_t *>(step.data_ptr()), gs, skip, on.stream));
  for (Py_ssize_t i = 0; i < n; i++) {
    if (grads[i] == Py_None) continue;
    written(THPVariable_Unpack(params[i]));
    if (copying) written(THPVariable_Unpack(copies[i]));
  }
  Py_RETURN_NONE;
}

// ---- the module ---------------------------------------------------------------------------------

PyObject *raise_status = nullptr;   // _capi.check
PyObject *out_of_memory = nullptr;  // torch.OutOfMemoryError

// Exceptions end here: a bad argument as ValueError, a status as _capi.check raises it.
template <PyObject *(*F)(PyObject *const *), int N>
PyObject *call(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != N) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  try {
    PyObject *r = F(args);
    if (PyErr_Occurred()) {
      Py_XDECREF(r);
      return nullptr;
    }
    return r;
  } catch (const BadValue &e) {
    PyErr_SetString(PyExc_ValueError, e.what.c_str());
  } catch (const Status &e) {
    PyObject *r = raise_status ? PyObject_CallFunction(raise_status, "i", e.rc) : nullptr;
    if (r) {
      Py_DECREF(r);
      PyErr_SetString(PyExc_RuntimeError, ig_last_error());
    }
  } catch (const c10::OutOfMemoryError &e) {
    PyErr_SetString(out_of_memory ? out_of_memory : PyExc_MemoryError, e.what_without_backtrace());
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

template <PyObject *(*F)(PyObject *const *), int N>
PyMethodDef method(const char *name) {
  return PyMethodDef{name, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&call<F, N>)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<layer_norm, 6>("layer_norm"),
                         method<layer_norm_backward, 8>("layer_norm_backward"),
                         method<gated_ff, 5>("gated_ff"),
                         method<gated_ff_backward, 9>("gated_ff_backward"),
                         method<adamw_step, 13>("adamw_step"),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops() {
  PyObject *m = PyModule_Create(&module);
  if (!m) return nullptr;
  auto attribute = [](const char *from, const char *name) {
    PyObject *mod = PyImport_ImportModule(from), *v = mod ? PyObject_GetAttrString(mod, name) : nullptr;
    Py_XDECREF(mod);
    return v;
  };
  raise_status = attribute("indecis_b200._capi", "check");
  out_of_memory = attribute("torch", "OutOfMemoryError");
  if (!raise_status || !out_of_memory) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
