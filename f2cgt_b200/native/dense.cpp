// The per-call part of f2cgt_b200/ops.py for the 8-bit products and the orthogonalised updates.
#include "native.h"

#include <vector>

#include <c10/core/AutogradState.h>
#include <torch/csrc/autograd/grad_mode.h>

namespace f2c_native {
namespace {

constexpr unsigned kFloats = bit(F2C_F32) | bit(F2C_F16) | bit(F2C_BF16);

// A CUDA matrix of one of `allowed` dtypes with contiguous rows, at any distance that keeps them apart.
const at::Tensor& matrix(PyObject* o, const char* name, unsigned allowed) {
  if (!THPVariable_Check(o)) fail(PyExc_TypeError, "%s must be a torch.Tensor", name);
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda()) fail(PyExc_RuntimeError, "%s must be a CUDA tensor", name);
  const int tag = dtype_tag(t.scalar_type());
  if (tag < 0 || !(allowed & bit(tag))) fail(PyExc_RuntimeError, "%s has unsupported dtype %s", name, c10::toString(t.scalar_type()));
  if (t.dim() != 2) fail(PyExc_RuntimeError, "%s must be 2-D", name);
  if ((t.size(1) > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < t.size(1))) fail(PyExc_RuntimeError, "%s must have contiguous rows", name);
  return t;
}

int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

void same_device(const at::Tensor& t, const at::Tensor& other, const char* name) {
  if (t.device() != other.device()) fail(PyExc_RuntimeError, "%s is on another device", name);
}

void no_gradient(const at::Tensor& t, const char* op, const char* name) {
  if (t.requires_grad() && at::GradMode::is_enabled())
    fail(PyExc_RuntimeError, "%s has no gradient: %s requires one (detach it, or call under torch.no_grad())", op, name);
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
    fail(PyExc_RuntimeError, "%s has no forward-mode derivative: %s has a tangent", op, name);
}

struct Rows {
  const at::Tensor* x1 = nullptr;
  const at::Tensor* x2 = nullptr;
  int64_t m() const { return x1->size(0); }
  int64_t k1() const { return x1->size(1); }
  int64_t k2() const { return x2 != nullptr ? x2->size(1) : 0; }
  const void* p2() const { return x2 != nullptr ? x2->const_data_ptr() : nullptr; }
  int64_t ld2() const { return x2 != nullptr ? row_stride(*x2) : 0; }
};

Rows rows(PyObject* a, PyObject* b, const char* op) {
  Rows r;
  r.x1 = &matrix(a, "x", kFloats);
  no_gradient(*r.x1, op, "x");
  if (b != Py_None) {
    r.x2 = &matrix(b, "x2", bit(dtype_tag(r.x1->scalar_type())));
    no_gradient(*r.x2, op, "x2");
    same_device(*r.x2, *r.x1, "x2");
    if (r.x2->size(0) != r.m()) fail(PyExc_RuntimeError, "x and x2 must have the same number of rows");
  }
  return r;
}

// The weights' codes and scales, and the bias (None: none).
struct Weights {
  const at::Tensor *w, *scales, *bias = nullptr;
  int64_t n() const { return w->size(0); }
  const float* b() const { return bias != nullptr ? bias->const_data_ptr<float>() : nullptr; }
};

Weights weights(PyObject* w, PyObject* s, PyObject* b, const at::Tensor& x, int64_t k, const char* op) {
  Weights r;
  r.w = &matrix(w, "w_codes", bit(F2C_I8));
  r.scales = &tensor(s, "w_scales", kF32);
  if (r.w->size(1) != k) fail(PyExc_RuntimeError, "w_codes must be [n, %lld]", (long long)k);
  if (r.scales->dim() != 1 || r.scales->size(0) != r.n()) fail(PyExc_RuntimeError, "w_scales must be [n]");
  same_device(*r.w, x, "w_codes");
  same_device(*r.scales, x, "w_scales");
  no_gradient(*r.scales, op, "w_scales");
  if (b != Py_None) {
    r.bias = &tensor(b, "bias", kF32);
    if (r.bias->dim() != 1 || r.bias->size(0) != r.n()) fail(PyExc_RuntimeError, "bias must be [n]");
    same_device(*r.bias, x, "bias");
    no_gradient(*r.bias, op, "bias");
  }
  return r;
}

at::ScalarType float_type(PyObject* o, at::ScalarType otherwise) {
  if (o == Py_None) return otherwise;
  if (!THPDtype_Check(o)) fail(PyExc_TypeError, "out_dtype must be a torch.dtype");
  const at::ScalarType t = reinterpret_cast<THPDtype*>(o)->scalar_type;
  const int tag = dtype_tag(t);
  if (tag < 0 || !(kFloats & bit(tag))) fail(PyExc_RuntimeError, "out_dtype %s is unsupported", c10::toString(t));
  return t;
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PythonError{};
  return v != 0;
}

PyObject* pair(at::Tensor a, at::Tensor b) {
  PyObject* x = THPVariable_Wrap(std::move(a));
  PyObject* y = THPVariable_Wrap(std::move(b));
  PyObject* r = x != nullptr && y != nullptr ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x); Py_XDECREF(y);
  return r;
}

PyObject* int8_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {  // x, x2
  return guarded([&]() -> PyObject* {
    arguments("int8_quantize", n, 2);
    const Rows r = rows(a[0], a[1], "int8_quantize");
    const int64_t k = r.k1() + r.k2(), ld = (k + 15) / 16 * 16;
    at::Tensor codes, scales;
    check_status(unlocked([&] {
      c10::cuda::CUDAGuard guard(r.x1->device());
      codes = empty({r.m(), ld}, at::kChar, r.x1->device());
      scales = empty({r.m()}, at::kFloat, r.x1->device());
      const int rc = f2c_int8_quantize(r.x1->const_data_ptr(), row_stride(*r.x1), r.k1(), r.p2(), r.ld2(), r.k2(), dtype_tag(r.x1->scalar_type()),
                                       r.m(), (int8_t*)codes.mutable_data_ptr(), ld, scales.mutable_data_ptr<float>(), stream_of(*r.x1));
      if (ld != k) codes = codes.narrow(1, 0, k);
      return rc;
    }));
    return pair(std::move(codes), std::move(scales));
  });
}

PyObject* int8_mm(PyObject*, PyObject* const* a, Py_ssize_t n) {  // codes, scales, w_codes, w_scales, bias, relu, out_dtype
  return guarded([&]() -> PyObject* {
    arguments("int8_mm", n, 7);
    const at::Tensor& q = matrix(a[0], "codes", bit(F2C_I8));
    const at::Tensor& s = tensor(a[1], "scales", kF32);
    if (s.dim() != 1 || s.size(0) != q.size(0)) fail(PyExc_RuntimeError, "scales must be [m]");
    same_device(s, q, "scales");
    no_gradient(s, "int8_mm", "scales");
    const Weights w = weights(a[2], a[3], a[4], q, q.size(1), "int8_mm");
    const bool relu = truth(a[5]);
    const at::ScalarType type = float_type(a[6], at::kFloat);
    at::Tensor out;
    check_status(unlocked([&] {
      c10::cuda::CUDAGuard guard(q.device());
      const int64_t m = q.size(0), cols = w.n(), k = q.size(1);
      const int8_t *qp = (const int8_t*)q.const_data_ptr(), *wp = (const int8_t*)w.w->const_data_ptr();
      out = empty({m, cols}, type, q.device());
      const int64_t bytes = f2c_int8_mm_workspace(qp, row_stride(q), wp, row_stride(*w.w), m, cols, k);
      at::Tensor ws;
      if (bytes > 0) ws = empty({bytes}, at::kByte, q.device());
      return f2c_int8_mm(qp, row_stride(q), s.const_data_ptr<float>(), wp, row_stride(*w.w), w.scales->const_data_ptr<float>(), w.b(), relu,
                         out.mutable_data_ptr(), dtype_tag(type), m, cols, k, bytes > 0 ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(q));
    }));
    return THPVariable_Wrap(std::move(out));
  });
}

PyObject* int8_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {  // x, x2, w_codes, w_scales, bias, relu, out_dtype
  return guarded([&]() -> PyObject* {
    arguments("int8_linear", n, 7);
    const Rows r = rows(a[0], a[1], "int8_linear");
    const Weights w = weights(a[2], a[3], a[4], *r.x1, r.k1() + r.k2(), "int8_linear");
    const bool relu = truth(a[5]);
    const at::ScalarType type = float_type(a[6], r.x1->scalar_type());
    at::Tensor out;
    check_status(unlocked([&] {
      c10::cuda::CUDAGuard guard(r.x1->device());
      const int64_t m = r.m(), cols = w.n();
      const int8_t* wp = (const int8_t*)w.w->const_data_ptr();
      out = empty({m, cols}, type, r.x1->device());
      const int64_t bytes = f2c_int8_linear_workspace(r.x1->const_data_ptr(), row_stride(*r.x1), r.k1(), r.p2(), r.ld2(), r.k2(),
                                                      dtype_tag(r.x1->scalar_type()), wp, row_stride(*w.w), m, cols);
      at::Tensor ws;
      if (bytes > 0) ws = empty({bytes}, at::kByte, r.x1->device());
      return f2c_int8_linear(r.x1->const_data_ptr(), row_stride(*r.x1), r.k1(), r.p2(), r.ld2(), r.k2(), dtype_tag(r.x1->scalar_type()), wp,
                             row_stride(*w.w), w.scales->const_data_ptr<float>(), w.b(), relu, out.mutable_data_ptr(), dtype_tag(type), m, cols,
                             bytes > 0 ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(*r.x1));
    }));
    return THPVariable_Wrap(std::move(out));
  });
}

// (a, b, c) for every step, or one triple per step
struct Steps {
  float co[3 * F2C_MAX_NS_STEPS];
  int count = 0;
};

struct Kept {  // a reference that is given back
  PyObject* o;
  ~Kept() { Py_XDECREF(o); }
};

Steps steps(PyObject* count, PyObject* coefficients) {
  Steps s;
  Kept all{PySequence_Fast(coefficients, "coefficients must be three numbers, or three for every step")};
  if (all.o == nullptr) throw PythonError{};
  const Py_ssize_t size = PySequence_Fast_GET_SIZE(all.o);
  const bool nested = size > 0 && PySequence_Check(PySequence_Fast_GET_ITEM(all.o, 0));
  const int64_t asked = integer(count);
  if (asked < 0 || asked > F2C_MAX_NS_STEPS) fail(PyExc_RuntimeError, "steps must be 0 to %d", F2C_MAX_NS_STEPS);
  if (nested ? size < asked : size != 3) fail(PyExc_RuntimeError, "coefficients must be three numbers, or three for every step");
  s.count = (int)asked;
  for (int t = 0; t < s.count; ++t) {
    Kept three{PySequence_Fast(nested ? PySequence_Fast_GET_ITEM(all.o, t) : all.o, "coefficients of a step must be three numbers")};
    if (three.o == nullptr) throw PythonError{};
    if (PySequence_Fast_GET_SIZE(three.o) != 3) fail(PyExc_RuntimeError, "coefficients of a step must be three numbers");
    for (int i = 0; i < 3; ++i) s.co[3 * t + i] = (float)real(PySequence_Fast_GET_ITEM(three.o, i));
  }
  return s;
}

PyObject* orthogonalize(PyObject*, PyObject* const* a, Py_ssize_t n) {  // g, steps, coefficients, eps, out
  return guarded([&]() -> PyObject* {
    arguments("orthogonalize", n, 5);
    const at::Tensor& g = tensor(a[0], "g", kFloats);
    no_gradient(g, "orthogonalize", "g");
    if (g.dim() < 2) fail(PyExc_RuntimeError, "g must be [..., rows, cols]");
    const Steps s = steps(a[1], a[2]);
    const double eps = real(a[3]);
    at::Tensor out;
    if (a[4] != Py_None) {
      out = tensor(a[4], "out", bit(dtype_tag(g.scalar_type())));
      no_gradient(out, "orthogonalize", "out");
      if (out.sizes() != g.sizes()) fail(PyExc_RuntimeError, "out must have the shape of g");
      same_device(out, g, "out");
    }
    check_status(unlocked([&] {
      c10::cuda::CUDAGuard guard(g.device());
      if (!out.defined()) out = empty(g.sizes(), g.scalar_type(), g.device());
      const int64_t rows = g.size(-2), cols = g.size(-1), batch = rows > 0 && cols > 0 ? g.numel() / (rows * cols) : 0;
      const int tag = dtype_tag(g.scalar_type());
      const int64_t bytes = f2c_orthogonalize_workspace(tag, batch, rows, cols);
      at::Tensor ws;
      if (bytes > 0) ws = empty({bytes}, at::kByte, g.device());
      return f2c_orthogonalize(g.const_data_ptr(), out.mutable_data_ptr(), tag, batch, rows, cols, s.co, s.count, (float)eps,
                               bytes > 0 ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(g));
    }));
    if (a[4] != Py_None) out.unsafeGetTensorImpl()->bump_version();
    return THPVariable_Wrap(std::move(out));
  });
}

// weights, grads, momenta (sequences), lr, momentum, nesterov, weight_decay, steps, coefficients, eps
PyObject* muon_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arguments("muon_step", n, 10);
    const char* names[3] = {"weights", "grads", "momenta"};
    Kept seq[3] = {{nullptr}, {nullptr}, {nullptr}};
    for (int i = 0; i < 3; ++i) {
      seq[i].o = PySequence_Fast(a[i], "muon_step takes sequences of weights, gradients and momenta");
      if (seq[i].o == nullptr) throw PythonError{};
      if (PySequence_Fast_GET_SIZE(seq[i].o) != PySequence_Fast_GET_SIZE(seq[0].o)) fail(PyExc_RuntimeError, "as many %s as weights are needed", names[i]);
    }
    const double lr = real(a[3]), mu = real(a[4]), decay = real(a[6]), eps = real(a[9]);
    const bool nesterov = truth(a[5]);
    const Steps s = steps(a[7], a[8]);
    const int count = (int)PySequence_Fast_GET_SIZE(seq[0].o);
    std::vector<f2c_muon_matrix> list((size_t)count);
    const at::Tensor* first = nullptr;
    for (int i = 0; i < count; ++i) {
      const at::Tensor& w = tensor(PySequence_Fast_GET_ITEM(seq[0].o, i), "weights", kFloats);
      if (first == nullptr) first = &w;
      const at::Tensor& g = tensor(PySequence_Fast_GET_ITEM(seq[1].o, i), "grads", bit(dtype_tag(w.scalar_type())));
      const at::Tensor& m = tensor(PySequence_Fast_GET_ITEM(seq[2].o, i), "momenta", kF32);
      no_gradient(w, "muon_step", "a weight"); no_gradient(g, "muon_step", "a gradient"); no_gradient(m, "muon_step", "a momentum");
      if (w.scalar_type() != first->scalar_type()) fail(PyExc_RuntimeError, "weights must have one dtype");
      if (w.dim() != 2 || g.sizes() != w.sizes() || m.sizes() != w.sizes()) fail(PyExc_RuntimeError, "weights, grads and momenta must be matrices of one shape");
      same_device(w, *first, "a weight"); same_device(g, *first, "a gradient"); same_device(m, *first, "a momentum");
      list[(size_t)i] = {w.mutable_data_ptr(), g.const_data_ptr(), m.mutable_data_ptr<float>(), w.size(0), w.size(1)};
    }
    if (count > 0) {
      check_status(unlocked([&] {
        c10::cuda::CUDAGuard guard(first->device());
        const int tag = dtype_tag(first->scalar_type());
        const int64_t bytes = f2c_muon_workspace(list.data(), count, tag);
        at::Tensor ws;
        if (bytes > 0) ws = empty({bytes}, at::kByte, first->device());
        return f2c_muon_step(list.data(), count, tag, (float)lr, (float)mu, nesterov, (float)decay, s.co, s.count, (float)eps,
                             bytes > 0 ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(*first));
      }));
      for (int i = 0; i < count; ++i)
        for (int j : {0, 2}) THPVariable_Unpack(PySequence_Fast_GET_ITEM(seq[j].o, i)).unsafeGetTensorImpl()->bump_version();
    }
    Py_RETURN_NONE;
  });
}

}  // namespace

PyMethodDef g_dense_methods[] = {{"int8_quantize", (PyCFunction)(void*)int8_quantize, METH_FASTCALL, nullptr},
                                 {"int8_mm", (PyCFunction)(void*)int8_mm, METH_FASTCALL, nullptr},
                                 {"int8_linear", (PyCFunction)(void*)int8_linear, METH_FASTCALL, nullptr},
                                 {"orthogonalize", (PyCFunction)(void*)orthogonalize, METH_FASTCALL, nullptr},
                                 {"muon_step", (PyCFunction)(void*)muon_step, METH_FASTCALL, nullptr},
                                 {nullptr, nullptr, 0, nullptr}};

}  // namespace f2c_native
