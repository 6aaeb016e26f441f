// The per-call part of f2cgt_b200/ops.py for layer norm, 8-bit activations and learned rows.
#include "native.h"

namespace f2c_native {
namespace {

constexpr int64_t kGroup = F2C_CHECKPOINT_GROUP;
int64_t groups_of(int64_t d) { return (d + kGroup - 1) / kGroup; }
int64_t bytes16(int64_t d) { return (d + 15) / 16 * 16; }

// A float vector [d], or None.
const float* vector(PyObject* o, const at::Tensor& x, int64_t d, const char* op, const char* name) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o, name, kF32);
  if (t.dim() != 1 || t.size(0) != d) fail(PyExc_RuntimeError, "%s must be [%lld]", name, (long long)d);
  same_device(t, x, name);
  no_gradient(t, op, name);
  return t.const_data_ptr<float>();
}

// A vector of one of `allowed` types [m] that must be there.
const at::Tensor& of_rows(PyObject* o, const at::Tensor& x, int64_t m, unsigned allowed, const char* op, const char* name) {
  const at::Tensor& t = tensor(o, name, allowed);
  if (t.dim() != 1 || t.size(0) != m) fail(PyExc_RuntimeError, "%s must be [%lld]", name, (long long)m);
  same_device(t, x, name);
  no_gradient(t, op, name);
  return t;
}

// 8-bit activations: codes [m, d] with rows of whole 16 bytes, scales [m, groups, 2].
struct Codes {
  const at::Tensor* codes = nullptr;
  const at::Tensor* scales = nullptr;
  int64_t ld = 0;
  const uint8_t* q() const { return codes != nullptr ? codes->const_data_ptr<uint8_t>() : nullptr; }
  const float* s() const { return codes != nullptr ? scales->const_data_ptr<float>() : nullptr; }
};

Codes codes_of(PyObject* c, PyObject* s, const char* op) {
  Codes r;
  r.codes = &matrix(c, "codes", bit(F2C_U8));
  r.scales = &tensor(s, "scales", kF32);
  const int64_t m = r.codes->size(0), d = r.codes->size(1);
  if (r.scales->dim() != 3 || r.scales->size(0) != m || r.scales->size(1) != groups_of(d) || r.scales->size(2) != 2)
    fail(PyExc_RuntimeError, "scales must be [%lld, %lld, 2]", (long long)m, (long long)groups_of(d));
  same_device(*r.scales, *r.codes, "scales");
  no_gradient(*r.scales, op, "scales");
  r.ld = m > 1 ? r.codes->stride(0) : bytes16(d);
  // (the kernels read whole 16 bytes of every row, the last one's too)
  if (m > 0 && d > 0 && (uint64_t)(r.codes->storage_offset() + (m - 1) * r.ld + bytes16(d)) > r.codes->storage().nbytes())
    fail(PyExc_RuntimeError, "codes must have rows of whole 16 bytes (as checkpoint_int8 lays them out)");
  return r;
}

struct NewCodes { at::Tensor codes, scales; int64_t ld; };
NewCodes new_codes(int64_t m, int64_t d, const at::Device& device) {
  const int64_t ld = bytes16(d);
  return {empty({m, ld}, at::kByte, device), empty({m, groups_of(d), 2}, at::kFloat, device), ld};
}

// A tuple of tensors; undefined ones are None.
template <typename... T>
PyObject* tuple_of(T&&... tensors) {
  at::Tensor all[] = {std::move(tensors)...};
  PyObject* r = PyTuple_New((Py_ssize_t)sizeof...(T));
  if (r == nullptr) return nullptr;
  for (size_t i = 0; i < sizeof...(T); ++i) {
    PyObject* o = all[i].defined() ? THPVariable_Wrap(std::move(all[i])) : Py_NewRef(Py_None);
    if (o == nullptr) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, (Py_ssize_t)i, o);
  }
  return r;
}

PyObject* checkpoint_int8(PyObject*, PyObject* const* a, Py_ssize_t n) {  // x
  return guarded([&]() -> PyObject* {
    arguments("checkpoint_int8", n, 1);
    const at::Tensor& x = matrix(a[0], "x", kFloats);
    no_gradient(x, "checkpoint_int8", "x");
    NewCodes c;
    check_status(unlocked([&] {
      c10::cuda::CUDAGuard guard(x.device());
      const int64_t m = x.size(0), d = x.size(1);
      c = new_codes(m, d, x.device());
      const int rc = f2c_checkpoint_int8(x.const_data_ptr(), row_stride(x), dtype_tag(x.scalar_type()), m, d, c.codes.mutable_data_ptr<uint8_t>(), c.ld,
                                         c.scales.mutable_data_ptr<float>(), stream_of(x));
      c.codes = c.codes.narrow(1, 0, d);
      return rc;
    }));
    return tuple_of(std::move(c.codes), std::move(c.scales));
  });
}

at::ScalarType float_type(PyObject* o) {
  if (!THPDtype_Check(o)) fail(PyExc_TypeError, "dtype must be a torch.dtype");
  const at::ScalarType t = reinterpret_cast<THPDtype*>(o)->scalar_type;
  const int tag = dtype_tag(t);
  if (tag < 0 || !(kFloats & bit(tag))) fail(PyExc_RuntimeError, "dtype %s is unsupported", c10::toString(t));
  return t;
}

PyObject* checkpoint_values(PyObject*, PyObject* const* a, Py_ssize_t n) {  // codes, scales, dtype
  return guarded([&]() -> PyObject* {
    arguments("checkpoint_values", n, 3);
    const Codes c = codes_of(a[0], a[1], "checkpoint_values");
    const at::ScalarType type = float_type(a[2]);
    at::Tensor out;
    check_status(unlocked([&] {
      c10::cuda::CUDAGuard guard(c.codes->device());
      const int64_t m = c.codes->size(0), d = c.codes->size(1);
      out = empty({m, d}, type, c.codes->device());
      return f2c_checkpoint_values(c.q(), c.ld, c.s(), m, d, out.mutable_data_ptr(), d, dtype_tag(type), stream_of(*c.codes));
    }));
    return THPVariable_Wrap(std::move(out));
  });
}

PyObject* checkpoint_weight_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {  // dy, codes, scales -> dw, db
  return guarded([&]() -> PyObject* {
    const char* op = "checkpoint_weight_grad";
    arguments(op, n, 3);
    const at::Tensor& dy = matrix(a[0], "dy", kFloats);
    no_gradient(dy, op, "dy");
    const Codes c = codes_of(a[1], a[2], op);
    same_device(*c.codes, dy, "codes");
    const int64_t m = dy.size(0), cols = dy.size(1), k = c.codes->size(1);
    if (c.codes->size(0) != m) fail(PyExc_RuntimeError, "dy must have as many rows as the input that was kept");
    at::Tensor dw, db;
    check_status(unlocked([&] {
      c10::cuda::CUDAGuard guard(dy.device());
      dw = empty({cols, k}, dy.scalar_type(), dy.device());
      db = empty({cols}, dy.scalar_type(), dy.device());
      const int64_t bytes = f2c_checkpoint_weight_grad_workspace(dy.const_data_ptr(), row_stride(dy), dtype_tag(dy.scalar_type()), m, cols, k);
      at::Tensor ws;
      if (bytes > 0) ws = empty({bytes}, at::kByte, dy.device());
      return f2c_checkpoint_weight_grad(dy.const_data_ptr(), row_stride(dy), dtype_tag(dy.scalar_type()), c.q(), c.ld, c.s(), m, cols, k, dw.mutable_data_ptr(), db.mutable_data_ptr(), 0,
                                        bytes > 0 ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(dy));
    }));
    return tuple_of(std::move(dw), std::move(db));
  });
}

// x, weight, bias, eps, relu, keep (0: nothing, 1: what goes with the rows, 2: and the rows in 8 bits)
// -> y, or y, mean, rstd, active, codes, scales (None: not wanted)
PyObject* layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    arguments("layer_norm", n, 6);
    const at::Tensor& x = matrix(a[0], "x", kFloats);
    no_gradient(x, "layer_norm", "x");
    const int64_t m = x.size(0), d = x.size(1);
    const float* weight = vector(a[1], x, d, "layer_norm", "weight");
    const float* bias = vector(a[2], x, d, "layer_norm", "bias");
    const double eps = real(a[3]);
    const bool relu = truth(a[4]);
    const int64_t keep = integer(a[5]);
    at::Tensor y, mean, rstd, active;
    NewCodes c;
    check_status(unlocked([&] {
      c10::cuda::CUDAGuard guard(x.device());
      y = empty({m, d}, x.scalar_type(), x.device());
      if (keep > 0) {
        mean = empty({m}, at::kFloat, x.device());
        rstd = empty({m}, at::kFloat, x.device());
        if (relu) active = empty({m, (d + 7) / 8}, at::kByte, x.device());
        if (keep > 1) c = new_codes(m, d, x.device());
      }
      const int rc = f2c_layer_norm(x.const_data_ptr(), row_stride(x), dtype_tag(x.scalar_type()), m, d, weight, bias, (float)eps, relu, y.mutable_data_ptr(),
                                    keep > 0 ? mean.mutable_data_ptr<float>() : nullptr, keep > 0 ? rstd.mutable_data_ptr<float>() : nullptr,
                                    active.defined() ? active.mutable_data_ptr<uint8_t>() : nullptr, keep > 1 ? c.codes.mutable_data_ptr<uint8_t>() : nullptr, c.ld,
                                    keep > 1 ? c.scales.mutable_data_ptr<float>() : nullptr, stream_of(x));
      if (keep > 1) c.codes = c.codes.narrow(1, 0, d);
      return rc;
    }));
    if (keep == 0) return THPVariable_Wrap(std::move(y));
    return tuple_of(std::move(y), std::move(mean), std::move(rstd), std::move(active), std::move(c.codes), std::move(c.scales));
  });
}

PyObject* layer_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {  // dy, x or codes, scales (None: x), mean, rstd, active, weight
  return guarded([&]() -> PyObject* {
    const char* op = "layer_norm_backward";
    arguments(op, n, 7);
    const at::Tensor& dy = matrix(a[0], "dy", kFloats);
    no_gradient(dy, op, "dy");
    const int64_t m = dy.size(0), d = dy.size(1);
    Codes c;
    const at::Tensor* x = nullptr;
    if (a[2] != Py_None) {
      c = codes_of(a[1], a[2], op);
      x = c.codes;
    } else {
      x = &matrix(a[1], "x", bit(dtype_tag(dy.scalar_type())));
      no_gradient(*x, op, "x");
    }
    if (x->sizes() != dy.sizes()) fail(PyExc_RuntimeError, "dy must have the shape of the rows that were kept");
    same_device(*x, dy, "the kept rows");
    const float* mean = of_rows(a[3], dy, m, kF32, op, "mean").const_data_ptr<float>();
    const float* rstd = of_rows(a[4], dy, m, kF32, op, "rstd").const_data_ptr<float>();
    const uint8_t* active = nullptr;
    if (a[5] != Py_None) {
      const at::Tensor& t = tensor(a[5], "active", bit(F2C_U8));
      if (t.dim() != 2 || t.size(0) != m || t.size(1) != (d + 7) / 8) fail(PyExc_RuntimeError, "active must be [%lld, %lld]", (long long)m, (long long)((d + 7) / 8));
      same_device(t, dy, "active");
      active = t.const_data_ptr<uint8_t>();
    }
    const float* weight = vector(a[6], dy, d, op, "weight");
    at::Tensor dx, dweight, dbias;
    check_status(unlocked([&] {
      c10::cuda::CUDAGuard guard(dy.device());
      dx = empty({m, d}, dy.scalar_type(), dy.device());
      dweight = empty({d}, at::kFloat, dy.device());
      dbias = empty({d}, at::kFloat, dy.device());
      const int64_t bytes = f2c_layer_norm_backward_workspace(m, d);
      at::Tensor ws;
      if (bytes > 0) ws = empty({bytes}, at::kByte, dy.device());
      return f2c_layer_norm_backward(dy.const_data_ptr(), row_stride(dy), dtype_tag(dy.scalar_type()), c.codes == nullptr ? x->const_data_ptr() : nullptr,
                                     c.codes == nullptr ? row_stride(*x) : 0, c.q(), c.ld, c.s(), mean, rstd, active, weight, m, d, dx.mutable_data_ptr(),
                                     dweight.mutable_data_ptr<float>(), dbias.mutable_data_ptr<float>(), bytes > 0 ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(dy));
    }));
    return tuple_of(std::move(dx), std::move(dweight), std::move(dbias));
  });
}

// Ids of any shape, without gaps; the dtype is checked.
const at::Tensor& ids_of(PyObject* o, const at::Tensor& other) {
  const at::Tensor& ids = tensor(o, "ids", kIndex);
  same_device(ids, other, "ids");
  return ids;
}

PyObject* embedding(PyObject*, PyObject* const* a, Py_ssize_t n) {  // table, ids, scale
  return guarded([&]() -> PyObject* {
    arguments("embedding", n, 3);
    const at::Tensor& table = matrix(a[0], "table", kFloats);
    no_gradient(table, "embedding", "table");
    const at::Tensor& ids = ids_of(a[1], table);
    const double scale = real(a[2]);
    at::Tensor out;
    check_status(unlocked([&] {
      c10::cuda::CUDAGuard guard(table.device());
      c10::DimVector shape(ids.sizes());
      shape.push_back(table.size(1));
      out = empty(shape, table.scalar_type(), table.device());
      return f2c_embedding(table.const_data_ptr(), row_stride(table), dtype_tag(table.scalar_type()), table.size(0), table.size(1), ids.const_data_ptr(),
                           dtype_tag(ids.scalar_type()), ids.numel(), (float)scale, out.mutable_data_ptr(), stream_of(table));
    }));
    return THPVariable_Wrap(std::move(out));
  });
}

// dy, ids, n_rows, scale, whether only the rows that were looked up -> the table's gradient; or looked_up, rows, count
PyObject* embedding_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const char* op = "embedding_backward";
    arguments(op, n, 5);
    if (!THPVariable_Check(a[0])) fail(PyExc_TypeError, "dy must be a torch.Tensor");
    const at::Tensor& given = THPVariable_Unpack(a[0]);
    // (a matrix may have its rows further apart)
    const at::Tensor& dy = given.dim() == 2 ? matrix(a[0], "dy", kFloats) : tensor(a[0], "dy", kFloats);
    no_gradient(dy, op, "dy");
    const at::Tensor& ids = ids_of(a[1], dy);
    const int64_t rows = integer(a[2]);
    const double scale = real(a[3]);
    const bool sparse = truth(a[4]);
    if (dy.dim() != ids.dim() + 1 || dy.sizes().slice(0, ids.dim()) != ids.sizes()) fail(PyExc_RuntimeError, "dy must be a row for every id");
    if (rows < 0) fail(PyExc_RuntimeError, "n_rows must not be negative");
    const int64_t m = ids.numel(), d = dy.size(-1);
    at::Tensor grad, looked_up, count;
    check_status(unlocked([&] {
      c10::cuda::CUDAGuard guard(dy.device());
      grad = empty({sparse ? m : rows, d}, dy.scalar_type(), dy.device());
      if (sparse) {
        looked_up = empty({m}, at::kLong, dy.device());
        count = empty({1}, at::kLong, dy.device());
      }
      const int64_t bytes = f2c_embedding_backward_workspace(m, rows, d);
      at::Tensor ws;
      if (bytes > 0) ws = empty({bytes}, at::kByte, dy.device());
      return f2c_embedding_backward(dy.const_data_ptr(), dy.dim() == 2 ? row_stride(dy) : d, dtype_tag(dy.scalar_type()), ids.const_data_ptr(), dtype_tag(ids.scalar_type()), m, rows,
                                    d, (float)scale, grad.mutable_data_ptr(), sparse ? looked_up.mutable_data_ptr<int64_t>() : nullptr,
                                    sparse ? count.mutable_data_ptr<int64_t>() : nullptr, bytes > 0 ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(dy));
    }));
    if (!sparse) return THPVariable_Wrap(std::move(grad));
    return tuple_of(std::move(looked_up), std::move(grad), std::move(count));
  });
}

}  // namespace

PyMethodDef g_learn_methods[] = {{"checkpoint_int8", (PyCFunction)(void*)checkpoint_int8, METH_FASTCALL, nullptr},
                                 {"checkpoint_values", (PyCFunction)(void*)checkpoint_values, METH_FASTCALL, nullptr},
                                 {"checkpoint_weight_grad", (PyCFunction)(void*)checkpoint_weight_grad, METH_FASTCALL, nullptr},
                                 {"layer_norm", (PyCFunction)(void*)layer_norm, METH_FASTCALL, nullptr},
                                 {"layer_norm_backward", (PyCFunction)(void*)layer_norm_backward, METH_FASTCALL, nullptr},
                                 {"embedding", (PyCFunction)(void*)embedding, METH_FASTCALL, nullptr},
                                 {"embedding_backward", (PyCFunction)(void*)embedding_backward, METH_FASTCALL, nullptr},
                                 {nullptr, nullptr, 0, nullptr}};

}  // namespace f2c_native
