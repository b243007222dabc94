// CPython module kernel._desc: tensor descriptors of an argument block in one
// call.
//
// fill(what, block, offsets, rows, device, refuse_grad, t0, t1, ...) writes the
// saf_tensor_t of each tensor (None: left as it is) at block + offsets[i].
// It raises where a tensor is not on HIP device `device`, has more than four
// dimensions or a dtype the library does not know, or (refuse_grad) needs a
// gradient while grad mode is on.  Bit i of `rows` asks for rows of tensor i
// (4-D, only read) to be 16-byte aligned with a unit last stride; the result
// has the bits of those that are not.
//
// The same through ctypes costs about 0.6 us a tensor, half of the host time
// of a single-token call; here the tensor's fields are read directly.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>

#include "saf_attn.h"

namespace {

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return SAF_F32;
    case at::kHalf: return SAF_F16;
    case at::kBFloat16: return SAF_BF16;
    case at::kInt: return SAF_I32;
    case at::kLong: return SAF_I64;
    default: return -1;
  }
}

bool rows_ok(const at::Tensor& x) {
  if (x.dim() != 4) return true;  // the library names the mistake
  const int64_t es = x.element_size();
  if (reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 || (x.size(3) > 1 && x.stride(3) != 1)) return false;
  for (int i = 0; i < 3; ++i)
    if (x.size(i) > 1 && x.stride(i) * es % 16) return false;
  return true;
}

PyObject* fill(PyObject*, PyObject* const* args, Py_ssize_t n) {
  constexpr Py_ssize_t kFixed = 6;
  if (n < kFixed || !PyTuple_Check(args[2]) || PyTuple_GET_SIZE(args[2]) != n - kFixed) {
    PyErr_SetString(PyExc_TypeError, "fill(what, block, offsets, rows, device, refuse_grad, *tensors)");
    return nullptr;
  }
  const char* what = PyUnicode_AsUTF8(args[0]);
  char* block = static_cast<char*>(PyLong_AsVoidPtr(args[1]));
  const long rows = PyLong_AsLong(args[3]), device = PyLong_AsLong(args[4]);
  const int refuse = PyObject_IsTrue(args[5]);
  if (what == nullptr || PyErr_Occurred()) return nullptr;
  long copies = 0;
  for (Py_ssize_t i = 0; i < n - kFixed; ++i) {
    PyObject* o = args[kFixed + i];
    if (o == Py_None) continue;
    if (!THPVariable_Check(o)) return PyErr_Format(PyExc_TypeError, "%s: a tensor is required, got %R", what, Py_TYPE(o));
    const at::Tensor& x = THPVariable_Unpack(o);
    if (!x.is_cuda() || x.device().index() != device)
      return PyErr_Format(PyExc_ValueError, "%s: a tensor is on %s, expected cuda:%ld", what, x.device().str().c_str(),
                          device);
    if (refuse && x.requires_grad() && at::GradMode::is_enabled())
      return PyErr_Format(PyExc_NotImplementedError, "%s has no backward: call it under torch.no_grad()", what);
    const int code = dtype_code(x.scalar_type());
    if (code < 0)
      return PyErr_Format(PyExc_NotImplementedError, "%s: unsupported dtype %s", what, c10::toString(x.scalar_type()));
    if (x.dim() > 4) return PyErr_Format(PyExc_ValueError, "%s: tensors have at most 4 dimensions", what);
    if (rows >> i & 1 && !rows_ok(x)) {
      copies |= 1L << i;
      continue;
    }
    saf_tensor_t* d = reinterpret_cast<saf_tensor_t*>(block + PyLong_AsLong(PyTuple_GET_ITEM(args[2], i)));
    *d = saf_tensor_t{};
    d->data = x.data_ptr();
    d->dtype = code;
    d->ndim = (int32_t)x.dim();
    for (int k = 0; k < d->ndim; ++k) {
      d->size[k] = x.size(k);
      d->stride[k] = x.stride(k);
    }
  }
  return PyLong_FromLong(copies);
}

PyObject* fill_checked(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  try {
    return fill(self, args, n);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyMethodDef methods[] = {
    {"fill", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fill_checked)), METH_FASTCALL,
     "fill(what, block, offsets, rows, device, refuse_grad, *tensors) -> mask of tensors whose rows need a copy"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_desc", "Tensor descriptors of libsafattn.so argument blocks.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__desc() { return PyModule_Create(&module); }
