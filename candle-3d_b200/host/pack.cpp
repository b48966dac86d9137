// Tensor descriptors and output allocations for the Python front end: one call
// describes all tensors of an operator as the bytes of l3d_tensor structures.
// A call on a few rows spends its time on the host; describing a tensor takes 0.8
// us in Python and 0.1 us here, allocating one 2.4 and about 1.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>

#include "l3d_ops.h"

namespace {

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return L3D_F32;
    case at::kHalf: return L3D_F16;
    case at::kBFloat16: return L3D_BF16;
    case at::kInt: return L3D_I32;
    case at::kLong: return L3D_I64;
    case at::kUInt32: return L3D_U32;
    case at::kByte: return L3D_U8;
    default: return -1;
  }
}

PyObject* describe(PyObject* o, bool on_device) {
  if (o == Py_None) Py_RETURN_NONE;
  if (!THPVariable_Check(o)) {
    PyErr_SetString(PyExc_TypeError, "a tensor or None expected");
    return nullptr;
  }
  const at::Tensor& t = THPVariable_Unpack(o);
  if (on_device && !t.is_cuda()) {
    PyErr_SetString(PyExc_ValueError, "libl3dops ops take CUDA tensors (no CPU implementation exists)");
    return nullptr;
  }
  const int code = dtype_code(t.scalar_type());
  if (code < 0) {
    PyErr_SetString(PyExc_TypeError, "unsupported tensor dtype");
    return nullptr;
  }
  if (t.dim() > L3D_MAX_DIMS) {
    PyErr_Format(PyExc_ValueError, "rank %d exceeds %d", int(t.dim()), int(L3D_MAX_DIMS));
    return nullptr;
  }
  l3d_tensor d{};
  d.data = t.data_ptr();  // the view's first element: offset 0
  d.dtype = code;
  d.ndim = int32_t(t.dim());
  for (int64_t i = 0; i < t.dim(); ++i) {
    d.dims[i] = t.size(i);
    d.strides[i] = t.stride(i);
  }
  return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(&d), sizeof(d));
}

// No C++ exception leaves an entry.
template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

PyObject* packed(PyObject*, PyObject* o) {
  return guarded([&] { return describe(o, false); });
}

PyObject* packs(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    PyObject* out = PyTuple_New(n);
    if (!out) return nullptr;
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* b = describe(args[i], true);
      if (!b) {
        Py_DECREF(out);
        return nullptr;
      }
      PyTuple_SET_ITEM(out, i, b);
    }
    return out;
  });
}

PyObject* empty(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n < 1 || n > 1 + L3D_MAX_DIMS || !THPVariable_Check(args[0])) {
      PyErr_SetString(PyExc_TypeError, "empty(like, *sizes)");
      return nullptr;
    }
    const at::Tensor& like = THPVariable_Unpack(args[0]);
    if (n == 1) return THPVariable_Wrap(at::empty(like.sizes(), like.options().requires_grad(false)));
    int64_t size[L3D_MAX_DIMS];
    for (Py_ssize_t i = 1; i < n; ++i) {
      size[i - 1] = PyLong_AsLongLong(args[i]);
      if (size[i - 1] == -1 && PyErr_Occurred()) return nullptr;
    }
    return THPVariable_Wrap(at::empty(at::IntArrayRef(size, size_t(n - 1)), like.options().requires_grad(false)));
  });
}

PyObject* workspace(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 2 || !THPVariable_Check(args[0])) {
      PyErr_SetString(PyExc_TypeError, "workspace(like, bytes)");
      return nullptr;
    }
    const int64_t bytes = PyLong_AsLongLong(args[1]);
    if (bytes == -1 && PyErr_Occurred()) return nullptr;
    return THPVariable_Wrap(at::empty({bytes}, THPVariable_Unpack(args[0]).options().dtype(at::kByte).requires_grad(false)));
  });
}

PyMethodDef methods[] = {
    {"packed", packed, METH_O, "l3d_tensor of a tensor view as bytes (None -> None)"},
    {"packs", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(packs)), METH_FASTCALL,
     "packed of each argument, which must be on a CUDA device, as a tuple"},
    {"empty", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(empty)), METH_FASTCALL,
     "contiguous tensor of the first argument's type and device, of its shape or the sizes given"},
    {"workspace", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(workspace)), METH_FASTCALL,
     "bytes on the first argument's device"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_l3dpack", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__l3dpack() { return PyModule_Create(&module); }
