// Tensor descriptors and output allocations for the Python front end: one call
// describes all tensors of an operator as the bytes of l3d_tensor structures.
// A call on a few rows spends its time on the host; describing a tensor takes 0.8
// us in Python and 0.1 us here, allocating one 2.4 and about 1.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

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

// `device`: ANY of them, the host too; CUDA; or a device's index.
constexpr int ANY = -2, CUDA = -1;

// False with a Python error set.
bool describe(const at::Tensor& t, int device, l3d_tensor* d) {
  if (device != ANY && !t.is_cuda()) {
    PyErr_SetString(PyExc_ValueError, "libl3dops ops take CUDA tensors (no CPU implementation exists)");
    return false;
  }
  if (device >= 0 && t.get_device() != device) {
    PyErr_Format(PyExc_ValueError, "a tensor lies on cuda:%d, the current device is cuda:%d", int(t.get_device()), device);
    return false;
  }
  const int code = dtype_code(t.scalar_type());
  if (code < 0) {
    PyErr_SetString(PyExc_TypeError, "unsupported tensor dtype");
    return false;
  }
  if (t.dim() > L3D_MAX_DIMS) {
    PyErr_Format(PyExc_ValueError, "rank %d exceeds %d", int(t.dim()), int(L3D_MAX_DIMS));
    return false;
  }
  *d = l3d_tensor{};
  d->data = t.data_ptr();  // the view's first element: offset 0
  d->dtype = code;
  d->ndim = int32_t(t.dim());
  for (int64_t i = 0; i < t.dim(); ++i) {
    d->dims[i] = t.size(i);
    d->strides[i] = t.stride(i);
  }
  return true;
}

PyObject* describe(PyObject* o, int device) {
  if (o == Py_None) Py_RETURN_NONE;
  if (!THPVariable_Check(o)) {
    PyErr_SetString(PyExc_TypeError, "a tensor or None expected");
    return nullptr;
  }
  l3d_tensor d;
  if (!describe(THPVariable_Unpack(o), device, &d)) return nullptr;
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
  return guarded([&] { return describe(o, ANY); });
}

PyObject* packs(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    PyObject* out = PyTuple_New(n);
    if (!out) return nullptr;
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* b = describe(args[i], CUDA);
      if (!b) {
        Py_DECREF(out);
        return nullptr;
      }
      PyTuple_SET_ITEM(out, i, b);
    }
    return out;
  });
}

// ---- whole calls.  ctypes takes some 0.2 us an argument; these entries, whose smallest calls are a launch or two,
// are called here: tensors described, output and workspace allocated, the entry (by its address) called.
// The descriptors of `n` arguments, which must be tensors on the current device, or None.
template <int N>
struct Descriptors {
  l3d_tensor at[N];
  const l3d_tensor* ptr[N];
  bool fill(PyObject* const* args) {
    int device = CUDA;
    // (Asked of the runtime only once a tensor is on a device: on a machine without one that is the error.)
    for (int i = 0; i < N && device == CUDA; ++i)
      if (THPVariable_Check(args[i]) && THPVariable_Unpack(args[i]).is_cuda()) {
        const c10::impl::VirtualGuardImpl impl(c10::DeviceType::CUDA);
        device = int(impl.getDevice().index());
      }
    for (int i = 0; i < N; ++i) {
      ptr[i] = nullptr;
      if (args[i] == Py_None) continue;
      if (!THPVariable_Check(args[i])) {
        PyErr_SetString(PyExc_TypeError, "a tensor or None expected");
        return false;
      }
      if (!describe(THPVariable_Unpack(args[i]), device, &at[i])) return false;
      ptr[i] = &at[i];
    }
    return true;
  }
};
template <typename F>
F entry(PyObject* address) {
  return reinterpret_cast<F>(PyLong_AsVoidPtr(address));
}
// An entry's status; the interpreter's lock is not held meanwhile.
template <typename F>
int without_lock(F f) {
  PyThreadState* st = PyEval_SaveThread();
  const int rc = f();
  PyEval_RestoreThread(st);
  return rc;
}
PyObject* refused(const char* what) {
  PyErr_SetString(PyExc_TypeError, what);
  return nullptr;
}
// (status, out) with out contiguous and shaped as q, or the tensor given.
PyObject* result(int rc, PyObject* out) {
  PyObject* t = PyTuple_New(2);
  if (t) {
    PyTuple_SET_ITEM(t, 0, PyLong_FromLong(rc));
    PyTuple_SET_ITEM(t, 1, out);
  } else {
    Py_DECREF(out);
  }
  return t;
}
// args[i] or, where it is None, a new tensor like args[like]; a new reference.
PyObject* out_or_new(PyObject* out, PyObject* like) {
  if (out != Py_None) {
    Py_INCREF(out);
    return out;
  }
  if (!THPVariable_Check(like)) return refused("a tensor expected");
  const at::Tensor& t = THPVariable_Unpack(like);
  return THPVariable_Wrap(at::empty(t.sizes(), t.options().requires_grad(false)));
}

// paged_append(entry, stream, eps, half, q, k, v, q_weight, k_weight, freqs, axes, positions, table, held, offsets,
//              out, k_pages, v_pages)
PyObject* paged_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 18) return refused("paged_append: 18 arguments");
    const auto fn = entry<decltype(&l3d_paged_append)>(a[0]);
    const auto stream = entry<l3d_stream>(a[1]);
    const double eps = PyFloat_AsDouble(a[2]);
    const long half = PyLong_AsLong(a[3]);
    if (PyErr_Occurred()) return nullptr;
    THPObjectPtr out(out_or_new(a[15], a[4]));
    if (!out) return nullptr;
    PyObject* args[14];
    for (int i = 0; i < 14; ++i) args[i] = i == 11 ? out.get() : a[4 + i];
    Descriptors<14> d;
    if (!d.fill(args)) return nullptr;
    const auto& p = d.ptr;
    return result(without_lock([&] {
                    return fn(p[0], p[1], p[2], p[3], p[4], float(eps), p[5], p[6], int(half), p[7], p[8], p[9], p[10],
                              p[11], p[12], p[13], stream);
                  }),
                  out.release());
  });
}

// A workspace of `bytes` on the tensor's device.
at::Tensor workspace_for(PyObject* like, size_t bytes) {
  return at::empty({int64_t(bytes)}, THPVariable_Unpack(like).options().dtype(at::kByte).requires_grad(false));
}

// paged_attention(entry, size entry, stream, scale, q, k_pages, v_pages, table, lengths, out); q and out with or
// without the dimension of the newest tokens
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 10) return refused("paged_attention: 10 arguments");
    const auto fn = entry<decltype(&l3d_paged_attention)>(a[0]);
    const auto size = entry<decltype(&l3d_paged_attention_workspace_size)>(a[1]);
    const auto stream = entry<l3d_stream>(a[2]);
    const double scale = PyFloat_AsDouble(a[3]);
    if (PyErr_Occurred()) return nullptr;
    THPObjectPtr out(out_or_new(a[9], a[4]));
    if (!out) return nullptr;
    PyObject* args[6] = {a[4], a[5], a[6], a[7], a[8], out.get()};
    Descriptors<6> d;
    if (!d.fill(args)) return nullptr;
    for (int i : {0, 5}) {  // one token each: [B, H, D] as [B, 1, H, D]
      l3d_tensor& t = d.at[i];
      if (!d.ptr[i] || t.ndim != 3) continue;
      for (int x = 3; x > 1; --x) {
        t.dims[x] = t.dims[x - 1];
        t.strides[x] = t.strides[x - 1];
      }
      t.dims[1] = 1;
      t.ndim = 4;
    }
    size_t need = 0;
    if (d.ptr[0] && d.ptr[1] && d.ptr[3] && d.at[0].ndim == 4 && d.at[1].ndim == 4 && d.at[3].ndim == 2)  // (else refused)
      need = size(d.at[0].dims[0], d.at[0].dims[2], d.at[1].dims[2], d.at[0].dims[1], d.at[3].dims[1] * d.at[1].dims[1],
                  d.at[0].dims[3]);
    at::Tensor ws;
    if (need) ws = workspace_for(out.get(), need);
    void* wp = need ? ws.data_ptr() : nullptr;
    const auto& p = d.ptr;
    return result(without_lock([&] { return fn(p[0], p[1], p[2], p[3], p[4], float(scale), p[5], wp, need, stream); }), out.release());
  });
}

// cross_attention(entry, size entry, stream, scale, q, k, v, k_offsets, q_offsets, out)
PyObject* cross_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 10) return refused("cross_attention: 10 arguments");
    const auto fn = entry<decltype(&l3d_cross_attention)>(a[0]);
    const auto size = entry<decltype(&l3d_cross_attention_workspace_size)>(a[1]);
    const auto stream = entry<l3d_stream>(a[2]);
    const double scale = PyFloat_AsDouble(a[3]);
    if (PyErr_Occurred()) return nullptr;
    THPObjectPtr out(out_or_new(a[9], a[4]));
    if (!out) return nullptr;
    PyObject* args[6] = {a[4], a[5], a[6], a[7], a[8], out.get()};
    Descriptors<6> d;
    if (!d.fill(args)) return nullptr;
    size_t need = 0;
    if (d.ptr[0] && d.ptr[1] && d.ptr[3] && d.at[0].ndim == 3 && d.at[1].ndim == 3 && d.at[3].ndim == 1)  // (else refused)
      need = size(d.at[3].dims[0] - 1, d.at[0].dims[0], d.at[1].dims[0], d.at[0].dims[1], d.at[1].dims[1], d.at[0].dims[2],
                  d.ptr[4] != nullptr);
    at::Tensor ws;
    if (need) ws = workspace_for(out.get(), need);
    void* wp = need ? ws.data_ptr() : nullptr;
    const auto& p = d.ptr;
    return result(without_lock([&] { return fn(p[0], p[1], p[2], p[3], p[4], float(scale), p[5], wp, need, stream); }), out.release());
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
    {"paged_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_append)), METH_FASTCALL,
     "l3d_paged_append, at the address given: (status, out)"},
    {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_attention)), METH_FASTCALL,
     "l3d_paged_attention, at the address given: (status, out)"},
    {"cross_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cross_attention)), METH_FASTCALL,
     "l3d_cross_attention, at the address given: (status, out)"},
    {"empty", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(empty)), METH_FASTCALL,
     "contiguous tensor of the first argument's type and device, of its shape or the sizes given"},
    {"workspace", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(workspace)), METH_FASTCALL,
     "bytes on the first argument's device"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_l3dpack", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__l3dpack() { return PyModule_Create(&module); }
