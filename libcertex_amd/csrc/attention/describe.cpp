// describe(first, tensors...): DLPack descriptions of torch tensors for the C API, written in one call.
//
// The operators' kernels take a few microseconds, and a Python call describes up to nine tensors: reading
// their fields in Python took 0.9 us each, here it is some tens of nanoseconds. The descriptions borrow the tensors'
// memory and lie in memory of the calling thread, where the next call of as many places overwrites them.
#include <torch/csrc/autograd/python_variable.h>

#include <dlpack/dlpack.h>

namespace {

constexpr int kPlaces = 16, kMaxDims = 4;

struct description {
  DLManagedTensor m;
  int64_t shape[kMaxDims], strides[kMaxDims];
};

bool type_of(at::ScalarType t, DLDataType* out)
{
  const auto set = [&](int code, int bits) {
    *out = {uint8_t(code), uint8_t(bits), 1};
    return true;
  };
  switch (t) {
    case at::kFloat: return set(kDLFloat, 32);
    case at::kHalf: return set(kDLFloat, 16);
    case at::kBFloat16: return set(kDLBfloat, 16);
    case at::kInt: return set(kDLInt, 32);
    case at::kLong: return set(kDLInt, 64);
    case at::kByte: return set(kDLUInt, 8);
    default: return false;
  }
}

/** The place of the first description, then tensors or None: a tuple of addresses (None for None). */
PyObject* describe(PyObject*, PyObject* const* args, Py_ssize_t n)
{
  static thread_local description places[kPlaces];
  const long first = n > 0 ? PyLong_AsLong(args[0]) : -1;
  if (first < 0 || first + n - 1 > kPlaces) {
    if (!PyErr_Occurred()) { PyErr_SetString(PyExc_ValueError, "too many tensors to describe"); }
    return nullptr;
  }
  PyObject* out = PyTuple_New(n - 1);
  if (out == nullptr) { return nullptr; }
  for (Py_ssize_t i = 1; i < n; ++i) {
    PyObject* item = Py_None;
    if (args[i] == Py_None) {
      Py_INCREF(item);
    } else {
      if (!THPVariable_Check(args[i])) {
        PyErr_SetString(PyExc_ValueError, "expected a tensor");
        Py_DECREF(out);
        return nullptr;
      }
      const at::Tensor& t = THPVariable_Unpack(args[i]);
      description& d      = places[first + i - 1];
      DLTensor& l         = d.m.dl_tensor;
      if (t.dim() > kMaxDims || t.layout() != at::kStrided || !type_of(t.scalar_type(), &l.dtype)) {
        PyErr_SetString(PyExc_ValueError, "a tensor has more than 4 dimensions, no strides, or an element type that is not used");
        Py_DECREF(out);
        return nullptr;
      }
      const bool gpu = t.is_cuda();
      l.data         = t.data_ptr();
      l.device       = {gpu ? kDLROCM : kDLCPU, gpu ? int32_t(t.get_device()) : 0};
      l.ndim         = int32_t(t.dim());
      l.byte_offset  = 0;
      l.shape        = d.shape;
      l.strides      = d.strides;
      for (int k = 0; k < l.ndim; ++k) {
        d.shape[k]   = t.size(k);
        d.strides[k] = t.stride(k);
      }
      d.m.manager_ctx = nullptr;
      d.m.deleter     = nullptr;
      item            = PyLong_FromVoidPtr(&d.m);
    }
    PyTuple_SET_ITEM(out, i - 1, item);
  }
  return out;
}

PyMethodDef methods[] = {{"describe", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(describe)), METH_FASTCALL,
                          "DLPack descriptions of tensors: (first place, tensors or None) -> addresses"},
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_describe", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__describe() { return PyModule_Create(&module); }
