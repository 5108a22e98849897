// Python module dgen_hip._tensor_args: the tests of a tensor argument and its
// address and strides, for dgen_hip/sequence.py.  A single frame's call is
// bound by them: about 0.75 us a tensor in Python, 0.15 here.  Each function
// takes (tensor, shape, type, device index), type as in dgen_hip.h (or
// kInt32), and returns None for what it turns down; the caller looks at that
// again and says why.
#include <torch/csrc/autograd/python_variable.h>

namespace {

constexpr long kF32 = 0, kBf16 = 1, kInt32 = 2;

// The tensor, if it has the type, device and shape (a tuple of integers).
const at::Tensor* tensor_of(PyObject* const* args, Py_ssize_t n) {
  if (n != 4 || !THPVariable_Check(args[0]) || !PyTuple_Check(args[1])) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(args[0]);
  const long type = PyLong_AsLong(args[2]), index = PyLong_AsLong(args[3]);
  const at::ScalarType want = type == kF32    ? at::kFloat
                              : type == kBf16 ? at::kBFloat16
                              : type == kInt32 ? at::kInt
                                               : at::ScalarType::Undefined;
  if (!t.defined() || t.scalar_type() != want || t.layout() != at::kStrided || !t.is_cuda() || t.get_device() != index)
    return nullptr;
  if (t.dim() != PyTuple_GET_SIZE(args[1])) return nullptr;
  for (int64_t d = 0; d < t.dim(); ++d)
    if (t.size(d) != PyLong_AsLongLong(PyTuple_GET_ITEM(args[1], d))) return nullptr;
  return &t;
}

PyObject* none_if_wrong() {
  PyErr_Clear();  // (a size that is no integer)
  Py_RETURN_NONE;
}

unsigned long long address(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()); }

template <class F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (...) {  // (a tensor without storage)
    return none_if_wrong();
  }
}

// Address of a contiguous tensor; 0 for None.
PyObject* dense(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n >= 1 && args[0] == Py_None) return PyLong_FromLong(0);
  return guarded([&]() -> PyObject* {
    const at::Tensor* t = tensor_of(args, n);
    if (!t || !t->is_contiguous()) return none_if_wrong();
    return PyLong_FromUnsignedLongLong(address(*t));
  });
}

// (address, batch stride, time stride) of a [batch][time][channel] tensor.
PyObject* sequence(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const at::Tensor* t = tensor_of(args, n);
    if (!t || t->dim() != 3 || (t->stride(2) != 1 && t->size(2) != 1)) return none_if_wrong();
    return Py_BuildValue("(KLL)", address(*t), (long long)t->stride(0), (long long)t->stride(1));
  });
}

// (address, row stride) of a matrix, or of a contiguous tensor's rows.
PyObject* rows(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const at::Tensor* t = tensor_of(args, n);
    if (!t || t->dim() < 1) return none_if_wrong();
    const int64_t width = t->size(t->dim() - 1);
    if (t->dim() == 2 && (t->stride(1) == 1 || width == 1))
      return Py_BuildValue("(KL)", address(*t), (long long)t->stride(0));
    if (t->dim() == 2 || !t->is_contiguous()) return none_if_wrong();
    return Py_BuildValue("(KL)", address(*t), (long long)width);
  });
}

PyMethodDef methods[] = {
    {"dense", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(dense)), METH_FASTCALL, nullptr},
    {"sequence", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(sequence)), METH_FASTCALL, nullptr},
    {"rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rows)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_args", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_args() { return PyModule_Create(&module); }
