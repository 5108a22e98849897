// Python module dgen_hip._tensor_args: the tests of a tensor argument and its
// address and strides, for dgen_hip/sequence.py.  A single frame's call is
// bound by them: about 0.75 us a tensor in Python, 0.15 here.  Each function
// takes (tensor, shape, type, device index), type as in dgen_hip.h (or
// kInt32), and returns None for what it turns down; the caller looks at that
// again and says why.  `covers` tells whether
// tensors share memory.
#include <c10/core/GradMode.h>
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
  if (t.requires_grad() && c10::GradMode::is_enabled()) return nullptr;  // (the caller warns)
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

// Bytes from a tensor's first element to past its last, along the axes whose
// steps are no multiples of `pitch` bytes (0: along all).
int64_t extent(const at::Tensor& t, int64_t pitch) {
  const int64_t item = (int64_t)t.itemsize();
  int64_t bytes = item;
  for (int64_t d = 0; d < t.dim(); ++d)
    if (pitch == 0 || t.stride(d) * item % pitch != 0) bytes += (t.size(d) - 1) * t.stride(d) * item;
  return bytes;
}

// Whether two tensors share memory: 0 no, 1 every element is the other's
// element of the same index, 2 otherwise (or it cannot be told).  Columns,
// rows or frames of one tensor side by side are apart: modulo the step of some
// axis each takes a range of the bytes.
int overlap_of(const at::Tensor& a, const at::Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return 0;
  const int64_t x = (int64_t)address(a), y = (int64_t)address(b);
  if (x + extent(a, 0) <= y || y + extent(b, 0) <= x) return 0;
  bool same = x == y && a.scalar_type() == b.scalar_type() && a.sizes() == b.sizes();
  for (int64_t d = 0; same && d < a.dim(); ++d) same = a.size(d) == 1 || a.stride(d) == b.stride(d);
  if (same) return 1;
  for (const at::Tensor* t : {&a, &b})
    for (int64_t d = 0; d < t->dim(); ++d) {
      const int64_t pitch = t->stride(d) * (int64_t)t->itemsize();
      if (t->size(d) == 1 || pitch == 0) continue;
      const int64_t between = ((y - x) % pitch + pitch) % pitch;
      if (between >= extent(a, pitch) && between + extent(b, pitch) <= pitch) return 0;
    }
  return 2;
}

// covers(k, t, *others): whether writing t changes what is read or written of
// the others; the first k may be t itself, element by element.  None is apart.
PyObject* covers(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n < 2 || !THPVariable_Check(args[1])) return none_if_wrong();
    const long may = PyLong_AsLong(args[0]);
    if (may == -1 && PyErr_Occurred()) return none_if_wrong();
    const at::Tensor& t = THPVariable_Unpack(args[1]);
    for (Py_ssize_t i = 2; i < n; ++i) {
      if (args[i] == Py_None) continue;
      if (!THPVariable_Check(args[i])) return none_if_wrong();
      if (overlap_of(t, THPVariable_Unpack(args[i])) > (i - 2 < may ? 1 : 0)) Py_RETURN_TRUE;
    }
    Py_RETURN_FALSE;
  });
}

PyMethodDef methods[] = {
    {"dense", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(dense)), METH_FASTCALL, nullptr},
    {"sequence", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(sequence)), METH_FASTCALL, nullptr},
    {"rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rows)), METH_FASTCALL, nullptr},
    {"covers", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(covers)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_args", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_args() { return PyModule_Create(&module); }
