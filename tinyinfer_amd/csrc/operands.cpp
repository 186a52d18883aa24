// What NativeOps asks of torch tensors, in one call each: a small call's time is Python's, and
// a check by attributes costs 0.05 us apiece.  Functions answer None where an operand is not
// acceptable; native_ops.py then goes through its checks one by one for the reason.
//
//   operand(x, dtype, index, rank, shape) -> address
//     a contiguous GPU tensor of 1 .. 2^31 - 1 elements without grad, of this dtype, on GPU
//     `index` (-2: any), of this rank (-1: any but 0) and shape (None: any);
//   rows(x, dtype, index, shape) -> (address, strides of the first three axes)
//     the same of rank 4 with contiguous values in the last axis alone;
//   empty(shape, like) -> an empty contiguous tensor of like's dtype and device;
//   empty_as(shape, dtype, like) -> of like's device;
//   record(tensors, stream id, GPU): the allocator learns that the stream uses them;
//   torch_version: the torch whose headers this was compiled with.  Under another one no
//     function here may be called (tensors are read through inlined accessors).
#include <Python.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <ATen/ops/empty.h>

namespace {

constexpr int64_t kMost = 2147483647;

bool has_shape(const at::Tensor& t, PyObject* shape) {
  if (shape == Py_None) return true;
  if (!PyTuple_Check(shape) || PyTuple_GET_SIZE(shape) != t.dim()) return false;
  for (int64_t i = 0; i < t.dim(); ++i)
    if (PyLong_AsLongLong(PyTuple_GET_ITEM(shape, i)) != t.size(i)) {
      PyErr_Clear();  // (an extent that is no number is another shape)
      return false;
    }
  return true;
}

// The tensor of an operand that is one of this dtype and place, or null.
const at::Tensor* tensor_of(PyObject* x, PyObject* dtype, long index) {
  if (!THPVariable_Check(x) || !THPDtype_Check(dtype)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(x);
  const int64_t n = t.numel();
  if (t.scalar_type() != reinterpret_cast<THPDtype*>(dtype)->scalar_type || !t.is_cuda() || (index != -2 && t.get_device() != index) ||
      t.requires_grad() || n <= 0 || n > kMost)
    return nullptr;
  return &t;
}

PyObject* operand(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 5) return PyErr_Format(PyExc_TypeError, "operand: 5 arguments");
  const long rank = PyLong_AsLong(args[3]);
  const at::Tensor* t = tensor_of(args[0], args[1], PyLong_AsLong(args[2]));
  if (!t || !t->is_contiguous() || t->dim() == 0 || (rank >= 0 && t->dim() != rank) || !has_shape(*t, args[4])) Py_RETURN_NONE;
  return PyLong_FromVoidPtr(t->data_ptr());
  END_HANDLE_TH_ERRORS
}

PyObject* rows(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 4) return PyErr_Format(PyExc_TypeError, "rows: 4 arguments");
  const at::Tensor* t = tensor_of(args[0], args[1], PyLong_AsLong(args[2]));
  if (!t || t->dim() != 4 || (t->stride(3) != 1 && t->size(3) != 1) || !has_shape(*t, args[3])) Py_RETURN_NONE;
  return Py_BuildValue("(KLLL)", reinterpret_cast<unsigned long long>(t->data_ptr()), static_cast<long long>(t->stride(0)),
                       static_cast<long long>(t->stride(1)), static_cast<long long>(t->stride(2)));
  END_HANDLE_TH_ERRORS
}

PyObject* empty(PyObject* shape, const at::TensorOptions& options) {
  if (!PyTuple_Check(shape)) return PyErr_Format(PyExc_TypeError, "empty: a tuple of extents");
  c10::SmallVector<int64_t, 6> extents;
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(shape); ++i) {
    const int64_t extent = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, i));
    if (extent < 0) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "empty: a negative extent");
    extents.push_back(extent);
  }
  at::Tensor y;
  {
    PyThreadState* state = PyEval_SaveThread();  // (an allocation may wait for the GPU)
    try {
      y = at::empty(extents, options);
    } catch (...) {
      PyEval_RestoreThread(state);
      throw;
    }
    PyEval_RestoreThread(state);
  }
  return THPVariable_Wrap(std::move(y));
}

PyObject* empty_like(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 2 || !THPVariable_Check(args[1])) return PyErr_Format(PyExc_TypeError, "empty: a shape and a tensor");
  const at::Tensor& like = THPVariable_Unpack(args[1]);
  return empty(args[0], at::TensorOptions().dtype(like.scalar_type()).device(like.device()));
  END_HANDLE_TH_ERRORS
}

PyObject* empty_as(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 3 || !THPDtype_Check(args[1]) || !THPVariable_Check(args[2]))
    return PyErr_Format(PyExc_TypeError, "empty_as: a shape, a dtype and a tensor");
  const at::Tensor& like = THPVariable_Unpack(args[2]);
  return empty(args[0], at::TensorOptions().dtype(reinterpret_cast<THPDtype*>(args[1])->scalar_type).device(like.device()));
  END_HANDLE_TH_ERRORS
}

PyObject* record(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 3 || !PyList_Check(args[0])) return PyErr_Format(PyExc_TypeError, "record: a list of tensors, a stream's number and a GPU's");
  const auto id = static_cast<c10::StreamId>(PyLong_AsLongLong(args[1]));
  const c10::Stream stream(c10::Stream::UNSAFE, c10::Device(c10::DeviceType::CUDA, static_cast<c10::DeviceIndex>(PyLong_AsLong(args[2]))), id);
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(args[0]); ++i) {
    PyObject* x = PyList_GET_ITEM(args[0], i);
    if (!THPVariable_Check(x)) return PyErr_Format(PyExc_TypeError, "record: a list of tensors");
    THPVariable_Unpack(x).record_stream(stream);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL
PyMethodDef methods[] = {{"operand", FAST(operand), nullptr},   {"rows", FAST(rows), nullptr},     {"empty", FAST(empty_like), nullptr},
                         {"empty_as", FAST(empty_as), nullptr}, {"record", FAST(record), nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_operands", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__operands() {
  PyObject* made = PyModule_Create(&module);
  if (made && PyModule_AddStringConstant(made, "torch_version", TIA_TORCH_VERSION) < 0) Py_CLEAR(made);
  return made;
}
