// The way from torch tensors to an entry that takes its views as one array of slots
// (include/intent_b200.h): types, shapes and devices are checked, outputs and scratch allocated, the slots
// packed and the entry called on torch's current stream, without a Python object a view.  A small call of ten
// views took 20 us of host time with ctypes and takes 10 this way; many of these kernels run for less.
#include <ATen/Functions.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cstdint>
#include <vector>

namespace {

constexpr int kMostSlots = 256;

// The extents that `shape`, a tuple of Python integers, asks for are the tensor's.
bool same_shape(const at::Tensor &tensor, PyObject *shape) {
  const Py_ssize_t rank = PyTuple_GET_SIZE(shape);
  if (tensor.dim() != rank) return false;
  for (Py_ssize_t i = 0; i < rank; ++i)
    if (PyLong_AsLongLong(PyTuple_GET_ITEM(shape, i)) != tensor.size(i)) return false;
  return true;
}

bool extents_of(PyObject *shape, std::vector<int64_t> &extents) {
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(shape); ++i) extents.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(shape, i)));
  return !PyErr_Occurred();
}

// invoke(entry, device, views, number, code, other) -> the tensors made, or a status: the entry's, or -1 - i if
// view i is not what it should be.  views: a tuple of
//     (name, tensor, dtype, shape)         a tensor that has to be that
//     (name, ..., dtype, shape)            one to be made and returned, contiguous
//     (name, ..., dtype, shape, True)      scratch: made, and given back to the allocator after the call, in
//                                          stream order
//     (name, None, rank)                   a view that is not there
// number: the entry's f32 argument, or None if it has none.
PyObject *invoke(PyObject *, PyObject *const *arguments, Py_ssize_t count) {
  if (count != 6 || !PyTuple_Check(arguments[2])) {
    PyErr_SetString(PyExc_TypeError, "invoke(entry, device, views, number, code, other)");
    return nullptr;
  }
  try {
    void *entry = PyLong_AsVoidPtr(arguments[0]);
    const long device = PyLong_AsLong(arguments[1]);
    PyObject *views = arguments[2];
    const double number = arguments[3] == Py_None ? 0.0 : PyFloat_AsDouble(arguments[3]);
    const long code = PyLong_AsLong(arguments[4]), other = PyLong_AsLong(arguments[5]);
    if (PyErr_Occurred()) return nullptr;
    // what is wrong is found before anything is made
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(views); ++i) {
      PyObject *view = PyTuple_GET_ITEM(views, i);
      if (!PyTuple_Check(view) || PyTuple_GET_SIZE(view) < 3) {
        PyErr_SetString(PyExc_TypeError, "a view is (name, tensor, dtype, shape) or (name, None, rank)");
        return nullptr;
      }
      PyObject *object = PyTuple_GET_ITEM(view, 1), *kind = PyTuple_GET_ITEM(view, 2);
      if (PyTuple_GET_SIZE(view) == 3) {
        if (object != Py_None || !PyLong_Check(kind)) return PyLong_FromSsize_t(-1 - i);
        continue;
      }
      PyObject *shape = PyTuple_GET_ITEM(view, 3);
      if (!THPDtype_Check(kind) || !PyTuple_Check(shape)) return PyLong_FromSsize_t(-1 - i);
      if (object == Py_Ellipsis) continue;
      if (!THPVariable_Check(object)) return PyLong_FromSsize_t(-1 - i);
      const at::Tensor &tensor = THPVariable_Unpack(object);
      if (tensor.layout() != at::kStrided || tensor.scalar_type() != reinterpret_cast<THPDtype *>(kind)->scalar_type ||
          !tensor.is_cuda() || tensor.get_device() != device || !same_shape(tensor, shape))
        return PyErr_Occurred() ? nullptr : PyLong_FromSsize_t(-1 - i);
    }
    int64_t slots[kMostSlots];
    int used = 0;
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
    std::vector<at::Tensor> made, scratch;
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(views); ++i) {
      PyObject *view = PyTuple_GET_ITEM(views, i), *object = PyTuple_GET_ITEM(view, 1);
      const bool absent = PyTuple_GET_SIZE(view) == 3;
      at::Tensor fresh;
      if (!absent && object == Py_Ellipsis) {
        std::vector<int64_t> extents;
        if (!extents_of(PyTuple_GET_ITEM(view, 3), extents)) return nullptr;
        fresh = at::empty(extents, at::TensorOptions()
                                       .dtype(reinterpret_cast<THPDtype *>(PyTuple_GET_ITEM(view, 2))->scalar_type)
                                       .device(at::kCUDA, static_cast<c10::DeviceIndex>(device)));
        (PyTuple_GET_SIZE(view) > 4 ? scratch : made).push_back(fresh);
      }
      const int64_t rank = absent ? PyLong_AsLong(PyTuple_GET_ITEM(view, 2)) : PyTuple_GET_SIZE(PyTuple_GET_ITEM(view, 3));
      if (rank < 0 || used + 1 + 2 * rank > kMostSlots) return PyLong_FromSsize_t(-1 - i);
      if (absent) {
        for (int64_t j = 0; j < 1 + 2 * rank; ++j) slots[used++] = 0;
        continue;
      }
      const at::Tensor &tensor = fresh.defined() ? fresh : THPVariable_Unpack(object);
      slots[used++] = reinterpret_cast<int64_t>(tensor.data_ptr());
      for (int64_t j = 0; j < rank; ++j) slots[used++] = tensor.size(j);
      for (int64_t j = 0; j < rank; ++j) slots[used++] = tensor.stride(j);
    }
    void *stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
    int status;
    if (arguments[3] == Py_None)
      status = reinterpret_cast<int (*)(const int64_t *, int64_t, int32_t, int32_t, void *)>(entry)(
          slots, used, static_cast<int32_t>(code), static_cast<int32_t>(other), stream);
    else
      status = reinterpret_cast<int (*)(const int64_t *, int64_t, float, int32_t, int32_t, void *)>(entry)(
          slots, used, static_cast<float>(number), static_cast<int32_t>(code), static_cast<int32_t>(other), stream);
    if (status != 0) return PyLong_FromLong(status);
    PyObject *result = PyTuple_New(static_cast<Py_ssize_t>(made.size()));
    for (size_t i = 0; result && i < made.size(); ++i) PyTuple_SET_ITEM(result, static_cast<Py_ssize_t>(i), THPVariable_Wrap(made[i]));
    return result;
  } catch (const std::exception &error) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, error.what());
    return nullptr;
  }
}

PyMethodDef methods[] = {
    {"invoke", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(invoke)), METH_FASTCALL,
     "invoke(entry, device, views, number, code, other) -> the tensors made, or a status"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef definition = {PyModuleDef_HEAD_INIT, "binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_binding(void) { return PyModule_Create(&definition); }
