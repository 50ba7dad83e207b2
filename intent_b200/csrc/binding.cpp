// The way from torch tensors to an entry that takes its views as one array of slots
// (include/intent_b200.h): types, shapes and devices are checked, outputs and scratch allocated, the slots
// packed and the entry called on torch's current stream, without a Python object a view.  A small call of ten
// views took 34 us of host time with ctypes and takes 6.7 this way; many of these kernels run for less.
#include <ATen/cuda/EmptyTensor.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cstdint>
#include <vector>

namespace {

constexpr int kMostSlots = 256, kMostSymbols = 16;

// What a view of a call may be.
enum Kind : long {
  kGiven = 0,     // a tensor
  kOutput = 1,    // a tensor, or ... for one to be made and returned
  kScratch = 2,   // made, and given back to the allocator after the call, in stream order
  kOptional = 3,  // a tensor, ... for one to be made and returned, or None for a view that is not there
};

// invoke(entry, device, plan, tensors, extents, number, code, other) -> the tensors made, or a status: the
// entry's, or -1 - i if view i is not what it should be.  plan: for each view (name, dtype, symbols, kind);
// dtype None is the type of the first such view.  A symbol, a small number, stands for an extent: the first
// of `extents` are given, others are those of the first view that has them, and later views have to agree.
// Everything made is contiguous and the call's own.  number: the entry's f32 argument, or None if it has none.
PyObject *invoke(PyObject *, PyObject *const *arguments, Py_ssize_t count) {
  if (count != 8 || !PyTuple_Check(arguments[2]) || !PyTuple_Check(arguments[3]) || !PyTuple_Check(arguments[4]) ||
      PyTuple_GET_SIZE(arguments[2]) != PyTuple_GET_SIZE(arguments[3])) {
    PyErr_SetString(PyExc_TypeError, "invoke(entry, device, plan, tensors, extents, number, code, other)");
    return nullptr;
  }
  HANDLE_TH_ERRORS   // an allocation that fails becomes torch.OutOfMemoryError, as it does of torch's own
    void *entry = PyLong_AsVoidPtr(arguments[0]);
    const long device = PyLong_AsLong(arguments[1]);
    PyObject *plan = arguments[2], *tensors = arguments[3], *extents = arguments[4];
    const double number = arguments[5] == Py_None ? 0.0 : PyFloat_AsDouble(arguments[5]);
    const long code = PyLong_AsLong(arguments[6]), other = PyLong_AsLong(arguments[7]);
    const Py_ssize_t views = PyTuple_GET_SIZE(plan), given = PyTuple_GET_SIZE(extents);
    int64_t known[kMostSymbols];
    for (int i = 0; i < kMostSymbols; ++i) known[i] = -1;
    for (Py_ssize_t i = 0; i < given && i < kMostSymbols; ++i) known[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(extents, i));
    if (PyErr_Occurred()) return nullptr;
    at::ScalarType call_type = at::ScalarType::Undefined;
    // what is wrong is found before anything is made
    for (Py_ssize_t i = 0; i < views; ++i) {
      PyObject *view = PyTuple_GET_ITEM(plan, i), *object = PyTuple_GET_ITEM(tensors, i);
      const long kind = PyLong_AsLong(PyTuple_GET_ITEM(view, 3));
      if (object == Py_Ellipsis && kind != kGiven) continue;
      if (object == Py_None && kind == kOptional) continue;
      if (kind == kScratch || !THPVariable_Check(object)) return PyLong_FromSsize_t(-1 - i);
      const at::Tensor &tensor = THPVariable_Unpack(object);
      PyObject *dtype = PyTuple_GET_ITEM(view, 1), *symbols = PyTuple_GET_ITEM(view, 2);
      if (dtype == Py_None && call_type == at::ScalarType::Undefined) call_type = tensor.scalar_type();
      const at::ScalarType wanted = dtype == Py_None ? call_type : reinterpret_cast<THPDtype *>(dtype)->scalar_type;
      const Py_ssize_t rank = PyTuple_GET_SIZE(symbols);
      if (tensor.layout() != at::kStrided || tensor.scalar_type() != wanted || !tensor.is_cuda() || tensor.get_device() != device ||
          tensor.dim() != rank)
        return PyLong_FromSsize_t(-1 - i);
      for (Py_ssize_t j = 0; j < rank; ++j) {
        int64_t &extent = known[PyLong_AsLong(PyTuple_GET_ITEM(symbols, j)) & (kMostSymbols - 1)];
        if (extent < 0) extent = tensor.size(j);
        if (extent != tensor.size(j)) return PyLong_FromSsize_t(-1 - i);
      }
    }
    int64_t slots[kMostSlots];
    int used = 0;
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
    std::vector<at::Tensor> made, scratch;
    for (Py_ssize_t i = 0; i < views; ++i) {
      PyObject *view = PyTuple_GET_ITEM(plan, i), *object = PyTuple_GET_ITEM(tensors, i), *symbols = PyTuple_GET_ITEM(view, 2);
      const int rank = static_cast<int>(PyTuple_GET_SIZE(symbols));
      if (used + 1 + 2 * rank > kMostSlots) return PyLong_FromSsize_t(-1 - i);
      if (object == Py_None) {
        for (int j = 0; j < 1 + 2 * rank; ++j) slots[used++] = 0;
        continue;
      }
      at::Tensor fresh;
      if (object == Py_Ellipsis) {
        PyObject *dtype = PyTuple_GET_ITEM(view, 1);
        int64_t shape[kMostSymbols];
        for (int j = 0; j < rank; ++j) {
          shape[j] = known[PyLong_AsLong(PyTuple_GET_ITEM(symbols, j)) & (kMostSymbols - 1)];
          if (shape[j] < 0) return PyLong_FromSsize_t(-1 - i);
        }
        fresh = at::detail::empty_cuda(at::IntArrayRef(shape, rank),
                                       dtype == Py_None ? call_type : reinterpret_cast<THPDtype *>(dtype)->scalar_type,
                                       at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(device)), std::nullopt);
        (PyLong_AsLong(PyTuple_GET_ITEM(view, 3)) == kScratch ? scratch : made).push_back(fresh);
      }
      const at::Tensor &tensor = fresh.defined() ? fresh : THPVariable_Unpack(object);
      slots[used++] = reinterpret_cast<int64_t>(tensor.data_ptr());
      for (int j = 0; j < rank; ++j) slots[used++] = tensor.size(j);
      for (int j = 0; j < rank; ++j) slots[used++] = tensor.stride(j);
    }
    if (PyErr_Occurred()) return nullptr;
    void *stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
    int status;
    if (arguments[5] == Py_None)
      status = reinterpret_cast<int (*)(const int64_t *, int64_t, int32_t, int32_t, void *)>(entry)(
          slots, used, static_cast<int32_t>(code), static_cast<int32_t>(other), stream);
    else
      status = reinterpret_cast<int (*)(const int64_t *, int64_t, float, int32_t, int32_t, void *)>(entry)(
          slots, used, static_cast<float>(number), static_cast<int32_t>(code), static_cast<int32_t>(other), stream);
    if (status != 0) return PyLong_FromLong(status);
    PyObject *result = PyTuple_New(static_cast<Py_ssize_t>(made.size()));
    for (size_t i = 0; result && i < made.size(); ++i) PyTuple_SET_ITEM(result, static_cast<Py_ssize_t>(i), THPVariable_Wrap(made[i]));
    return result;
  END_HANDLE_TH_ERRORS
}

// zeroed(device, words) -> int32 zeros that are there when it returns and belong to no graph, also if the
// current stream is being captured: they are made on a stream of their own, and waited for.
PyObject *zeroed(PyObject *, PyObject *const *arguments, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  const long device = count == 2 ? PyLong_AsLong(arguments[0]) : -1;
  const long long words = count == 2 ? PyLong_AsLongLong(arguments[1]) : -1;
  if (PyErr_Occurred()) return nullptr;
  if (device < 0 || words < 0) {
    PyErr_SetString(PyExc_TypeError, "zeroed(device, words)");
    return nullptr;
  }
  const c10::DeviceIndex index = static_cast<c10::DeviceIndex>(device);
  const c10::cuda::CUDAGuard guard(index);
  // memory may be allocated and another stream waited for while a graph is being captured
  const c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
  c10::cuda::CUDAStream stream = c10::cuda::getStreamFromPool(false, index);
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  for (int i = 0; i < 64; ++i) {   // the pool's streams go round, and the one being captured may be among them
    C10_CUDA_CHECK(cudaStreamIsCapturing(stream.stream(), &status));
    if (status == cudaStreamCaptureStatusNone) break;
    stream = c10::cuda::getStreamFromPool(false, index);
  }
  const c10::cuda::CUDAStreamGuard on(stream);
  const int64_t shape[1] = {words};
  at::Tensor space = at::detail::empty_cuda(at::IntArrayRef(shape, 1), at::kInt, at::Device(at::kCUDA, index), std::nullopt);
  C10_CUDA_CHECK(cudaMemsetAsync(space.data_ptr(), 0, static_cast<size_t>(words) * 4, stream.stream()));
  C10_CUDA_CHECK(cudaStreamSynchronize(stream.stream()));
  return THPVariable_Wrap(space);
  END_HANDLE_TH_ERRORS
}

// What build.py and _native.py look for in the file.
const char built_for[] = "built for " B200_BUILT_FOR ";";

PyMethodDef methods[] = {
    {"zeroed", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(zeroed)), METH_FASTCALL,
     "zeroed(device, words) -> int32 zeros outside any graph"},
    {"invoke", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(invoke)), METH_FASTCALL,
     "invoke(entry, device, plan, tensors, extents, number, code, other) -> the tensors made, or a status"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef definition = {PyModuleDef_HEAD_INIT, "binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_binding(void) {
  PyObject *module = PyModule_Create(&definition);
  if (module && PyModule_AddStringConstant(module, "built_for", built_for) < 0) {
    Py_DECREF(module);
    return nullptr;
  }
  return module;
}
