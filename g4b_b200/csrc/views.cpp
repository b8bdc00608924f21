// The Python side's argument packing in C++: torch tensors into the C views of include/g4b_attn.h, and the call itself.
//
// A call of the packed step has 8 to 14 tensors (page copies: dozens of pools).  Asked through Python a tensor's pointer,
// extents, strides, type and device cost 0.8 us, which for small steps is more than the launches; here they are plain
// reads.  What is not a torch tensor, or wrong, is left to the Python code of _cabi.py (the functions return None),
// so that checks and messages stand in one place.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include <cstring>

#include "../../include/g4b_attn.h"

namespace {

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return G4B_F32;
    case at::kHalf: return G4B_F16;
    case at::kBFloat16: return G4B_BF16;
    case at::kInt: return G4B_I32;
    case at::kLong: return G4B_I64;
    case at::kByte: return G4B_U8;
    case at::kFloat8_e4m3fn: return G4B_FP8_E4M3;
    default: return -1;
  }
}

// A CUDA tensor of the current device, or any tensor where the device is not checked.
bool device_fits(const at::Tensor& t, bool check_device) {
  return !check_device || (t.is_cuda() && t.get_device() == c10::cuda::current_device());
}

// false: not for this code (the Python code takes it, or says what is wrong)
bool fill(PyObject* o, G4bTensor& out, bool check_device) {
  std::memset(&out, 0, sizeof(out));
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  const int code = t.defined() && t.layout() == at::kStrided ? dtype_code(t.scalar_type()) : -1;
  if (code < 0 || t.dim() > 5 || !device_fits(t, check_device)) return false;
  out.ptr = t.data_ptr();
  out.ndim = (int32_t)t.dim();
  out.dtype = code;
  for (int i = 0; i < out.ndim; ++i) { out.shape[i] = t.size(i); out.stride[i] = t.stride(i); }
  return true;
}

constexpr int kMostTensors = 32, kMostTail = 64, kMostPools = 1024;

// The stream to launch on: an int, or None for torch's current one.
bool stream_of(PyObject* o, void*& out) {
  if (o == Py_None) {
    out = (void*)c10::cuda::getCurrentCUDAStream().stream();
    return true;
  }
  out = PyLong_AsVoidPtr(o);
  return !(out == nullptr && PyErr_Occurred());
}

// call(function address, check devices, stream, tail of the argument struct, tensors) -> status, or None
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  try {
    if (n != 5 || !PyBytes_Check(args[3]) || !PyTuple_Check(args[4])) { PyErr_SetString(PyExc_TypeError, "call(address, check, stream, tail, tensors)"); return nullptr; }
    const Py_ssize_t count = PyTuple_GET_SIZE(args[4]), tail = PyBytes_GET_SIZE(args[3]);
    if (count > kMostTensors || tail > kMostTail) Py_RETURN_NONE;
    alignas(16) char block[kMostTensors * sizeof(G4bTensor) + kMostTail];
    const bool check = PyObject_IsTrue(args[1]) == 1;
    for (Py_ssize_t i = 0; i < count; ++i)
      if (!fill(PyTuple_GET_ITEM(args[4], i), *reinterpret_cast<G4bTensor*>(block + i * sizeof(G4bTensor)), check)) Py_RETURN_NONE;
    std::memcpy(block + count * sizeof(G4bTensor), PyBytes_AS_STRING(args[3]), (size_t)tail);
    void* fn = PyLong_AsVoidPtr(args[0]);
    if (fn == nullptr) { if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "no function"); return nullptr; }
    void* stream = nullptr;
    if (!stream_of(args[2], stream)) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = reinterpret_cast<int (*)(const void*, void*)>(fn)(block, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// page_copy(function address, check devices, stream, pools, src, dst) -> status, or None
PyObject* page_copy(PyObject*, PyObject* const* args, Py_ssize_t n) {
  try {
    if (n != 6 || !PyList_Check(args[3])) { PyErr_SetString(PyExc_TypeError, "page_copy(address, check, stream, pools, src, dst)"); return nullptr; }
    const Py_ssize_t count = PyList_GET_SIZE(args[3]);
    if (count > kMostPools) Py_RETURN_NONE;
    const bool check = PyObject_IsTrue(args[1]) == 1;
    G4bPagePool pools[kMostPools];
    G4bPageCopyArgs a;
    std::memset(&a, 0, sizeof(a));
    for (Py_ssize_t i = 0; i < count; ++i) {
      PyObject* o = PyList_GET_ITEM(args[3], i);
      if (!THPVariable_Check(o)) Py_RETURN_NONE;
      const at::Tensor& t = THPVariable_Unpack(o);
      if (!t.defined() || t.layout() != at::kStrided || t.dim() < 1 || !t.is_contiguous() || !device_fits(t, check)) Py_RETURN_NONE;
      if (i == 0) a.num_pages = t.size(0);
      if (t.size(0) != a.num_pages) Py_RETURN_NONE;
      pools[i].ptr = t.data_ptr();
      pools[i].page_bytes = a.num_pages > 0 ? (int64_t)t.nbytes() / a.num_pages : 0;
    }
    if (!fill(args[4], a.src_pages, check) || !fill(args[5], a.dst_pages, check)) Py_RETURN_NONE;
    a.pools = pools;
    a.num_pools = (int32_t)count;
    void* fn = PyLong_AsVoidPtr(args[0]);
    if (fn == nullptr) { if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "no function"); return nullptr; }
    void* stream = nullptr;
    if (!stream_of(args[2], stream)) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = reinterpret_cast<int (*)(const void*, void*)>(fn)(&a, stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// views(check devices, tensors) -> the C views behind one another, or None
PyObject* views(PyObject*, PyObject* const* args, Py_ssize_t n) {
  try {
    if (n != 2 || !PyTuple_Check(args[1])) { PyErr_SetString(PyExc_TypeError, "views(check, tensors)"); return nullptr; }
    const Py_ssize_t count = PyTuple_GET_SIZE(args[1]);
    if (count > kMostTensors) Py_RETURN_NONE;
    G4bTensor block[kMostTensors];
    const bool check = PyObject_IsTrue(args[0]) == 1;
    for (Py_ssize_t i = 0; i < count; ++i)
      if (!fill(PyTuple_GET_ITEM(args[1], i), block[i], check)) Py_RETURN_NONE;
    return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(block), count * (Py_ssize_t)sizeof(G4bTensor));
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyMethodDef methods[] = {
    {"call", (PyCFunction)(void*)call, METH_FASTCALL, nullptr},
    {"page_copy", (PyCFunction)(void*)page_copy, METH_FASTCALL, nullptr},
    {"views", (PyCFunction)(void*)views, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_views", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// built_for: the torch and the Python whose headers this was compiled with.  A tensor is read through their inlined
// layouts, so the module is used with no other (_cabi.py compares).
PyMODINIT_FUNC PyInit__views(void) {
  PyObject* m = PyModule_Create(&module);
  if (m != nullptr && PyModule_AddStringConstant(m, "built_for", G4B_BUILT_FOR) != 0) { Py_DECREF(m); return nullptr; }
  return m;
}
