// The host path of one q35_run call from Python, without Python: `run(role, stream=None, **tensors)` binds the tensors by
// name into the C ABI's IO table (include/q35b200.h) and issues the call on their device's current stream.
//
// What it does is what _lib.py's run_checked does in 6 to 10 us of interpreter time, in less than 2.  It only takes calls
// that bind as they are: tensors, contiguous, on one GPU, of types the ABI has a code for.  Anything else goes to
// run_checked, which names what is wrong.  The library's entry points come as addresses, so that this module links
// against nothing of it.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include "../../include/q35b200.h"

namespace {

using RunFn = int (*)(const char*, const q35_io*, int, void*);
using BytesFn = int64_t (*)(const char*, const q35_io*, int);
RunFn g_run = nullptr;
BytesFn g_bytes = nullptr;
PyObject* g_checked = nullptr;  // run_checked(role, stream=..., **tensors)
PyObject* g_scratch = nullptr;  // scratch(device, bytes, stream) -> (address, owner)
PyObject* g_error = nullptr;    // error(status) raises

constexpr int kMax = 48;

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kByte: case at::kChar: return Q35_U8;
    case at::kFloat: return Q35_F32;
    case at::kInt: return Q35_I32;
    case at::kBFloat16: return Q35_BF16;
    case at::kHalf: return Q35_F16;
    case at::kFloat8_e4m3fn: return Q35_E4M3;
    case at::kFloat8_e8m0fnu: return Q35_U8;
    default: return 0;
  }
}

// false: not a call for the fast path (no Python error set)
bool bind(const char* name, PyObject* v, q35_io* io, int* device) {
  if (!name || !THPVariable_Check(v)) return false;
  const at::Tensor& t = THPVariable_Unpack(v);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.is_contiguous() || t.dim() > Q35_MAX_DIMS) return false;
  const int code = code_of(t.scalar_type()), dev = t.get_device();
  if (code == 0 || (*device >= 0 && dev != *device)) return false;
  *device = dev;
  io->name = name;
  io->ptr = t.data_ptr();
  io->bytes = size_t(t.numel()) * t.element_size();
  io->dtype = code;
  io->ndim = int(t.dim());
  for (int d = 0; d < io->ndim; ++d) io->shape[d] = t.size(d);
  return true;
}

PyObject* run(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  try {
    const Py_ssize_t nkw = kwnames ? PyTuple_GET_SIZE(kwnames) : 0;
    q35_io ios[kMax + 1];
    int n = 0, device = -1;
    bool fast = nargs >= 1 && nargs <= 2 && nkw <= kMax && PyUnicode_Check(args[0]), has_workspace = false;
    PyObject* stream_arg = nargs == 2 ? args[1] : Py_None;
    const char* role = fast ? PyUnicode_AsUTF8(args[0]) : nullptr;
    for (Py_ssize_t i = 0; fast && i < nkw; ++i) {
      const char* name = PyUnicode_AsUTF8(PyTuple_GET_ITEM(kwnames, i));
      if (!name) return nullptr;
      if (strcmp(name, "stream") == 0) {
        stream_arg = args[nargs + i];
        continue;
      }
      fast = bind(name, args[nargs + i], &ios[n++], &device);
      has_workspace |= fast && strcmp(name, "workspace") == 0;
    }
    if (!fast || !role || device < 0) return PyObject_Vectorcall(g_checked, args, nargs, kwnames);
    c10::cuda::OptionalCUDAGuard guard;
    if (c10::cuda::current_device() != device) guard.set_index(c10::DeviceIndex(device));
    void* stream;
    if (stream_arg == Py_None) {
      stream = c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(device)).stream();
    } else {
      stream = PyLong_AsVoidPtr(stream_arg);
      if (!stream && PyErr_Occurred()) return nullptr;
    }
    PyObject* owner = nullptr;  // of the scratch, until the call is issued
    if (!has_workspace) {
      const int64_t need = g_bytes(role, ios, n);
      if (need < 0) return PyObject_CallFunction(g_error, "i", int(-need));
      if (need > 0) {
        owner = PyObject_CallFunction(g_scratch, "iLK", device, (long long)need, (unsigned long long)(uintptr_t)stream);
        if (!owner) return nullptr;
        void* p = PyTuple_Check(owner) ? PyLong_AsVoidPtr(PyTuple_GET_ITEM(owner, 0)) : nullptr;
        if (!p) {
          Py_DECREF(owner);
          if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "no scratch memory");
          return nullptr;
        }
        q35_io& io = ios[n++];
        io.name = "workspace";
        io.ptr = p;
        io.bytes = size_t(need);
        io.dtype = Q35_U8;
        io.ndim = 1;
        io.shape[0] = need;
      }
    }
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = g_run(role, ios, n, stream);
    Py_END_ALLOW_THREADS
    Py_XDECREF(owner);
    if (status != 0) return PyObject_CallFunction(g_error, "i", status);
    Py_RETURN_NONE;
  } catch (const std::exception& e) {  // a C++ exception must not cross into the interpreter
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyObject* init(PyObject*, PyObject* args) {
  unsigned long long run_at, bytes_at;
  PyObject *checked, *scratch, *error;
  if (!PyArg_ParseTuple(args, "KKOOO", &run_at, &bytes_at, &checked, &scratch, &error)) return nullptr;
  g_run = reinterpret_cast<RunFn>(uintptr_t(run_at));
  g_bytes = reinterpret_cast<BytesFn>(uintptr_t(bytes_at));
  Py_INCREF(checked); Py_INCREF(scratch); Py_INCREF(error);
  Py_XDECREF(g_checked); Py_XDECREF(g_scratch); Py_XDECREF(g_error);
  g_checked = checked; g_scratch = scratch; g_error = error;
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"run", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(run)), METH_FASTCALL | METH_KEYWORDS,
     "run(role, stream=None, **tensors): q35_run with the tensors bound by name"},
    {"init", init, METH_VARARGS, "init(address of q35_run, address of q35_workspace_bytes, run_checked, scratch, error)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind() {
  PyObject* m = PyModule_Create(&kModule);
  // the torch whose object layouts this file was compiled with: the host compares it before the first call
  if (m && PyModule_AddStringConstant(m, "built_for", Q35_BUILT_FOR) < 0) Py_CLEAR(m);
  return m;
}
