// Host side of a repeated direct call (conductor_b200/ops.py): checks that the tensors are the ones the call was
// prepared for, takes the output and the scratch from torch's caching allocator, fills in the pointers and
// calls the library.  A decode step's kernels take 9 us; host time of the call: 14 us with these steps in Python, 8 us so.
// Holds no kernel and no pointer of a tensor between calls.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <memory>
#include <vector>

#include "../../include/conductor_b200.h"

namespace {

typedef int (*LaunchMany)(const cdr_launch_item*, int, void*, int*);

struct Expected {
  std::vector<int64_t> sizes, strides;
  at::ScalarType dtype;
  c10::Device device = c10::Device(c10::kCPU);
  bool aligned;                 // rank >= 3: read in 16-byte pieces
};

struct CallState {
  std::vector<Expected> ins;
  std::vector<int64_t> out_sizes;
  cdr_launch_item* item = nullptr;       // owned by the Python object that made the call
  cdr_tensor* in_desc = nullptr;
  cdr_tensor* out_desc = nullptr;
  LaunchMany launch = nullptr;
};

// What only the dispatcher can serve: modes and tracers that record a call, wrappers of function transforms, and views
// whose elements are not what the memory holds.
constexpr c10::DispatchKeySet kDispatched({
    c10::DispatchKey::Python, c10::DispatchKey::PythonDispatcher, c10::DispatchKey::PythonTLSSnapshot, c10::DispatchKey::PreDispatch,
    c10::DispatchKey::Tracer, c10::DispatchKey::Functionalize, c10::DispatchKey::FuncTorchDynamicLayerFrontMode,
    c10::DispatchKey::FuncTorchDynamicLayerBackMode, c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::FuncTorchBatched,
    c10::DispatchKey::FuncTorchBatchedDecomposition, c10::DispatchKey::FuncTorchVmapMode, c10::DispatchKey::BatchedNestedTensor,
    c10::DispatchKey::VmapMode, c10::DispatchKey::Conjugate, c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor});

bool calls_are_dispatched() {
  const c10::impl::LocalDispatchKeySet tls = c10::impl::tls_local_dispatch_key_set();
  return (tls.included_ - tls.excluded_).has_any(kDispatched);
}

bool needs_gradient(const at::Tensor& t) {
  const c10::AutogradState& state = c10::AutogradState::get_tls_state();
  return (state.get_grad_mode() && t.requires_grad()) || (state.get_fw_grad_mode() && t._fw_grad(0).defined());
}

struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

struct CallObject {
  PyObject_HEAD
  CallState* state;
};

// Call(item address, input descriptors, output descriptor, address of cdr_launch_many, tensors)
PyObject* call_new(PyTypeObject* type, PyObject* args, PyObject*) {
  HANDLE_TH_ERRORS
  unsigned long long item = 0, in_desc = 0, out_desc = 0, launch = 0;
  PyObject* tensors = nullptr;
  if (!PyArg_ParseTuple(args, "KKKKO!", &item, &in_desc, &out_desc, &launch, &PyTuple_Type, &tensors)) return nullptr;
  std::unique_ptr<CallState> st(new CallState);
  st->item = reinterpret_cast<cdr_launch_item*>(item);
  st->in_desc = reinterpret_cast<cdr_tensor*>(in_desc);
  st->out_desc = reinterpret_cast<cdr_tensor*>(out_desc);
  st->launch = reinterpret_cast<LaunchMany>(launch);
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(tensors); ++i) {
    PyObject* o = PyTuple_GET_ITEM(tensors, i);
    if (!THPVariable_Check(o)) { PyErr_SetString(PyExc_TypeError, "expected tensors"); return nullptr; }
    const at::Tensor& t = THPVariable_Unpack(o);
    Expected e;
    e.sizes = t.sizes().vec();
    e.strides = t.strides().vec();
    e.dtype = t.scalar_type();
    e.device = t.device();
    e.aligned = t.dim() >= 3;
    st->ins.push_back(std::move(e));
  }
  st->out_sizes.assign(st->out_desc->shape, st->out_desc->shape + st->out_desc->rank);
  PyObject* self = type->tp_alloc(type, 0);
  if (!self) return nullptr;
  reinterpret_cast<CallObject*>(self)->state = st.release();
  return self;
  END_HANDLE_TH_ERRORS
}

void call_dealloc(PyObject* self) {
  delete reinterpret_cast<CallObject*>(self)->state;
  Py_TYPE(self)->tp_free(self);
}

// run(*tensors): the output; None where the call was made for other tensors, would need gradients or is one for the
// dispatcher; the library's status where it refused.
PyObject* call_run(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  CallState& st = *reinterpret_cast<CallObject*>(self)->state;
  if (n != static_cast<Py_ssize_t>(st.ins.size())) Py_RETURN_NONE;
  if (calls_are_dispatched()) Py_RETURN_NONE;
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (!THPVariable_CheckExact(args[i])) Py_RETURN_NONE;
    const at::Tensor& t = THPVariable_Unpack(args[i]);
    const Expected& e = st.ins[i];
    if (t.device() != e.device || t.scalar_type() != e.dtype || t.sizes() != at::IntArrayRef(e.sizes) ||
        t.strides() != at::IntArrayRef(e.strides) || t.key_set().has_any(kDispatched) || needs_gradient(t))
      Py_RETURN_NONE;
    void* p = const_cast<void*>(t.const_data_ptr());
    if (e.aligned && (reinterpret_cast<uintptr_t>(p) & 15u)) Py_RETURN_NONE;
    st.in_desc[i].data = p;
  }
  at::Tensor out;
  int rc = 0;
  {
    NoGil no_gil;                 // a full launch queue must not keep other threads from Python
    const c10::Device device = st.ins[0].device;
    c10::cuda::OptionalCUDAGuard guard;
    if (c10::cuda::current_device() != device.index()) guard.set_device(device);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    out = at::empty(st.out_sizes, at::TensorOptions().dtype(st.ins[0].dtype).device(device));
    st.out_desc->data = out.data_ptr();
    // scratch of this call alone: it goes back to the stream's pool once the launch is enqueued
    void* ws = st.item->workspace_bytes ? c10::cuda::CUDACachingAllocator::raw_alloc_with_stream(st.item->workspace_bytes, stream) : nullptr;
    st.item->workspace = ws;
    rc = st.launch(st.item, 1, stream, nullptr);
    if (ws) c10::cuda::CUDACachingAllocator::raw_delete(ws);
  }
  if (rc != 0) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// is_dispatched(*tensors): the call is one for the dispatcher.
PyObject* is_dispatched(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  bool any = calls_are_dispatched();
  for (Py_ssize_t i = 0; i < n && !any; ++i) any = THPVariable_Check(args[i]) && THPVariable_Unpack(args[i]).key_set().has_any(kDispatched);
  return PyBool_FromLong(any);
  END_HANDLE_TH_ERRORS
}

PyMethodDef module_methods[] = {
    {"is_dispatched", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(is_dispatched)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyMethodDef call_methods[] = {
    {"run", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(call_run)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyTypeObject call_type = {PyVarObject_HEAD_INIT(nullptr, 0) "_cdr_torch.Call", sizeof(CallObject)};

PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_cdr_torch", nullptr, -1, module_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__cdr_torch(void) {
  call_type.tp_flags = Py_TPFLAGS_DEFAULT;
  call_type.tp_new = call_new;
  call_type.tp_dealloc = call_dealloc;
  call_type.tp_methods = call_methods;
  if (PyType_Ready(&call_type) < 0) return nullptr;
  PyObject* m = PyModule_Create(&module_def);
  if (!m) return nullptr;
  if (PyModule_AddStringConstant(m, "built_for", CDR_BUILT_FOR) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  Py_INCREF(&call_type);
  if (PyModule_AddObject(m, "Call", reinterpret_cast<PyObject*>(&call_type)) < 0) {
    Py_DECREF(&call_type);
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
