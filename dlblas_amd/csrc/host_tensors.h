// What the native entry points share: which tensors make a plain call, allocation, device and stream, the op event, the scope
// without the interpreter lock.
#pragma once

#include <Python.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/Tensor.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/record_function.h>
#include <c10/core/DefaultDtype.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <cstring>
#include <string>
#include <unordered_map>
#include <utility>
#include <vector>

#include "../../include/dlblas_decoder.h"
#include "../../include/dlblas_fp8_gemm.h"
#include "../../include/dlblas_fp8_moe.h"

namespace {

constexpr int64_t kBlock = 128;

// ---- what a plain call is ---------------------------------------------------------------------------------------------

const c10::DispatchKeySet kPlainKeys({c10::DispatchKey::CUDA, c10::DispatchKey::AutogradCUDA, c10::DispatchKey::ADInplaceOrView, c10::DispatchKey::AutocastCUDA});
const c10::DispatchKeySet kPlainIncluded({c10::DispatchKey::BackendSelect, c10::DispatchKey::ADInplaceOrView, c10::DispatchKey::AutocastCUDA});

// (raw bits: set difference on DispatchKeySet leaves the backend bits alone)
bool within(c10::DispatchKeySet keys, c10::DispatchKeySet allowed) { return (keys.raw_repr() & ~allowed.raw_repr()) == 0; }

bool no_modes() { return within(c10::impl::tls_local_dispatch_key_set().included_, kPlainIncluded) && !at::impl::torch_function_mode_enabled(); }

// A dense GPU tensor that nothing but its own storage stands behind; nullptr otherwise.  *grad, where asked for: whether a gradient is
// wanted for it; otherwise such a tensor is not plain.
const at::Tensor* plain(PyObject* o, bool* grad = nullptr) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || !within(t.key_set(), kPlainKeys)) return nullptr;
  const bool wanted = c10::GradMode::is_enabled() && t.requires_grad();
  if (t.is_conj() || t.is_neg() || (wanted && !grad) || t._fw_grad(0).defined()) return nullptr;
  if (wanted) *grad = true;
  return &t;
}

template <size_t N>
bool all_plain(PyObject* const* args, const at::Tensor* (&out)[N]) {
  if (!no_modes()) return false;
  for (size_t i = 0; i < N; ++i) {
    out[i] = plain(args[i]);
    if (!out[i] || out[i]->get_device() != out[0]->get_device()) return false;
  }
  return true;
}

// Makes the tensors' device current for the scope (a no-op in the usual case).
struct DeviceScope {
  c10::DeviceIndex before, dev;
  explicit DeviceScope(const at::Tensor& t) : before(c10::hip::current_device()), dev(t.get_device()) {
    if (dev != before) c10::hip::set_device(dev);
  }
  ~DeviceScope() {
    if (dev != before) c10::hip::set_device(before);
  }
};

hipStream_t stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

at::Tensor empty(at::IntArrayRef size, at::ScalarType dtype, const at::Tensor& like) {
  return at::Tensor(at::detail::empty_cuda(size, dtype, like.device(), std::nullopt));
}
at::Tensor empty_strided(at::IntArrayRef size, at::IntArrayRef stride, at::ScalarType dtype, const at::Tensor& like) {
  return at::Tensor(at::detail::empty_strided_cuda(size, stride, dtype, like.device()));
}

// A custom op that mutates an argument moves its version counter on.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void* ptr(const at::Tensor& t) { return t.numel() > 0 ? t.data_ptr() : nullptr; }
float* fptr(const at::Tensor& t) { return static_cast<float*>(ptr(t)); }
int32_t* iptr(const at::Tensor& t) { return static_cast<int32_t*>(ptr(t)); }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool is_f8(const at::Tensor& t) { return t.scalar_type() == at::kFloat8_e4m3fn; }
bool is_f32(const at::Tensor& t) { return t.scalar_type() == at::kFloat; }
int out_code(at::ScalarType t) { return t == at::kBFloat16 ? DLB_OUT_BF16 : t == at::kFloat ? DLB_OUT_F32 : -1; }
int in_code(at::ScalarType t) { return t == at::kBFloat16 ? DLB_IN_BF16 : t == at::kHalf ? DLB_IN_F16 : t == at::kFloat ? DLB_IN_F32 : -1; }
int idx_code(at::ScalarType t) { return t == at::kInt ? DLB_IDX_I32 : t == at::kLong ? DLB_IDX_I64 : -1; }

// An op event of torch's profiler, as the custom ops of the Python path leave one; nothing when nobody records.
struct OpRecord {
  at::RecordFunction guard{at::RecordScope::FUNCTION};
  std::vector<c10::IValue> inputs;
  template <size_t N>
  OpRecord(const char* name, const at::Tensor* const (&t)[N]) {
    if (!guard.isActive()) return;
    if (guard.needsInputs())
      for (const at::Tensor* x : t)
        if (x) inputs.emplace_back(*x);
    guard.before(name, c10::ArrayRef<const c10::IValue>(inputs.data(), inputs.size()));
  }
};

// Allocations and launches run without the GIL: a launch waits while the hardware queue is full.  No Python object is touched
// in such a scope.
class NoGil {
 public:
  NoGil() : state_(PyEval_SaveThread()) {}
  ~NoGil() { PyEval_RestoreThread(state_); }
  NoGil(const NoGil&) = delete;
  NoGil& operator=(const NoGil&) = delete;

 private:
  PyThreadState* state_;
};

#define NOT_PLAIN Py_RETURN_NONE
// An exception raised in Python, by a hook on saved tensors for one, goes on as what it is: checkpointing ends a recomputation with
// one of its own.
#define HANDLE_EXCEPTIONS_BEGIN try {
#define HANDLE_EXCEPTIONS_END                          \
  }                                                    \
  catch (const c10::OutOfMemoryError& e) {             \
    NOT_PLAIN; /* the Python path raises torch's own */ \
  }                                                    \
  catch (py::error_already_set & e) {                  \
    e.restore();                                       \
    return nullptr;                                    \
  }                                                    \
  catch (python_error & e) {                           \
    e.restore();                                       \
    return nullptr;                                    \
  }                                                    \
  catch (const std::exception& e) {                    \
    PyErr_SetString(PyExc_RuntimeError, e.what());     \
    return nullptr;                                    \
  }

}  // namespace

// The functions of host_steps.cpp, added to the module by PyInit__host; the last entry is empty.
extern PyMethodDef host_step_methods[];
