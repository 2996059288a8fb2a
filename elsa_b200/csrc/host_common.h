// What the native host paths (host.cpp, host_decoder.cpp) share: which calls they cover, views, allocation, statuses.
#pragma once

#define PY_SSIZE_T_CLEAN
#include <torch/csrc/python_headers.h>

#include <functional>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/dynamo/compiled_autograd.h>

#include "../../include/elsa_b200.h"

namespace elsa_host {

// (set by bind)
extern decltype(&elsa_strerror) f_strerror;
extern decltype(&elsa_last_cuda_error) f_last_cuda_error;

inline void check_status(int rc, const char* what) {
  if (rc == ELSA_OK) return;
  std::string msg = std::string(what) + ": " + f_strerror(rc);
  if (rc == ELSA_ERR_CUDA) msg += " [cudaError " + std::to_string(f_last_cuda_error()) + "]";
  if (rc == ELSA_ERR_INVALID_ARGUMENT || rc == ELSA_ERR_UNSUPPORTED) TORCH_CHECK_VALUE(false, msg);
  throw std::runtime_error(msg);
}

inline int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? ELSA_F32 : t == at::kHalf ? ELSA_F16 : t == at::kBFloat16 ? ELSA_BF16 : -1;
}

struct View {                 // a [B, H, N, D] operand: first element and {batch, head, row} element strides
  char* p = nullptr;
  int64_t st[3] = {0, 0, 0};
};

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline char* data_of(const at::Tensor& t) { return static_cast<char*>(const_cast<void*>(t.const_data_ptr())); }

// fills *v; true when the kernels can read `t` in place
inline bool in_place_view(const at::Tensor& t, View* v) {
  const auto sz = t.sizes();
  const auto st = t.strides();
  v->p = data_of(t);
  for (int i = 0; i < 3; ++i) v->st[i] = sz[i] > 1 ? st[i] : sz[3] * 8;   // (a size-1 axis may have any stride)
  if ((sz[3] > 1 && st[3] != 1) || !aligned16(v->p)) return false;
  return ((v->st[0] | v->st[1] | v->st[2]) % 8 == 0) && v->st[0] > 0 && v->st[1] > 0 && v->st[2] >= sz[3];
}

inline at::Tensor aligned(const at::Tensor& t) {
  at::Tensor c = t.contiguous();
  return aligned16(c.const_data_ptr()) ? c : c.clone();
}

inline at::Tensor new_tensor(at::IntArrayRef sizes, const at::Tensor& like, at::ScalarType dtype) {
  return at::detail::empty_cuda(sizes, dtype, like.device(), std::nullopt);
}

// an uninitialised [B, H, N, D] tensor in row-major [B, N, H, D] memory
inline at::Tensor new_bnhd(const at::Tensor& like, int64_t b, int64_t h, int64_t n, int64_t d) {
  return at::detail::empty_strided_cuda({b, h, n, d}, {n * h * d, d, h * d, 1}, like.scalar_type(), like.device());
}

inline bool plain(const at::Tensor& t) {
  // wrappers of function transforms, Python-dispatched and functional tensors keep to the general path
  constexpr c10::DispatchKeySet special({c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::FuncTorchBatched,
                                         c10::DispatchKey::FuncTorchVmapMode, c10::DispatchKey::Python,
                                         c10::DispatchKey::Functionalize, c10::DispatchKey::Batched});
  // (a forward-mode tangent too: the autograd functions of the general path refuse it, a result without one would be wrong)
  return t.is_cuda() && t.layout() == at::kStrided && !t.key_set().has_any(special) && !t._fw_grad(/*level=*/0).defined();
}

// dispatch modes, and torch.jit.trace: the general path's autograd functions are recorded as operations of the graph, while
// the output of a native call would be recorded as a constant
inline bool modes_active() { return c10::impl::TorchDispatchModeTLS::any_modes_set() || at::tracer::impl::is_dispatch_enabled(); }

inline c10::DataPtr workspace(int64_t bytes) { return c10::cuda::CUDACachingAllocator::get()->allocate(static_cast<size_t>(bytes)); }

// A saved tensor as the backward may use it: saved-tensor hooks may return the values in another memory layout (a copy
// built from the sizes alone, an unaligned slice), so nothing but the values is taken for granted.
inline void check_unpacked(const at::Tensor& t, at::IntArrayRef sizes, at::ScalarType dtype, c10::Device dev) {
  TORCH_CHECK(t.defined() && plain(t) && t.device() == dev && t.scalar_type() == dtype && t.sizes() == sizes,
              "a saved tensor of the attention came back from its unpack hook with another shape, dtype or device");
}

inline bool get_tensor(PyObject* o, at::Tensor* t) {
  if (o == Py_None) return true;
  if (!THPVariable_CheckExact(o)) return false;
  *t = THPVariable_Unpack(o);
  return true;
}

struct NoGil {
  PyThreadState* s = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(s); }
};

// host_decoder.cpp
void bind_decoder(const std::function<void*(const char*)>& at_name);
PyObject* py_rotary(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* py_shared_prefix(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* py_differential(PyObject*, PyObject* const* a, Py_ssize_t n);

}  // namespace elsa_host
