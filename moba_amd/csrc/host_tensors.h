// What the functions of the extension module that take tensors have in common: which they read where they lie, new ones, errors.
#pragma once
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/EmptyTensor.h>
#include <Python.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include "../../include/moba_hip.h"

inline decltype(&moba_strerror) str_error = nullptr;   // (bind_layer)

namespace {

using at::Tensor;

constexpr int64_t kMostHeads = 1 << 16;

// Other threads go on while a call allocates and launches.
struct NoGil {
  PyThreadState* const state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

const Tensor* plain_tensor(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

// an optional tensor: false if it is something else
bool optional_tensor(PyObject* o, Tensor& t) {
  if (o == Py_None) return true;
  const Tensor* p = plain_tensor(o);
  if (p) t = *p;
  return p != nullptr;
}

bool aligned(const Tensor& t, int bytes) { return ((uintptr_t)t.const_data_ptr() & (bytes - 1)) == 0; }

// [tokens, heads, head_dim] of 16-bit elements that is read where it lies: its token and head strides, multiples of `step`.
// The stride of a dimension of one entry says nothing and is the packed one.
bool rows_in_place(const Tensor& t, int step, int bytes, int64_t* strides) {
  const auto size = t.sizes(), stride = t.strides();
  strides[0] = size[0] > 1 ? stride[0] : size[1] * size[2];
  strides[1] = size[1] > 1 ? stride[1] : size[2];
  return stride[2] == 1 && strides[0] % step == 0 && strides[1] % step == 0 && aligned(t, bytes);
}

bool half_type(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }
int type_code(const Tensor& t) { return t.scalar_type() == at::kHalf ? MOBA_DTYPE_F16 : MOBA_DTYPE_BF16; }
hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

bool frequencies_fit(const Tensor& f, const at::Device& device, int64_t d) {
  return f.scalar_type() == at::kFloat && f.dim() == 1 && f.is_contiguous() && f.device() == device && f.numel() % 4 == 0 &&
         f.numel() > 0 && 2 * f.numel() <= d && aligned(f, 4);
}

// A new tensor, without the way through the dispatcher (which is a third of what at::empty takes).
Tensor fresh(at::IntArrayRef size, at::ScalarType type, const at::Device& device) {
  return Tensor(at::detail::empty_cuda(size, type, device, std::nullopt));
}
Tensor fresh_like(const Tensor& t) { return fresh(t.sizes(), t.scalar_type(), t.device()); }   // (packed, whatever t's strides)
Tensor bytes(size_t count, const at::Device& device) { return fresh({(int64_t)count}, at::kByte, device); }

// whether a forward-mode tangent comes with it (there are no such derivatives)
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }

void check(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed with code ", rc, ": ", str_error(rc)); }

const void* pointer(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* mutable_pointer(Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }


// ---- the paged cache (whose tensors its class has checked)
bool wants_derivative(const Tensor& t) {   // (there are none)
  return t.defined() && ((t.requires_grad() && at::GradMode::is_enabled()) || has_tangent(t));
}

// autograd learns that a tensor has changed (an inference tensor keeps no such number)
void written(const Tensor& t) {
  if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

struct Cache {
  const Tensor *k, *v;
  Tensor k_scales, v_scales;
  bool take(PyObject* const* args) {
    k = plain_tensor(args[0]);
    v = plain_tensor(args[1]);
    return k && v && optional_tensor(args[2], k_scales) && optional_tensor(args[3], v_scales) && k->is_cuda() && k->dim() == 4 &&
           !wants_derivative(*k) && !wants_derivative(*v) && !wants_derivative(k_scales) && !wants_derivative(v_scales);
  }
  bool takes_rows(const Tensor& x) const {
    return !wants_derivative(x) && half_type(x) && (k_scales.defined() || x.scalar_type() == k->scalar_type()) && x.dim() == 3 &&
           x.size(2) == k->size(3) && x.device() == k->device();
  }
};

struct Index {
  const Tensor *table, *lengths, *cu;
  bool take(PyObject* const* args, const at::Device& device) {
    table = plain_tensor(args[0]);
    lengths = plain_tensor(args[1]);
    cu = plain_tensor(args[2]);
    if (!table || !lengths || !cu) return false;
    for (const Tensor* t : {table, lengths, cu})
      if (t->scalar_type() != at::kInt || t->device() != device) return false;
    if (table->dim() != 2 || lengths->dim() != 1 || cu->dim() != 1 || !lengths->is_contiguous() || !cu->is_contiguous()) return false;
    const int64_t b = table->size(0);
    return b > 0 && b < INT32_MAX && table->size(1) > 0 && table->size(1) <= INT32_MAX && (table->stride(1) == 1 || table->size(1) == 1) && lengths->size(0) == b &&
           cu->size(0) == b + 1;
  }
};

}  // namespace
