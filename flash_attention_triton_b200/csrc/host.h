// What the files of the Python module `_host` share.
#pragma once
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>

#include "../../include/fa2_b200.h"

namespace fa2_host {

// Raises _lib.Fa2Error for a non-zero code.  Called without the interpreter lock.
void check_code(const char* fn, int code);

// FA2_B200_CHECK_STATUS=1: raises _lib.Fa2Error when the status word of the device is set.  Called with the interpreter lock.
void check_status_if_asked(const char* fn, const at::Tensor& on);

inline int dtype_code(const at::Tensor& t) { return t.scalar_type() == at::kHalf ? FA2_DTYPE_FP16 : FA2_DTYPE_BF16; }
inline bool is_16bit(const at::Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }

// A tensor argument, or an undefined one for None where that is allowed; TypeError for anything else.  What stands for
// another tensor (in a transform, under a fake-tensor mode) or carries a forward-mode tangent is refused, not computed without it.
inline at::Tensor tensor_argument(PyObject* arg, const char* name, bool optional = false) {
  if (optional && arg == Py_None) return {};
  TORCH_CHECK_TYPE(THPVariable_Check(arg), name, " must be a tensor", optional ? " or None" : "");
  const at::Tensor& t = THPVariable_Unpack(arg);
  TORCH_CHECK_VALUE(t.defined() && t.layout() == at::kStrided, name, " must be a dense tensor");
  TORCH_CHECK_VALUE(t.has_storage() && !t.unsafeGetTensorImpl()->is_python_dispatch() && !t._fw_grad(0).defined(), name,
                    " must be a plain tensor: there is no form for transforms, fake tensors and forward-mode differentiation");
  return t.is_neg() ? t.resolve_neg() : t;
}
// A tensor that the call writes: not a view that negates what it shows.
inline at::Tensor written_argument(PyObject* arg, const char* name) {
  TORCH_CHECK_VALUE(!THPVariable_Check(arg) || !THPVariable_Unpack(arg).is_neg(), name, " must not be a negating view");
  return tensor_argument(arg, name);
}

// The softmax scale of a call: None and 0.0 mean 1 / sqrt(head dim).
inline double scale_argument(PyObject* arg, int64_t head_dim) {
  const double scale = arg == Py_None ? 0.0 : PyFloat_AsDouble(arg);
  if (scale == -1.0 && PyErr_Occurred()) throw python_error();
  return scale == 0.0 ? 1.0 / std::sqrt(static_cast<double>(head_dim)) : scale;
}

// Kernels read a [rows, H, D] tensor through its own strides: unit last stride, 16-byte aligned base, row and head
// strides that are multiples of 8 elements and at least D (those of dimensions of size 1 do not matter).
bool rows_readable(const at::Tensor& t);
// What cannot be read so is copied (a tensor that is dense but not aligned, too).
inline at::Tensor rows_input(const at::Tensor& t) { return rows_readable(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

// AssertionError as flash_attention_v2 raises it, for what is not a CUDA tensor; ValueError for another device.
void check_devices(std::initializer_list<std::pair<const at::Tensor*, const char*>> tensors);

void check_int32(const at::Tensor& t, const char* name, int dims);  // contiguous in its last dimension

PyObject* packed(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* kv_append(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* decode(PyObject*, PyObject* const* args, Py_ssize_t nargs);

}  // namespace fa2_host
