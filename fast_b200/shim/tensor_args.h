// What the torch-level modules over the libfast_b200 C ABI share: checks of
// tensor arguments (bad ones raise ValueError), library errors as
// fast_b200.capi.FastB200Error, outputs from torch's allocator, launch counts.
// Included once by each module.
#pragma once
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "fast_b200.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

[[noreturn]] void refuse(const std::string &what) { throw py::value_error(what); }

void check(int rc) {
  if (rc == FB_OK) return;
  const py::object cls = py::module_::import("fast_b200.capi").attr("FastB200Error");
  PyErr_SetString(cls.ptr(), (std::string("fast_b200: ") + fb_last_error()).c_str());
  throw py::error_already_set();
}

// Adds the kernels launched in its lifetime to the list given to count_into
// (how many a call takes depends on its sizes).  The list is never freed.
py::handle &count_list() {
  static py::handle list;
  return list;
}
struct Count {
  const int64_t before = fb_launches();
  ~Count() {
    PyObject *list = count_list().ptr();
    if (!list) return;
    const long long now = PyLong_AsLongLong(PyList_GET_ITEM(list, 0)) + (fb_launches() - before);
    PyList_SetItem(list, 0, PyLong_FromLongLong(now));
  }
};

const char *type_name(at::ScalarType t) { return t == at::kFloat ? "fp32" : (t == at::kBFloat16 ? "bf16" : "int64"); }

int head_type(const Tensor &t, const char *name) {
  if (t.scalar_type() == at::kFloat) return FB_F32;
  if (t.scalar_type() == at::kBFloat16) return FB_BF16;
  refuse(std::string(name) + " must be fp32 or bf16");
}

// A matrix of `type` on `like`'s GPU, rows of unit column stride that do not
// overlap, [r, c] when given (-1: any).
void rows(const Tensor &t, const char *name, at::ScalarType type, const Tensor &like, int64_t r = -1, int64_t c = -1) {
  if (t.scalar_type() != type || t.dim() != 2 || !t.is_cuda() || t.get_device() != like.get_device())
    refuse(std::string(name) + " must be a CUDA " + type_name(type) + " matrix on the inputs' device");
  const int64_t n = t.size(0), d = t.size(1);
  if ((r >= 0 && n != r) || (c >= 0 && d != c))
    refuse(std::string(name) + " must have shape [" + (r < 0 ? "n" : std::to_string(r)) + ", " +
           (c < 0 ? "D" : std::to_string(c)) + "], not [" + std::to_string(n) + ", " + std::to_string(d) + "]");
  if (d > 1 && t.stride(1) != 1) refuse(std::string(name) + " must have unit column stride");
  if (n > 1 && t.stride(0) < d) refuse(std::string(name) + " must have rows that do not overlap");
}

// Leading dimension (a single row's stride says nothing).
int64_t ld(const Tensor &t) { return t.size(0) > 1 ? t.stride(0) : std::max(t.stride(0), t.size(1)); }

void vec(const Tensor &t, const char *name, at::ScalarType type, const Tensor &like, int64_t n) {
  if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != n || !t.is_cuda() ||
      t.get_device() != like.get_device() || !t.is_contiguous())
    refuse(std::string(name) + " must be a contiguous CUDA " + type_name(type) + " vector of " + std::to_string(n) +
           " on the inputs' device");
}

void *ptr(const Tensor &t) { return t.data_ptr(); }
void *ptr(const OptTensor &t) { return t ? t->data_ptr() : nullptr; }

Tensor empty(at::IntArrayRef size, const Tensor &like, at::ScalarType type) {
  return at::empty(size, like.options().dtype(type));
}

cudaStream_t stream_of(const Tensor &t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

}  // namespace
