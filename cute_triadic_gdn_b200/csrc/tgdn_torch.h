// What the translation units of the host path share: the package's errors, autograd functions that keep their classes, pointers and
// optional tensors.
#pragma once

#include <torch/extension.h>
#include <torch/csrc/Exceptions.h>
#include <torch/library.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <cstdlib>
#include <cstring>
#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>
#include <vector>

#include "tgdn_host.h"

namespace tgdn_torch {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ---- errors -----------------------------------------------------------------------------------------------------------
// The package raises AssertionError from the argument checks of the core (as the reference does), ValueError for
// packed-row and device / E problems, and TgdnError (_lib.py) when the library rejects a call.
struct AssertFail : std::runtime_error { using std::runtime_error::runtime_error; };
struct LibraryFail : std::runtime_error { using std::runtime_error::runtime_error; };

inline py::handle library_error;                                  // TgdnError, set by _lib.py
inline void set_python_error(const AssertFail& e) { PyErr_SetString(PyExc_AssertionError, e.what()); }
inline void set_python_error(const LibraryFail& e) { PyErr_SetString(library_error ? library_error.ptr() : PyExc_RuntimeError, e.what()); }

// Impl::forward and Impl::backward as an autograd function.  A backward runs under torch's engine, which keeps the class of a Python
// error only: the two above are turned into one there (elsewhere the module's translator does it).
template <typename Impl>
struct Differentiable : public torch::autograd::Function<Differentiable<Impl>> {
  template <typename... Args>
  static auto forward(AutogradContext* ctx, Args&&... args) { return Impl::forward(ctx, std::forward<Args>(args)...); }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    try {
      return Impl::backward(ctx, std::move(grads));
    } catch (const AssertFail& e) {
      rethrow(e);
    } catch (const LibraryFail& e) {
      rethrow(e);
    }
  }
  template <typename Fail>
  [[noreturn]] static void rethrow(const Fail& e) {
    py::gil_scoped_acquire gil;
    set_python_error(e);
    python_error error;
    error.persist();
    throw error;
  }
};

inline void check_rc(int rc, const char* what) {
  if (rc != 0) throw LibraryFail(std::string(what) + ": " + tgdn_error_string(rc) + " (code " + std::to_string(rc) + ")");
}

inline std::string shape_of(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}

#define TGDN_ASSERT(cond, ...) do { if (!(cond)) throw AssertFail(c10::str(__VA_ARGS__)); } while (0)

template <typename T = void>
T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }
template <typename T = void>
T* ptr(const OptTensor& t) { return t.has_value() ? ptr<T>(*t) : nullptr; }
inline const float* fptr(const Tensor& t) { return ptr<float>(t); }
inline bool has(const OptTensor& t) { return t.has_value() && t->defined(); }

inline void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

inline Tensor empty(at::IntArrayRef sizes, const Tensor& like, at::ScalarType dtype) { return at::empty(sizes, like.options().dtype(dtype)); }

inline Tensor or_undefined(const OptTensor& t) { return has(t) ? *t : Tensor(); }
inline OptTensor or_nullopt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

inline bool any_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->requires_grad()) return true;
  return false;
}

// The operators around the core (tgdn_torch_block.cpp), as functions of the module.
void bind_block_operators(py::module_& m);

}  // namespace tgdn_torch
