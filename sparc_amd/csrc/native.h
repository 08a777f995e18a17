// What the torch bindings share: checks, addresses, and what torch has to be told.
#ifndef SPARC_NATIVE_H
#define SPARC_NATIVE_H

#include <stdexcept>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include "sparc_hip.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Tensors = std::vector<Tensor>;

sparc_stream_t stream_of(const Tensor& t) {
  return reinterpret_cast<sparc_stream_t>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}
void check(sparc_status s, const char* what) {
  if (s != SPARC_OK)
    throw std::runtime_error(std::string(what) + " failed (sparc_status " + std::to_string(s) +
                             "): " + sparc_last_error());
}
bool is_io(const Tensor& t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16; }
int32_t code_of(at::ScalarType t) { return t == at::kFloat ? SPARC_F32 : SPARC_BF16; }
// whether t is a dense tensor on the device of the GPU tensor ``with``
bool beside(const Tensor& t, const Tensor& with) {
  return t.layout() == at::kStrided && t.is_cuda() && t.device() == with.device();
}
bool beside(const optional<Tensor>& t, const Tensor& with) { return !t || beside(*t, with); }
void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor scratch(size_t bytes, const Tensor& like) {
  return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}
// The values as they lie in memory: not those of a view that conjugates or negates
// when torch reads it (z.conj(), and its imaginary part)
bool is_literal(const Tensor& t) { return !t.is_conj() && !t.is_neg(); }
Tensor contiguous(const Tensor& t) {
  return is_literal(t) ? t.contiguous() : t.clone(at::MemoryFormat::Contiguous);
}
Tensor contiguous(const optional<Tensor>& t) { return t ? contiguous(*t) : Tensor(); }
// torch.jit.trace would record the allocation of a result and nothing that fills it.
void refuse_tracing(const char* what) {
  if (at::tracer::impl::is_dispatch_enabled())
    throw std::runtime_error(std::string(what) + " cannot be traced");
}
// Bytes from the first value of a tensor with values to behind its last
int64_t reach_of(const Tensor& t) {
  int64_t reach = 1;
  for (int64_t d = 0; d < t.dim(); ++d) reach += (t.size(d) - 1) * t.stride(d);
  return reach * static_cast<int64_t>(t.element_size());
}
// No operator has a forward-mode derivative; without this a dual tensor that needs no
// gradient would lose its tangent.  (Also under no_grad, which leaves that mode on.)
void refuse_tangents(const char* what, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if (t && t->_fw_grad(0).defined())
      throw std::runtime_error(std::string(what) + " has no forward-mode derivative");
}
void refuse_tangents(const char* what, const Tensors& tensors) {
  for (const Tensor& t : tensors) refuse_tangents(what, {&t});
}
// The same for calls without a backward: a graph must not end in them unnoticed.
void refuse_gradients(const char* what, std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : tensors)
    if (t && t->requires_grad())
      throw std::runtime_error(std::string(what) + " has no backward, and one of its tensors requires grad: call it "
                               "under torch.no_grad() or on detached tensors");
}
void refuse_gradients(const char* what, const Tensors& tensors) {
  for (const Tensor& t : tensors) refuse_gradients(what, {&t});
}
const Tensor* pointer(const optional<Tensor>& t) { return t ? &*t : nullptr; }
// Tensors that a call writes through their addresses: a backward that has saved one
// must find that it is no longer what it was.  (Before the launch: torch refuses
// inference tensors here, as in its own in-place operators.)
void mark_written(const Tensors& tensors) {
  for (const Tensor& t : tensors) t.unsafeGetTensorImpl()->bump_version();
}

}  // namespace

// The operators of a linear attention block (native_block.cpp)
void bind_block(pybind11::module_& m);

#endif  // SPARC_NATIVE_H
