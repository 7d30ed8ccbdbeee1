// Refusal of tensors without memory of their own (fake tensors and other subclasses, tensors
// wrapped by a function transform): their data pointers are null or not what they stand for.
#pragma once

#include <torch/extension.h>

namespace nori {

inline void check_plain(const torch::Tensor& t, const char* what) {
  using c10::DispatchKey;
  constexpr c10::DispatchKeySet wrapped(
      {DispatchKey::Python, DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper, DispatchKey::Functionalize});
  TORCH_CHECK(!t.unsafeGetTensorImpl()->key_set().has_any(wrapped), what, ": a plain tensor expected, not a wrapped one");
}
inline void check_plain(const c10::optional<torch::Tensor>& t, const char* what) {
  if (t.has_value() && t->defined()) check_plain(*t, what);
}

// Whether two contiguous tensors share memory.
inline bool overlap(const torch::Tensor& a, const torch::Tensor& b) {
  const char *pa = static_cast<const char*>(a.const_data_ptr()), *pb = static_cast<const char*>(b.const_data_ptr());
  return pa < pb + b.nbytes() && pb < pa + a.nbytes();
}

}  // namespace nori
