// Refusal of tensors without memory of their own (fake tensors and other subclasses, tensors
// wrapped by a function transform): their data pointers are null or not what they stand for.
#pragma once

#include <torch/extension.h>

#include <algorithm>
#include <array>
#include <vector>

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

// Whether elements of two strided tensors share memory (other than by their ranges meeting: columns of one buffer
// side by side do not).  Looks for a place that both reach, stride by stride from the largest: where strides are
// nested, as views of a buffer have them, one or two steps each are left.  A layout that takes more than 10^5 steps
// counts as shared.  `self`: whether two elements of `a` do.
inline bool shares_memory(const torch::Tensor& a, const torch::Tensor& b, bool self = false) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const int64_t at = static_cast<const char*>(b.const_data_ptr()) - static_cast<const char*>(a.const_data_ptr());
  const int64_t ea = a.element_size(), eb = b.element_size();
  const auto span = [](const torch::Tensor& t) {
    int64_t last = 0;
    for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
    return (last + 1) * t.element_size();
  };
  if (at >= span(a) || -at >= span(b)) return false;
  struct Term {  // stride x, lo <= x <= hi
    int64_t stride, lo, hi;
  };
  std::vector<Term> terms;
  const auto add = [&](const torch::Tensor& t, int64_t down, int64_t up) {
    for (int64_t d = 0; d < t.dim(); ++d) {
      const int64_t most = t.size(d) - 1, stride = t.stride(d) * t.element_size();
      if (most == 0 || (stride == 0 && !self)) continue;
      auto same = std::find_if(terms.begin(), terms.end(), [&](const Term& x) { return !self && x.stride == stride; });
      if (same == terms.end()) same = terms.insert(terms.end(), Term{stride, 0, 0});
      same->lo -= down * most, same->hi += up * most;
    }
  };
  add(b, self ? 1 : 0, 1);  // (of itself: differences of two elements)
  if (!self) add(a, 1, 0);
  std::sort(terms.begin(), terms.end(), [](const Term& x, const Term& y) { return x.stride > y.stride; });
  // what the strides from k on can still add
  std::vector<std::array<int64_t, 2>> rest(terms.size() + 1, {0, 0});
  for (int64_t k = static_cast<int64_t>(terms.size()) - 1; k >= 0; --k)
    rest[k] = {rest[k + 1][0] + terms[k].stride * terms[k].lo, rest[k + 1][1] + terms[k].stride * terms[k].hi};
  int64_t steps = 0;
  // b's element starts less than eb before or ea behind a's
  const auto meet = [&](const auto& go, size_t k, int64_t r, bool moved) -> bool {
    if (k == terms.size()) return r > -eb && r < ea && (moved || !self);
    const Term& t = terms[k];
    int64_t lo = t.lo, hi = t.hi;
    if (t.stride > 0) {
      const auto floor_div = [&](int64_t n) { return n >= 0 ? n / t.stride : -((-n + t.stride - 1) / t.stride); };
      lo = std::max(lo, -floor_div(r + rest[k + 1][1] + eb - 1));
      hi = std::min(hi, floor_div(ea - 1 - r - rest[k + 1][0]));
    }
    for (int64_t x = lo; x <= hi; ++x)
      if (++steps > 100000 || go(go, k + 1, r + t.stride * x, moved || x != 0)) return true;
    return false;
  };
  return meet(meet, 0, self ? 0 : at, false);
}

}  // namespace nori
