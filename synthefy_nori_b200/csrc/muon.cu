// Entry points of the Muon operators: which matrices run in one CTA each and which over the
// whole GPU, and the checks of the arguments.
#include "muon.cuh"

#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <c10/cuda/CUDAStream.h>

#include <cmath>

namespace nori {
namespace muon {

constexpr int64_t kMaxDim = 1 << 20;

static Coeffs make_coeffs(int64_t steps, double eps, const std::vector<double>& c, const char* who) {
  TORCH_CHECK(steps >= 1 && steps <= 64, who, ": steps must be in 1..64");
  TORCH_CHECK(eps >= 0.0, who, ": eps must not be negative");
  // below 1 the small directions shrink from step to step and the iterate's scale has no bound
  TORCH_CHECK(c.size() == 3 && c[0] >= 1.0 && c[0] <= 1024.0 && std::isfinite(c[1]) && std::isfinite(c[2]), who,
              ": three finite coefficients, the first in 1..1024, expected");
  return {static_cast<int>(steps), static_cast<float>(eps), static_cast<float>(c[0]), static_cast<float>(c[1] / c[0]),
          static_cast<float>(c[2] / c[0])};
}

static const float* opt_scalar(const c10::optional<torch::Tensor>& t, const torch::Device& dev, const char* what) {
  if (!t.has_value() || !t->defined()) return nullptr;
  TORCH_CHECK(t->device() == dev && t->scalar_type() == at::kFloat && t->numel() == 1, what,
              ": one fp32 value on the same device expected");
  return t->data_ptr<float>();
}

}  // namespace muon

// Newton-Schulz of every matrix of contiguous g [.., rows, cols] (fp32, bf16 or fp16), into
// `out` (contiguous, of g's shape) or a new tensor of `out_type`.
torch::Tensor newton_schulz(const torch::Tensor& g, const c10::optional<torch::Tensor>& out_opt,
                            c10::optional<c10::ScalarType> out_type, int64_t steps, double eps,
                            std::vector<double> coeffs, const torch::Tensor& status) {
  using namespace muon;
  check_plain(g, "newton_schulz");
  TORCH_CHECK(g.is_cuda() && g.dim() >= 2 && g.is_contiguous(), "newton_schulz: contiguous CUDA [.., rows, cols]");
  auto kind = [](c10::ScalarType s, const char* what) {
    TORCH_CHECK(s == at::kFloat || s == at::kBFloat16 || s == at::kHalf, "newton_schulz: ", what,
                " must be fp32, bf16 or fp16");
    return s == at::kFloat ? 0 : s == at::kBFloat16 ? 1 : 2;
  };
  const Coeffs k = make_coeffs(steps, eps, coeffs, "newton_schulz");
  const int src = kind(g.scalar_type(), "g");
  const int64_t rows = g.size(-2), cols = g.size(-1);
  TORCH_CHECK(rows < kMaxDim && cols < kMaxDim, "newton_schulz: at most 2^20 rows and columns");
  const at::cuda::CUDAGuard guard(g.device());
  torch::Tensor out = out_opt.has_value() && out_opt->defined()
                          ? *out_opt
                          : torch::empty(g.sizes(), g.options().dtype(out_type.value_or(g.scalar_type())));
  check_plain(out, "newton_schulz: out");
  TORCH_CHECK(out.device() == g.device() && out.is_contiguous() && out.sizes() == g.sizes(),
              "newton_schulz: out must be contiguous, of g's shape and device");
  const int dst = kind(out.scalar_type(), "out");
  // matrix i is written while others are still read: in place, or apart
  TORCH_CHECK((out.const_data_ptr() == g.const_data_ptr() && dst == src) || !overlap(out, g),
              "newton_schulz: out must be g itself or share no memory with it");
  if (g.numel() == 0) return out;
  const int64_t batch = g.numel() / (rows * cols);
  TORCH_CHECK(batch <= INT_MAX, "newton_schulz: at most 2^31 - 1 matrices");
  const Fit fit = single_fit(static_cast<int>(rows), static_cast<int>(cols));
  if (fit.ok)
    run_single(src, g.data_ptr(), dst, out.data_ptr(), StepArgs{}, 0, batch, static_cast<int>(rows),
               static_cast<int>(cols), fit.smem, k, status);
  else
    run_large(src, g.data_ptr(), dst, out.data_ptr(), StepArgs{},
              {Shape{0, batch, static_cast<int>(rows), static_cast<int>(cols)}}, k, status, g.options(),
              nullptr);
  return out;
}

// One Muon step on the matrices of a plan: `table` [count, 4] int64 on the device (offset in
// the flat buffers, offset in the momentum buffer, rows, cols), `groups` (first, count, rows,
// cols) runs of equal shape in it.
void muon_step(torch::Tensor& data, const torch::Tensor& grad, torch::Tensor& mom,
               const c10::optional<torch::Tensor>& ema, const torch::Tensor& table, std::vector<int64_t> groups,
               double lr, double wd, double momentum, bool nesterov, int64_t steps, double eps,
               std::vector<double> coeffs, int64_t adjust, const c10::optional<torch::Tensor>& norm_sq,
               double max_norm, const c10::optional<torch::Tensor>& skip, double ema_decay,
               const torch::Tensor& status) {
  using namespace muon;
  for (const auto& t : {data, grad, mom, table, status}) check_plain(t, "muon_step");
  for (const auto& t : {ema, norm_sq, skip}) check_plain(t, "muon_step");
  for (const torch::Tensor* t : std::initializer_list<const torch::Tensor*>{&data, &grad, &mom})
    TORCH_CHECK(t->is_cuda() && t->device() == data.device() && t->scalar_type() == at::kFloat && t->dim() == 1 &&
                    t->is_contiguous(),
                "muon_step: flat contiguous fp32 buffers on one CUDA device expected");
  TORCH_CHECK(grad.numel() == data.numel(), "muon_step: data and grad must have the same length");
  TORCH_CHECK(table.device() == data.device() && table.scalar_type() == at::kLong && table.is_contiguous(),
              "muon_step: the plan is on another device than the parameters");
  const Coeffs k = make_coeffs(steps, eps, coeffs, "muon_step");
  StepArgs s{};
  s.data = data.data_ptr<float>();
  s.grad = grad.data_ptr<float>();
  s.mom = mom.data_ptr<float>();
  if (ema.has_value() && ema->defined()) {
    TORCH_CHECK(ema->device() == data.device() && ema->scalar_type() == at::kFloat && ema->dim() == 1 &&
                    ema->is_contiguous() && ema->numel() == data.numel(),
                "muon_step: ema must be a flat fp32 buffer of data's length");
    s.ema = ema->data_ptr<float>();
  }
  const torch::Tensor* written[3] = {&data, &mom, s.ema != nullptr ? &*ema : nullptr};
  for (int i = 0; i < 3; ++i) {
    if (written[i] == nullptr) continue;
    bool shared = overlap(*written[i], grad);
    for (int j = 0; j < i; ++j) shared = shared || overlap(*written[i], *written[j]);
    TORCH_CHECK(!shared, "muon_step: data, grad, momentum and ema must not share memory");
  }
  s.table = reinterpret_cast<const Mat*>(table.data_ptr<int64_t>());
  s.norm_sq = opt_scalar(norm_sq, data.device(), "muon_step: norm_sq");
  s.skip = opt_scalar(skip, data.device(), "muon_step: skip");
  if (!(max_norm > 0.0)) s.norm_sq = nullptr;
  s.lr = static_cast<float>(lr);
  s.wd = static_cast<float>(wd);
  s.momentum = static_cast<float>(momentum);
  s.max_norm = static_cast<float>(max_norm);
  s.ema_w = static_cast<float>(1.0 - ema_decay);
  s.nesterov = nesterov ? 1 : 0;
  s.adjust = static_cast<int>(adjust);
  const at::cuda::CUDAGuard guard(data.device());
  // the matrices that fit one CTA each in one launch (a plan keeps them together), the others
  // over the whole GPU, in one launch as well
  std::vector<Shape> large;
  int64_t run_first = 0, run_count = 0;
  int run_smem = 0;
  auto flush = [&]() {
    if (run_count > 0)
      run_single(kSrcMuon, nullptr, kOutMuon, nullptr, s, run_first, run_count, 0, 0, run_smem, k, status);
    run_count = 0;
    run_smem = 0;
  };
  for (size_t i = 0; i + 3 < groups.size(); i += 4) {
    const int rows = static_cast<int>(groups[i + 2]), cols = static_cast<int>(groups[i + 3]);
    const Fit fit = single_fit(rows, cols);
    if (!fit.ok) {
      large.push_back(Shape{groups[i], groups[i + 1], rows, cols});
      continue;
    }
    if (run_count > 0 && groups[i] != run_first + run_count) flush();
    if (run_count == 0) run_first = groups[i];
    run_count += groups[i + 1];
    run_smem = std::max(run_smem, fit.smem);
  }
  if (large.empty()) {
    flush();
    return;
  }
  auto whole = [&](at::cuda::CUDAEvent* ready) {
    run_large(kSrcMuon, nullptr, kOutMuon, nullptr, s, large, k, status, data.options(), ready);
  };
  if (run_count == 0 || at::cuda::currentStreamCaptureStatusMayInitCtx() != at::cuda::CaptureStatus::None) {
    whole(nullptr);
    flush();
    return;
  }
  // The two sets touch different matrices, and the products of the large ones, a chain that
  // seldom fills the GPU, need all their CTAs at once: they start first, the single CTAs beside
  // them on another stream.  (Not under capture, where a stream of the pool could belong to
  // someone else.)
  const auto main = at::cuda::getCurrentCUDAStream();
  const auto side = at::cuda::getStreamFromPool(false, data.get_device());
  at::cuda::CUDAEvent ready, join;
  whole(&ready);
  ready.block(side);
  {
    c10::cuda::CUDAStreamGuard on(side);
    flush();
  }
  join.record(side);
  join.block(main);
}

// Whether a matrix of this shape runs its whole step in one CTA.
bool muon_single_cta(int64_t rows, int64_t cols) {
  return muon::single_fit(static_cast<int>(rows), static_cast<int>(cols)).ok;
}

}  // namespace nori
