// LayerNorm forward for rows of any width: fp32, bf16 or fp16 in, the same type or fp32 out
// (fp32 from 16-bit rows is what bf16 autocast asks of a norm: no cast pass before it),
// optional weight and bias, strided rows.  Memory bound: a row is read once and written once.
//
// Reference counterpart: model/layer.py:219-230, model/encoders.py:432-585 (torch LayerNorm).
#include "layer_norm.cuh"

namespace nori {
namespace ln {

template <typename T, typename U, int VEC, int TPR, int VPL>
__global__ void __launch_bounds__(kThreads) fwd_kernel(const T* __restrict__ x, int64_t ldx, int64_t R, int C,
                                                       const float* __restrict__ w, const float* __restrict__ b,
                                                       float eps, U* __restrict__ y, float* __restrict__ mean_out,
                                                       float* __restrict__ rstd_out) {
  constexpr int CH = VPL / VEC, RPB = kThreads / TPR;
  __shared__ float sh[32];
  const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const float inv_c = 1.f / static_cast<float>(C);
  int flip = 0;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * RPB; base < R; base += static_cast<int64_t>(gridDim.x) * RPB) {
    const int64_t row = base + g;
    const bool ok = row < R;
    float v[VPL];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int c = VEC * (t + TPR * j);
      if (ok && c < C) {
        load_vec<T, VEC>(x + row * ldx + c, v + VEC * j);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[VEC * j + i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) s += v[VEC * j + i];
    }
    const float mean = row_sum<TPR>(s, sh + flip * 16) * inv_c;
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      if (VEC * (t + TPR * j) < C) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          v[VEC * j + i] -= mean;
          ss += v[VEC * j + i] * v[VEC * j + i];
        }
      }
    }
    const float rstd = rsqrtf(row_sum<TPR>(ss, sh + flip * 16 + 8) * inv_c + eps);
    flip ^= 1;  // the other half of `sh`: this row's sums may still be read
    if (!ok) continue;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int c = VEC * (t + TPR * j);
      if (c < C) {
        float o[VEC], wv[VEC], bv[VEC];
        if (w != nullptr) load_vec<float, VEC>(w + c, wv);
        if (b != nullptr) load_vec<float, VEC>(b + c, bv);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          o[i] = v[VEC * j + i] * rstd;
          if (w != nullptr) o[i] *= wv[i];
          if (b != nullptr) o[i] += bv[i];
        }
        store_vec<U, VEC>(y + row * static_cast<int64_t>(C) + c, o);
      }
    }
    if (t == 0) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
  }
}

// Rows wider than the registers of a CTA: three passes over the row (the second and third
// hit L2 for all but the widest).
template <typename T, typename U>
__global__ void __launch_bounds__(kThreads) fwd_wide_kernel(const T* __restrict__ x, int64_t ldx, int64_t R, int C,
                                                            const float* __restrict__ w, const float* __restrict__ b,
                                                            float eps, U* __restrict__ y,
                                                            float* __restrict__ mean_out,
                                                            float* __restrict__ rstd_out) {
  __shared__ float sh[32];
  const float inv_c = 1.f / static_cast<float>(C);
  int flip = 0;
  for (int64_t row = blockIdx.x; row < R; row += gridDim.x) {
    const T* xr = x + row * ldx;
    float s = 0.f;
    for (int c = threadIdx.x; c < C; c += kThreads) s += to_f32<T>(xr[c]);
    const float mean = row_sum<kThreads>(s, sh + flip * 16) * inv_c;
    float ss = 0.f;
    for (int c = threadIdx.x; c < C; c += kThreads) {
      const float d = to_f32<T>(xr[c]) - mean;
      ss += d * d;
    }
    const float rstd = rsqrtf(row_sum<kThreads>(ss, sh + flip * 16 + 8) * inv_c + eps);
    flip ^= 1;
    for (int c = threadIdx.x; c < C; c += kThreads) {
      float o = (to_f32<T>(xr[c]) - mean) * rstd;
      if (w != nullptr) o *= w[c];
      if (b != nullptr) o += b[c];
      y[row * static_cast<int64_t>(C) + c] = from_f32<U>(o);
    }
    if (threadIdx.x == 0) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
  }
}

template <typename T, typename U, int VEC>
static void launch(const T* x, int64_t ldx, int64_t R, int C, const float* w, const float* b, float eps, U* y,
                   float* mean, float* rstd) {
  auto stream = at::cuda::getCurrentCUDAStream();
  const int64_t cap = 148 * 8;
#define NORI_LN_FWD(TPR, VPL)                                                                                       \
  fwd_kernel<T, U, VEC, TPR, VPL>                                                                                   \
      <<<static_cast<unsigned>(std::min<int64_t>((R + kThreads / TPR - 1) / (kThreads / TPR), cap)), kThreads, 0,  \
         stream>>>(x, ldx, R, C, w, b, eps, y, mean, rstd)
  if (C <= 64) NORI_LN_FWD(8, 8);
  else if (C <= 256) NORI_LN_FWD(32, 8);
  else if (C <= 512) NORI_LN_FWD(32, 16);
  else if (C <= 1024) NORI_LN_FWD(32, 32);
  else if (C <= 2048) NORI_LN_FWD(256, 8);
  else if (C <= 4096) NORI_LN_FWD(256, 16);
  else if (C <= kMaxRegCols) NORI_LN_FWD(256, 32);
  else
    fwd_wide_kernel<T, U><<<static_cast<unsigned>(std::min<int64_t>(R, cap)), kThreads, 0, stream>>>(
        x, ldx, R, C, w, b, eps, y, mean, rstd);
#undef NORI_LN_FWD
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

template <typename T, typename U>
static void run(const torch::Tensor& x, const float* w, const float* b, float eps, torch::Tensor& y,
                torch::Tensor& mean, torch::Tensor& rstd) {
  constexpr int VEC = sizeof(T) == 4 || sizeof(U) == 4 ? 4 : 8;  // 16-byte accesses of the wider type
  const T* xp = reinterpret_cast<const T*>(x.data_ptr());
  U* yp = reinterpret_cast<U*>(y.data_ptr());
  const int64_t R = x.size(0), C = x.size(1), ldx = x.stride(0);
  const bool vec = vec_ok(xp, ldx, C, sizeof(T), VEC) && vec_ok(yp, C, C, sizeof(U), VEC) &&
                   vec_ok(w, 0, C, 4, 4) && vec_ok(b, 0, C, 4, 4) &&
                   (VEC == 4 || (vec_ok(w, 0, C, 4, 8) && vec_ok(b, 0, C, 4, 8)));
  if (vec)
    launch<T, U, VEC>(xp, ldx, R, static_cast<int>(C), w, b, eps, yp, mean.data_ptr<float>(), rstd.data_ptr<float>());
  else
    launch<T, U, 1>(xp, ldx, R, static_cast<int>(C), w, b, eps, yp, mean.data_ptr<float>(), rstd.data_ptr<float>());
}

}  // namespace ln

// (y [R, C], mean [R], rstd [R]) of x [R, C]; y has x's type, or fp32 with out_f32.
std::vector<torch::Tensor> layer_norm_fwd(const torch::Tensor& x, const c10::optional<torch::Tensor>& w,
                                          const c10::optional<torch::Tensor>& b, double eps, bool out_f32) {
  using namespace ln;
  check_rows(x, "layer_norm_fwd: x");
  TORCH_CHECK(eps >= 0.0, "layer_norm_fwd: eps must not be negative");
  const float* wp = opt_vec(w, x.size(1), x.device(), "layer_norm_fwd: weight");
  const float* bp = opt_vec(b, x.size(1), x.device(), "layer_norm_fwd: bias");
  const at::cuda::CUDAGuard guard(x.device());
  auto y = torch::empty({x.size(0), x.size(1)}, x.options().dtype(out_f32 ? at::kFloat : x.scalar_type()));
  auto mean = torch::empty({x.size(0)}, x.options().dtype(at::kFloat));
  auto rstd = torch::empty({x.size(0)}, x.options().dtype(at::kFloat));
  if (x.size(0) == 0) return {y, mean, rstd};
  const float e = static_cast<float>(eps);
  if (x.scalar_type() == at::kFloat)
    run<float, float>(x, wp, bp, e, y, mean, rstd);
  else if (x.scalar_type() == at::kBFloat16)
    out_f32 ? run<__nv_bfloat16, float>(x, wp, bp, e, y, mean, rstd)
            : run<__nv_bfloat16, __nv_bfloat16>(x, wp, bp, e, y, mean, rstd);
  else
    out_f32 ? run<__half, float>(x, wp, bp, e, y, mean, rstd) : run<__half, __half>(x, wp, bp, e, y, mean, rstd);
  return {y, mean, rstd};
}

}  // namespace nori
