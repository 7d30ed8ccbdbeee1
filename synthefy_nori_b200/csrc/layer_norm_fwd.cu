// LayerNorm forward for rows of any width: fp32, bf16 or fp16 in, the same type or fp32 out
// (fp32 from 16-bit rows is what bf16 autocast asks of a norm: no cast pass before it),
// optional weight and bias, strided rows.  Memory bound: a row is read once and written once.
// 403200 x 448 bf16 to fp32 in 187 - 204 us, 82 - 89% of the device's copy rate.  24 warps an SM with two
// rows each did better than 32 with spilled registers or 40 with one (143, 166, 149 us bf16 to
// bf16) and than one row with the next one's loads held in registers (189).
//
// Reference counterpart: model/layer.py:219-230, model/encoders.py:432-585 (torch LayerNorm).
#include "layer_norm.cuh"

namespace nori {
namespace ln {

template <typename T, typename U, typename W, int VEC, int TPR>
__global__ void __launch_bounds__(kCta<TPR>, 768 / kCta<TPR>) fwd_kernel(const T* __restrict__ x, int64_t ldx, int64_t R, int C,
                                                        const W* __restrict__ w, const W* __restrict__ b,
                                                        float eps, U* __restrict__ y, float* __restrict__ mean_out,
                                                        float* __restrict__ rstd_out) {
  constexpr int CH = kValues / VEC, RPB = kCta<TPR> / TPR;
  __shared__ float sh[2][2][16];
  const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const float inv_c = 1.f / static_cast<float>(C);
  int flip = 0;
  // a CTA's rows: 2 RPB neighbours, RPB apart within a group
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * (2 * RPB); base < R;
       base += static_cast<int64_t>(gridDim.x) * (2 * RPB)) {
    const int64_t row = base + g, ahead = row + static_cast<int64_t>(gridDim.x) * (2 * RPB) + t * RPB;
    if (t < 2 && ahead < R) prefetch_row(x + ahead * ldx, C);
    float v[2][kValues], s[2] = {0.f, 0.f}, mean[2], rstd[2];
    {
      Row<T, VEC, TPR> r[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) r[k].load(x, ldx, row + k * RPB, R, C, t);
#pragma unroll
      for (int k = 0; k < 2; ++k) r[k].values(v[k]);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) s[k] = pairwise_sum(v[k]);
    row_sum<TPR, 2>(s, sh, flip);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      mean[k] = s[k] * inv_c;
      s[k] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      if (VEC * (t + TPR * j) < C) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if constexpr (VEC > 1) {
            const F2 m = f2(-mean[k], -mean[k]);
            F2 ss = f2(0.f, 0.f);
#pragma unroll
            for (int i = VEC * j; i < VEC * (j + 1); i += 2) {
              const F2 d = add2(f2(v[k][i], v[k][i + 1]), m);
              ss = fma2(d, d, ss);
              unpack(d, v[k][i], v[k][i + 1]);
            }
            float lo, hi;
            unpack(ss, lo, hi);
            s[k] += lo + hi;
          } else {
            v[k][j] -= mean[k];
            s[k] += v[k][j] * v[k][j];
          }
        }
      }
    }
    row_sum<TPR, 2>(s, sh, flip);
#pragma unroll
    for (int k = 0; k < 2; ++k) rstd[k] = rsqrtf(s[k] * inv_c + eps);
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int c = VEC * (t + TPR * j);
      if (c < C) {
        float wv[VEC], bv[VEC];
        load_columns<VEC, W>(w, c, 1.f, wv);
        load_columns<VEC, W>(b, c, 0.f, bv);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (row + k * RPB < R) {
            float o[VEC];
            if constexpr (VEC > 1) {
              const F2 r = f2(rstd[k], rstd[k]);
#pragma unroll
              for (int i = 0; i < VEC; i += 2)
                unpack(fma2(mul2(f2(v[k][VEC * j + i], v[k][VEC * j + i + 1]), r), f2(wv[i], wv[i + 1]),
                            f2(bv[i], bv[i + 1])),
                       o[i], o[i + 1]);
            } else {
              o[0] = v[k][j] * rstd[k] * wv[0] + bv[0];
            }
            store_vec<U, VEC>(y + (row + k * RPB) * static_cast<int64_t>(C) + c, o);
          }
        }
      }
    }
    if (t == 0) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (row + k * RPB < R) {
          mean_out[row + k * RPB] = mean[k];
          rstd_out[row + k * RPB] = rstd[k];
        }
      }
    }
  }
}

// Rows wider than the registers of a CTA: three passes over the row (the second and third
// hit L2 for all but the widest).
template <typename T, typename U, typename W>
__global__ void __launch_bounds__(512) fwd_wide_kernel(const T* __restrict__ x, int64_t ldx, int64_t R, int C,
                                                       const W* __restrict__ w, const W* __restrict__ b,
                                                       float eps, U* __restrict__ y, float* __restrict__ mean_out,
                                                       float* __restrict__ rstd_out) {
  __shared__ float sh[2][1][16];
  const float inv_c = 1.f / static_cast<float>(C);
  int flip = 0;
  for (int64_t row = blockIdx.x; row < R; row += gridDim.x) {
    const T* xr = x + row * ldx;
    float s[1] = {0.f};
    for (int c = threadIdx.x; c < C; c += 512) s[0] += to_f32<T>(xr[c]);
    row_sum<512, 1>(s, sh, flip);
    const float mean = s[0] * inv_c;
    s[0] = 0.f;
    for (int c = threadIdx.x; c < C; c += 512) {
      const float d = to_f32<T>(xr[c]) - mean;
      s[0] += d * d;
    }
    row_sum<512, 1>(s, sh, flip);
    const float rstd = rsqrtf(s[0] * inv_c + eps);
    for (int c = threadIdx.x; c < C; c += 512) {
      float o = (to_f32<T>(xr[c]) - mean) * rstd;
      if (w != nullptr) o *= to_f32<W>(w[c]);
      if (b != nullptr) o += to_f32<W>(b[c]);
      y[row * static_cast<int64_t>(C) + c] = from_f32<U>(o);
    }
    if (threadIdx.x == 0) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
  }
}

template <typename T, typename U, typename W, int VEC>
static void launch(const T* x, int64_t ldx, int64_t R, int C, const W* w, const W* b, float eps, U* y,
                   float* mean, float* rstd) {
  auto stream = at::cuda::getCurrentCUDAStream();
  const int64_t sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
#define NORI_LN_FWD(TPR)                                                                                            \
  fwd_kernel<T, U, W, VEC, TPR>                                                                                        \
      <<<static_cast<unsigned>(std::min<int64_t>((R + 2 * kCta<TPR> / TPR - 1) / (2 * kCta<TPR> / TPR),            \
                                                 sms * (768 / kCta<TPR>))),                                      \
         kCta<TPR>, 0, stream>>>(x, ldx, R, C, w, b, eps, y, mean, rstd)
  if (C <= 128) NORI_LN_FWD(8);
  else if (C <= 512) NORI_LN_FWD(32);
  else if (C <= 2048) NORI_LN_FWD(128);
  else if (C <= kMaxRegCols) NORI_LN_FWD(512);
  else
    fwd_wide_kernel<T, U, W><<<static_cast<unsigned>(std::min<int64_t>(R, sms * 4)), 512, 0, stream>>>(
        x, ldx, R, C, w, b, eps, y, mean, rstd);
#undef NORI_LN_FWD
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

template <typename T, typename U, typename W>
static void run(const torch::Tensor& x, const Affine& a, float eps, torch::Tensor& y, torch::Tensor& mean,
                torch::Tensor& rstd) {
  constexpr int VEC = sizeof(T) == 4 || sizeof(U) == 4 ? 4 : 8;  // 16-byte accesses of the wider type
  const T* xp = reinterpret_cast<const T*>(x.data_ptr());
  U* yp = reinterpret_cast<U*>(y.data_ptr());
  const W *w = static_cast<const W*>(a.wp()), *b = static_cast<const W*>(a.bp());
  const int64_t R = x.size(0), C = x.size(1), ldx = x.stride(0);
  const bool vec = vec_ok(xp, ldx, C, sizeof(T), VEC) && vec_ok(yp, C, C, sizeof(U), VEC) &&
                   vec_ok_columns<W>(w, C, VEC) && vec_ok_columns<W>(b, C, VEC);
  if (vec)
    launch<T, U, W, VEC>(xp, ldx, R, static_cast<int>(C), w, b, eps, yp, mean.data_ptr<float>(), rstd.data_ptr<float>());
  else
    launch<T, U, W, 1>(xp, ldx, R, static_cast<int>(C), w, b, eps, yp, mean.data_ptr<float>(), rstd.data_ptr<float>());
}
template <typename T>
static void run_half(const torch::Tensor& x, const Affine& a, float eps, bool out_f32, torch::Tensor& y,
                     torch::Tensor& mean, torch::Tensor& rstd) {
  if (out_f32)
    a.f32 ? run<T, float, float>(x, a, eps, y, mean, rstd) : run<T, float, T>(x, a, eps, y, mean, rstd);
  else
    a.f32 ? run<T, T, float>(x, a, eps, y, mean, rstd) : run<T, T, T>(x, a, eps, y, mean, rstd);
}

}  // namespace ln

// (y [R, C], mean [R], rstd [R]) of x [R, C]; y has x's type, or fp32 with out_f32.  Weight and bias
// are read as they are in fp32 or in x's type, and cast to fp32 otherwise.
std::vector<torch::Tensor> layer_norm_fwd(const torch::Tensor& x, const c10::optional<torch::Tensor>& w,
                                          const c10::optional<torch::Tensor>& b, double eps, bool out_f32) {
  using namespace ln;
  check_rows(x, "layer_norm_fwd: x");
  TORCH_CHECK(eps >= 0.0, "layer_norm_fwd: eps must not be negative");
  const at::cuda::CUDAGuard guard(x.device());
  const Affine a = affine_of(x, w, b, "layer_norm_fwd");
  auto y = torch::empty({x.size(0), x.size(1)}, x.options().dtype(out_f32 ? at::kFloat : x.scalar_type()));
  auto mean = torch::empty({x.size(0)}, x.options().dtype(at::kFloat));
  auto rstd = torch::empty({x.size(0)}, x.options().dtype(at::kFloat));
  check_plain(y, "layer_norm_fwd");  // (a real x under a mode that makes fake tensors)
  if (x.size(0) == 0) return {y, mean, rstd};
  const float e = static_cast<float>(eps);
  if (x.scalar_type() == at::kFloat)
    run<float, float, float>(x, a, e, y, mean, rstd);
  else if (x.scalar_type() == at::kBFloat16)
    run_half<__nv_bfloat16>(x, a, e, out_f32, y, mean, rstd);
  else
    run_half<__half>(x, a, e, out_f32, y, mean, rstd);
  return {y, mean, rstd};
}

}  // namespace nori
