// LayerNorm backward: the row gradient and the reduction of the weight's and bias's gradients.
//
//   q = dy w,  xhat = (x - mean) rstd
//   dx = rstd (q - mean(q) - xhat mean(q xhat));  dw = sum_rows dy xhat;  db = sum_rows dy
//
// One pass over x and dy: each thread keeps the sums of its own columns over all rows that it
// visits in fp32 registers; a CTA adds its row groups in a fixed order and writes one partial
// row, and a second kernel adds the partial rows in a fixed order.  No atomics: the same
// inputs give the same bits.
//
// Reference counterpart: torch LayerNorm's autograd (model/layer.py:219-230).
#include "layer_norm.cuh"

namespace nori {
namespace ln {

template <typename T, typename U, int VEC, int TPR, int VPL>
__global__ void __launch_bounds__(kThreads)
    bwd_kernel(const U* __restrict__ dy, int64_t ldy, const T* __restrict__ x, int64_t ldx, int64_t R, int C,
               const float* __restrict__ mean_in, const float* __restrict__ rstd_in, const float* __restrict__ w,
               T* __restrict__ dx, float* __restrict__ part_w, float* __restrict__ part_b) {
  constexpr int CH = VPL / VEC, RPB = kThreads / TPR;
  extern __shared__ float acc_sh[];  // [RPB][C] when a CTA holds several row groups
  __shared__ float sh[32];
  const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const float inv_c = 1.f / static_cast<float>(C);
  float gw[VPL], gb[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) gw[i] = gb[i] = 0.f;
  int flip = 0;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * RPB; base < R; base += static_cast<int64_t>(gridDim.x) * RPB) {
    const int64_t row = base + g;
    const bool ok = row < R;
    const float mean = ok ? mean_in[row] : 0.f, rstd = ok ? rstd_in[row] : 0.f;
    float h[VPL], q[VPL];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int c = VEC * (t + TPR * j);
      if (ok && c < C) {
        load_vec<T, VEC>(x + row * ldx + c, h + VEC * j);
        load_vec<U, VEC>(dy + row * ldy + c, q + VEC * j);
        float wv[VEC];
        if (w != nullptr) load_vec<float, VEC>(w + c, wv);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const int k = VEC * j + i;
          h[k] = (h[k] - mean) * rstd;
          gw[k] += q[k] * h[k];
          gb[k] += q[k];
          if (w != nullptr) q[k] *= wv[i];
          s1 += q[k];
          s2 += q[k] * h[k];
        }
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) h[VEC * j + i] = q[VEC * j + i] = 0.f;
      }
    }
    s1 = row_sum<TPR>(s1, sh + flip * 16) * inv_c;
    s2 = row_sum<TPR>(s2, sh + flip * 16 + 8) * inv_c;
    flip ^= 1;
    if (!ok) continue;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int c = VEC * (t + TPR * j);
      if (c < C) {
        float o[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = rstd * (q[VEC * j + i] - s1 - h[VEC * j + i] * s2);
        store_vec<T, VEC>(dx + row * static_cast<int64_t>(C) + c, o);
      }
    }
  }
  // this CTA's partial rows
  for (int pass = 0; pass < 2; ++pass) {
    float* out = pass == 0 ? part_w : part_b;
    if (out == nullptr) continue;
    out += static_cast<int64_t>(blockIdx.x) * C;
    if constexpr (RPB == 1) {
#pragma unroll
      for (int k = 0; k < VPL; ++k) {
        const int c = VEC * (t + TPR * (k / VEC)) + k % VEC;
        if (c < C) out[c] = pass == 0 ? gw[k] : gb[k];
      }
    } else {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < VPL; ++k) {
        const int c = VEC * (t + TPR * (k / VEC)) + k % VEC;
        if (c < C) acc_sh[g * C + c] = pass == 0 ? gw[k] : gb[k];
      }
      __syncthreads();
      for (int c = threadIdx.x; c < C; c += kThreads) {
        float s = 0.f;
        for (int i = 0; i < RPB; ++i) s += acc_sh[i * C + c];
        out[c] = s;
      }
    }
  }
}

// Rows wider than the registers of a CTA: dx in two passes over the row ...
template <typename T, typename U>
__global__ void __launch_bounds__(kThreads)
    bwd_wide_kernel(const U* __restrict__ dy, int64_t ldy, const T* __restrict__ x, int64_t ldx, int64_t R, int C,
                    const float* __restrict__ mean_in, const float* __restrict__ rstd_in, const float* __restrict__ w,
                    T* __restrict__ dx) {
  __shared__ float sh[32];
  const float inv_c = 1.f / static_cast<float>(C);
  int flip = 0;
  for (int64_t row = blockIdx.x; row < R; row += gridDim.x) {
    const float mean = mean_in[row], rstd = rstd_in[row];
    const T* xr = x + row * ldx;
    const U* dyr = dy + row * ldy;
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < C; c += kThreads) {
      const float q = to_f32<U>(dyr[c]) * (w != nullptr ? w[c] : 1.f);
      s1 += q;
      s2 += q * ((to_f32<T>(xr[c]) - mean) * rstd);
    }
    s1 = row_sum<kThreads>(s1, sh + flip * 16) * inv_c;
    s2 = row_sum<kThreads>(s2, sh + flip * 16 + 8) * inv_c;
    flip ^= 1;
    for (int c = threadIdx.x; c < C; c += kThreads) {
      const float q = to_f32<U>(dyr[c]) * (w != nullptr ? w[c] : 1.f);
      const float h = (to_f32<T>(xr[c]) - mean) * rstd;
      dx[row * static_cast<int64_t>(C) + c] = from_f32<T>(rstd * (q - s1 - h * s2));
    }
  }
}

// ... and the column sums by a pass down the columns: 32 columns x 8 row lanes per CTA, one
// partial row per blockIdx.y.
template <typename T, typename U>
__global__ void __launch_bounds__(kThreads)
    colgrad_kernel(const U* __restrict__ dy, int64_t ldy, const T* __restrict__ x, int64_t ldx, int64_t R, int C,
                   const float* __restrict__ mean_in, const float* __restrict__ rstd_in, float* __restrict__ part_w,
                   float* __restrict__ part_b) {
  __shared__ float sw[8][33], sb[8][33];
  const int lane = threadIdx.x % 32, ry = threadIdx.x / 32;
  const int c = blockIdx.x * 32 + lane;
  const int64_t per = (R + gridDim.y - 1) / gridDim.y;
  const int64_t r0 = blockIdx.y * per, r1 = min(R, r0 + per);
  float gw = 0.f, gb = 0.f;
  if (c < C) {
    for (int64_t r = r0 + ry; r < r1; r += 8) {
      const float d = to_f32<U>(dy[r * ldy + c]);
      gw += d * ((to_f32<T>(x[r * ldx + c]) - mean_in[r]) * rstd_in[r]);
      gb += d;
    }
  }
  sw[ry][lane] = gw;
  sb[ry][lane] = gb;
  __syncthreads();
  if (ry == 0 && c < C) {
    float a = 0.f, e = 0.f;
    for (int i = 0; i < 8; ++i) {
      a += sw[i][lane];
      e += sb[i][lane];
    }
    if (part_w != nullptr) part_w[static_cast<int64_t>(blockIdx.y) * C + c] = a;
    if (part_b != nullptr) part_b[static_cast<int64_t>(blockIdx.y) * C + c] = e;
  }
}

// out[c] = sum_p part[p][c], in a fixed order: 32 columns x 8 partial lanes per CTA; blockIdx.y
// picks the weight's or the bias's sums.
__global__ void __launch_bounds__(kThreads) reduce_kernel(const float* __restrict__ part_w,
                                                          const float* __restrict__ part_b, int P, int C,
                                                          float* __restrict__ dw, float* __restrict__ db) {
  __shared__ float sh[8][33];
  const float* part = blockIdx.y == 0 ? part_w : part_b;
  float* out = blockIdx.y == 0 ? dw : db;
  if (out == nullptr) return;
  const int lane = threadIdx.x % 32, py = threadIdx.x / 32;
  const int c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < C)
    for (int p = py; p < P; p += 8) s += part[static_cast<int64_t>(p) * C + c];
  sh[py][lane] = s;
  __syncthreads();
  if (py == 0 && c < C) {
    float a = 0.f;
    for (int i = 0; i < 8; ++i) a += sh[i][lane];
    out[c] = a;
  }
}

struct BwdArgs {
  int64_t ldy, ldx, R;
  int C;
  const float *mean, *rstd, *w;
  bool want_w, want_b;
};

template <typename T, typename U, int VEC>
static void launch(const U* dy, const T* x, T* dx, const BwdArgs& a, torch::Tensor& dw, torch::Tensor& db) {
  auto stream = at::cuda::getCurrentCUDAStream();
  const int C = a.C;
  const int tpr = C <= 64 ? 8 : C <= 1024 ? 32 : 256, rpb = kThreads / tpr;
  const bool wide = C > kMaxRegCols;
  const int64_t cap = 148 * 2;
  const int P = static_cast<int>(wide ? std::min<int64_t>(16, (a.R + 63) / 64)
                                      : std::min<int64_t>(cap, (a.R + rpb - 1) / rpb));
  const bool grads = a.want_w || a.want_b;
  torch::Tensor part;
  float *pw = nullptr, *pb = nullptr;
  if (grads) {
    part = torch::empty({2, P, C}, dw.options());
    pw = a.want_w ? part.data_ptr<float>() : nullptr;
    pb = a.want_b ? part.data_ptr<float>() + static_cast<int64_t>(P) * C : nullptr;
  }
  const size_t smem = rpb > 1 && grads ? static_cast<size_t>(rpb) * C * sizeof(float) : 0;
#define NORI_LN_BWD(TPR, VPL)                                                                                  \
  bwd_kernel<T, U, VEC, TPR, VPL>                                                                              \
      <<<P, kThreads, smem, stream>>>(dy, a.ldy, x, a.ldx, a.R, C, a.mean, a.rstd, a.w, dx, pw, pb)
  if (C <= 64) NORI_LN_BWD(8, 8);
  else if (C <= 256) NORI_LN_BWD(32, 8);
  else if (C <= 512) NORI_LN_BWD(32, 16);
  else if (C <= 1024) NORI_LN_BWD(32, 32);
  else if (C <= 2048) NORI_LN_BWD(256, 8);
  else if (C <= 4096) NORI_LN_BWD(256, 16);
  else if (C <= kMaxRegCols) NORI_LN_BWD(256, 32);
  else {
    bwd_wide_kernel<T, U><<<static_cast<unsigned>(std::min<int64_t>(a.R, 148 * 8)), kThreads, 0, stream>>>(
        dy, a.ldy, x, a.ldx, a.R, C, a.mean, a.rstd, a.w, dx);
    if (grads) {
      C10_CUDA_KERNEL_LAUNCH_CHECK();
      colgrad_kernel<T, U><<<dim3((C + 31) / 32, P), kThreads, 0, stream>>>(dy, a.ldy, x, a.ldx, a.R, C, a.mean,
                                                                            a.rstd, pw, pb);
    }
  }
#undef NORI_LN_BWD
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (grads) {
    reduce_kernel<<<dim3((C + 31) / 32, 2), kThreads, 0, stream>>>(pw, pb, P, C, a.want_w ? dw.data_ptr<float>() : nullptr,
                                                                   a.want_b ? db.data_ptr<float>() : nullptr);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
}

template <typename T, typename U>
static void run(const torch::Tensor& dy, const torch::Tensor& x, torch::Tensor& dx, const BwdArgs& a,
                torch::Tensor& dw, torch::Tensor& db) {
  constexpr int VEC = sizeof(T) == 4 || sizeof(U) == 4 ? 4 : 8;
  const U* dyp = reinterpret_cast<const U*>(dy.data_ptr());
  const T* xp = reinterpret_cast<const T*>(x.data_ptr());
  T* dxp = reinterpret_cast<T*>(dx.data_ptr());
  const bool vec = vec_ok(dyp, a.ldy, a.C, sizeof(U), VEC) && vec_ok(xp, a.ldx, a.C, sizeof(T), VEC) &&
                   vec_ok(dxp, a.C, a.C, sizeof(T), VEC) && vec_ok(a.w, 0, a.C, 4, VEC);
  if (vec)
    launch<T, U, VEC>(dyp, xp, dxp, a, dw, db);
  else
    launch<T, U, 1>(dyp, xp, dxp, a, dw, db);
}

}  // namespace ln

// (dx [R, C] of x's type, dw [C], db [C] fp32; an unwanted one is empty) from dy [R, C] (x's
// type or fp32), x and the forward's mean and rstd.
std::vector<torch::Tensor> layer_norm_bwd(const torch::Tensor& dy, const torch::Tensor& x, const torch::Tensor& mean,
                                          const torch::Tensor& rstd, const c10::optional<torch::Tensor>& w,
                                          bool weight_grad, bool bias_grad) {
  using namespace ln;
  check_rows(x, "layer_norm_bwd: x");
  check_rows(dy, "layer_norm_bwd: dy");
  TORCH_CHECK(dy.device() == x.device() && dy.sizes() == x.sizes(), "layer_norm_bwd: dy must be of x's shape and device");
  TORCH_CHECK(dy.scalar_type() == x.scalar_type() || dy.scalar_type() == at::kFloat,
              "layer_norm_bwd: dy must have x's type or fp32");
  const int64_t R = x.size(0), C = x.size(1);
  for (const torch::Tensor* t : std::initializer_list<const torch::Tensor*>{&mean, &rstd})
    TORCH_CHECK(t->device() == x.device() && t->scalar_type() == at::kFloat && t->is_contiguous() && t->numel() == R,
                "layer_norm_bwd: mean and rstd must be the forward's fp32 rows");
  BwdArgs a;
  a.w = opt_vec(w, C, x.device(), "layer_norm_bwd: weight");
  const at::cuda::CUDAGuard guard(x.device());
  auto f32 = x.options().dtype(at::kFloat);
  auto dx = torch::empty({R, C}, x.options());
  auto dw = weight_grad ? torch::empty({C}, f32) : torch::empty({0}, f32);
  auto db = bias_grad ? torch::empty({C}, f32) : torch::empty({0}, f32);
  if (R == 0) {
    dw.zero_();
    db.zero_();
    return {dx, dw, db};
  }
  a.ldy = dy.stride(0);
  a.ldx = x.stride(0);
  a.R = R;
  a.C = static_cast<int>(C);
  a.mean = mean.data_ptr<float>();
  a.rstd = rstd.data_ptr<float>();
  a.want_w = weight_grad;
  a.want_b = bias_grad;
  const bool f = dy.scalar_type() == at::kFloat;
  if (x.scalar_type() == at::kFloat)
    run<float, float>(dy, x, dx, a, dw, db);
  else if (x.scalar_type() == at::kBFloat16)
    f ? run<__nv_bfloat16, float>(dy, x, dx, a, dw, db) : run<__nv_bfloat16, __nv_bfloat16>(dy, x, dx, a, dw, db);
  else
    f ? run<__half, float>(dy, x, dx, a, dw, db) : run<__half, __half>(dy, x, dx, a, dw, db);
  return {dx, dw, db};
}

}  // namespace nori
