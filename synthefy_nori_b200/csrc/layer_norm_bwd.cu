// LayerNorm backward: the row gradient and the reduction of the weight's and bias's gradients.
//
//   q = dy w,  xhat = (x - mean) rstd
//   dx = rstd (q - mean(q) - xhat mean(q xhat));  dw = sum_rows dy xhat;  db = sum_rows dy
//
// One pass over x and dy: each thread keeps the sums of its own columns over all rows that it
// visits in fp32 registers; a CTA adds its row groups in a fixed order and writes one partial
// row, and a second kernel adds the partial rows in a fixed order.  Where the partial rows
// would be more traffic than reading x and dy (from L2) once more, the columns are summed by a
// pass of their own (257 x 8192 fp16, forward and backward: 39 us with partial rows, 22 with the pass).
// 403200 x 448 bf16 in 220 us against 167 at the copy rate: 16 warps an SM issue 2.3
// instructions a cycle.  No atomics: the same inputs give the same bits.
//
// Reference counterpart: torch LayerNorm's autograd (model/layer.py:219-230).
#include "layer_norm.cuh"

namespace nori {
namespace ln {

template <typename T, typename U, typename W, int VEC, int TPR, bool GRADS>
__global__ void __launch_bounds__(kCta<TPR>, 512 / kCta<TPR>)
    bwd_kernel(const U* __restrict__ dy, int64_t ldy, const T* __restrict__ x, int64_t ldx, int64_t R, int C,
               const float* __restrict__ mean_in, const float* __restrict__ rstd_in, const W* __restrict__ w,
               T* __restrict__ dx, float* __restrict__ part_w, float* __restrict__ part_b) {
  constexpr int CH = kValues / VEC, RPB = kCta<TPR> / TPR;
  extern __shared__ float acc_sh[];  // [RPB][C] where a CTA holds several row groups
  __shared__ float sh[2][4][16];
  const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
  const float inv_c = 1.f / static_cast<float>(C);
  int flip = 0;
  constexpr int H = kValues / 2;
  F2 gw[H], gb[H];
#pragma unroll
  for (int i = 0; i < H; ++i) gw[i] = gb[i] = f2(0.f, 0.f);
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * (2 * RPB); base < R;
       base += static_cast<int64_t>(gridDim.x) * (2 * RPB)) {
    const int64_t row = base + g, ahead = row + static_cast<int64_t>(gridDim.x) * (2 * RPB) + t % 2 * RPB;
    if (t < 4 && ahead < R) {
      if (t < 2)
        prefetch_row(x + ahead * ldx, C);
      else
        prefetch_row(dy + ahead * ldy, C);
    }
    F2 h[2][H], q[2][H];
    float s[4], rstd[2];
    {
      Row<T, VEC, TPR> rx[2];
      Row<U, VEC, TPR> ry[2];
      float mean[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        rx[k].load(x, ldx, row + k * RPB, R, C, t);
        ry[k].load(dy, ldy, row + k * RPB, R, C, t);
        mean[k] = row + k * RPB < R ? mean_in[row + k * RPB] : 0.f;
        rstd[k] = row + k * RPB < R ? rstd_in[row + k * RPB] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const F2 m = f2(-mean[k], -mean[k]), r = f2(rstd[k], rstd[k]);
        float vx[kValues], vy[kValues];
        rx[k].values(vx);
        ry[k].values(vy);
#pragma unroll
        for (int i = 0; i < H; ++i) {
          h[k][i] = mul2(add2(f2(vx[2 * i], vx[2 * i + 1]), m), r);
          q[k][i] = f2(vy[2 * i], vy[2 * i + 1]);
        }
      }
    }
    float wv[kValues];
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int c = VEC * (t + TPR * j);
      if (c < C) {
        load_columns<VEC, W>(w, c, 1.f, wv + VEC * j);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) wv[VEC * j + i] = 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {  // dy is 0 beyond the last row and column
      F2 s1 = f2(0.f, 0.f), s2 = f2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < H; ++i) {
        if constexpr (GRADS) {
          gw[i] = fma2(q[k][i], h[k][i], gw[i]);
          gb[i] = add2(gb[i], q[k][i]);
        }
        q[k][i] = mul2(q[k][i], f2(wv[2 * i], wv[2 * i + 1]));
        s1 = add2(s1, q[k][i]);
        s2 = fma2(q[k][i], h[k][i], s2);
      }
      float lo, hi;
      unpack(s1, lo, hi);
      s[2 * k] = lo + hi;
      unpack(s2, lo, hi);
      s[2 * k + 1] = lo + hi;
    }
    row_sum<TPR, 4>(s, sh, flip);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (row + k * RPB < R) {
        const float a1 = -s[2 * k] * inv_c, a2 = -s[2 * k + 1] * inv_c;
        const F2 n1 = f2(a1, a1), n2 = f2(a2, a2), r = f2(rstd[k], rstd[k]);
        float o[kValues];
#pragma unroll
        for (int i = 0; i < H; ++i)
          unpack(mul2(r, fma2(h[k][i], n2, add2(q[k][i], n1))), o[2 * i], o[2 * i + 1]);
        T* dxr = dx + (row + k * RPB) * static_cast<int64_t>(C);
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          const int c = VEC * (t + TPR * j);
          if (c < C) store_vec<T, VEC>(dxr + c, o + VEC * j);
        }
      }
    }
  }
  if constexpr (GRADS) {  // this CTA's partial rows
    for (int pass = 0; pass < 2; ++pass) {
      float* out = pass == 0 ? part_w : part_b;
      if (out == nullptr) continue;
      out += static_cast<int64_t>(blockIdx.x) * C;
      if constexpr (RPB > 1) __syncthreads();
#pragma unroll
      for (int k = 0; k < kValues; ++k) {
        const int c = VEC * (t + TPR * (k / VEC)) + k % VEC;
        float lo, hi;
        unpack(pass == 0 ? gw[k / 2] : gb[k / 2], lo, hi);
        if (c < C) (RPB > 1 ? acc_sh + g * C : out)[c] = k % 2 == 0 ? lo : hi;
      }
      if constexpr (RPB > 1) {
        __syncthreads();
        for (int c = threadIdx.x; c < C; c += kCta<TPR>) {
          float v = 0.f;
          for (int i = 0; i < RPB; ++i) v += acc_sh[i * C + c];
          out[c] = v;
        }
      }
    }
  }
}

// Rows wider than the registers of a CTA: dx in two passes over the row.
template <typename T, typename U, typename W>
__global__ void __launch_bounds__(512)
    bwd_wide_kernel(const U* __restrict__ dy, int64_t ldy, const T* __restrict__ x, int64_t ldx, int64_t R, int C,
                    const float* __restrict__ mean_in, const float* __restrict__ rstd_in, const W* __restrict__ w,
                    T* __restrict__ dx) {
  __shared__ float sh[2][2][16];
  const float inv_c = 1.f / static_cast<float>(C);
  int flip = 0;
  for (int64_t row = blockIdx.x; row < R; row += gridDim.x) {
    const float mean = mean_in[row], rstd = rstd_in[row];
    const T* xr = x + row * ldx;
    const U* dyr = dy + row * ldy;
    float s[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < C; c += 512) {
      const float q = to_f32<U>(dyr[c]) * (w != nullptr ? to_f32<W>(w[c]) : 1.f);
      s[0] += q;
      s[1] += q * ((to_f32<T>(xr[c]) - mean) * rstd);
    }
    row_sum<512, 2>(s, sh, flip);
    const float s1 = s[0] * inv_c, s2 = s[1] * inv_c;
    for (int c = threadIdx.x; c < C; c += 512) {
      const float q = to_f32<U>(dyr[c]) * (w != nullptr ? to_f32<W>(w[c]) : 1.f);
      const float h = (to_f32<T>(xr[c]) - mean) * rstd;
      dx[row * static_cast<int64_t>(C) + c] = from_f32<T>(rstd * (q - s1 - h * s2));
    }
  }
}

// The column sums by a pass down the columns: 64 columns (2 a lane) x 16 row lanes per CTA,
// one partial row per blockIdx.y (the result itself where there is only one).
template <typename T, typename U>
__global__ void __launch_bounds__(512)
    colgrad_kernel(const U* __restrict__ dy, int64_t ldy, const T* __restrict__ x, int64_t ldx, int64_t R, int C,
                   const float* __restrict__ mean_in, const float* __restrict__ rstd_in, float* __restrict__ part_w,
                   float* __restrict__ part_b) {
  __shared__ float sw[16][65], sb[16][65];
  const int lane = threadIdx.x % 32, ry = threadIdx.x / 32;
  const int c = blockIdx.x * 64 + lane;  // and c + 32
  const int64_t per = (R + gridDim.y - 1) / gridDim.y;
  const int64_t r0 = blockIdx.y * per, r1 = min(R, r0 + per);
  float gw[2] = {0.f, 0.f}, gb[2] = {0.f, 0.f};
#pragma unroll 4
  for (int64_t r = r0 + ry; r < r1; r += 16) {
    const float mean = mean_in[r], rstd = rstd_in[r];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (c + 32 * k < C) {
        const float d = to_f32<U>(dy[r * ldy + c + 32 * k]);
        gw[k] += d * ((to_f32<T>(x[r * ldx + c + 32 * k]) - mean) * rstd);
        gb[k] += d;
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    sw[ry][lane + 32 * k] = gw[k];
    sb[ry][lane + 32 * k] = gb[k];
  }
  __syncthreads();
  const int col = threadIdx.x;
  if (col < 64 && blockIdx.x * 64 + col < C) {
    float a = 0.f, e = 0.f;
    for (int i = 0; i < 16; ++i) {
      a += sw[i][col];
      e += sb[i][col];
    }
    const int64_t at = static_cast<int64_t>(blockIdx.y) * C + blockIdx.x * 64 + col;
    if (part_w != nullptr) part_w[at] = a;
    if (part_b != nullptr) part_b[at] = e;
  }
}

// out[c] = sum_p part[p][c], in a fixed order: 32 columns x 32 partial lanes per CTA;
// blockIdx.y picks the weight's or the bias's sums.
template <typename O>
__global__ void __launch_bounds__(1024) reduce_kernel(const float* __restrict__ part_w,
                                                      const float* __restrict__ part_b, int P, int C,
                                                      O* __restrict__ dw, O* __restrict__ db) {
  __shared__ float sh[32][33];
  const float* part = blockIdx.y == 0 ? part_w : part_b;
  O* out = blockIdx.y == 0 ? dw : db;
  if (out == nullptr) return;
  const int lane = threadIdx.x % 32, py = threadIdx.x / 32;
  const int c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < C) {
#pragma unroll 4
    for (int p = py; p < P; p += 32) s += part[static_cast<int64_t>(p) * C + c];
  }
  sh[py][lane] = s;
  __syncthreads();
  s = sh[lane][py];  // column py of this CTA
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0 && blockIdx.x * 32 + py < C) out[blockIdx.x * 32 + py] = from_f32<O>(s);
}

struct BwdArgs {
  int64_t ldy, ldx, R;
  int C;
  const float *mean, *rstd;
  const void* w;
  bool want_w, want_b;
};

template <typename T, typename U, typename W, int VEC, int TPR>
static void launch_rows(const U* dy, const T* x, T* dx, const BwdArgs& a, int P, float* pw, float* pb) {
  auto stream = at::cuda::getCurrentCUDAStream();
  constexpr int RPB = kCta<TPR> / TPR;
  const W* w = static_cast<const W*>(a.w);
  const size_t smem = RPB > 1 ? static_cast<size_t>(RPB) * a.C * sizeof(float) : 0;
  if (pw != nullptr || pb != nullptr)
    bwd_kernel<T, U, W, VEC, TPR, true><<<P, kCta<TPR>, smem, stream>>>(dy, a.ldy, x, a.ldx, a.R, a.C, a.mean, a.rstd,
                                                                        w, dx, pw, pb);
  else
    bwd_kernel<T, U, W, VEC, TPR, false><<<P, kCta<TPR>, 0, stream>>>(dy, a.ldy, x, a.ldx, a.R, a.C, a.mean, a.rstd, w,
                                                                      dx, nullptr, nullptr);
}

template <typename T, typename U, typename W, int VEC>
static void launch(const U* dy, const T* x, T* dx, const BwdArgs& a, torch::Tensor& dw, torch::Tensor& db) {
  auto stream = at::cuda::getCurrentCUDAStream();
  const int C = a.C;
  const int64_t sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const int tpr = C <= 128 ? 8 : C <= 512 ? 32 : C <= 2048 ? 128 : 512, cta = tpr > 256 ? tpr : 256;
  const int64_t ctas = std::min<int64_t>(sms * (512 / cta), (a.R + 2 * cta / tpr - 1) / (2 * cta / tpr));
  const bool grads = a.want_w || a.want_b;
  // partial rows are written and read in fp32 (16 bytes a column and CTA); a second pass over
  // x and dy reads them again
  const bool columns =
      grads && (C > kMaxRegCols || ctas * 16 > a.R * static_cast<int64_t>(sizeof(T) + sizeof(U)));
  const int P = static_cast<int>(
      !columns ? ctas : std::max<int64_t>(1, std::min<int64_t>(a.R / 256, 4 * sms / ((C + 63) / 64))));
  // where the sums (or the partial rows) go
  const bool direct = P == 1 && dw.scalar_type() == at::kFloat;
  float *pw = direct && a.want_w ? dw.data_ptr<float>() : nullptr, *pb = direct && a.want_b ? db.data_ptr<float>() : nullptr;
  torch::Tensor part;
  if (grads && !direct) {
    part = torch::empty({2, P, C}, dw.options().dtype(at::kFloat));
    pw = a.want_w ? part.data_ptr<float>() : nullptr;
    pb = a.want_b ? part.data_ptr<float>() + static_cast<int64_t>(P) * C : nullptr;
  }
  float *rw = columns ? nullptr : pw, *rb = columns ? nullptr : pb;
  const int n = static_cast<int>(ctas);
  if (C <= 128) launch_rows<T, U, W, VEC, 8>(dy, x, dx, a, n, rw, rb);
  else if (C <= 512) launch_rows<T, U, W, VEC, 32>(dy, x, dx, a, n, rw, rb);
  else if (C <= 2048) launch_rows<T, U, W, VEC, 128>(dy, x, dx, a, n, rw, rb);
  else if (C <= kMaxRegCols) launch_rows<T, U, W, VEC, 512>(dy, x, dx, a, n, rw, rb);
  else
    bwd_wide_kernel<T, U, W><<<static_cast<unsigned>(std::min<int64_t>(a.R, sms * 4)), 512, 0, stream>>>(
        dy, a.ldy, x, a.ldx, a.R, C, a.mean, a.rstd, static_cast<const W*>(a.w), dx);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (columns) {
    colgrad_kernel<T, U><<<dim3((C + 63) / 64, P), 512, 0, stream>>>(dy, a.ldy, x, a.ldx, a.R, C, a.mean, a.rstd, pw,
                                                                     pb);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  if (grads && !direct) {
    const dim3 grid((C + 31) / 32, 2);
    auto reduce = [&](auto kind) {
      using O = decltype(kind);
      reduce_kernel<O><<<grid, 1024, 0, stream>>>(pw, pb, P, C, a.want_w ? static_cast<O*>(dw.data_ptr()) : nullptr,
                                                  a.want_b ? static_cast<O*>(db.data_ptr()) : nullptr);
    };
    if (dw.scalar_type() == at::kFloat)
      reduce(float{});
    else if (dw.scalar_type() == at::kBFloat16)
      reduce(__nv_bfloat16{});
    else
      reduce(__half{});
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
}

template <typename T, typename U, typename W>
static void run(const torch::Tensor& dy, const torch::Tensor& x, torch::Tensor& dx, const BwdArgs& a,
                torch::Tensor& dw, torch::Tensor& db) {
  constexpr int VEC = sizeof(T) == 4 || sizeof(U) == 4 ? 4 : 8;
  const U* dyp = reinterpret_cast<const U*>(dy.data_ptr());
  const T* xp = reinterpret_cast<const T*>(x.data_ptr());
  T* dxp = reinterpret_cast<T*>(dx.data_ptr());
  const bool vec = vec_ok(dyp, a.ldy, a.C, sizeof(U), VEC) && vec_ok(xp, a.ldx, a.C, sizeof(T), VEC) &&
                   vec_ok(dxp, a.C, a.C, sizeof(T), VEC) && vec_ok_columns<W>(a.w, a.C, VEC);
  if (vec)
    launch<T, U, W, VEC>(dyp, xp, dxp, a, dw, db);
  else
    launch<T, U, W, 1>(dyp, xp, dxp, a, dw, db);
}
template <typename T>
static void run_half(const torch::Tensor& dy, const torch::Tensor& x, torch::Tensor& dx, const BwdArgs& a, bool w_f32,
                     torch::Tensor& dw, torch::Tensor& db) {
  if (dy.scalar_type() == at::kFloat)
    w_f32 ? run<T, float, float>(dy, x, dx, a, dw, db) : run<T, float, T>(dy, x, dx, a, dw, db);
  else
    w_f32 ? run<T, T, float>(dy, x, dx, a, dw, db) : run<T, T, T>(dy, x, dx, a, dw, db);
}

}  // namespace ln

// (dx [R, C] of x's type, dw [C], db [C] of `grad_type`, fp32 or x's; an unwanted one is empty) from
// dy [R, C] (x's type or fp32), x and the forward's mean and rstd.
std::vector<torch::Tensor> layer_norm_bwd(const torch::Tensor& dy, const torch::Tensor& x, const torch::Tensor& mean,
                                          const torch::Tensor& rstd, const c10::optional<torch::Tensor>& w,
                                          bool weight_grad, bool bias_grad, c10::ScalarType grad_type) {
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
  check_plain(mean, "layer_norm_bwd: mean");
  check_plain(rstd, "layer_norm_bwd: rstd");
  TORCH_CHECK(grad_type == at::kFloat || grad_type == x.scalar_type(),
              "layer_norm_bwd: the weight's gradients are fp32 or of x's type");
  BwdArgs a;
  const at::cuda::CUDAGuard guard(x.device());
  const Affine affine = affine_of(x, w, c10::nullopt, "layer_norm_bwd");
  a.w = affine.wp();
  auto vec = x.options().dtype(grad_type);
  auto dx = torch::empty({R, C}, x.options());
  auto dw = weight_grad ? torch::empty({C}, vec) : torch::empty({0}, vec);
  auto db = bias_grad ? torch::empty({C}, vec) : torch::empty({0}, vec);
  check_plain(dx, "layer_norm_bwd");
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
  if (x.scalar_type() == at::kFloat)
    run<float, float, float>(dy, x, dx, a, dw, db);
  else if (x.scalar_type() == at::kBFloat16)
    run_half<__nv_bfloat16>(dy, x, dx, a, affine.f32, dw, db);
  else
    run_half<__half>(dy, x, dx, a, affine.f32, dw, db);
  return {dx, dw, db};
}

}  // namespace nori
