// Muon on sm_100a: momentum, orthogonalisation by Newton-Schulz products and the weight
// update for a ragged set of matrices, and the orthogonalisation alone.
//
// For one matrix G (rows x cols; n = max, m = min of the two, taken tall, i.e. n x m):
//   X_0 = G / (|G|_F + eps)
//   A = X^T X,   C = (b A + c A^2) / a,   X <- a (X + X C)          (repeated `steps` times)
//
// Numerics.  The kernels carry Z_k = X_k / xi_k with xi_0 = f 2^-8, f = |G|_F / (|G|_F + eps), so
// that one step is Z <- Z + Z C, xi <- a xi, and the leading term needs no multiplication.  X
// stays of size 1 while xi grows by a (3.4 with the usual coefficients) a step, so Z would shrink
// to nothing in fp16: where xi has grown past 1 (|Z| < |X|) a power of two, exact in all that holds Z,
// goes from xi to Z (`renorm`), and any number of steps keeps its digits; five steps with the usual
// coefficients never get there.  As long as X itself is still growing (|G| far below eps) xi is
// below 1 and Z stays as it is.
// Z is held in fp32 (one CTA a matrix) or as a pair of fp16 (high, low: 22 significant bits;
// over the whole GPU); the three products read fp16 operands (the high parts, A and C: 11
// bits) and accumulate in fp32.  A small singular value of G lives in the pair and is only
// multiplied by 1 + C, so it keeps its 22 bits, while the rounding of the products' operands
// (2^-11 relative at most) perturbs the dominant directions only and is not amplified: five steps are
// 1e-3 .. 3e-3 (2-norm) from the exact iteration for flat, power-law, exponential and
// rank-deficient spectra alike, about the rounding of a bf16 result, and 64 steps about 1e-2.  With iterates rounded
// to bf16 the noise 2^-8 |G|_F is amplified by up to a^5 = 485 in the small directions: 1e-2
// for a flat spectrum and 0.1 .. 1 for steep ones.  Products of fp16 pairs (three MMAs each)
// give 1e-6 for three times the tensor work; the single-CTA kernel takes them up to 32 columns,
// where the work is nothing and few roundings average out.
//
// Reference counterpart: training/optim.py:60-85 (Newton-Schulz), 180-319 (Muon step).
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAEvent.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>
#include <torch/extension.h>

#include <algorithm>
#include <climits>
#include <type_traits>
#include <vector>

#include "plain.h"
#include "sm100.cuh"
#include "tma_host.h"

namespace nori {
namespace muon {

constexpr float kZScale = 256.f;

// Takes a power of two out of xi once it is above 1, leaving it in [2^-9, 2^-8), and returns that
// power for Z to be multiplied by (1 where there is nothing to do, or xi is NaN).
__device__ __forceinline__ float renorm(float& xi) {
  if (!(xi > 1.f)) return 1.f;
  const int e = (__float_as_int(xi) >> 23) - (127 - 9);
  xi *= __int_as_float((127 - e) << 23);
  return __int_as_float((127 + e) << 23);
}

enum OutType : int { kOutF32 = 0, kOutBF16 = 1, kOutF16 = 2, kOutMuon = 3 };
enum SrcType : int { kSrcF32 = 0, kSrcBF16 = 1, kSrcF16 = 2, kSrcMuon = 3 };

// Learning-rate factor of the orthogonalised update, by shape.
enum Adjust : int { kMatchRms = 0, kOriginal = 1, kNd = 2 };

// One row of the plan's device table.
struct Mat {
  int64_t off;   // first element in the flat parameter / gradient / average buffers
  int64_t moff;  // first element in the momentum buffer
  int64_t rows, cols;
};

struct Coeffs {
  int steps;
  float eps, a, ba, ca;  // the coefficients a, b / a, c / a
};

struct StepArgs {
  float* data;
  const float* grad;
  float* mom;
  float* ema;  // or null
  const Mat* table;
  const float* norm_sq;  // or null
  const float* skip;     // or null
  float lr, wd, momentum, max_norm, ema_w;
  int nesterov, adjust;
};

// Whether a wait of an earlier kernel has run out (nothing is read or written from then on, until the
// host has seen it).  The word can change at any time, so the CTA's threads settle on one answer:
// with some gone and some not, tensor memory would be used before it is there.
__device__ __forceinline__ bool timed_out(const int* status) {
  return __syncthreads_or(*reinterpret_cast<const volatile int*>(status) != 0) != 0;
}

// A step that the trainer rejected on the device, or one whose gradient norm is not finite,
// leaves weights, momentum and average as they are (as adamw_ema_kernel does).
__device__ __forceinline__ bool step_rejected(const StepArgs& s) {
  if (s.skip != nullptr && *s.skip > 0.f) return true;
  return s.norm_sq != nullptr && !(*s.norm_sq < INFINITY);
}

__device__ __forceinline__ float clip_factor(const StepArgs& s) {
  if (s.norm_sq == nullptr) return 1.f;
  return fminf(1.f, s.max_norm / (sqrtf(*s.norm_sq) + 1e-6f));
}

__device__ __forceinline__ float lr_factor(int adjust, int rows, int cols) {
  const float r = static_cast<float>(rows), c = static_cast<float>(cols);
  if (adjust == kMatchRms) return 0.2f * sqrtf(fmaxf(r, c));
  if (adjust == kOriginal) return sqrtf(fmaxf(1.f, r / c));
  return sqrtf(fmaxf(r, c) / fminf(r, c));
}

template <int SRC>
__device__ __forceinline__ float load_src(const void* g, int64_t i) {
  if constexpr (SRC == kSrcF32) return static_cast<const float*>(g)[i];
  if constexpr (SRC == kSrcBF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(g)[i]);
  if constexpr (SRC == kSrcF16) return __half2float(static_cast<const __half*>(g)[i]);
  return 0.f;
}

// Where one element of the result goes: a plain output tensor, or the weights.
struct Sink {
  int type;      // OutType
  void* out;     // plain output of this matrix's batch, or null
  int64_t base;  // first element of the matrix
  float lr_o;    // kOutMuon: lr times the shape's factor
};
// Values o[0 .. cnt) go to elements e0, e0 + stride, ...: every load of the weights is issued
// before the first store (the compiler may not move one past the other), so a thread waits
// for memory once, not once per element.
template <typename T, int N>
__device__ __forceinline__ void store_strided(T* p, int64_t stride, int cnt, const float* o) {
#pragma unroll
  for (int i = 0; i < N; ++i, p += stride)
    if (i < cnt) {
      if constexpr (sizeof(T) == 4)
        *p = o[i];
      else if constexpr (std::is_same<T, __nv_bfloat16>::value)
        *p = __float2bfloat16(o[i]);
      else
        *p = __float2half_rn(o[i]);
    }
}
template <int N>
__device__ __forceinline__ void emit(const Sink& k, const StepArgs& s, int64_t e0, int64_t stride, int cnt,
                                     const float* o) {
  e0 += k.base;
  if (k.type == kOutMuon) {
    float p[N], e[N];
    float* w = s.data + e0;
    float* av = s.ema + e0;  // used where there is one
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = i < cnt ? w[i * stride] : 0.f;
    if (s.ema != nullptr) {
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = i < cnt ? av[i * stride] : 0.f;
    }
    const float keep = 1.f - s.lr * s.wd;
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = p[i] * keep - k.lr_o * o[i];
    store_strided<float, N>(w, stride, cnt, p);
    if (s.ema != nullptr) {
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] += s.ema_w * (p[i] - e[i]);
      store_strided<float, N>(av, stride, cnt, e);
    }
  } else if (k.type == kOutF32) {
    store_strided<float, N>(static_cast<float*>(k.out) + e0, stride, cnt, o);
  } else if (k.type == kOutBF16) {
    store_strided<__nv_bfloat16, N>(static_cast<__nv_bfloat16*>(k.out) + e0, stride, cnt, o);
  } else {
    store_strided<__half, N>(static_cast<__half*>(k.out) + e0, stride, cnt, o);
  }
}

// The same for N groups of 4 consecutive values, `stride` apart, where sink4() allows it.
__device__ __forceinline__ bool sink4(const Sink& k, const StepArgs& s) {
  if (k.type == kOutMuon)
    return ((reinterpret_cast<uintptr_t>(s.data + k.base) |
             (s.ema != nullptr ? reinterpret_cast<uintptr_t>(s.ema + k.base) : 0)) & 15) == 0;
  if (k.type == kOutF32) return (reinterpret_cast<uintptr_t>(static_cast<float*>(k.out) + k.base) & 15) == 0;
  return (reinterpret_cast<uintptr_t>(static_cast<__half*>(k.out) + k.base) & 7) == 0;
}
template <int N>
__device__ __forceinline__ void emit4(const Sink& k, const StepArgs& s, int64_t e0, int64_t stride, int cnt,
                                      const float4* o) {
  e0 += k.base;
  if (k.type == kOutMuon) {
    float4 p[N], e[N];
    float* w = s.data + e0;
    float* av = s.ema + e0;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < cnt) p[i] = *reinterpret_cast<const float4*>(w + i * stride);
    if (s.ema != nullptr) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < cnt) e[i] = *reinterpret_cast<const float4*>(av + i * stride);
    }
    const float keep = 1.f - s.lr * s.wd;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < cnt) {
        p[i].x = p[i].x * keep - k.lr_o * o[i].x;
        p[i].y = p[i].y * keep - k.lr_o * o[i].y;
        p[i].z = p[i].z * keep - k.lr_o * o[i].z;
        p[i].w = p[i].w * keep - k.lr_o * o[i].w;
        *reinterpret_cast<float4*>(w + i * stride) = p[i];
      }
    if (s.ema != nullptr) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < cnt) {
          e[i].x += s.ema_w * (p[i].x - e[i].x);
          e[i].y += s.ema_w * (p[i].y - e[i].y);
          e[i].z += s.ema_w * (p[i].z - e[i].z);
          e[i].w += s.ema_w * (p[i].w - e[i].w);
          *reinterpret_cast<float4*>(av + i * stride) = e[i];
        }
    }
  } else if (k.type == kOutF32) {
    float* d = static_cast<float*>(k.out) + e0;
#pragma unroll
    for (int i = 0; i < N; ++i, d += stride)
      if (i < cnt) *reinterpret_cast<float4*>(d) = o[i];
  } else if (k.type == kOutBF16) {
    __nv_bfloat16* d = static_cast<__nv_bfloat16*>(k.out) + e0;
#pragma unroll
    for (int i = 0; i < N; ++i, d += stride)
      if (i < cnt) *reinterpret_cast<uint2*>(d) = make_uint2(pack_bf16x2(o[i].x, o[i].y), pack_bf16x2(o[i].z, o[i].w));
  } else {
    __half* d = static_cast<__half*>(k.out) + e0;
#pragma unroll
    for (int i = 0; i < N; ++i, d += stride)
      if (i < cnt) {
        uint2 u;
        *reinterpret_cast<__half2*>(&u.x) = __floats2half2_rn(o[i].x, o[i].y);
        *reinterpret_cast<__half2*>(&u.y) = __floats2half2_rn(o[i].z, o[i].w);
        *reinterpret_cast<uint2*>(d) = u;
      }
  }
}

// The update's input at elements e0, e0 + stride, ... (the momentum brought up to date on the
// way), loads before stores as in emit.
template <int SRC, int N>
__device__ __forceinline__ void fetch(const void* g, const StepArgs& s, int64_t base, int64_t mbase, float clip,
                                      int64_t e0, int64_t stride, int cnt, float* v) {
  if constexpr (SRC == kSrcMuon) {
    float m[N];
    const float* gr = s.grad + base + e0;
    float* mo = s.mom + mbase + e0;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < cnt ? gr[i * stride] * clip : 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) m[i] = i < cnt ? mo[i * stride] : 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      m[i] = s.momentum * m[i] + v[i];
      v[i] = s.nesterov ? v[i] + s.momentum * m[i] : m[i];
    }
    store_strided<float, N>(mo, stride, cnt, m);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < cnt ? load_src<SRC>(g, base + e0 + i * stride) : 0.f;
  }
}

// 4 consecutive values of the update's input, where aligned4() allows it.
template <int SRC>
__device__ __forceinline__ void load4(const void* g, int64_t i, float* v) {
  if constexpr (SRC == kSrcF32) {
    const float4 u = *reinterpret_cast<const float4*>(static_cast<const float*>(g) + i);
    v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
  } else if constexpr (SRC == kSrcBF16) {
    const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(g) + i);
    v[0] = bf16lo(u.x), v[1] = bf16hi(u.x), v[2] = bf16lo(u.y), v[3] = bf16hi(u.y);
  } else if constexpr (SRC == kSrcF16) {
    const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const __half*>(g) + i);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  }
}
template <int SRC>
__device__ __forceinline__ bool aligned4(const void* g, const StepArgs& s, int64_t base, int64_t mbase) {
  if constexpr (SRC == kSrcMuon)
    return ((reinterpret_cast<uintptr_t>(s.grad + base) | reinterpret_cast<uintptr_t>(s.mom + mbase)) & 15) == 0;
  if constexpr (SRC == kSrcF32) return (reinterpret_cast<uintptr_t>(static_cast<const float*>(g) + base) & 15) == 0;
  return (reinterpret_cast<uintptr_t>(static_cast<const __half*>(g) + base) & 7) == 0;
}
// N groups of 4 consecutive values, `stride` apart.
template <int SRC, int N>
__device__ __forceinline__ void fetch4(const void* g, const StepArgs& s, int64_t base, int64_t mbase, float clip,
                                       int64_t e0, int64_t stride, int cnt, float* v) {
  if constexpr (SRC == kSrcMuon) {
    float m[4 * N];
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) v[i] = m[i] = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < cnt) load4<kSrcF32>(s.grad, base + e0 + i * stride, v + 4 * i);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < cnt) load4<kSrcF32>(s.mom, mbase + e0 + i * stride, m + 4 * i);
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) {
      v[i] *= clip;
      m[i] = s.momentum * m[i] + v[i];
      v[i] = s.nesterov ? v[i] + s.momentum * m[i] : m[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < cnt)
        *reinterpret_cast<float4*>(s.mom + mbase + e0 + i * stride) =
            make_float4(m[4 * i], m[4 * i + 1], m[4 * i + 2], m[4 * i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) v[i] = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < cnt) load4<SRC>(g, base + e0 + i * stride, v + 4 * i);
  }
}

// From a matrix's sum of squares v: 2^8 / norm as a product of two floats (it may lie outside
// fp32's range; powers of two from the exponent, the rest is in [2^7, 2^8]), and
// f = norm / (norm + eps).  All zero for a zero matrix; f is NaN where the sum is not finite.
__device__ __forceinline__ void z_scale(double v, float eps, float& s0, float& s1, float& f) {
  if (!(v > 0.0) || !(v < INFINITY)) {
    s0 = s1 = 0.f;
    f = v == 0.0 ? 0.f : NAN;
    return;
  }
  const int k = (((__double2hiint(v) >> 20) & 0x7ff) - 1023) >> 1;  // norm is in [2^k, 2^(k+1))
  const float r = rsqrtf(static_cast<float>(v * __hiloint2double((1023 - 2 * k) << 20, 0)));  // 2^k / norm
  const int k0 = k / 2, k1 = k - k0;
  s0 = __int_as_float((127 - k0) << 23);
  const float t = __int_as_float((127 - k1) << 23) * r;
  s1 = kZScale * t;
  f = 1.f / (1.f + eps * s0 * t);
}

// kind::f16 with fp16 operands, fp32 accumulators, M = 128.
__device__ __forceinline__ uint32_t idesc_f16(int N, bool mn_major) {
  return (1u << 4) | (mn_major ? (1u << 15) | (1u << 16) : 0u) | (static_cast<uint32_t>(N >> 3) << 17) | (8u << 24);
}

__device__ __forceinline__ uint4 pack8(const float* v) {
  uint4 u;
  __half2* h = reinterpret_cast<__half2*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
  return u;
}
__device__ __forceinline__ void unpack8(uint4 u, float* v) {
  const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// ------------------------------------------------------------------ one matrix per CTA
constexpr int kSingleThreads = 512;
constexpr int kSingleMaxTiles = 12;
constexpr int kSingleStage = 16 * 32 * 17 * 4;  // one [32][17] tile per warp, in the operands' place

struct Fit {
  int n, m, mp, tiles, panels;
  int smem, tmem;
  bool ok;
};
__host__ __device__ inline Fit single_fit(int rows, int cols) {
  Fit f;
  f.n = rows > cols ? rows : cols;
  f.m = rows > cols ? cols : rows;
  f.mp = (f.m + 15) / 16 * 16;
  f.tiles = (f.n + 127) / 128;
  f.panels = (f.mp + 63) / 64;
  f.smem = (f.tiles + 1) * f.panels * 16384;
  if (f.smem < kSingleStage) f.smem = kSingleStage;
  f.tmem = (f.tiles + 1) * f.mp;
  f.ok = f.m <= 128 && f.tiles <= kSingleMaxTiles && f.smem <= 220 * 1024 && f.tmem <= 512;
  return f;
}

// Matrices first .. first + count of a set that all fit one CTA; `smem` is the largest need.
void run_single(int src, const void* g, int out_type, void* out, const StepArgs& s, int64_t first, int64_t count,
                int rows, int cols, int smem, const Coeffs& k, const torch::Tensor& status);

// ------------------------------------------------------------------ matrices over the whole GPU
struct Shape {
  int64_t first, count;  // matrices of the plan's table (or of the batch)
  int rows, cols;
};
// `ready`, if given, is recorded once the norms and Z_0 are under way and before the products.
void run_large(int src, const void* g, int out_type, void* out, const StepArgs& s, const std::vector<Shape>& shapes,
               const Coeffs& k, const torch::Tensor& status, const at::TensorOptions& dev, at::cuda::CUDAEvent* ready);

}  // namespace muon
}  // namespace nori
