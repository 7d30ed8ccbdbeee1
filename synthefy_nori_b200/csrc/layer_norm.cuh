// Shared pieces of the LayerNorm forward and backward kernels.
//
//   y = (x - mean) rstd w + b,  mean and variance over a row's C values (two passes over
//   registers: the variance sums squares of differences, never a difference of sums)
//
// A row belongs to TPR threads (8, a warp, 128 or 512), each holding up to 16 values in chunks
// of VEC consecutive columns, so a row is read from memory once in each direction.  The threads
// work on two rows at a time: both rows' loads are in flight together, their reductions overlap
// and the weight is read (from L1) once for both.
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <torch/extension.h>

#include <algorithm>

#include "plain.h"
#include "sm100.cuh"

namespace nori {
namespace ln {

constexpr int kValues = 16;         // of one row in a thread
constexpr int kMaxRegCols = 8192;   // 512 threads x 16 values
template <int TPR>
constexpr int kCta = TPR > 256 ? TPR : 256;

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) {
  return __half2float(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}

// VEC consecutive values as one memory access (VEC * sizeof(T) is 2, 4, 8 or 16 bytes).
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float* v) {
  const Pack<T, VEC> u = *reinterpret_cast<const Pack<T, VEC>*>(p);
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = to_f32<T>(u.v[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float* v) {
  Pack<T, VEC> u;
#pragma unroll
  for (int i = 0; i < VEC; ++i) u.v[i] = from_f32<T>(v[i]);
  *reinterpret_cast<Pack<T, VEC>*>(p) = u;
}

// Two fp32 values in one instruction (add, mul, fma; each rounded as the scalar one): the
// backward spends about 11 of these an element and is bound by instruction issue otherwise.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack(F2 x, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v));
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// A thread's chunks of one row; zero beyond the last row or column.
template <typename T, int VEC, int TPR>
struct Row {
  static constexpr int CH = kValues / VEC;
  Pack<T, VEC> p[CH];
  __device__ __forceinline__ void load(const T* x, int64_t ld, int64_t row, int64_t R, int C, int t) {
    const T* xr = x + row * ld;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int c = VEC * (t + TPR * j);
      if (row < R && c < C) {
        p[j] = *reinterpret_cast<const Pack<T, VEC>*>(xr + c);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) p[j].v[i] = from_f32<T>(0.f);
      }
    }
  }
  __device__ __forceinline__ void values(float* v) const {
#pragma unroll
    for (int j = 0; j < CH; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[VEC * j + i] = to_f32<T>(p[j].v[i]);
  }
};
// Brings a row's whole 16-byte pieces to L2: one instruction, no registers held.  A CTA asks for
// its next rows before it works on the ones at hand, so its loads wait for L2 and not for DRAM.
template <typename T>
__device__ __forceinline__ void prefetch_row(const T* row, int C) {
  const uintptr_t a = (reinterpret_cast<uintptr_t>(row) + 15) & ~uintptr_t(15);
  const uintptr_t e = reinterpret_cast<uintptr_t>(row + C) & ~uintptr_t(15);
  if (e > a)
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(a), "r"(static_cast<uint32_t>(e - a)) : "memory");
}

// VEC columns of a weight vector (`fill` where there is none).
template <int VEC, typename W>
__device__ __forceinline__ void load_columns(const W* w, int c, float fill, float* v) {
  constexpr int N = VEC * sizeof(W) > 16 ? 16 / sizeof(W) : VEC;  // of one access
#pragma unroll
  for (int i = 0; i < VEC; i += N) {
    if (w == nullptr) {
#pragma unroll
      for (int k = 0; k < N; ++k) v[i + k] = fill;
    } else {
      load_vec<W, N>(w + c + i, v + i);
    }
  }
}

// The sum of a thread's values.  Sums are pairwise throughout, so a row of 2^k equal values has them
// for its mean, exactly, and gives the bias.
__device__ __forceinline__ float pairwise_sum(const float (&v)[kValues]) {
  float a[kValues / 2];
#pragma unroll
  for (int i = 0; i < kValues / 2; ++i) a[i] = v[2 * i] + v[2 * i + 1];
#pragma unroll
  for (int n = kValues / 4; n > 0; n >>= 1)
#pragma unroll
    for (int i = 0; i < n; ++i) a[i] += a[i + n];
  return a[0];
}

// Sums of N values over the TPR threads of a row; every one of them gets them.  Rows wider
// than a warp add their warps' sums through `sh`, which alternates between two places from one
// use to the next, so one barrier is enough.
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (&sh)[2][N][16], int& flip) {
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if constexpr (TPR > 32) {
    const int warp = threadIdx.x / 32, w0 = warp / (TPR / 32) * (TPR / 32);
    if (threadIdx.x % 32 == 0)
#pragma unroll
      for (int k = 0; k < N; ++k) sh[flip][k][warp] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float a[TPR / 32];
#pragma unroll
      for (int i = 0; i < TPR / 32; ++i) a[i] = sh[flip][k][w0 + i];
#pragma unroll
      for (int n = TPR / 64; n > 0; n >>= 1)
#pragma unroll
        for (int i = 0; i < n; ++i) a[i] += a[i + n];
      v[k] = a[0];
    }
    flip ^= 1;
  }
}

// 16-byte accesses need rows that start on 16 bytes and a width that is a whole number of them.
inline bool vec_ok(const void* p, int64_t ld, int64_t C, int64_t elem, int vec) {
  return C % vec == 0 && (ld * elem) % (vec * elem) == 0 && reinterpret_cast<uintptr_t>(p) % (vec * elem) == 0;
}

// The weight and the bias as the kernels read them: in x's type where both have it, else in fp32.
struct Affine {
  torch::Tensor w, b;  // undefined where there is none
  bool f32;
  const void* wp() const { return w.defined() ? w.data_ptr() : nullptr; }
  const void* bp() const { return b.defined() ? b.data_ptr() : nullptr; }
};
inline Affine affine_of(const torch::Tensor& x, const c10::optional<torch::Tensor>& w,
                        const c10::optional<torch::Tensor>& b, const char* what) {
  Affine a;
  a.f32 = x.scalar_type() == at::kFloat;
  for (const auto* t : {&w, &b}) {
    if (!t->has_value() || !(*t)->defined()) continue;
    check_plain(**t, what);
    TORCH_CHECK((*t)->device() == x.device() && at::isFloatingType((*t)->scalar_type()) && (*t)->numel() == x.size(1), what,
                ": weight and bias must be floating vectors of the row width on x's device");
    if ((*t)->scalar_type() != x.scalar_type()) a.f32 = true;
  }
  const auto type = a.f32 ? at::kFloat : x.scalar_type();
  auto plain = [&](const torch::Tensor& t) {
    return t.scalar_type() == type && t.is_contiguous() ? t : t.detach().to(type).contiguous();
  };
  if (w.has_value() && w->defined()) a.w = plain(*w);
  if (b.has_value() && b->defined()) a.b = plain(*b);
  return a;
}
template <typename W>
inline bool vec_ok_columns(const void* p, int64_t C, int vec) {
  return vec_ok(p, 0, C, sizeof(W), std::min<int>(vec, 16 / sizeof(W)));
}

// rows of `t`: [R, C] with unit column stride, any row stride
inline void check_rows(const torch::Tensor& t, const char* what) {
  check_plain(t, what);
  TORCH_CHECK(t.is_cuda() && t.dim() == 2, what, ": a CUDA matrix [rows, cols] expected");
  const auto s = t.scalar_type();
  TORCH_CHECK(s == at::kFloat || s == at::kBFloat16 || s == at::kHalf, what, ": fp32, bf16 or fp16 expected");
  TORCH_CHECK(t.size(1) >= 1 && t.size(1) < (int64_t{1} << 30), what, ": 1 to 2^30 columns expected");
  TORCH_CHECK(t.size(1) == 1 || t.stride(1) == 1, what, ": columns must be contiguous");
  TORCH_CHECK(t.stride(0) >= 0, what, ": negative row stride");
}

}  // namespace ln
}  // namespace nori
