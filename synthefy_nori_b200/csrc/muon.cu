// Muon on sm_100a: momentum, orthogonalisation by Newton-Schulz products and the weight
// update for a ragged set of matrices, and the orthogonalisation alone.
//
// For one matrix G (rows x cols; n = max, m = min of the two, taken tall, i.e. n x m):
//   X_0 = G / (|G|_F + eps)
//   A = X^T X,   C = (b A + c A^2) / a,   X <- a (X + X C)          (repeated `steps` times)
//
// Numerics.  The kernels carry Z_k = 2^8 X_k / (f a^k) with f = |G|_F / (|G|_F + eps), so
// that one step is Z <- Z + Z C and the leading term needs no multiplication: X_k = xi_k Z_k
// with xi_0 = f 2^-8 and xi_{k+1} = a xi_k.  Z is held as a pair of fp16 (high, low: 22
// significant bits); the three products read fp16 operands (the high parts, A and C: 11
// bits) and accumulate in fp32.  A small singular value of G lives in the pair and is only
// multiplied by 1 + C, so it keeps its 22 bits, while the rounding of the products' operands
// (2^-12 relative) perturbs the dominant directions only and is not amplified: the result is
// 2e-4 .. 2e-3 (2-norm) from the exact iteration for flat, power-law, exponential and
// rank-deficient spectra alike, about the rounding of a bf16 result.  With iterates rounded
// to bf16 the noise 2^-9 |G|_F is amplified by up to a^5 = 485 in the small directions: 1e-2
// for a flat spectrum and 0.1 .. 1 for steep ones.  Products of fp16 pairs (three MMAs each)
// would give 1e-6 for three times the tensor work.
//
// Reference counterpart: training/optim.py:60-85 (Newton-Schulz), 180-319 (Muon step).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>
#include <torch/extension.h>

#include <algorithm>
#include <climits>

#include "sm100.cuh"
#include "tma_host.h"

namespace nori {
namespace muon {

constexpr int kThreads = 320;     // TMA warp, MMA warp, 8 epilogue warps
constexpr int kStages = 4;
constexpr int kStageBytes = 48 * 1024;  // 128 x 64 and up to 256 x 64 fp16 operands
constexpr int kTileFloats = 32 * 33;    // one epilogue warp's transposition tile
constexpr int kSmemBytes = kStages * kStageBytes + 8 * kTileFloats * 4 + 1024 + 256;
constexpr float kZScale = 256.f;

enum Phase : int { kGram = 0, kPoly = 1, kUpdate = 2 };
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
template <int N>
__device__ __forceinline__ void emit(const Sink& k, const StepArgs& s, int64_t e0, int64_t stride, int cnt,
                                     const float* o) {
  e0 += k.base;
  if (k.type == kOutMuon) {
    float p[N], e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = i < cnt ? s.data[e0 + i * stride] : 0.f;
    if (s.ema != nullptr) {
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = i < cnt ? s.ema[e0 + i * stride] : 0.f;
    }
    const float keep = 1.f - s.lr * s.wd;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      p[i] = p[i] * keep - k.lr_o * o[i];
      if (i < cnt) s.data[e0 + i * stride] = p[i];
    }
    if (s.ema != nullptr) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < cnt) s.ema[e0 + i * stride] = e[i] + s.ema_w * (p[i] - e[i]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i < cnt) {
      if (k.type == kOutF32)
        static_cast<float*>(k.out)[e0 + i * stride] = o[i];
      else if (k.type == kOutBF16)
        static_cast<__nv_bfloat16*>(k.out)[e0 + i * stride] = __float2bfloat16(o[i]);
      else
        static_cast<__half*>(k.out)[e0 + i * stride] = __float2half_rn(o[i]);
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
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < cnt ? s.grad[base + e0 + i * stride] * clip : 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) m[i] = i < cnt ? s.mom[mbase + e0 + i * stride] : 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      m[i] = s.momentum * m[i] + v[i];
      if (i < cnt) s.mom[mbase + e0 + i * stride] = m[i];
      v[i] = s.nesterov ? v[i] + s.momentum * m[i] : m[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < cnt ? load_src<SRC>(g, base + e0 + i * stride) : 0.f;
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

// ------------------------------------------------------------------ norm (and momentum)
// Partial sums of squares of the update's input, one per (matrix, slice), in double: no fp32
// gradient overflows or vanishes in its own norm.  With kSrcMuon the momentum buffer is
// brought up to date on the way.
template <int SRC>
__global__ void __launch_bounds__(256) norm_kernel(const void* __restrict__ g, StepArgs s, int first, int64_t numel,
                                                   double* __restrict__ partial) {
  if constexpr (SRC == kSrcMuon) {
    if (step_rejected(s)) return;
  }
  const int mat = blockIdx.y;
  double acc = 0.0;
  const int64_t per = (numel + gridDim.x - 1) / gridDim.x;
  const int64_t i0 = blockIdx.x * per, i1 = min(numel, i0 + per);
  if constexpr (SRC == kSrcMuon) {
    const Mat t = s.table[first + mat];
    const float clip = clip_factor(s);
    for (int64_t i = i0 + threadIdx.x; i < i1; i += blockDim.x) {
      const float gi = s.grad[t.off + i] * clip;
      const float m = s.momentum * s.mom[t.moff + i] + gi;
      s.mom[t.moff + i] = m;
      const float e = s.nesterov ? gi + s.momentum * m : m;
      acc += static_cast<double>(e) * e;
    }
  } else {
    for (int64_t i = i0 + threadIdx.x; i < i1; i += blockDim.x) {
      const float e = load_src<SRC>(g, mat * numel + i);
      acc += static_cast<double>(e) * e;
    }
  }
  __shared__ double sh[8];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    double v = 0.0;
    for (int w = 0; w < 8; ++w) v += sh[w];
    partial[static_cast<int64_t>(mat) * gridDim.x + blockIdx.x] = v;
  }
}

// ------------------------------------------------------------------ Z_0
// Z_0 = 2^8 G / |G|_F as a pair of fp16 [n, ldz], tall (a wide G is transposed on the way),
// and f = |G|_F / (|G|_F + eps).  A zero matrix stays zero.
template <int SRC>
__global__ void __launch_bounds__(256) scale_kernel(const void* __restrict__ g, StepArgs s, int first, int rows,
                                                    int cols, int slices, const double* __restrict__ partial,
                                                    float eps, __half* __restrict__ zh, __half* __restrict__ zl,
                                                    int ldz, float* __restrict__ f) {
  if constexpr (SRC == kSrcMuon) {
    if (step_rejected(s)) return;
  }
  __shared__ float tile[64][65];
  __shared__ float scale[2];
  const int mat = blockIdx.y;
  if (threadIdx.x == 0) {
    double v = 0.0;
    for (int i = 0; i < slices; ++i) v += partial[static_cast<int64_t>(mat) * slices + i];
    float fm;
    z_scale(v, eps, scale[0], scale[1], fm);
    if (blockIdx.x == 0) f[mat] = fm;
  }
  __syncthreads();
  const float s0 = scale[0], s1 = scale[1];
  const bool wide = rows < cols;
  const int n = wide ? cols : rows, m = wide ? rows : cols;
  const int tiles_c = (cols + 63) / 64;
  const int r0 = blockIdx.x / tiles_c * 64, c0 = blockIdx.x % tiles_c * 64;  // in G
  int64_t base = 0, mbase = 0;
  float clip = 1.f;
  if constexpr (SRC == kSrcMuon) {
    const Mat t = s.table[first + mat];
    base = t.off;
    mbase = t.moff;
    clip = clip_factor(s);
  } else {
    base = static_cast<int64_t>(mat) * rows * cols;
  }
  for (int i = threadIdx.x; i < 64 * 64; i += 256) {
    const int r = r0 + i / 64, c = c0 + i % 64;
    float v = 0.f;
    if (r < rows && c < cols) {
      const int64_t at = static_cast<int64_t>(r) * cols + c;
      if constexpr (SRC == kSrcMuon) {
        const float mo = s.mom[mbase + at];
        v = s.nesterov ? s.grad[base + at] * clip + s.momentum * mo : mo;
      } else {
        v = load_src<SRC>(g, base + at);
      }
    }
    tile[i / 64][i % 64] = v * s0 * s1;
  }
  __syncthreads();
  __half* zhb = zh + static_cast<int64_t>(mat) * n * ldz;
  __half* zlb = zl + static_cast<int64_t>(mat) * n * ldz;
  const int zr0 = wide ? c0 : r0, zc0 = wide ? r0 : c0;
  for (int i = threadIdx.x; i < 64 * 64; i += 256) {
    const int zr = i / 64, zc = i % 64;
    if (zr0 + zr < n && zc0 + zc < m) {
      const float v = wide ? tile[zc][zr] : tile[zr][zc];
      const __half h = __float2half_rn(v);
      const int64_t at = static_cast<int64_t>(zr0 + zr) * ldz + zc0 + zc;
      zhb[at] = h;
      zlb[at] = __float2half_rn(v - __half2float(h));
    }
  }
}

// ------------------------------------------------------------------ the products
struct NsParams {
  int n, m, ldz, batch;
  int bn;             // column tile of the update
  int phase, it, steps;
  float a, ba, ca;    // the coefficients a, b / a, c / a
  __half* zh_out;     // the other Z (high) buffer
  const __half* zh;   // this step's
  __half* zl;         // updated in place
  __half* A;
  __half* C;
  const float* f;
  int out_type;
  void* out;          // [batch, rows, cols], or null with kOutMuon
  int rows, cols, first;
  StepArgs s;
  int* status;
};

// kind::f16 with fp16 operands, fp32 accumulators, M = 128.
__device__ __forceinline__ uint32_t idesc_f16(int N, bool mn_major) {
  return (1u << 4) | (mn_major ? (1u << 15) | (1u << 16) : 0u) | (static_cast<uint32_t>(N >> 3) << 17) | (8u << 24);
}

struct Item {
  int mat, ti, tj;
};

// Tiles of the symmetric products: 128 x 128 with ti <= tj (the other half is mirrored);
// of the update: 128 rows x bn columns.
__device__ __forceinline__ Item decode(const NsParams& p, int t) {
  Item it;
  if (p.phase == kUpdate) {
    const int tn = (p.m + p.bn - 1) / p.bn, per = (p.n + 127) / 128 * tn;
    it.mat = t / per;
    const int r = t % per;
    it.ti = r / tn;
    it.tj = r % tn;
  } else {
    const int nt = (p.m + 127) / 128, per = nt * (nt + 1) / 2;
    it.mat = t / per;
    int r = t % per, i = 0;
    while (r >= nt - i) {
      r -= nt - i;
      ++i;
    }
    it.ti = i;
    it.tj = i + r;
  }
  return it;
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

// One of the three products over all matrices of a shape, persistent and warp-specialised:
// one warp loads 128B-swizzled boxes by TMA into a 4-stage ring, one thread issues
// tcgen05.mma (M = 128, N <= 256, K = 16) into two TMEM accumulators, eight warps run the
// epilogue of the previous tile.  The Gram product reads Z as an MN-major operand on both
// sides (the sum runs over Z's rows), the other two read K-major rows; A and C are
// symmetric, so only tiles on and above the diagonal are computed and then mirrored.
__global__ void __launch_bounds__(kThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap tmZ, const __grid_constant__ CUtensorMap tmA,
                   const __grid_constant__ CUtensorMap tmC, NsParams p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* tiles = reinterpret_cast<float*>(smem + kStages * kStageBytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(tiles + 8 * kTileFloats);
  uint64_t* empty = full + kStages;
  uint64_t* tfull = empty + kStages;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (*reinterpret_cast<volatile int*>(p.status) != 0) return;
  if (p.out_type == kOutMuon && step_rejected(p.s)) return;

  const int nt = (p.m + 127) / 128;
  const int per_mat = p.phase == kUpdate ? (p.n + 127) / 128 * ((p.m + p.bn - 1) / p.bn) : nt * (nt + 1) / 2;
  const int items = per_mat * p.batch;
  const int K = p.phase == kGram ? p.n : p.m;
  const int num_kb = (K + 63) / 64;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 8);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < items && ok; t += gridDim.x) {
        const Item it = decode(p, t);
        const bool diag = p.phase != kUpdate && it.ti == it.tj;  // both operands are the same rows
        const uint32_t bytes = 16384u + (p.phase == kUpdate ? p.bn * 128u : diag ? 0u : 16384u);
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1, p.status, kTimeoutProducer, abort_flag)) {
            ok = false;
            break;
          }
          uint8_t* sa = smem + stage * kStageBytes;
          uint8_t* sb = sa + 16384;
          mbar_arrive_expect_tx(&full[stage], bytes);
          if (p.phase == kGram) {
            tma_load_3d(sa, &tmZ, &full[stage], it.ti * 128, kb * 64, it.mat);
            tma_load_3d(sa + 8192, &tmZ, &full[stage], it.ti * 128 + 64, kb * 64, it.mat);
            if (!diag) {
              tma_load_3d(sb, &tmZ, &full[stage], it.tj * 128, kb * 64, it.mat);
              tma_load_3d(sb + 8192, &tmZ, &full[stage], it.tj * 128 + 64, kb * 64, it.mat);
            }
          } else if (p.phase == kPoly) {
            tma_load_3d(sa, &tmA, &full[stage], kb * 64, it.ti * 128, it.mat);
            tma_load_3d(sa + 8192, &tmA, &full[stage], kb * 64, it.ti * 128 + 64, it.mat);
            if (!diag) {
              tma_load_3d(sb, &tmA, &full[stage], kb * 64, it.tj * 128, it.mat);
              tma_load_3d(sb + 8192, &tmA, &full[stage], kb * 64, it.tj * 128 + 64, it.mat);
            }
          } else {
            tma_load_3d(sa, &tmZ, &full[stage], kb * 64, it.ti * 128, it.mat);
            tma_load_3d(sa + 8192, &tmZ, &full[stage], kb * 64, it.ti * 128 + 64, it.mat);
            tma_load_3d(sb, &tmC, &full[stage], kb * 64, it.tj * p.bn, it.mat);
          }
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < items && ok; t += gridDim.x) {
        const Item it = decode(p, t);
        const bool diag = p.phase != kUpdate && it.ti == it.tj;
        const int tile_n = p.phase == kUpdate ? p.bn : 128;
        const int N = min(tile_n, (p.m - it.tj * tile_n + 15) / 16 * 16);
        const uint32_t idesc = idesc_f16(N, p.phase == kGram);
        if (!mbar_wait(&tempty[acc], acc_phase ^ 1, p.status, kTimeoutMma, abort_flag)) break;
        tc_fence_after();
        const uint32_t d = tmem + acc * 256;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&full[stage], phase, p.status, kTimeoutMma, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * kStageBytes);
          const uint32_t sb = diag ? sa : sa + 16384;
          const int k16 = min(4, (K - kb * 64 + 15) / 16);  // the rest of the box is zero fill
          for (int k = 0; k < k16; ++k) {
            uint64_t da, db;
            if (p.phase == kGram) {
              da = umma_smem_desc(sa + k * 2048, 8192, 1024, 2);
              db = umma_smem_desc(sb + k * 2048, 8192, 1024, 2);
            } else {
              da = umma_desc_kmajor_sw128(sa + k * 32);
              db = umma_desc_kmajor_sw128(sb + k * 32);
            }
            umma_bf16_ss(d, da, db, idesc, (kb > 0 || k > 0) ? 1u : 0u);
          }
          umma_commit(&empty[stage]);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        umma_commit(&tfull[acc]);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
    }
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;
    float* tile = tiles + (warp - 2) * kTileFloats;
    const bool final_step = p.phase == kUpdate && p.it == p.steps - 1;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int t = blockIdx.x; t < items; t += gridDim.x) {
      const Item it = decode(p, t);
      const int tile_n = p.phase == kUpdate ? p.bn : 128;
      const int n0 = it.tj * tile_n, ncols = min(tile_n, p.ldz - n0);  // columns kept (padding included)
      const int rows = p.phase == kUpdate ? p.n : p.m;
      const int row = it.ti * 128 + q * 32 + lane;
      const bool row_ok = row < rows;
      float xi = p.f[it.mat] * (1.f / kZScale);
      for (int k = 0; k < p.it; ++k) xi *= p.a;
      if (!mbar_wait_warp(&tfull[acc], acc_phase, p.status, kTimeoutEpilogue, abort_flag)) break;
      tc_fence_after();
      const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16) + acc * 256;
      for (int c = half; c * 32 < ncols; c += 2) {
        uint32_t r[32];
        tmem_ld32(taddr + c * 32, r);
        tmem_wait_ld();
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
        const int col = n0 + c * 32, left = ncols - c * 32;  // left is a multiple of 8
        if (p.phase != kUpdate) {
          const int64_t at = (static_cast<int64_t>(it.mat) * p.m + row) * p.ldz + col;
          __half* dst = p.phase == kGram ? p.A : p.C;
          if (p.phase == kGram) {
            const float x2 = xi * xi;
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] *= x2;
          } else if (row_ok) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (8 * j < left) {
                float s[8];
                unpack8(*reinterpret_cast<const uint4*>(p.A + at + 8 * j), s);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[8 * j + i] = p.ba * s[i] + p.ca * v[8 * j + i];
              }
            }
          }
          if (row_ok) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (8 * j < left) *reinterpret_cast<uint4*>(dst + at + 8 * j) = pack8(v + 8 * j);
            if (it.ti != it.tj) {  // the mirrored tile: consecutive lanes are consecutive columns
              __half* mir = dst + (static_cast<int64_t>(it.mat) * p.m + col) * p.ldz + row;
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (col + i < p.m && i < left) mir[static_cast<int64_t>(i) * p.ldz] = __float2half_rn(v[i]);
            }
          }
        } else {
          const int64_t at = (static_cast<int64_t>(it.mat) * p.n + row) * p.ldz + col;
          if (row_ok) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (8 * j < left) {
                float h[8], l[8];
                unpack8(*reinterpret_cast<const uint4*>(p.zh + at + 8 * j), h);
                unpack8(*reinterpret_cast<const uint4*>(p.zl + at + 8 * j), l);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[8 * j + i] += h[i] + l[i];
              }
            }
          }
          if (!final_step) {
            if (row_ok) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                if (8 * j < left) {
                  const uint4 hi = pack8(v + 8 * j);
                  float h[8], l[8];
                  unpack8(hi, h);
#pragma unroll
                  for (int i = 0; i < 8; ++i) l[i] = v[8 * j + i] - h[i];
                  *reinterpret_cast<uint4*>(p.zh_out + at + 8 * j) = hi;
                  *reinterpret_cast<uint4*>(p.zl + at + 8 * j) = pack8(l);
                }
              }
            }
          } else {
            // the result in G's orientation: rows through shared memory (tall), or as they
            // lie, consecutive lanes being consecutive columns of a wide G
            const float xo = xi * p.a;
            const bool wide = p.rows < p.cols;
            const Sink sink = {p.out_type, p.out,
                               p.out_type == kOutMuon ? p.s.table[p.first + it.mat].off
                                                      : static_cast<int64_t>(it.mat) * p.rows * p.cols,
                               p.s.lr * lr_factor(p.s.adjust, p.rows, p.cols)};
            if (wide) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] *= xo;
              const int cnt = row_ok ? min(left, p.m - col) : 0;
              emit<16>(sink, p.s, static_cast<int64_t>(col) * p.n + row, p.n, cnt, v);
              emit<16>(sink, p.s, static_cast<int64_t>(col + 16) * p.n + row, p.n, cnt - 16, v + 16);
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i) tile[lane * 33 + i] = v[i] * xo;
              __syncwarp();
              const int r0 = it.ti * 128 + q * 32;
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = tile[i * 33 + lane];
              __syncwarp();
              const int cnt = col + lane < p.m && lane < left ? p.n - r0 : 0;
              emit<16>(sink, p.s, static_cast<int64_t>(r0) * p.m + col + lane, p.m, cnt, v);
              emit<16>(sink, p.s, static_cast<int64_t>(r0 + 16) * p.m + col + lane, p.m, cnt - 16, v + 16);
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[acc]);
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
  }
  // every MMA of this CTA was waited for by its epilogue (or the CTA has given up)
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------ one matrix per CTA
// Matrices that fit one SM run their whole step in one CTA, and a ragged set of them in one
// launch.  The iterate stays in fp32 in tensor memory, where the update's MMAs add to it in
// place (Z <- Z + Z C); its fp16 copy lies in shared memory once, as 128B-swizzled rows of 64
// columns, and serves the Gram product (read MN-major, the sum running over rows) and the
// update (read K-major).  A and then C take one 128-row tile beside it.  Nothing but the
// matrix itself and its result crosses memory.  The chain of 3 x steps dependent products
// bounds it: each is issued by one thread, waited for by all, read back by tcgen05.ld.
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

struct SingleParams {
  int first, rows, cols;
  Coeffs k;
  int out_type;
  void* out;
  StepArgs s;
  int* status;
};

template <int SRC>
__global__ void __launch_bounds__(kSingleThreads, 1) single_kernel(const void* __restrict__ g, SingleParams p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ uint64_t bar[1 + kSingleMaxTiles];
  __shared__ double red[16];
  __shared__ uint32_t tmem_slot;
  if (*reinterpret_cast<volatile int*>(p.status) != 0) return;
  int rows = p.rows, cols = p.cols;
  int64_t base, mbase = 0;
  float clip = 1.f;
  if constexpr (SRC == kSrcMuon) {
    if (step_rejected(p.s)) return;
    const Mat t = p.s.table[p.first + blockIdx.x];
    rows = static_cast<int>(t.rows);
    cols = static_cast<int>(t.cols);
    base = t.off;
    mbase = t.moff;
    clip = clip_factor(p.s);
  } else {
    base = static_cast<int64_t>(blockIdx.x) * rows * cols;
  }
  const Fit fit = single_fit(rows, cols);
  const bool wide = rows < cols;
  const int n = fit.n, m = fit.m, mp = fit.mp, tiles = fit.tiles, chunks = mp / 16;
  uint8_t* zh = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ac = zh + tiles * fit.panels * 16384;
  const int zpanel = tiles * 16384;  // bytes between two 64-column panels of Z

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int q = warp & 3, grp = warp >> 2;  // lane quarter; 16-column chunks are dealt to 4 groups
  float* stage = reinterpret_cast<float*>(zh) + warp * 32 * 17;
  uint32_t tmem_cols = 32;
  while (tmem_cols < static_cast<uint32_t>(fit.tmem)) tmem_cols *= 2;
  if (warp == 0) tmem_alloc(&tmem_slot, tmem_cols);
  if (threadIdx.x == 0) {
    for (int i = 0; i <= kSingleMaxTiles; ++i) mbar_init(&bar[i], 1);
    fence_barrier_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const uint32_t tlane = tmem + (static_cast<uint32_t>(q * 32) << 16);
  const int cl = lane & 15, rl = lane >> 4;  // a 16-column chunk in memory: two rows per warp access
  // this group's first (tile, chunk), and the one after
  auto first = [&](int& t, int& c) {
    t = 0;
    c = grp;
    while (c >= chunks) {
      c -= chunks;
      ++t;
    }
  };
  auto next = [&](int& t, int& c) {
    c += 4;
    while (c >= chunks) {
      c -= chunks;
      ++t;
    }
  };

  // the update's input, tall, raw, into tensor memory; its sum of squares
  double acc = 0.0;
  int t, c;
  for (first(t, c); t < tiles; next(t, c)) {
    const int c0 = c * 16, r0 = t * 128 + q * 32;
    float v[16];
    if (wide) {  // consecutive lanes are consecutive columns of G
      fetch<SRC, 16>(g, p.s, base, mbase, clip, static_cast<int64_t>(c0) * n + r0 + lane, n,
                     r0 + lane < n ? m - c0 : 0, v);
    } else {     // turned in shared memory
      fetch<SRC, 16>(g, p.s, base, mbase, clip, static_cast<int64_t>(r0 + rl) * m + c0 + cl, 2 * m,
                     c0 + cl < m ? (n - r0 - rl + 1) / 2 : 0, v);
#pragma unroll
      for (int i = 0; i < 16; ++i) stage[(2 * i + rl) * 17 + cl] = v[i];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = stage[lane * 17 + i];
      __syncwarp();
    }
    uint32_t r[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      acc += static_cast<double>(v[i]) * v[i];
      r[i] = __float_as_uint(v[i]);
    }
    tmem_st16(tlane + t * mp + c0, r);
  }
  tmem_wait_st();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if (lane == 0) red[warp] = acc;
  __syncthreads();
  acc = 0.0;
#pragma unroll
  for (int i = 0; i < 16; ++i) acc += red[i];
  float s0, s1, xi;
  z_scale(acc, p.k.eps, s0, s1, xi);
  xi *= 1.f / kZScale;

  // 16 columns of row r as fp16 in the swizzled rows at `panel0`
  auto put16 = [&](uint8_t* panel0, int pstride, int r, int c0, const float* v) {
    uint8_t* d = panel0 + (c0 >> 6) * pstride + r * 128;
    const int k = (c0 & 63) >> 3, x = r & 7;
    *reinterpret_cast<uint4*>(d + ((k ^ x) << 4)) = pack8(v);
    *reinterpret_cast<uint4*>(d + (((k + 1) ^ x) << 4)) = pack8(v + 8);
  };
  auto get16 = [&](const uint8_t* panel0, int pstride, int r, int c0, float* v) {
    const uint8_t* d = panel0 + (c0 >> 6) * pstride + r * 128;
    const int k = (c0 & 63) >> 3, x = r & 7;
    unpack8(*reinterpret_cast<const uint4*>(d + ((k ^ x) << 4)), v);
    unpack8(*reinterpret_cast<const uint4*>(d + (((k + 1) ^ x) << 4)), v + 8);
  };
  auto ld16 = [&](uint32_t addr, float* v) {
    uint32_t r[16];
    tmem_ld16(addr, r);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
  };

  const uint32_t zs = smem_u32(zh), as = smem_u32(ac);
  const uint32_t d_a = tmem + tiles * mp;  // A's (and A^2's) accumulator
  const uint32_t idesc_mn = idesc_f16(mp, true), idesc_k = idesc_f16(mp, false);
  // with one panel the MMA's rows 64..127 are padding: let them read the next rows
  const uint32_t lbo = fit.panels == 2 ? zpanel : 1024;
  const int row = q * 32 + lane;
  const Sink sink = {p.out_type, p.out, base, p.s.lr * lr_factor(p.s.adjust, rows, cols)};
  bool ok = true;
  // All that the threads wrote to shared memory is there for the MMAs that one thread issues
  // next; false once a wait of any thread has run out.
  auto publish = [&]() -> bool {
    tc_fence_before();
    fence_proxy_async_smem();
    ok = !__syncthreads_or(!ok);
    tc_fence_after();
    return ok;
  };
  // A += Z^T Z over the rows of tile t
  auto gram = [&](int t) {
    if (warp == 0 && elect_one()) {
      const int k1 = min(8, (n - t * 128 + 15) / 16);
      for (int k = 0; k < k1; ++k) {
        const uint64_t d = umma_smem_desc(zs + (t * 8 + k) * 2048, lbo, 1024, 2);
        umma_bf16_ss(d_a, d, d, idesc_mn, t > 0 || k > 0 ? 1u : 0u);
      }
      if (t == tiles - 1) umma_commit(&bar[0]);
    }
    __syncwarp();
  };

  // the fp16 copy of Z_0 (and Z_0 itself, scaled in place)
  for (first(t, c); t < tiles; next(t, c)) {
    float v[16];
    uint32_t r[16];
    ld16(tlane + t * mp + c * 16, v);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      v[i] = v[i] * s0 * s1;
      r[i] = __float_as_uint(v[i]);
    }
    tmem_st16(tlane + t * mp + c * 16, r);
    put16(zh, zpanel, t * 128 + q * 32 + lane, c * 16, v);
  }
  tmem_wait_st();
  if (publish()) {
    for (int i = 0; i < tiles; ++i) gram(i);
    for (int it = 0; it < p.k.steps; ++it) {
      // A = xi^2 Z^T Z
      ok = mbar_wait_warp(&bar[0], 0, p.status, kTimeoutEpilogue, nullptr);
      tc_fence_after();
      const float x2 = xi * xi;
      for (int j = grp; j < chunks; j += 4) {
        float v[16];
        ld16(tlane + tiles * mp + j * 16, v);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = (row < m && j * 16 + i < m) ? v[i] * x2 : 0.f;
        put16(ac, 16384, row, j * 16, v);
      }
      if (!publish()) break;
      if (warp == 0 && elect_one()) {
        for (int k = 0; k < chunks; ++k) {
          const uint64_t d = umma_desc_kmajor_sw128(as + (k >> 2) * 16384 + (k & 3) * 32);
          umma_bf16_ss(d_a, d, d, idesc_k, k > 0 ? 1u : 0u);
        }
        umma_commit(&bar[0]);
      }
      __syncwarp();
      // C = (b A + c A^2) / a
      ok = mbar_wait_warp(&bar[0], 1, p.status, kTimeoutEpilogue, nullptr);
      tc_fence_after();
      for (int j = grp; j < chunks; j += 4) {
        float v[16], s[16];
        ld16(tlane + tiles * mp + j * 16, v);
        get16(ac, 16384, row, j * 16, s);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          v[i] = (row < m && j * 16 + i < m) ? p.k.ba * s[i] + p.k.ca * v[i] : 0.f;
        put16(ac, 16384, row, j * 16, v);
      }
      if (!publish()) break;
      // Z += Z C, tile by tile
      if (warp == 0 && elect_one()) {
        for (int i = 0; i < tiles; ++i) {
          for (int k = 0; k < chunks; ++k) {
            const uint64_t da = umma_desc_kmajor_sw128(zs + (k >> 2) * zpanel + i * 16384 + (k & 3) * 32);
            const uint64_t db = umma_desc_kmajor_sw128(as + (k >> 2) * 16384 + (k & 3) * 32);
            umma_bf16_ss(tmem + i * mp, da, db, idesc_k, 1u);
          }
          umma_commit(&bar[1 + i]);
        }
      }
      __syncwarp();
      xi *= p.k.a;
      if (it == p.k.steps - 1) break;
      // the fp16 copy of each finished tile, and its share of the next A behind it
      first(t, c);
      for (int i = 0; i < tiles; ++i) {
        ok = ok && mbar_wait_warp(&bar[1 + i], it & 1, p.status, kTimeoutEpilogue, nullptr);
        tc_fence_after();
        for (; t == i; next(t, c)) {
          float v[16];
          ld16(tlane + t * mp + c * 16, v);
          put16(zh, zpanel, t * 128 + q * 32 + lane, c * 16, v);
        }
        if (!publish()) break;  // every warp's part of the tile
        gram(i);
      }
      if (!ok) break;
    }
    // the result: the operands' place is free once the last tile is done
    ok = ok && mbar_wait_warp(&bar[tiles], (p.k.steps - 1) & 1, p.status, kTimeoutEpilogue, nullptr);
    tc_fence_after();
    if (ok) {
      for (first(t, c); t < tiles; next(t, c)) {
        const int c0 = c * 16, r0 = t * 128 + q * 32;
        float v[16];
        ld16(tlane + t * mp + c0, v);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] *= xi;
        if (wide) {
          emit<16>(sink, p.s, static_cast<int64_t>(c0) * n + r0 + lane, n, r0 + lane < n ? m - c0 : 0, v);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) stage[lane * 17 + i] = v[i];
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = stage[(2 * i + rl) * 17 + cl];
          __syncwarp();
          emit<16>(sink, p.s, static_cast<int64_t>(r0 + rl) * m + c0 + cl, 2 * m,
                   c0 + cl < m ? (n - r0 - rl + 1) / 2 : 0, v);
        }
      }
    }
  }
  // every product was waited for (or a wait has run out)
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
}

// ------------------------------------------------------------------ host
static CUtensorMap map_f16(const __half* base, int cols, int rows, int ld, int batch, int box_rows) {
  const int64_t dims[3] = {cols, rows, batch};
  const int64_t strides[2] = {static_cast<int64_t>(ld) * 2, static_cast<int64_t>(ld) * rows * 2};
  const int box[3] = {64, box_rows, 1};
  return make_tmap_nd_bf16(const_cast<__half*>(base), 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_DATA_TYPE_FLOAT16);
}

static int64_t align_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }


// Orthogonalise `batch` matrices of one shape: Newton-Schulz output into `out`, or with
// kSrcMuon / kOutMuon the whole step.  Work buffers come from PyTorch's allocator (per call
// and stream, so concurrent calls and captured graphs never share them).
static void run_group(int src, const void* g, int out_type, void* out, const StepArgs& s, int first, int batch,
                      int rows, int cols, const Coeffs& k, const torch::Tensor& status, const at::TensorOptions& dev) {
  const int n = std::max(rows, cols), m = std::min(rows, cols), ldz = static_cast<int>(align_up(m, 8));
  const int64_t numel = static_cast<int64_t>(rows) * cols;
  const int slices = static_cast<int>(std::min<int64_t>(64, (numel + 4095) / 4096));
  const int64_t z_bytes = align_up(static_cast<int64_t>(batch) * n * ldz * 2, 1024);
  const int64_t a_bytes = align_up(static_cast<int64_t>(batch) * m * ldz * 2, 1024);
  const int64_t p_bytes = align_up(static_cast<int64_t>(batch) * slices * 8, 1024);
  const int64_t f_bytes = align_up(static_cast<int64_t>(batch) * 4, 1024);
  auto ws = torch::empty({3 * z_bytes + 2 * a_bytes + p_bytes + f_bytes}, dev.dtype(at::kByte));
  uint8_t* w = ws.data_ptr<uint8_t>();
  __half* z[2] = {reinterpret_cast<__half*>(w), reinterpret_cast<__half*>(w + z_bytes)};
  __half* zl = reinterpret_cast<__half*>(w + 2 * z_bytes);
  __half* A = reinterpret_cast<__half*>(w + 3 * z_bytes);
  __half* C = reinterpret_cast<__half*>(w + 3 * z_bytes + a_bytes);
  double* partial = reinterpret_cast<double*>(w + 3 * z_bytes + 2 * a_bytes);
  float* f = reinterpret_cast<float*>(w + 3 * z_bytes + 2 * a_bytes + p_bytes);
  auto stream = at::cuda::getCurrentCUDAStream();
  const int n_sm = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;

  const dim3 tiles(static_cast<unsigned>(((rows + 63) / 64) * ((cols + 63) / 64)), batch);
#define NORI_MUON_SRC(S)                                                                                           \
  norm_kernel<S><<<dim3(slices, batch), 256, 0, stream>>>(g, s, first, numel, partial);                          \
  C10_CUDA_KERNEL_LAUNCH_CHECK();                                                                                  \
  scale_kernel<S><<<tiles, 256, 0, stream>>>(g, s, first, rows, cols, slices, partial, k.eps, z[0], zl, ldz, f);   \
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (src == kSrcF32) {
    NORI_MUON_SRC(kSrcF32)
  } else if (src == kSrcBF16) {
    NORI_MUON_SRC(kSrcBF16)
  } else if (src == kSrcF16) {
    NORI_MUON_SRC(kSrcF16)
  } else {
    NORI_MUON_SRC(kSrcMuon)
  }
#undef NORI_MUON_SRC

  const int nb = (m + 255) / 256;
  NsParams p{};
  p.n = n;
  p.m = m;
  p.ldz = ldz;
  p.batch = batch;
  p.bn = static_cast<int>(align_up((m + nb - 1) / nb, 16));
  p.steps = k.steps;
  p.a = k.a;
  p.ba = k.ba;
  p.ca = k.ca;
  p.zl = zl;
  p.A = A;
  p.C = C;
  p.f = f;
  p.out_type = out_type;
  p.out = out;
  p.rows = rows;
  p.cols = cols;
  p.first = first;
  p.s = s;
  p.status = status.data_ptr<int>();
  const CUtensorMap mz[2] = {map_f16(z[0], m, n, ldz, batch, 64), map_f16(z[1], m, n, ldz, batch, 64)};
  const CUtensorMap ma = map_f16(A, m, m, ldz, batch, 64), mc = map_f16(C, m, m, ldz, batch, p.bn);
  C10_CUDA_CHECK(cudaFuncSetAttribute(product_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
  const int nt = (m + 127) / 128;
  for (int it = 0; it < k.steps; ++it) {
    p.it = it;
    p.zh = z[it & 1];
    p.zh_out = z[(it & 1) ^ 1];
    for (int ph = 0; ph < 3; ++ph) {
      p.phase = ph;
      const int64_t items =
          static_cast<int64_t>(batch) * (ph == kUpdate ? (n + 127) / 128 * ((m + p.bn - 1) / p.bn) : nt * (nt + 1) / 2);
      const int grid = static_cast<int>(std::min<int64_t>(items, persistent_sms(n_sm)));
      product_kernel<<<grid, kThreads, kSmemBytes, stream>>>(mz[it & 1], ma, mc, p);
      C10_CUDA_KERNEL_LAUNCH_CHECK();
    }
  }
}

// Matrices first .. first + count of a set that all fit one CTA; `smem` is the largest need.
static void run_single(int src, const void* g, int out_type, void* out, const StepArgs& s, int64_t first,
                       int64_t count, int rows, int cols, int smem, const Coeffs& k, const torch::Tensor& status) {
  SingleParams p{};
  p.first = static_cast<int>(first);
  p.rows = rows;
  p.cols = cols;
  p.k = k;
  p.out_type = out_type;
  p.out = out;
  p.s = s;
  p.status = status.data_ptr<int>();
  auto kernel = src == kSrcF32    ? single_kernel<kSrcF32>
                : src == kSrcBF16 ? single_kernel<kSrcBF16>
                : src == kSrcF16  ? single_kernel<kSrcF16>
                                  : single_kernel<kSrcMuon>;
  smem += 1024;
  C10_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 221 * 1024));
  kernel<<<static_cast<unsigned>(count), kSingleThreads, smem, at::cuda::getCurrentCUDAStream()>>>(g, p);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

constexpr int64_t kMaxDim = 1 << 20, kMaxBatch = 65535;

static Coeffs make_coeffs(int64_t steps, double eps, const std::vector<double>& c, const char* who) {
  TORCH_CHECK(steps >= 1 && steps <= 64, who, ": steps must be in 1..64");
  TORCH_CHECK(eps >= 0.0, who, ": eps must not be negative");
  TORCH_CHECK(c.size() == 3 && c[0] > 0.0, who, ": three coefficients with a positive first one expected");
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

// O = Newton-Schulz(G) for contiguous G [batch, rows, cols] (fp32, bf16 or fp16) into out.
void newton_schulz(const torch::Tensor& g, torch::Tensor& out, int64_t steps, double eps, std::vector<double> coeffs,
                   const torch::Tensor& status) {
  using namespace muon;
  TORCH_CHECK(g.is_cuda() && g.dim() == 3 && g.is_contiguous(), "newton_schulz: contiguous CUDA [batch, rows, cols]");
  TORCH_CHECK(out.device() == g.device() && out.is_contiguous() && out.sizes() == g.sizes(),
              "newton_schulz: out must be contiguous, of g's shape and device");
  auto kind = [](const torch::Tensor& t, const char* what) {
    const auto s = t.scalar_type();
    TORCH_CHECK(s == at::kFloat || s == at::kBFloat16 || s == at::kHalf, "newton_schulz: ", what,
                " must be fp32, bf16 or fp16");
    return s == at::kFloat ? 0 : s == at::kBFloat16 ? 1 : 2;
  };
  const int src = kind(g, "g"), dst = kind(out, "out");
  const Coeffs k = make_coeffs(steps, eps, coeffs, "newton_schulz");
  TORCH_CHECK(g.size(1) < kMaxDim && g.size(2) < kMaxDim, "newton_schulz: at most 2^20 rows and columns");
  if (g.numel() == 0) return;
  const at::cuda::CUDAGuard guard(g.device());
  const int64_t numel = g.size(1) * g.size(2);
  const Fit fit = single_fit(static_cast<int>(g.size(1)), static_cast<int>(g.size(2)));
  if (fit.ok) {
    TORCH_CHECK(g.size(0) <= INT_MAX, "newton_schulz: at most 2^31 - 1 matrices");
    run_single(src, g.data_ptr(), dst, out.data_ptr(), StepArgs{}, 0, g.size(0), static_cast<int>(g.size(1)),
               static_cast<int>(g.size(2)), fit.smem, k, status);
    return;
  }
  for (int64_t b0 = 0; b0 < g.size(0); b0 += kMaxBatch) {
    const int nb = static_cast<int>(std::min(kMaxBatch, g.size(0) - b0));
    run_group(src, static_cast<const char*>(g.data_ptr()) + b0 * numel * g.element_size(), dst,
              static_cast<char*>(out.data_ptr()) + b0 * numel * out.element_size(), StepArgs{}, 0, nb,
              static_cast<int>(g.size(1)), static_cast<int>(g.size(2)), k, status, g.options());
  }
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
  // runs of groups whose matrices fit one CTA go in one launch
  int64_t run_first = 0, run_count = 0;
  int run_smem = 0;
  auto flush = [&]() {
    if (run_count > 0)
      run_single(kSrcMuon, nullptr, kOutMuon, nullptr, s, run_first, run_count, 0, 0, run_smem, k, status);
    run_count = 0;
    run_smem = 0;
  };
  for (size_t i = 0; i + 3 < groups.size(); i += 4) {
    const Fit fit = single_fit(static_cast<int>(groups[i + 2]), static_cast<int>(groups[i + 3]));
    if (fit.ok) {
      if (run_count == 0) run_first = groups[i];
      run_count += groups[i + 1];
      run_smem = std::max(run_smem, fit.smem);
      continue;
    }
    flush();
    for (int64_t b0 = 0; b0 < groups[i + 1]; b0 += kMaxBatch)
      run_group(kSrcMuon, nullptr, kOutMuon, nullptr, s, static_cast<int>(groups[i] + b0),
                static_cast<int>(std::min(kMaxBatch, groups[i + 1] - b0)), static_cast<int>(groups[i + 2]),
                static_cast<int>(groups[i + 3]), k, status, data.options());
  }
  flush();
}

// Whether a matrix of this shape runs its whole step in one CTA.
bool muon_single_cta(int64_t rows, int64_t cols) {
  return muon::single_fit(static_cast<int>(rows), static_cast<int>(cols)).ok;
}

}  // namespace nori
