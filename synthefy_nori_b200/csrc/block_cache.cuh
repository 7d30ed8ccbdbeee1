// Shared by the kernels of the context cache in 8 bits with block scales: what they are given,
// and the exact widening of stored values to fp16.
//
// Storage: rows of W = D up to a multiple of 8 bytes, [batch, heads, capacity, W], int8 or e4m3,
// one fp32 scale per (sequence, head, block of rows); a value is q * scale.  The capacity is a
// multiple of 128 rows and every row of 8 bytes' alignment, so a tile of 128 rows is one
// contiguous, 16-byte aligned piece of memory for every width (no padding to TMA's strides).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace nori {
namespace bc {

constexpr int kMaxWidth = 64;  // head width, as in the framework's other attention kernels
constexpr int kTile = 128;     // rows of a key tile; the capacity is a multiple

enum Float : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

struct View {
  uint8_t *k, *v;
  float *k_scale, *v_scale;
  int batch, heads;
  int64_t cap;
  int width, stored;  // D, W
  int block_log2;
  bool fp8;
  __host__ __device__ __forceinline__ int64_t blocks() const { return cap >> block_log2; }
  __device__ __forceinline__ uint8_t* data(int which) const { return which ? v : k; }
  __device__ __forceinline__ float* scale(int which) const { return which ? v_scale : k_scale; }
};

// [b0, b1, n, h, d] with contiguous d; sequence b = b0 * n1 + b1
struct Rows {
  void* p;
  int64_t s0, s1, sn, sh;
  int n1;
  __device__ __forceinline__ int64_t offset(int b, int64_t n, int h) const {
    return (b / n1) * s0 + (b % n1) * s1 + n * sn + h * sh;
  }
};

// How many bytes of 16-bit rows can be read and written at a time: 16, 4 or 2.
inline int access_bytes(const Rows& r, int width) {
  for (int a : {8, 2})
    if (width % a == 0 && reinterpret_cast<uintptr_t>(r.p) % (2 * a) == 0 && r.s0 % a == 0 && r.s1 % a == 0 &&
        r.sn % a == 0 && r.sh % a == 0)
      return 2 * a;
  return 2;
}

// One value for all sequences or one of each, on the device.
struct PerSequence {
  const int* dev;
  int64_t all;
  __device__ __forceinline__ int64_t at(int b) const { return dev != nullptr ? dev[b] : all; }
};

struct Attention {
  Rows q, o;
  int type;  // of q and o (kBF16, kF16)
  View c;
  PerSequence length;
  int64_t n;        // query rows
  int group;        // query heads of one K/V head
  int64_t rows;     // n * group: the rows that read one K/V head; this call's are first .. rows - 1
  int64_t first;
  float scale_log2; // softmax scale * log2(e)
  float* lse;       // [batch, query heads, n] or null
  int64_t whole;    // cells, a (sequence, K/V head) and a tile of query rows each, that one CTA takes whole
  int splits;       // of the key range of the others
  int cluster;      // splits that are joined on the way (kernel for few rows), a divisor of splits
  float* part_o;    // [cells - whole, parts, tile rows, 64], unnormalised; parts = splits / cluster
  float2* part_ml;  // [cells - whole, parts, tile rows] (maximum, sum)
  int* status;
};

// Weights are 2^(t - m + kLift): fp16 keeps 11 bits of them down to 2^-21 of the largest, and below that its
// values are 2^-31 of the largest apart (a million keys off by half of that: 2^-12 at most).  A maximum that
// lags by up to kLazy (no rescale of the sums) stays below fp16's largest value.  4 and 11 instead rescale a
// dozen times a row where scores spread by a few units: 1024 rows x 10,000 733 us for 698.
constexpr float kLift = 7.f;
constexpr float kLazy = 8.f;

#ifdef __CUDACC__
// A contiguous piece (16-byte aligned, a multiple of 16 bytes) to shared memory; arrives on `bar`.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src), "r"(bytes), "r"(static_cast<uint32_t>(__cvta_generic_to_shared(bar)))
               : "memory");
}

__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Four codes (bytes of x, int8 ones biased by 128) -> two fp16 pairs, exact.
// int8: 0x64uu is the fp16 1024 + u, minus 1152.  e4m3: the conversion instruction (the same by shifts
// and masks is three times as many instructions: 220 for 180 us a row x 168 x 50,000).
template <bool FP8>
__device__ __forceinline__ void widen(uint32_t x, uint32_t& lo, uint32_t& hi) {
  if (FP8) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(x));
  } else {
    lo = hsub2(__byte_perm(x, 0x64646464u, 0x4140), 0x64806480u);
    hi = hsub2(__byte_perm(x, 0x64646464u, 0x4342), 0x64806480u);
  }
}
template <bool FP8>
__device__ __forceinline__ uint32_t biased(uint32_t x) {
  return FP8 ? x : x ^ 0x80808080u;
}

// A power of two that brings a row's largest magnitude near 2^14 and its inverse (both normal
// numbers); a row with an infinity or a NaN gets a NaN inverse.
__device__ __forceinline__ void row_scale(float top, float& up, float& down) {
  if (!(top < INFINITY)) {
    up = 1.f;
    down = __uint_as_float(0x7fc00000u);
    return;
  }
  int e = 14 - (static_cast<int>(__float_as_uint(top) >> 23) - 127);
  e = min(max(e, -120), 120);
  up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
  down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
}

// The V scale that a block counts with: one whose log2 and inverse are finite (a block that was never written has
// scale 0 and holds zeros), and 2^-100 of the largest so far at least.  Weights carry the scale (t = score + log2 s_v)
// and the sum divides by it, so keys of a block whose values are tiny beside the largest can be all of the sum and
// nothing of the result: with a log2 further below, 2^t would leave fp32's range.  The sum does not mind which scale
// it is; the result is off by 2^-100 of the largest value at most.
constexpr float kLeastScale = 0x1p-80f;  // (written ones are 2^-49 or more)
__device__ __forceinline__ void raise_floor(float& least, float s) { least = fmaxf(least, s * 0x1p-100f); }  // (not by a NaN)
__device__ __forceinline__ float safe_scale(float s, float least) {  // a NaN stays one
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(s), "f"(least));
  return r;
}

// A sum times h^2 = 2^d, d <= 0, in two steps: 2^d alone may lie below fp32's range where the sum, which divides by
// scales down to 2^-47, lies as far above 1.
__device__ __forceinline__ float lowered(float sum, float h) { return sum * h * h; }

// The natural log-sum-exp of a row from its maximum and its sum (which carries kLift).
__device__ __forceinline__ float row_lse(float m, float l) {
  return l != 0.f ? 0.6931471805599453f * (m + log2f(l) - kLift) : -INFINITY;
}
#endif

cudaError_t launch_write(const View& c, const Rows& k, const Rows& v, int type, const PerSequence& start,
                         const PerSequence& count, int64_t n, cudaStream_t stream);
cudaError_t launch_read(const View& c, void* k, void* v, int type, int64_t start, int64_t n, cudaStream_t stream);
// rows of a tile of the kernel for few rows, and how many of its CTAs an SM holds
int few_tile_rows(int64_t rows);
int few_resident(int64_t rows);
// beside: it may start while the kernel before it on the stream, which it does not depend on, still runs
cudaError_t launch_few(const Attention& a, bool beside, cudaStream_t stream);
// rows of a tile pair of the kernel for many rows; one CTA per SM
constexpr int kPairRows = 256;
cudaError_t launch_tc(const Attention& a, cudaStream_t stream);
cudaError_t launch_combine(const Attention& a, int tile_rows, cudaStream_t stream);

}  // namespace bc
}  // namespace nori
