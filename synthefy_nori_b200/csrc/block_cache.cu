// Context cache in 8 bits with a scale for each block of rows and head: rows quantised as they
// are written, and read back.
//
// Write.  For one (sequence, head, block) of K or V, with Q = 127 (int8) or 448 (e4m3):
//   s  = max(max(|x| of the block's new rows, 1e-12) / Q, s_old)   s_old where earlier rows stay
//   q  = round(x * (1 / s)),   rows that stay: q' = round(q * (s_old * (1 / s)))
// every operation in fp32 with one rounding, ties to even.  A block with an infinity or a NaN gets
// a NaN scale: all of it reads as NaN, rather than as something finite.
// A CTA takes 64 rows (128 for blocks of 128) of one (sequence, head), K and V, twice as many threads a
// block as it has rows, its new rows in registers between the maximum and the rounding: each new value
// is read once (2 bytes, or 4) and written once (1 byte).  All heads of a row are neighbouring CTAs, so the
// pieces of a cache line that different heads own are read together.  168 x 2048 x 8 x 56 bf16 take
// 155 us, 6.0 TB/s; a CTA each for K and V spent its instructions on finding its place (222 us, issue slots
// 81% taken), CTAs of 128 rows for every block length left too few loads in flight (275 us).
//
// Read.  x = q * s, rounded once to the result's type: 8 values a thread and step.
//
// Reference counterpart: per-vector int8 quantisation (kv_cache_scaling.py:29-41).
#include "block_cache.cuh"

namespace nori {
namespace bc {
namespace {

constexpr int write_rows(int block) { return block > 64 ? block : 64; }  // of a CTA

template <int TYPE>
struct Raw;  // eight values as they were loaded
template <>
struct Raw<kF32> {
  uint32_t r[8];
};
template <>
struct Raw<kBF16> {
  uint32_t r[4];
};
template <>
struct Raw<kF16> {
  uint32_t r[4];
};

// Eight values from p, the first `have` of them there (the rest 0), in pieces of ALIGN values.
template <int TYPE, int ALIGN>
__device__ __forceinline__ Raw<TYPE> load8(const void* base, int64_t at, int have) {
  Raw<TYPE> x;
  if constexpr (TYPE == kF32) {
    const uint32_t* p = static_cast<const uint32_t*>(base) + at;
    if constexpr (ALIGN >= 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4 v = 4 * i < have ? __ldg(reinterpret_cast<const uint4*>(p) + i) : make_uint4(0, 0, 0, 0);
        x.r[4 * i] = v.x, x.r[4 * i + 1] = v.y, x.r[4 * i + 2] = v.z, x.r[4 * i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x.r[i] = i < have ? __ldg(p + i) : 0u;
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(base) + at;
    if constexpr (ALIGN == 8) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
      x.r[0] = v.x, x.r[1] = v.y, x.r[2] = v.z, x.r[3] = v.w;
    } else if constexpr (ALIGN == 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint2 v = 4 * i < have ? __ldg(reinterpret_cast<const uint2*>(p) + i) : make_uint2(0, 0);
        x.r[2 * i] = v.x, x.r[2 * i + 1] = v.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = 2 * i < have ? __ldg(p + 2 * i) : 0u, b = 2 * i + 1 < have ? __ldg(p + 2 * i + 1) : 0u;
        x.r[i] = a | b << 16;
      }
    }
  }
  return x;
}

template <int TYPE>
__device__ __forceinline__ float value(const Raw<TYPE>& x, int i) {
  if constexpr (TYPE == kF32) return __uint_as_float(x.r[i]);
  const uint32_t w = x.r[i / 2];
  if constexpr (TYPE == kBF16) return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
  return __half2float(__ushort_as_half(static_cast<uint16_t>(i & 1 ? w >> 16 : w)));
}

// The largest magnitude so far as bits (ordered like the magnitudes, infinities and NaN on top):
// 16-bit types in both halves of a word.
template <int TYPE>
__device__ __forceinline__ uint32_t top_bits(const Raw<TYPE>& x, uint32_t m) {
  if constexpr (TYPE == kF32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, x.r[i] & 0x7fffffffu);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __vmaxu2(m, x.r[i] & 0x7fff7fffu);
  }
  return m;
}
template <int TYPE>
__device__ __forceinline__ float top_value(uint32_t m) {
  if constexpr (TYPE == kF32) return __uint_as_float(m);
  const uint32_t h = max(m & 0xffffu, m >> 16);
  if constexpr (TYPE == kBF16) return __uint_as_float(h << 16);
  return __half2float(__ushort_as_half(static_cast<uint16_t>(h)));
}

// Four values as codes: round to nearest even.  |y| <= Q (1 + 2^-22), so int8 needs no clamp.
template <bool FP8>
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  if (FP8) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
  }
  // adding 1.5 * 2^23 leaves the rounded integer in the low bits (two's complement)
  constexpr float kRound = 12582912.f;
  const uint32_t x = __float_as_uint(__fadd_rn(a, kRound)), y = __float_as_uint(__fadd_rn(b, kRound));
  const uint32_t z = __float_as_uint(__fadd_rn(c, kRound)), w = __float_as_uint(__fadd_rn(d, kRound));
  return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
}

template <bool FP8>
__device__ __forceinline__ float code_value(uint32_t byte) {
  if (FP8) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3);
    return __half2float(*reinterpret_cast<const __half*>(&h));
  }
  return static_cast<float>(static_cast<int8_t>(byte));
}

// Row and eight-column unit of the i-th piece of a block (i < 1024, up to 8 units a row).
struct Pieces {
  int units;
  uint32_t inverse;  // 65536 / units + 1
  __device__ __forceinline__ void at(int i, int& row, int& unit) const {
    row = static_cast<int>(static_cast<uint32_t>(i) * inverse >> 16);
    unit = i - row * units;
  }
};

template <int TYPE, bool FP8, int ALIGN, int BLOCK>
__global__ void __launch_bounds__(2 * write_rows(BLOCK))
    write_kernel(View c, Rows rk, Rows rv, PerSequence start, PerSequence count, int64_t n, uint32_t per_seq,
                 Pieces pieces) {
  constexpr int kRows = write_rows(BLOCK), kGroup = 2 * BLOCK, kEach = kMaxWidth / 16;  // threads of a block, pieces (of up to 8 a row) of a thread
  constexpr float kTop = FP8 ? 448.f : 127.f;
  uint32_t rest = blockIdx.x / static_cast<uint32_t>(c.heads);  // (32 bits: a division in 64 takes longer than the loads)
  const int h = static_cast<int>(blockIdx.x - rest * static_cast<uint32_t>(c.heads));
  const int b = static_cast<int>(rest / per_seq);
  const int64_t j = rest - static_cast<uint32_t>(b) * per_seq;
  const int64_t first = start.at(b), m = min(max(count.at(b), int64_t{0}), n);
  const int64_t lo = max(first, int64_t{0}), hi = min(first + m, c.cap);  // rows of the cache that get values
  const int t = threadIdx.x % kGroup;
  const int64_t row0 = (lo / kRows + j) * kRows + threadIdx.x / kGroup * BLOCK;  // of this thread's block
  // its rows r0 .. r1 - 1 get values (none where it is not touched)
  const int r0 = static_cast<int>(min(max(lo - row0, int64_t{0}), int64_t{BLOCK}));
  const int r1 = static_cast<int>(min(max(hi - row0, int64_t{0}), int64_t{BLOCK}));
  const bool touched = r0 < r1;
  const int64_t bh = static_cast<int64_t>(b) * c.heads + h;
  const int64_t dst_at = (bh * c.cap + row0) * c.stored, scale_at = bh * c.blocks() + (row0 >> c.block_log2);

  // K, then V: all their values in flight together
  Raw<TYPE> x[2][kEach];
  uint32_t top[2] = {0, 0};
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const Rows& src = w ? rv : rk;
    const int64_t from = src.offset(b, row0 - first, h);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      int row, u;
      pieces.at(t + e * kGroup, row, u);
      if (row >= r0 && row < r1) x[w][e] = load8<TYPE, ALIGN>(src.p, from + row * src.sn + u * 8, c.width - u * 8);
    }
  }
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      int row, u;
      pieces.at(t + e * kGroup, row, u);
      if (row >= r0 && row < r1) top[w] = top_bits<TYPE>(x[w][e], top[w]);
    }
  // over the block: magnitudes order like their bits
  float old[2] = {0.f, 0.f};
  if (touched && r0 > 0) old[0] = c.k_scale[scale_at], old[1] = c.v_scale[scale_at];  // rows before r0 stay
  __shared__ uint32_t tops[2][2 * kRows / 32];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    top[w] = __reduce_max_sync(0xffffffffu, __float_as_uint(top_value<TYPE>(top[w])));
    if (threadIdx.x % 32 == 0) tops[w][threadIdx.x / 32] = top[w];
  }
  __syncthreads();
  if (!touched) return;
  const int w0 = threadIdx.x / kGroup * (kGroup / 32);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
#pragma unroll
    for (int i = 0; i < kGroup / 32; ++i) top[w] = max(top[w], tops[w][w0 + i]);
    const float amax = __uint_as_float(top[w]), was = old[w];
    float s = __fdiv_rn(fmaxf(amax, 1e-12f), kTop);
    s = was > s ? was : s;
    if (!(amax < INFINITY) || was != was) s = __uint_as_float(0x7fc00000u);
    const float inv = __frcp_rn(s);
    uint8_t* dst = c.data(w) + dst_at;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      int row, u;
      pieces.at(t + e * kGroup, row, u);
      if (row >= r0 && row < r1) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = __fmul_rn(value<TYPE>(x[w][e], i), inv);
        // (W = 8 units: piece t + e * kGroup of the block lies at 8 times that)
        *reinterpret_cast<uint2*>(dst + (t + e * kGroup) * 8) =
            make_uint2(codes4<FP8>(y[0], y[1], y[2], y[3]), codes4<FP8>(y[4], y[5], y[6], y[7]));
      }
    }
    if (r0 > 0 && s != was) {  // the rows that stay, under the new scale
      const float ratio = __fmul_rn(was, inv);
#pragma unroll 1
      for (int i = t; i < r0 * pieces.units; i += kGroup) {
        uint2* p = reinterpret_cast<uint2*>(dst) + i;
        const uint2 q = *p;
        float y[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          y[k] = __fmul_rn(code_value<FP8>(((k < 4 ? q.x : q.y) >> 8 * (k & 3)) & 0xffu), ratio);
        *p = make_uint2(codes4<FP8>(y[0], y[1], y[2], y[3]), codes4<FP8>(y[4], y[5], y[6], y[7]));
      }
    }
    if (t == 0) c.scale(w)[scale_at] = s;
  }
}

// ------------------------------------------------------------------ read back
constexpr int kReadThreads = 256, kReadEach = 4;
constexpr int kReadRows = kReadThreads * kReadEach / (kMaxWidth / 8);  // rows of a CTA

template <int TYPE, int ALIGN>
__device__ __forceinline__ void store8(void* base, int64_t at, const float (&y)[8], int have) {
  if constexpr (TYPE == kF32) {
    float* p = static_cast<float*>(base) + at;
    if constexpr (ALIGN >= 4) {
      *reinterpret_cast<float4*>(p) = make_float4(y[0], y[1], y[2], y[3]);
      if (have > 4) *reinterpret_cast<float4*>(p + 4) = make_float4(y[4], y[5], y[6], y[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < have) p[i] = y[i];
    }
  } else {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (TYPE == kBF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(y[2 * i], y[2 * i + 1]);
        r[i] = *reinterpret_cast<const uint32_t*>(&v);
      } else {
        const __half2 v = __floats2half2_rn(y[2 * i], y[2 * i + 1]);
        r[i] = *reinterpret_cast<const uint32_t*>(&v);
      }
    }
    uint16_t* p = static_cast<uint16_t*>(base) + at;
    if constexpr (ALIGN == 8) {
      *reinterpret_cast<uint4*>(p) = make_uint4(r[0], r[1], r[2], r[3]);
    } else if constexpr (ALIGN == 4) {
      *reinterpret_cast<uint2*>(p) = make_uint2(r[0], r[1]);
      if (have > 4) *reinterpret_cast<uint2*>(p + 4) = make_uint2(r[2], r[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < have) p[i] = static_cast<uint16_t>(r[i / 2] >> 16 * (i & 1));
    }
  }
}

// k, v [batch, heads, n, D]; one CTA: kReadRows rows of one (sequence, head)
template <int TYPE, bool FP8, int ALIGN>
__global__ void __launch_bounds__(kReadThreads)
    read_kernel(View c, void* k, void* v, int64_t start, int64_t n, uint32_t chunks, Pieces pieces) {
  const uint32_t unit = blockIdx.x / chunks, chunk = blockIdx.x - unit * chunks;
  const int which = static_cast<int>(unit & 1);
  const int64_t bh = unit >> 1, row0 = static_cast<int64_t>(chunk) * kReadRows;
  const int rows = static_cast<int>(min(n - row0, int64_t{kReadRows})), total = rows * pieces.units;
  const uint2* src = reinterpret_cast<const uint2*>(c.data(which) + (bh * c.cap + start + row0) * c.stored);
  const float* scale = c.scale(which) + bh * c.blocks();
  void* out = which ? v : k;
  const int64_t to = (bh * n + row0) * c.width;
  uint2 q[kReadEach];
  float s[kReadEach];
  int row[kReadEach], u[kReadEach];
#pragma unroll
  for (int e = 0; e < kReadEach; ++e) {
    const int i = threadIdx.x + e * kReadThreads;
    pieces.at(i, row[e], u[e]);
    if (i < total) {
      q[e] = __ldg(src + i);
      s[e] = __ldg(scale + ((start + row0 + row[e]) >> c.block_log2));
    }
  }
#pragma unroll
  for (int e = 0; e < kReadEach; ++e) {
    if (static_cast<int>(threadIdx.x) + e * kReadThreads < total) {
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        y[j] = __fmul_rn(code_value<FP8>(((j < 4 ? q[e].x : q[e].y) >> 8 * (j & 3)) & 0xffu), s[e]);
      store8<TYPE, ALIGN>(out, to + row[e] * c.width + u[e] * 8, y, c.width - u[e] * 8);
    }
  }
}

// How many values each access may take: rows, heads and the base all on that boundary.
int alignment(int type, int width, const Rows& r) {
  const int size = type == kF32 ? 4 : 2;
  for (int a : {8, 4}) {
    const int64_t bytes = a * size > 16 ? 16 : a * size;
    const int64_t values = bytes / size;
    if (width % a == 0 && reinterpret_cast<uintptr_t>(r.p) % bytes == 0 && r.s0 % values == 0 && r.s1 % values == 0 &&
        r.sn % values == 0 && r.sh % values == 0)
      return a;
  }
  return 1;
}

template <int TYPE, bool FP8, int ALIGN>
cudaError_t write_typed(const View& c, const Rows& k, const Rows& v, const PerSequence& start, const PerSequence& count,
                        int64_t n, cudaStream_t stream) {
  const int units = c.stored / 8;
  const Pieces pieces{units, 65536u / units + 1};
  auto go = [&](auto block) -> cudaError_t {
    constexpr int kRows = write_rows(block.value);
    // runs of kRows rows that n rows can touch, wherever they begin
    const int64_t most = c.cap / kRows;
    const int64_t span = start.dev == nullptr ? (start.all + n - 1) / kRows - start.all / kRows + 1 : (n - 1) / kRows + 2;
    const int64_t per_seq = span < most ? span : most, grid = static_cast<int64_t>(c.batch) * per_seq * c.heads;
    if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
    write_kernel<TYPE, FP8, ALIGN, block.value><<<static_cast<unsigned>(grid), 2 * kRows, 0, stream>>>(
        c, k, v, start, count, n, static_cast<uint32_t>(per_seq), pieces);
    return cudaGetLastError();
  };
  if (c.block_log2 == 5) return go(std::integral_constant<int, 32>());
  if (c.block_log2 == 6) return go(std::integral_constant<int, 64>());
  return go(std::integral_constant<int, 128>());
}

template <int TYPE, bool FP8, int ALIGN>
cudaError_t read_typed(const View& c, void* k, void* v, int64_t start, int64_t n, cudaStream_t stream) {
  const int64_t chunks = (n + kReadRows - 1) / kReadRows, grid = chunks * 2 * c.batch * c.heads;
  if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
  const int units = c.stored / 8;
  read_kernel<TYPE, FP8, ALIGN><<<static_cast<unsigned>(grid), kReadThreads, 0, stream>>>(
      c, k, v, start, n, static_cast<uint32_t>(chunks), Pieces{units, 65536u / units + 1});
  return cudaGetLastError();
}

// calls f<TYPE, FP8, ALIGN> for values known at run time
template <typename F>
cudaError_t dispatch(int type, bool fp8, int align, F&& f) {
  auto by_align = [&](auto t, auto q) {
    if (align == 8) return f(t, q, std::integral_constant<int, 8>());
    if (align == 4) return f(t, q, std::integral_constant<int, 4>());
    return f(t, q, std::integral_constant<int, 1>());
  };
  auto by_code = [&](auto t) { return fp8 ? by_align(t, std::true_type()) : by_align(t, std::false_type()); };
  if (type == kF32) return by_code(std::integral_constant<int, kF32>());
  if (type == kBF16) return by_code(std::integral_constant<int, kBF16>());
  return by_code(std::integral_constant<int, kF16>());
}

}  // namespace

cudaError_t launch_write(const View& c, const Rows& k, const Rows& v, int type, const PerSequence& start,
                         const PerSequence& count, int64_t n, cudaStream_t stream) {
  const int ak = alignment(type, c.width, k), av = alignment(type, c.width, v);
  return dispatch(type, c.fp8, ak < av ? ak : av, [&](auto t, auto q, auto a) {
    return write_typed<t.value, q.value, a.value>(c, k, v, start, count, n, stream);
  });
}

cudaError_t launch_read(const View& c, void* k, void* v, int type, int64_t start, int64_t n, cudaStream_t stream) {
  // rows of the result follow one another, so the width alone decides (the base is an allocation's)
  const int align = c.width % 8 == 0 ? 8 : c.width % 4 == 0 ? 4 : 1;
  return dispatch(type, c.fp8, align, [&](auto t, auto q, auto a) {
    return read_typed<t.value, q.value, a.value>(c, k, v, start, n, stream);
  });
}

}  // namespace bc
}  // namespace nori
