// Muon for matrices that fit one SM: the whole step of a matrix in one CTA.
#include "muon.cuh"

namespace nori {
namespace muon {

// ------------------------------------------------------------------ one matrix per CTA
// Matrices that fit one SM run their whole step in one CTA, and a ragged set of them in one
// launch.  The iterate stays in fp32 in tensor memory, where the update's MMAs add to it in
// place (Z <- Z + Z C); its fp16 copy lies in shared memory once, as 128B-swizzled rows of 64
// columns, and serves the Gram product (read MN-major, the sum running over rows) and the
// update (read K-major).  A and then C take one 128-row tile beside it.  Nothing but the
// matrix itself and its result crosses memory.  The chain of 3 x steps dependent products bounds
// it: each is issued by one thread, waited for by all, read back by tcgen05.ld and published
// again: about 1,300 cycles a product at 64 x 56 (16 us in all) and 3,000 at 384 x 128 (41 us).
// Up to 32 columns, where few roundings average
// out (fp16 operands leave up to 1e-2 of a 2 x 2 matrix), the other half of the 64-column rows
// holds the low parts of Z, A and C, and every product is three (high high, high low, low high:
// 22-bit operands, 1e-5 or less).
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
  if (timed_out(p.status)) return;
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
  const bool pair = mp <= 32;        // low parts in columns 32 ..

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
  // a 16-column chunk in memory: 2 rows of single values, or 8 rows of groups of 4, per access
  const int cl = lane & 15, rl = lane >> 4, c4 = (lane & 3) * 4, r8 = lane >> 2;
  const bool in4 = m % 4 == 0 && aligned4<SRC>(g, p.s, base, mbase);
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

  // what this CTA reads now, and what it updates at the end, on its way to L2
  auto prefetch = [&](const void* at, int64_t bytes) {
    const char* line = reinterpret_cast<const char*>(at);
    for (int64_t i = threadIdx.x * 128; i < bytes; i += kSingleThreads * 128)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(line + i));
  };
  const int64_t numel = static_cast<int64_t>(rows) * cols;
  if constexpr (SRC == kSrcMuon) {
    prefetch(p.s.grad + base, numel * 4);
    prefetch(p.s.mom + mbase, numel * 4);
    prefetch(p.s.data + base, numel * 4);
    if (p.s.ema != nullptr) prefetch(p.s.ema + base, numel * 4);
  } else {
    constexpr int size = SRC == kSrcF32 ? 4 : 2;
    prefetch(static_cast<const char*>(g) + base * size, numel * size);
  }

  // the update's input, tall, raw, into tensor memory; its sum of squares
  double acc = 0.0;
  int t, c;
  for (first(t, c); t < tiles; next(t, c)) {
    const int c0 = c * 16, r0 = t * 128 + q * 32;
    float v[16];
    if (wide) {  // consecutive lanes are consecutive columns of G
      const int cnt = r0 + lane < n ? m - c0 : 0;
#pragma unroll
      for (int k = 0; k < 16; k += 8)
        fetch<SRC, 8>(g, p.s, base, mbase, clip, static_cast<int64_t>(c0 + k) * n + r0 + lane, n, cnt - k, v + k);
    } else {     // turned in shared memory
      if (in4) {  // 4 lanes of 4 columns a row, 8 rows at a time
        fetch4<SRC, 4>(g, p.s, base, mbase, clip, static_cast<int64_t>(r0 + r8) * m + c0 + c4, 8 * m,
                       c0 + c4 < m ? (n - r0 - r8 + 7) / 8 : 0, v);
#pragma unroll
        for (int i = 0; i < 16; ++i) stage[((i & ~3) * 2 + r8) * 17 + c4 + (i & 3)] = v[i];
      } else {    // 16 lanes a row, 2 rows at a time
        const int cnt = c0 + cl < m ? (n - r0 - rl + 1) / 2 : 0;
#pragma unroll
        for (int k = 0; k < 16; k += 8)
          fetch<SRC, 8>(g, p.s, base, mbase, clip, static_cast<int64_t>(r0 + rl + 2 * k) * m + c0 + cl, 2 * m, cnt - k,
                        v + k);
#pragma unroll
        for (int i = 0; i < 16; ++i) stage[(2 * i + rl) * 17 + cl] = v[i];
      }
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
  // v's high parts at c0 and, for pairs, its low parts beside them
  auto put = [&](uint8_t* panel0, int pstride, int r, int c0, float* v) {
    put16(panel0, pstride, r, c0, v);
    if (pair) {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] -= __half2float(__float2half_rn(v[i]));
      put16(panel0, pstride, r, c0 + 32, v);
    }
  };
  auto ld16 = [&](uint32_t addr, float* v) {
    uint32_t r[16];
    tmem_ld16(addr, r);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
  };

  // operand descriptors (addresses in their low 14 bits, in 16-byte units): Z's rows along K,
  // Z's columns along K, and A's (then C's) rows
  const uint32_t z16 = smem_u32(zh) >> 4, a16 = smem_u32(ac) >> 4, zp16 = zpanel >> 4;
  const uint32_t d_a = tmem + tiles * mp;  // A's (and A^2's) accumulator
  const uint32_t idesc_mn = idesc_f16(mp, true), idesc_k = idesc_f16(mp, false);
  // with one panel the MMA's rows 64..127 are padding: let them read the next rows
  const uint64_t dz_mn = umma_smem_desc(0, fit.panels == 2 ? zpanel : 1024, 1024, 2) + z16;
  const uint64_t dz_k = umma_smem_desc(0, 16, 1024, 2) + z16, da_k = umma_smem_desc(0, 16, 1024, 2) + a16;
  const int row = q * 32 + lane;
  const Sink sink = {p.out_type, p.out, base, p.s.lr * lr_factor(p.s.adjust, rows, cols)};
  const bool out4 = m % 4 == 0 && sink4(sink, p.s);
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
  // D (+)= x y^T for one step along K of the operands at `x`, `y` (low parts 64 bytes on)
  auto mma3 = [&](uint32_t d, uint64_t x, uint64_t y, uint32_t idesc, uint32_t more) {
    umma_bf16_ss(d, x, y, idesc, more);
    umma_bf16_ss(d, x, y + 4, idesc, 1u);
    umma_bf16_ss(d, x + 4, y, idesc, 1u);
  };
  // zeros in A and C beyond the matrix (chunk j of this thread's row)
  auto clear = [&](float* v, int j) {
    const int keep = row < m ? m - j * 16 : 0;
    if (keep < 16) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i >= keep) v[i] = 0.f;
    }
  };
  // A += Z^T Z over the rows of tile t
  auto gram = [&](int t) {
    if (warp == 0 && elect_one()) {
      const int k1 = (n - t * 128 + 15) / 16;
      const uint64_t d = dz_mn + t * 1024;
      if (pair) {
        for (int k = 0; k < min(k1, 8); ++k)
          mma3(d_a, d + k * 128, d + k * 128, idesc_mn, t > 0 || k > 0 ? 1u : 0u);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < k1) umma_bf16_ss(d_a, d + k * 128, d + k * 128, idesc_mn, t > 0 || k > 0 ? 1u : 0u);
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
    put(zh, zpanel, t * 128 + q * 32 + lane, c * 16, v);
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
        for (int i = 0; i < 16; ++i) v[i] *= x2;
        clear(v, j);
        put(ac, 16384, row, j * 16, v);
      }
      if (!publish()) break;
      if (warp == 0 && elect_one()) {
        if (pair) {
          for (int k = 0; k < chunks; ++k) mma3(d_a, da_k + k * 2, da_k + k * 2, idesc_k, k > 0 ? 1u : 0u);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint64_t d = da_k + (k >> 2) * 1024 + (k & 3) * 2;
            if (k < chunks) umma_bf16_ss(d_a, d, d, idesc_k, k > 0 ? 1u : 0u);
          }
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
        if (pair) {
          float l[16];
          get16(ac, 16384, row, j * 16 + 32, l);
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] += l[i];
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = p.k.ba * s[i] + p.k.ca * v[i];
        clear(v, j);
        put(ac, 16384, row, j * 16, v);
      }
      if (!publish()) break;
      // Z += Z C, tile by tile
      if (warp == 0 && elect_one()) {
        for (int i = 0; i < tiles; ++i) {
          const uint64_t d = dz_k + i * 1024;
          if (pair) {
            for (int k = 0; k < chunks; ++k) mma3(tmem + i * mp, d + k * 2, da_k + k * 2, idesc_k, 1u);
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (k < chunks)
                umma_bf16_ss(tmem + i * mp, d + (k >> 2) * zp16 + (k & 3) * 2, da_k + (k >> 2) * 1024 + (k & 3) * 2,
                             idesc_k, 1u);
          }
          umma_commit(&bar[1 + i]);
        }
      }
      __syncwarp();
      xi *= p.k.a;
      if (it == p.k.steps - 1) break;
      const float up = renorm(xi);
      // the fp16 copy of each finished tile, and its share of the next A behind it
      first(t, c);
      for (int i = 0; i < tiles; ++i) {
        ok = ok && mbar_wait_warp(&bar[1 + i], it & 1, p.status, kTimeoutEpilogue, nullptr);
        tc_fence_after();
        for (; t == i; next(t, c)) {
          float v[16];
          ld16(tlane + t * mp + c * 16, v);
          if (up != 1.f) {
            uint32_t r[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              v[k] *= up;
              r[k] = __float_as_uint(v[k]);
            }
            tmem_st16(tlane + t * mp + c * 16, r);
          }
          put(zh, zpanel, t * 128 + q * 32 + lane, c * 16, v);
        }
        tmem_wait_st();
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
          const int cnt = r0 + lane < n ? m - c0 : 0;
#pragma unroll
          for (int k = 0; k < 16; k += 8)
            emit<8>(sink, p.s, static_cast<int64_t>(c0 + k) * n + r0 + lane, n, cnt - k, v + k);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) stage[lane * 17 + i] = v[i];
          __syncwarp();
          if (out4) {
            float4 o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float* at = stage + (8 * i + r8) * 17 + c4;
              o[i] = make_float4(at[0], at[1], at[2], at[3]);
            }
            emit4<4>(sink, p.s, static_cast<int64_t>(r0 + r8) * m + c0 + c4, 8 * m,
                     c0 + c4 < m ? (n - r0 - r8 + 7) / 8 : 0, o);
          } else {
            const int cnt = c0 + cl < m ? (n - r0 - rl + 1) / 2 : 0;
#pragma unroll
            for (int k = 0; k < 16; k += 8) {
              float o[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) o[i] = stage[(2 * (k + i) + rl) * 17 + cl];
              emit<8>(sink, p.s, static_cast<int64_t>(r0 + rl + 2 * k) * m + c0 + cl, 2 * m, cnt - k, o);
            }
          }
          __syncwarp();
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

// Matrices first .. first + count of a set that all fit one CTA; `smem` is the largest need.
void run_single(int src, const void* g, int out_type, void* out, const StepArgs& s, int64_t first,
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
  if (smem > 48 * 1024)
    C10_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 221 * 1024));
  kernel<<<static_cast<unsigned>(count), kSingleThreads, smem, at::cuda::getCurrentCUDAStream()>>>(g, p);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace muon
}  // namespace nori
