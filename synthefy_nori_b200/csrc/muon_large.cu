// Muon for matrices that need the whole GPU: norms, Z_0, and all steps' products of all shapes
// of a call in one persistent kernel.
#include "muon.cuh"

namespace nori {
namespace muon {

constexpr int kMaxShapes = 16;   // shapes of one launch (their tensor maps are kernel arguments)
constexpr int kSlice = 8192;     // values of one partial sum of squares

// ------------------------------------------------------------------ arguments
struct Group {
  int first, count;              // matrices of the plan's table
  int rows, cols, n, m, ldz;
  int nt, tm;                    // tiles of 128 along m and n
  int base;                      // first matrix's index among all of the call
  int slices, norm_cta, scale_cta;  // partial sums of a matrix; first CTA of the group in each pre-pass
  int scale_tiles;
  __half *z[2], *zl, *A, *C;
};
struct Pre {
  int groups;
  double* partial;               // [matrix][slices], the groups one after the other
  float2* scale;                 // [matrix][step]: xi before the step, and the power of two after it
  int* done;
  const int* status;
  Group g[kMaxShapes];
};

__device__ __forceinline__ const double* partials(const Pre& p, int gi, int mat) {
  int64_t at = 0;
  for (int i = 0; i < gi; ++i) at += static_cast<int64_t>(p.g[i].count) * p.g[i].slices;
  return p.partial + at + static_cast<int64_t>(mat) * p.g[gi].slices;
}

// ------------------------------------------------------------------ norm (and momentum)
// Partial sums of squares of the update's input, one CTA per 8192 values of a matrix, in
// double: no fp32 gradient overflows or vanishes in its own norm.  With kSrcMuon the momentum
// is brought up to date on the way.  Memory bound: 4 or 2 bytes a value (12 with momentum).
template <int SRC>
__global__ void __launch_bounds__(256) norm_kernel(const void* __restrict__ g, StepArgs s,
                                                   const __grid_constant__ Pre p) {
  if constexpr (SRC == kSrcMuon) {  // the momentum stays where the weights will
    if (timed_out(p.status) || step_rejected(s)) return;
  }
  int gi = 0;
  while (gi + 1 < p.groups && static_cast<int>(blockIdx.x) >= p.g[gi + 1].norm_cta) ++gi;
  const Group& q = p.g[gi];
  const int mat = (blockIdx.x - q.norm_cta) / q.slices, slice = (blockIdx.x - q.norm_cta) % q.slices;
  const int64_t numel = static_cast<int64_t>(q.rows) * q.cols;
  int64_t base, mbase = 0;
  float clip = 1.f;
  if constexpr (SRC == kSrcMuon) {
    const Mat t = s.table[q.first + mat];
    base = t.off;
    mbase = t.moff;
    clip = clip_factor(s);
  } else {
    base = mat * numel;
  }
  const int64_t i0 = static_cast<int64_t>(slice) * kSlice;
  const int len = static_cast<int>(min(static_cast<int64_t>(kSlice), numel - i0));
  double acc = 0.0;
  if (aligned4<SRC>(g, s, base, mbase) && len % 4 == 0) {
    for (int j = threadIdx.x * 4; j < len; j += 256 * 4 * 4) {  // 4 x 4 values in flight
      float v[4][4], m[4][4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int k = j + u * 1024;
        if (k < len) {
          if constexpr (SRC == kSrcMuon) {
            load4<kSrcF32>(s.grad, base + i0 + k, v[u]);
            load4<kSrcF32>(s.mom, mbase + i0 + k, m[u]);
          } else {
            load4<SRC>(g, base + i0 + k, v[u]);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int k = j + u * 1024;
        if (k < len) {
          if constexpr (SRC == kSrcMuon) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float gi4 = v[u][i] * clip;
              m[u][i] = s.momentum * m[u][i] + gi4;
              v[u][i] = s.nesterov ? gi4 + s.momentum * m[u][i] : m[u][i];
            }
            *reinterpret_cast<float4*>(s.mom + mbase + i0 + k) = make_float4(m[u][0], m[u][1], m[u][2], m[u][3]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) acc += static_cast<double>(v[u][i]) * v[u][i];
        }
      }
    }
  } else {
    for (int j = threadIdx.x; j < len; j += 256 * 8) {
      float v[8];
      fetch<SRC, 8>(g, s, base, mbase, clip, i0 + j, 256, (len - j + 255) / 256, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc += static_cast<double>(v[i]) * v[i];
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
    const_cast<double*>(partials(p, gi, mat))[slice] = v;
    if (slice == 0) p.done[q.base + mat] = 0;
  }
}

// ------------------------------------------------------------------ Z_0
// Z_0 = 2^8 G / |G|_F as a pair of fp16 [n, ldz], tall (a wide G is turned in shared memory),
// and its scales over the steps, from f = |G|_F / (|G|_F + eps).  One CTA per 64 x 64 tile.
template <int SRC>
__global__ void __launch_bounds__(256) scale_kernel(const void* __restrict__ g, StepArgs s, Coeffs k,
                                                    const __grid_constant__ Pre p) {
  if constexpr (SRC == kSrcMuon) {
    if (step_rejected(s)) return;
  }
  __shared__ float tile[64][65];
  __shared__ double total;
  int gi = 0;
  while (gi + 1 < p.groups && static_cast<int>(blockIdx.x) >= p.g[gi + 1].scale_cta) ++gi;
  const Group& q = p.g[gi];
  const int mat = (blockIdx.x - q.scale_cta) / q.scale_tiles, ti = (blockIdx.x - q.scale_cta) % q.scale_tiles;
  const bool wide = q.rows < q.cols;
  const int tiles_c = (q.cols + 63) / 64;
  const int r0 = ti / tiles_c * 64, c0 = ti % tiles_c * 64;  // in G
  int64_t base, mbase = 0;
  float clip = 1.f;
  if constexpr (SRC == kSrcMuon) {
    const Mat t = s.table[q.first + mat];
    base = t.off;
    mbase = t.moff;
    clip = clip_factor(s);
  } else {
    base = static_cast<int64_t>(mat) * q.rows * q.cols;
  }
  // this thread's values: rows tid / 16 + 16 i, columns 4 (tid % 16) .. + 3
  const int lr = threadIdx.x / 16, lc = threadIdx.x % 16 * 4;
  float v[4][4], mo[4][4];
  const bool vec = q.cols % 4 == 0 && aligned4<SRC>(g, s, base, mbase);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + lr + 16 * i, c = c0 + lc;
    const int64_t at = static_cast<int64_t>(r) * q.cols + c;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[i][k] = mo[i][k] = 0.f;
    if (r < q.rows && vec) {
      if (c < q.cols) {
        if constexpr (SRC == kSrcMuon) {
          load4<kSrcF32>(s.mom, mbase + at, mo[i]);
          if (s.nesterov) load4<kSrcF32>(s.grad, base + at, v[i]);
        } else {
          load4<SRC>(g, base + at, v[i]);
        }
      }
    } else if (r < q.rows) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (c + k < q.cols) {
          if constexpr (SRC == kSrcMuon) {
            mo[i][k] = s.mom[mbase + at + k];
            if (s.nesterov) v[i][k] = s.grad[base + at + k];
          } else {
            v[i][k] = load_src<SRC>(g, base + at + k);
          }
        }
      }
    }
  }
  if (threadIdx.x < 32) {  // the same order in every CTA of the matrix
    const double* part = partials(p, gi, mat);
    double a = 0.0;
    for (int i = threadIdx.x; i < q.slices; i += 32) a += part[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    if (threadIdx.x == 0) total = a;
  }
  __syncthreads();
  float s0, s1, f;
  z_scale(total, k.eps, s0, s1, f);
  if (ti == 0 && threadIdx.x == 0) {
    float2* d = p.scale + static_cast<int64_t>(q.base + mat) * k.steps;
    float xi = f * (1.f / kZScale);
    for (int it = 0; it < k.steps; ++it) {
      float next = xi * k.a;
      d[it] = make_float2(xi, renorm(next));
      xi = next;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float u = SRC == kSrcMuon ? (s.nesterov ? v[i][k] * clip + s.momentum * mo[i][k] : mo[i][k]) : v[i][k];
      tile[lr + 16 * i][lc + k] = u * s0 * s1;
    }
  __syncthreads();
  const int64_t zoff = static_cast<int64_t>(mat) * q.n * q.ldz;
  const int zr0 = wide ? c0 : r0, zc0 = wide ? r0 : c0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int zr = threadIdx.x / 8 + 32 * i, zc = threadIdx.x % 8 * 8;
    if (zr0 + zr < q.n && zc0 + zc < q.ldz) {
      float x[8], h[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = wide ? tile[zc + k][zr] : tile[zr][zc + k];
      const uint4 hi = pack8(x);
      unpack8(hi, h);
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] -= h[k];
      const int64_t at = zoff + static_cast<int64_t>(zr0 + zr) * q.ldz + zc0 + zc;
      *reinterpret_cast<uint4*>(q.z[0] + at) = hi;
      *reinterpret_cast<uint4*>(q.zl + at) = pack8(x);
    }
  }
}

// ------------------------------------------------------------------ the products
// One persistent CTA per SM walks the tiles of all products of all steps in one order that
// every CTA shares:
//
//   blocks of matrices (their buffers fit L2 together; every shape spread over all blocks)
//     steps
//       A = xi^2 Z^T Z        128 x 128 tiles on and above the diagonal, then mirrored
//       I + C = I + (b A + c A^2) / a   the same tiles
//       Z <- Z (I + C)        all 128 x 128 tiles (the last step writes the result instead)
//
// A tile needs all tiles of its own matrix's previous product: a counter per matrix, raised
// when a tile's stores are complete, tells (release / acquire at GPU scope).  Tiles of other
// matrices lie between the two, so a CTA seldom waits, and small shapes or a lone large matrix
// fill in among the others.  The launch is cooperative (every CTA resident), and a tile only
// waits for tiles before it in the shared order, so the oldest unfinished tile can always run.
//
// Roles (448 threads).  Warp 10 walks ahead and waits for tiles' inputs (an acquire at GPU
// scope and a proxy fence: 1,300 cycles even when they are there).  Warp 0 loads operands by
// TMA (128B-swizzled) into a ring of four 32 KB stages: 64 rows of Z for the Gram product
// (both operands MN-major: the sum runs over rows), 64 columns of the rows of A, or of Z and C,
// otherwise (K-major).  One thread of warp 1 issues tcgen05.mma (M = 128, N <= 128, K = 16) into
// four TMEM accumulators.  Warps 2..9 run the epilogue on 64-column boxes and touch only tensor
// and shared memory: warp 11 loads the boxes that it reads (Z's low half, or A), warps 12 and 13
// store, for alternate tiles, what it leaves there (Z's pair, or A / C and their mirror image)
// and count the tile once its stores are complete, all by TMA.
//
// What bounds a tile is latency at every hand-over rather than a rate (at 81 x 1344 x 448, 838 us
// under ncu, the tensor core runs at 24%, L2 at 36% and DRAM at 41% of their peaks; a 128 x 128 tile of the
// update takes 5,000 - 6,000 cycles to load and 3,000 in its epilogue), so the choices below keep
// many small pieces in flight: 128 x 128 tiles (with 128 x 256 ones the epilogue's boxes queued behind
// 144 KB of operands, and a lone matrix had half as many tiles), two storing warps (one would
// wait 2,000 cycles a tile for its stores), three boxes.  C is kept as I + C, so that Z's high
// half comes out of the product itself and only the low half is loaded and added.  (Rounding the
// diagonal of I + C to fp16 scales Z's columns by 1 + 2^-11 at most: an error like the other
// operands'.)
constexpr int kThreads = 448;
constexpr int kStages = 4, kStageBytes = 32768;
constexpr int kAccs = 4;                        // TMEM accumulators of 128 columns
constexpr int kReady = 4;                       // tiles whose inputs are known to be there
constexpr int kSlots = 3, kSlotBytes = 32768;   // boxes of 128 x 64, two halves each
constexpr int kSmemBytes = kStages * kStageBytes + kSlots * kSlotBytes + 1024 + 512;

enum Phase : int { kGram = 0, kPoly = 1, kUpdate = 2 };

struct alignas(64) Maps {
  CUtensorMap z[2], zl, A, C;    // boxes of 64 columns x 64 rows: MN-major operands, the epilogue's
  CUtensorMap zk[2], Ak, Ck;     // of 128 rows: K-major operands
};
struct Args {
  Maps maps[kMaxShapes];
  Group g[kMaxShapes];
  int groups, blocks;
  Coeffs k;
  const float2* scale;
  int* done;
  int out_type;
  void* out;
  StepArgs s;
  int* status;
};

// Walks the shared order: segments (block, step, product, shape), each `size` tiles.
struct Cursor {
  int b, it, ph, g, base, size, per, c0;

  __device__ __forceinline__ void segment(const Args& a) {
    const Group& q = a.g[g];
    c0 = static_cast<int>(static_cast<int64_t>(q.count) * b / a.blocks);
    const int c1 = static_cast<int>(static_cast<int64_t>(q.count) * (b + 1) / a.blocks);
    per = ph == kUpdate ? q.tm * q.nt : q.nt * (q.nt + 1) / 2;
    size = (c1 - c0) * per;
  }
  __device__ __forceinline__ void start(const Args& a) {
    b = it = ph = g = base = 0;
    segment(a);
  }
  __device__ __forceinline__ bool seek(const Args& a, int t) {
    while (t - base >= size) {
      base += size;
      if (++g == a.groups) {
        g = 0;
        if (++ph == 3) {
          ph = 0;
          if (++it == a.k.steps) {
            it = 0;
            if (++b == a.blocks) return false;
          }
        }
      }
      segment(a);
    }
    return true;
  }
};

struct Item {
  int g, mat, it, ph, ti, tj;
  int n0, ncols;                 // first column of the tile, columns up to the matrix's edge
  int need;                      // finished tiles of this matrix that it waits for
  bool diag, last;
};
__device__ __forceinline__ Item item_of(const Args& a, const Cursor& c, int t) {
  Item x;
  const Group& q = a.g[c.g];
  x.g = c.g;
  x.it = c.it;
  x.ph = c.ph;
  x.mat = c.c0 + (t - c.base) / c.per;
  int r = (t - c.base) % c.per;
  const int tri = q.nt * (q.nt + 1) / 2;
  x.need = c.it * (2 * tri + q.tm * q.nt) + c.ph * tri;
  x.last = c.ph == kUpdate && c.it == a.k.steps - 1;
  if (c.ph == kUpdate) {
    x.ti = r / q.nt;
    x.tj = r % q.nt;
    x.diag = false;
  } else {
    int i = 0;
    while (r >= q.nt - i) {
      r -= q.nt - i;
      ++i;
    }
    x.ti = i;
    x.tj = i + r;
    x.diag = x.ti == x.tj;
  }
  x.n0 = x.tj * 128;
  x.ncols = min(128, q.m - x.n0);
  return x;
}

// Bounded wait until the matrix's counter reaches `need`; what its producers stored through
// the async proxy is then visible to this thread's TMA loads.
__device__ __forceinline__ bool wait_done(const Args& a, const Item& x, volatile int* abort) {
  const int* c = a.done + a.g[x.g].base + x.mat;
  uint64_t t0 = 0;
  for (uint32_t spins = 0;; ++spins) {
    int v;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(c) : "memory");
    if (v >= x.need) break;
    if (spins == 0) t0 = globaltimer_ns();
    if ((spins & 63u) == 63u) {
      if (*abort) return false;
      if (*reinterpret_cast<volatile int*>(a.status) != 0) {  // another CTA has given up
        *abort = 1;
        return false;
      }
      if (globaltimer_ns() - t0 > kWaitLimitNs) {
        record_status(a.status, kTimeoutProducer);
        *abort = 1;
        return false;
      }
    }
    __nanosleep(20);
  }
  asm volatile("fence.proxy.async;" ::: "memory");
  return true;
}

// TMA tiled store of one box (3-D map).
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* smem_src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(smem_src)), "r"(x), "r"(y), "r"(z)
               : "memory");
}

__global__ void __launch_bounds__(kThreads, 1) product_kernel(const __grid_constant__ Args a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* slots = stages + kStages * kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(slots + kSlots * kSlotBytes);
  uint64_t* empty = full + kStages;
  uint64_t* tfull = empty + kStages;
  uint64_t* tempty = tfull + kAccs;
  uint64_t* ready = tempty + kAccs; // a tile's inputs are there
  uint64_t* rfree = ready + kReady; // both loading warps know
  uint64_t* sfull = rfree + kReady; // a slot is the epilogue's (its loads have landed)
  uint64_t* sdone = sfull + kSlots; // the epilogue has left it
  uint64_t* sfree = sdone + kSlots; // its stores have read it
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sfree + kSlots);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (timed_out(a.status)) return;
  if (a.out_type == kOutMuon && step_rejected(a.s)) return;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kAccs; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 8);
    }
    for (int i = 0; i < kReady; ++i) {
      mbar_init(&ready[i], 1);
      mbar_init(&rfree[i], 2);
    }
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&sfull[i], 1);
      mbar_init(&sdone[i], 8);
      mbar_init(&sfree[i], 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Cursor cur;
  cur.start(a);
  // this role's place in a ring of `n` (stages, accumulators, ready tiles or slots)
  auto advance = [](int& i, uint32_t& phase, int n) {
    if (++i == n) {
      i = 0;
      phase ^= 1;
    }
  };
  // a role that has given up waits (again with a limit) until what it last started in each place of
  // its ring is complete: no copy or product is under way when the CTA's memory goes to another
  auto drain = [&](uint64_t* bars, int i, uint32_t phase, int n) {
    for (int k = 0; k < n; ++k)
      mbar_wait(&bars[k], k < i ? phase : phase ^ 1, a.status, kTimeoutProducer, nullptr);
  };
  int re = 0;
  uint32_t rp = 0;

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && cur.seek(a, t); t += gridDim.x) {
        const Item x = item_of(a, cur, t);
        const Group& q = a.g[x.g];
        const Maps& mp = a.maps[x.g];
        if (!mbar_wait(&ready[re], rp, a.status, kTimeoutProducer, abort_flag)) break;
        mbar_arrive(&rfree[re]);
        advance(re, rp, kReady);
        const bool gram = x.ph == kGram;
        const int K = gram ? q.n : q.m, row = x.ti * 128;
        const CUtensorMap* ma = gram ? &mp.z[x.it & 1] : x.ph == kPoly ? &mp.Ak : &mp.zk[x.it & 1];
        const CUtensorMap* mb = x.ph == kPoly ? &mp.Ak : &mp.Ck;
        for (int k0 = 0; k0 < K; k0 += 64) {
          ok = mbar_wait(&empty[stage], phase ^ 1, a.status, kTimeoutProducer, abort_flag);
          if (!ok) break;
          uint8_t* sa = stages + stage * kStageBytes;
          uint64_t* bar = &full[stage];
          mbar_arrive_expect_tx(bar, x.diag ? 16384 : 32768);
          if (gram) {
            tma_load_3d(sa, ma, bar, row, k0, x.mat);
            tma_load_3d(sa + 8192, ma, bar, row + 64, k0, x.mat);
            if (!x.diag) {
              tma_load_3d(sa + 16384, ma, bar, x.n0, k0, x.mat);
              tma_load_3d(sa + 24576, ma, bar, x.n0 + 64, k0, x.mat);
            }
          } else {
            tma_load_3d(sa, ma, bar, k0, row, x.mat);
            if (!x.diag) tma_load_3d(sa + 16384, mb, bar, k0, x.n0, x.mat);
          }
          advance(stage, phase, kStages);
        }
      }
      drain(full, stage, phase, kStages);
    }
  } else if (warp == 1) {
    if (elect_one()) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      const uint32_t stages_lo = smem_u32(stages) >> 4;
      bool ok = true;
      for (int t = blockIdx.x; ok && cur.seek(a, t); t += gridDim.x) {
        const Item x = item_of(a, cur, t);
        const Group& q = a.g[x.g];
        const bool gram = x.ph == kGram;
        const int K = gram ? q.n : q.m;
        const uint32_t idesc = idesc_f16((x.ncols + 15) / 16 * 16, gram);
        // descriptors without the address (their low 14 bits, in 16-byte units), and the steps
        // of 16 along K: 16 rows of an MN-major panel, 32 bytes of a K-major row; a tile on the
        // diagonal multiplies its rows by themselves
        const uint64_t dbase = umma_smem_desc(0, gram ? 8192 : 16, 1024, 2);
        const uint32_t inc = gram ? 2048 / 16 : 32 / 16;
        const uint32_t second = x.diag ? 0 : 16384 / 16;
        if (!mbar_wait(&tempty[acc], acc_phase ^ 1, a.status, kTimeoutMma, abort_flag)) break;
        tc_fence_after();
        const uint32_t d = tmem + acc * 128;
        for (int k0 = 0; k0 < K; k0 += 64) {
          ok = mbar_wait(&full[stage], phase, a.status, kTimeoutMma, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint64_t da = dbase + (stages_lo + stage * (kStageBytes / 16)), db = da + second;
          const uint32_t more = k0 > 0 ? 1u : 0u;
          const int steps = (min(64, K - k0) + 15) / 16;  // the rest of the boxes is zero fill
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (k < steps) umma_bf16_ss(d, da + k * inc, db + k * inc, idesc, k > 0 ? 1u : more);
          umma_commit(&empty[stage]);
          advance(stage, phase, kStages);
        }
        if (!ok) break;
        umma_commit(&tfull[acc]);
        advance(acc, acc_phase, kAccs);
      }
      drain(empty, stage, phase, kStages);
    }
  } else if (warp == 10) {
    if (elect_one()) {
      for (int t = blockIdx.x; cur.seek(a, t); t += gridDim.x) {
        const Item x = item_of(a, cur, t);
        if (!mbar_wait(&rfree[re], rp ^ 1, a.status, kTimeoutProducer, abort_flag)) break;
        if (!wait_done(a, x, abort_flag)) break;
        mbar_arrive(&ready[re]);
        advance(re, rp, kReady);
      }
    }
  } else if (warp < 10) {
    const int q4 = warp & 3, half = (warp - 2) >> 2;  // lane quarter, 32-column half of a box
    const int rt = q4 * 32 + lane;                    // row inside the tile
    const int x7 = rt & 7;                            // 128B swizzle of this row
    int acc = 0, slot = 0;
    uint32_t acc_phase = 0, s_phase = 0;
    bool ok = true;
    for (int t = blockIdx.x; ok && cur.seek(a, t); t += gridDim.x) {
      const Item x = item_of(a, cur, t);
      const Group& q = a.g[x.g];
      const float2 sc = a.scale[static_cast<int64_t>(q.base + x.mat) * a.k.steps + x.it];
      const float xi = sc.x, up = sc.y;
      if (!mbar_wait_warp(&tfull[acc], acc_phase, a.status, kTimeoutEpilogue, abort_flag)) break;
      tc_fence_after();
      const uint32_t taddr = tmem + (static_cast<uint32_t>(q4 * 32) << 16) + acc * 128 + half * 32;
      for (int c = 0; c < x.ncols; c += 64) {
        uint8_t* s0 = slots + slot * kSlotBytes;
        uint8_t* s1 = s0 + 16384;
        uint8_t* row0 = s0 + rt * 128;
        uint8_t* row1 = s1 + rt * 128;
        ok = mbar_wait_warp(&sfull[slot], s_phase, a.status, kTimeoutEpilogue, abort_flag);
        if (!ok) break;
        uint32_t r[32];
        tmem_ld32(taddr + c, r);
        tmem_wait_ld();
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
        if (x.ph != kUpdate) {
          const float x2 = xi * xi;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint4* cell = reinterpret_cast<uint4*>(row0 + (((half * 4 + j) ^ x7) << 4));
            if (x.ph == kGram) {
#pragma unroll
              for (int i = 0; i < 8; ++i) v[8 * j + i] *= x2;
            } else {
              float s[8];
              unpack8(*cell, s);
#pragma unroll
              for (int i = 0; i < 8; ++i) v[8 * j + i] = a.k.ba * s[i] + a.k.ca * v[8 * j + i];
              if (x.diag) {  // I + C
#pragma unroll
                for (int i = 0; i < 8; ++i)
                  if (c + half * 32 + 8 * j + i == rt) v[8 * j + i] += 1.f;
              }
            }
            *cell = pack8(v + 8 * j);
          }
          if (!x.diag) {  // the mirrored box: row = column here, two 64-column panels
            uint8_t* mir = s1 + (rt >> 6) * 8192 + (rt & 7) * 2;
            const int ch = (rt & 63) >> 3;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const int mr = half * 32 + i;
              *reinterpret_cast<__half*>(mir + mr * 128 + ((ch ^ (mr & 7)) << 4)) = __float2half_rn(v[i]);
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int off = ((half * 4 + j) ^ x7) << 4;
            float l[8];
            unpack8(*reinterpret_cast<const uint4*>(row1 + off), l);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[8 * j + i] += l[i];
            if (!x.last) {
              float h[8];
              if (up != 1.f) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[8 * j + i] *= up;
              }
              const uint4 hi = pack8(v + 8 * j);
              unpack8(hi, h);
#pragma unroll
              for (int i = 0; i < 8; ++i) l[i] = v[8 * j + i] - h[i];
              *reinterpret_cast<uint4*>(row0 + off) = hi;
              *reinterpret_cast<uint4*>(row1 + off) = pack8(l);
            }
          }
          if (x.last) {
            // the result in G's orientation: as it lies, consecutive lanes being consecutive
            // columns of a wide G, or turned in the slot's cells that this warp alone uses
            const float xo = xi * a.k.a;
            const Sink sink = {a.out_type, a.out,
                               a.out_type == kOutMuon ? a.s.table[q.first + x.mat].off
                                                      : static_cast<int64_t>(x.mat) * q.rows * q.cols,
                               a.s.lr * lr_factor(a.s.adjust, q.rows, q.cols)};
            const int col = x.n0 + c + half * 32, r0 = x.ti * 128 + q4 * 32;
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] *= xo;
            if (q.rows < q.cols) {
              const int64_t e0 = static_cast<int64_t>(col) * q.n + r0 + lane;
              const int cnt = r0 + lane < q.n ? q.m - col : 0;
#pragma unroll
              for (int k = 0; k < 32; k += 8) emit<8>(sink, a.s, e0 + static_cast<int64_t>(k) * q.n, q.n, cnt - k, v + k);
            } else {
              // 16-byte cell j of row rr among the ones that this warp alone uses
              auto cell = [&](int rr, int j) -> float4* {
                const int rl = q4 * 32 + rr;
                return reinterpret_cast<float4*>((j < 4 ? s0 : s1) + rl * 128 + (((half * 4 + (j & 3)) ^ (rl & 7)) << 4));
              };
              __syncwarp();
#pragma unroll
              for (int j = 0; j < 8; ++j) *cell(lane, j) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
              __syncwarp();
              if (q.m % 4 == 0 && sink4(sink, a.s)) {  // 8 lanes of 4 columns a row, 4 rows at a time
                const int rr = lane >> 3, cc = col + (lane & 7) * 4;
                const int cnt = cc < q.m ? (q.n - r0 - rr + 3) / 4 : 0;
                const int64_t e0 = static_cast<int64_t>(r0 + rr) * q.m + cc;
#pragma unroll 1
                for (int k = 0; k < 8; k += 4) {
                  float4 o[4];
#pragma unroll
                  for (int i = 0; i < 4; ++i) o[i] = *cell(4 * (k + i) + rr, lane & 7);
                  emit4<4>(sink, a.s, e0 + 4ll * k * q.m, 4ll * q.m, cnt - k, o);
                }
              } else {
                const int cnt = col + lane < q.m ? q.n - r0 : 0;
                const int64_t e0 = static_cast<int64_t>(r0) * q.m + col + lane;
#pragma unroll 1
                for (int k = 0; k < 32; k += 8) {
                  float o[8];
#pragma unroll
                  for (int i = 0; i < 8; ++i) o[i] = reinterpret_cast<const float*>(cell(k + i, lane >> 2))[lane & 3];
                  emit<8>(sink, a.s, e0 + static_cast<int64_t>(k) * q.m, q.m, cnt - k, o);
                }
              }
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sdone[slot]);
        advance(slot, s_phase, kSlots);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[acc]);
      advance(acc, acc_phase, kAccs);
    }
  } else if (warp == 11) {
    if (elect_one()) {
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && cur.seek(a, t); t += gridDim.x) {
        const Item x = item_of(a, cur, t);
        const Maps& mp = a.maps[x.g];
        if (!mbar_wait(&ready[re], rp, a.status, kTimeoutProducer, abort_flag)) break;
        mbar_arrive(&rfree[re]);
        advance(re, rp, kReady);
        for (int c = 0; c < x.ncols; c += 64) {
          ok = mbar_wait(&sfree[slot], phase ^ 1, a.status, kTimeoutProducer, abort_flag);
          if (!ok) break;
          uint8_t* s0 = slots + slot * kSlotBytes;
          uint64_t* bar = &sfull[slot];
          const int col = x.n0 + c, row = x.ti * 128;
          if (x.ph == kGram) {
            mbar_arrive(bar);
          } else {
            const CUtensorMap* m = x.ph == kPoly ? &mp.A : &mp.zl;
            uint8_t* d = x.ph == kPoly ? s0 : s0 + 16384;
            mbar_arrive_expect_tx(bar, 16384);
            tma_load_3d(d, m, bar, col, row, x.mat);
            tma_load_3d(d + 8192, m, bar, col, row + 64, x.mat);
          }
          advance(slot, phase, kSlots);
        }
      }
      drain(sfull, slot, phase, kSlots);
    }
  } else {
    if (elect_one()) {
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true, mine = warp == 12;
      for (int t = blockIdx.x; ok && cur.seek(a, t); t += gridDim.x, mine = !mine) {
        const Item x = item_of(a, cur, t);
        const Group& q = a.g[x.g];
        const Maps& mp = a.maps[x.g];
        int before = -1;  // the slot that the box before this one left
        for (int c = 0; c < x.ncols; c += 64, advance(slot, phase, kSlots)) {
          if (!mine) continue;
          ok = mbar_wait(&sdone[slot], phase, a.status, kTimeoutEpilogue, abort_flag);
          if (!ok) break;
          uint8_t* s0 = slots + slot * kSlotBytes;
          const int col = x.n0 + c, row = x.ti * 128;
          if (x.ph != kUpdate) {
            const CUtensorMap* mo = x.ph == kGram ? &mp.A : &mp.C;
            tma_store_3d(mo, s0, col, row, x.mat);
            if (row + 64 < q.m) tma_store_3d(mo, s0 + 8192, col, row + 64, x.mat);
            if (!x.diag) {
              tma_store_3d(mo, s0 + 16384, row, col, x.mat);
              if (row + 64 < q.m) tma_store_3d(mo, s0 + 24576, row + 64, col, x.mat);
            }
          } else if (!x.last) {
            const CUtensorMap* mo = &mp.z[(x.it & 1) ^ 1];
            tma_store_3d(mo, s0, col, row, x.mat);
            tma_store_3d(&mp.zl, s0 + 16384, col, row, x.mat);
            if (row + 64 < q.n) {
              tma_store_3d(mo, s0 + 8192, col, row + 64, x.mat);
              tma_store_3d(&mp.zl, s0 + 24576, col, row + 64, x.mat);
            }
          }
          bulk_commit();
          if (before >= 0) {
            asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            mbar_arrive(&sfree[before]);
          }
          before = slot;
        }
        if (!ok || !mine) continue;
        bulk_wait_read0();
        mbar_arrive(&sfree[before]);
        if (!x.last) {  // the tile is in memory: count it
          bulk_wait0();
          asm volatile("fence.proxy.async;" ::: "memory");
          __threadfence();
          atomicAdd(a.done + q.base + x.mat, 1);
        }
      }
      bulk_wait0();
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

// ------------------------------------------------------------------ host
static CUtensorMap map_f16(const __half* base, int cols, int rows, int ld, int batch, int box_rows) {
  const int64_t dims[3] = {cols, rows, batch};
  const int64_t strides[2] = {static_cast<int64_t>(ld) * 2, static_cast<int64_t>(ld) * rows * 2};
  const int box[3] = {64, box_rows, 1};
  return make_tmap_nd_bf16(const_cast<__half*>(base), 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_DATA_TYPE_FLOAT16);
}

static int64_t align_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

// Work buffers of the matrices of a block.  Wide blocks put more tiles between a product and the
// one that needs it, narrow ones stay in L2: calls of 81 x 1344 x 448 in a loop take 977 us with 100 MB, 922
// with 200, 940 with 400 or more; 52 x 896 x 448 450, 433 and 433.
constexpr int64_t kBlockBytes = 200ll << 20;

static void run_shapes(int src, const void* g, int out_type, void* out, const StepArgs& s, const Shape* shapes, int ns,
                       const Coeffs& k, const torch::Tensor& status, const at::TensorOptions& dev,
                       at::cuda::CUDAEvent* ready) {
  Args a{};
  Pre p{};
  int64_t bytes = 0, mats = 0, parts = 0, norm_ctas = 0, scale_ctas = 0, items = 0;
  auto take = [&](int64_t n) {
    const int64_t at = bytes;
    bytes += align_up(n, 1024);
    return at;
  };
  std::vector<std::array<int64_t, 5>> at(ns);
  for (int i = 0; i < ns; ++i) {
    Group& q = p.g[i];
    const int64_t count = shapes[i].count, numel = static_cast<int64_t>(shapes[i].rows) * shapes[i].cols;
    q.first = static_cast<int>(shapes[i].first);
    q.count = static_cast<int>(count);
    q.rows = shapes[i].rows;
    q.cols = shapes[i].cols;
    q.n = std::max(q.rows, q.cols);
    q.m = std::min(q.rows, q.cols);
    q.ldz = static_cast<int>(align_up(q.m, 8));
    q.nt = (q.m + 127) / 128;
    q.tm = (q.n + 127) / 128;
    q.base = static_cast<int>(mats);
    q.slices = static_cast<int>((numel + kSlice - 1) / kSlice);
    q.scale_tiles = ((q.rows + 63) / 64) * ((q.cols + 63) / 64);
    q.norm_cta = static_cast<int>(norm_ctas);
    q.scale_cta = static_cast<int>(scale_ctas);
    mats += count;
    parts += count * q.slices;
    norm_ctas += count * q.slices;
    scale_ctas += count * q.scale_tiles;
    items += count * k.steps * (static_cast<int64_t>(q.nt) * (q.nt + 1) + static_cast<int64_t>(q.tm) * q.nt);
    const int64_t zb = count * q.n * q.ldz * 2, ab = count * q.m * q.ldz * 2;
    at[i] = {take(zb), take(zb), take(zb), take(ab), take(ab)};
    TORCH_CHECK(mats < INT_MAX && norm_ctas < INT_MAX && scale_ctas < INT_MAX && items < INT_MAX - (1 << 20),
                "muon: too many matrices for one call");
  }
  const int64_t work = bytes;
  const int64_t p_at = take(parts * 8), s_at = take(mats * k.steps * 8), d_at = take(mats * 4);
  auto ws = torch::empty({bytes}, dev.dtype(at::kByte));
  check_plain(ws, "muon");
  uint8_t* w = ws.data_ptr<uint8_t>();
  for (int i = 0; i < ns; ++i) {
    Group& q = p.g[i];
    q.z[0] = reinterpret_cast<__half*>(w + at[i][0]);
    q.z[1] = reinterpret_cast<__half*>(w + at[i][1]);
    q.zl = reinterpret_cast<__half*>(w + at[i][2]);
    q.A = reinterpret_cast<__half*>(w + at[i][3]);
    q.C = reinterpret_cast<__half*>(w + at[i][4]);
    Maps& mp = a.maps[i];
    for (int j = 0; j < 2; ++j) {
      mp.z[j] = map_f16(q.z[j], q.m, q.n, q.ldz, q.count, 64);
      mp.zk[j] = map_f16(q.z[j], q.m, q.n, q.ldz, q.count, 128);
    }
    mp.zl = map_f16(q.zl, q.m, q.n, q.ldz, q.count, 64);
    mp.A = map_f16(q.A, q.m, q.m, q.ldz, q.count, 64);
    mp.Ak = map_f16(q.A, q.m, q.m, q.ldz, q.count, 128);
    mp.C = map_f16(q.C, q.m, q.m, q.ldz, q.count, 64);
    mp.Ck = map_f16(q.C, q.m, q.m, q.ldz, q.count, 128);
    a.g[i] = q;
  }
  p.groups = ns;
  p.partial = reinterpret_cast<double*>(w + p_at);
  p.scale = reinterpret_cast<float2*>(w + s_at);
  p.done = reinterpret_cast<int*>(w + d_at);
  p.status = status.data_ptr<int>();
  a.groups = ns;
  a.blocks = static_cast<int>(std::max<int64_t>(1, (work + kBlockBytes - 1) / kBlockBytes));
  a.k = k;
  a.scale = p.scale;
  a.done = p.done;
  a.out_type = out_type;
  a.out = out;
  a.s = s;
  a.status = status.data_ptr<int>();
  auto stream = at::cuda::getCurrentCUDAStream();
#define NORI_MUON_SRC(S)                                                                    \
  norm_kernel<S><<<static_cast<unsigned>(norm_ctas), 256, 0, stream>>>(g, s, p);           \
  C10_CUDA_KERNEL_LAUNCH_CHECK();                                                           \
  scale_kernel<S><<<static_cast<unsigned>(scale_ctas), 256, 0, stream>>>(g, s, k, p);      \
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
  C10_CUDA_CHECK(cudaFuncSetAttribute(product_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
  // no more CTAs than the widest product has tiles
  int64_t widest = 1;
  for (int ph = 0; ph < 2; ++ph) {
    int64_t n = 0;
    for (int i = 0; i < ns; ++i) {
      const Group& q = p.g[i];
      n += (q.count + a.blocks - 1) / a.blocks * static_cast<int64_t>(ph == 0 ? q.nt * (q.nt + 1) / 2 : q.tm * q.nt);
    }
    widest = std::max(widest, n);
  }
  const int sms = persistent_sms(at::cuda::getCurrentDeviceProperties()->multiProcessorCount);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(widest, sms));
  if (ready != nullptr) ready->record(stream);
  void* argv[] = {&a};
  C10_CUDA_CHECK(cudaLaunchCooperativeKernel(reinterpret_cast<const void*>(product_kernel), dim3(grid), dim3(kThreads),
                                             argv, kSmemBytes, stream));
}

void run_large(int src, const void* g, int out_type, void* out, const StepArgs& s, const std::vector<Shape>& shapes,
               const Coeffs& k, const torch::Tensor& status, const at::TensorOptions& dev, at::cuda::CUDAEvent* ready) {
  for (size_t i = 0; i < shapes.size(); i += kMaxShapes)
    run_shapes(src, g, out_type, out, s, shapes.data() + i,
               static_cast<int>(std::min<size_t>(kMaxShapes, shapes.size() - i)), k, status, dev,
               i == 0 ? ready : nullptr);
}

}  // namespace muon
}  // namespace nori
