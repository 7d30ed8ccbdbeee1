// Attention of many query rows over a context cache in 8 bits with block scales, on the 5th-generation
// tensor cores.
//
// Persistent, one CTA of 16 warps per SM; a work item is 256 query rows (two tiles of 128, one per
// softmax group) against a range of the keys of one (sequence, K/V head).  Roles:
//   warp 0        copies the codes of 128-key tiles of K and V, each one contiguous piece of the
//                 cache, into two rings (untiled bulk copies: no stride rules, so any width);
//   warps 12..15  widen the codes to fp16, exactly, into the swizzled tiles that the products read;
//                 both groups use them, so a code is widened once for 256 query rows;
//   warp 1        issues S_g = Q_g K^T (128 x 128 x 64) and O_g += P_g V (A = P_g from TMEM); S_g of
//                 the next tile goes out as soon as group g has S_g in registers;
//   warps 4..11   softmax: thread = query row (its TMEM lane), the whole score row in registers; P_g
//                 (fp16 pairs) has TMEM columns of its own, so scores never wait for P . V.
//
// Scales cost nothing per value: with c = scale log2(e) s_k 2^-e (2^e brings the query row into
// fp16's range, exactly) and t = c (q . k) + log2 s_v,
//   w = 2^(t - max t),  O = sum w v_code,  l = sum over blocks of (sum of w) / s_v.
// The maximum is lazy (O is rescaled when it grows by more than 2^4); w is kept at up to 2^15 so
// that fp16 holds 11 bits down to 2^-25 of the largest weight.  Half of the exponentials run on the
// MUFU, half as a polynomial on the FMA pipe.  Scores, sums and O are fp32.
//
// Every wait is bounded (sm100.cuh); on a timeout the CTA records it in the status word, waits for
// its own copies and products, frees its TMEM and returns.
//
// Reference counterpart: attention over a quantised context cache (model/layer.py:747-934).
#include "block_cache.cuh"
#include "sm100.cuh"

namespace nori {
namespace bc {
namespace {

constexpr int kM = 128, kN = kTile, kD = kMaxWidth;
static_assert(kPairRows == 2 * kM);
constexpr int kThreads = 512;
constexpr int kRing = 3;                 // stages of each ring (codes and fp16 tiles, K and V)
constexpr int kTile16 = kN * kD * 2;     // bytes of an fp16 tile of 128 x 64 (Q, K or V)
constexpr int kTile8 = kN * kD;          // room for a tile of codes
constexpr int kSmem = kTile16 * (2 + 2 * kRing) + kTile8 * 2 * kRing + 512 + 1024;
// S 0..255 (128 a group), P 256..383 (64 a group), O 384..511 (64 a group)
constexpr uint32_t kTmemCols = 512, kPcol = 256, kOcol = 384;
constexpr int kConvertWarps = 4, kGroupWarps = 4;
// registers of a thread: launch 128 (512 threads); the softmax warps take what the others give up
constexpr uint32_t kRegsLow = 56, kRegsSoftmax = 200;
static_assert(8 * 32 * (kRegsLow + kRegsSoftmax) <= kThreads * 128, "register split over the launch total");

constexpr uint32_t idesc_f16(int M, int N, bool b_mn_major) {  // fp16 A and B, fp32 D
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// ------------------------------------------------------------------ 2^x
__device__ __forceinline__ float exp2_mufu(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint64_t f2pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2unpack(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t f2fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t f2add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2sub(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^x of a pair without the MUFU: x = n + f, n by adding 1.5 * 2^23, 2^f by a polynomial of degree 4
// fitted for the smallest relative error on [-0.5, 0.5] (2.7e-6), n added to the exponent.  x is
// held at -125 and above so that the result stays a normal number.
__device__ __forceinline__ void exp2_poly2(uint64_t x2, float& e0, float& e1) {
  constexpr float kRound = 12582912.0f;
  float x0, x1;
  f2unpack(x2, x0, x1);
  x2 = f2pack(fmaxf(x0, -125.0f), fmaxf(x1, -125.0f));
  const uint64_t r2 = f2pack(kRound, kRound);
  const uint64_t t2 = f2add(x2, r2);
  const uint64_t f2 = f2sub(x2, f2sub(t2, r2));
  uint64_t p = f2fma(f2, f2pack(0.009570102207362652f, 0.009570102207362652f),
                     f2pack(0.05591785907745361f, 0.05591785907745361f));
  p = f2fma(p, f2, f2pack(0.240247443318367f, 0.240247443318367f));
  p = f2fma(p, f2, f2pack(0.6931217908859253f, 0.6931217908859253f));
  p = f2fma(p, f2, f2pack(0.9999992847442627f, 0.9999992847442627f));
  float p0, p1, t0, t1;
  f2unpack(p, p0, p1);
  f2unpack(t2, t0, t1);
  e0 = __uint_as_float(__float_as_uint(p0) + (__float_as_uint(t0) << 23));
  e1 = __uint_as_float(__float_as_uint(p1) + (__float_as_uint(t1) << 23));
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float max32(const uint32_t (&v)[32], int valid) {
  if (valid >= 32) {
    float m[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      m[i] = max3(__uint_as_float(v[i]), __uint_as_float(v[i + 8]), __uint_as_float(v[i + 16]));
#pragma unroll
    for (int i = 0; i < 8; ++i) m[i] = fmaxf(m[i], __uint_as_float(v[i + 24]));
    return max3(max3(m[0], m[1], m[2]), max3(m[3], m[4], m[5]), fmaxf(m[6], m[7]));
  }
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (i < valid) m = fmaxf(m, __uint_as_float(v[i]));
  return m;
}

// w = 2^(s c + shift) for 32 columns as fp16 pairs; returns their sum in fp32.  Columns at or past
// `valid` give 0.
__device__ __forceinline__ float weights32(const uint32_t (&v)[32], int valid, float c, float shift, uint32_t (&pk)[16]) {
  if (valid >= 32) {
    const uint64_t c2 = f2pack(c, c), s2 = f2pack(shift, shift);
    uint64_t ra = 0, rb = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint64_t xa = f2fma(f2pack(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1])), c2, s2);
      const uint64_t xb = f2fma(f2pack(__uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3])), c2, s2);
      float x0, x1, e2, e3;
      f2unpack(xa, x0, x1);
      const float e0 = exp2_mufu(x0), e1 = exp2_mufu(x1);
      exp2_poly2(xb, e2, e3);
      pk[2 * i] = pack_half2(e0, e1);
      pk[2 * i + 1] = pack_half2(e2, e3);
      ra = f2add(ra, f2pack(e0, e1));
      rb = f2add(rb, f2pack(e2, e3));
    }
    float r0, r1;
    f2unpack(f2add(ra, rb), r0, r1);
    return r0 + r1;
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float e0 = 2 * i < valid ? exp2_mufu(fmaf(__uint_as_float(v[2 * i]), c, shift)) : 0.f;
    const float e1 = 2 * i + 1 < valid ? exp2_mufu(fmaf(__uint_as_float(v[2 * i + 1]), c, shift)) : 0.f;
    pk[i] = pack_half2(e0, e1);
    sum += e0 + e1;
  }
  return sum;
}

struct Item {
  int b, h, split;
  int64_t bh, row0, key0;  // first query row, first key
  int64_t len;             // keys of the sequence
  int tiles;               // key tiles of this item
  int groups;              // query tiles with rows in them (1 or 2)
};

__device__ __forceinline__ Item item_at(const Attention& a, int64_t w) {
  Item it;
  const int64_t pairs = (a.rows + kPairRows - 1) / kPairRows;
  it.row0 = w % pairs * kPairRows;
  w /= pairs;
  it.split = static_cast<int>(w % a.splits);
  it.bh = w / a.splits;
  it.b = static_cast<int>(it.bh / a.c.heads);
  it.h = static_cast<int>(it.bh % a.c.heads);
  it.len = min(max(a.length.at(it.b), int64_t{0}), a.c.cap);
  const int64_t all = (it.len + kN - 1) / kN, each = (all + a.splits - 1) / a.splits;
  const int64_t t0 = min(it.split * each, all);
  it.key0 = t0 * kN;
  it.tiles = static_cast<int>(min(t0 + each, all) - t0);
  it.groups = it.row0 + kM < a.rows ? 2 : 1;
  return it;
}

template <bool FP8>
__global__ void __launch_bounds__(kThreads, 1) tc_kernel(const __grid_constant__ Attention a, int64_t items, bool q_vec,
                                                         bool o_vec) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                     // [group]
  uint8_t* sK = sQ + 2 * kTile16;         // [kRing] fp16, swizzled
  uint8_t* sV = sK + kRing * kTile16;     // [kRing]
  uint8_t* rK = sV + kRing * kTile16;     // [kRing] codes
  uint8_t* rV = rK + kRing * kTile8;      // [kRing]
  uint64_t* bars = reinterpret_cast<uint64_t*>(rV + kRing * kTile8);
  uint64_t* rk_full = bars;               // codes have arrived
  uint64_t* rk_empty = rk_full + kRing;   // codes are widened
  uint64_t* rv_full = rk_empty + kRing;
  uint64_t* rv_empty = rv_full + kRing;
  uint64_t* k_full = rv_empty + kRing;    // fp16 tile is there
  uint64_t* k_empty = k_full + kRing;     // the products that read it are done
  uint64_t* v_full = k_empty + kRing;
  uint64_t* v_empty = v_full + kRing;
  uint64_t* q_full = v_empty + kRing;     // [group] per item
  uint64_t* s_full = q_full + 2;          // [group] per tile
  uint64_t* s_free = s_full + 2;          // [group] scores are in registers
  uint64_t* p_full = s_free + 2;          // [group]
  uint64_t* o_full = p_full + 2;          // [group] P . V of a tile is done
  uint64_t* o_free = o_full + 2;          // [group] per item: O is in registers
  uint64_t* done = o_free + 2;            // every product of this CTA
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((8 * kRing + 13) * 8 + 8 <= 512, "barriers fit their room");

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (*reinterpret_cast<volatile int*>(a.status) != 0) return;  // another CTA or kernel timed out

  if (threadIdx.x == 0) {
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&rk_full[i], 1);
      mbar_init(&rv_full[i], 1);
      mbar_init(&rk_empty[i], kConvertWarps);
      mbar_init(&rv_empty[i], kConvertWarps);
      mbar_init(&k_full[i], kConvertWarps);
      mbar_init(&v_full[i], kConvertWarps);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(&q_full[g], kGroupWarps);
      mbar_init(&s_full[g], 1);
      mbar_init(&s_free[g], kGroupWarps);
      mbar_init(&p_full[g], kGroupWarps);
      mbar_init(&o_full[g], 1);
      mbar_init(&o_free[g], kGroupWarps);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  // columns past the width are never written again: zero everywhere (finite, and 0 in Q)
  for (int i = threadIdx.x; i < kTile16 * (2 + 2 * kRing) / 16; i += kThreads)
    reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  if (warp == 1) tmem_alloc(tmem_slot, kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    setmaxnreg_dec<kRegsLow>();
    if (elect_one()) {
      const uint32_t bytes = static_cast<uint32_t>(kN * a.c.stored);
      uint32_t nk = 0, nv = 0;  // tiles asked for so far
      bool ok = true;
      for (int64_t w = blockIdx.x; ok && w < items; w += gridDim.x) {
        const Item it = item_at(a, w);
        const int64_t at = (it.bh * a.c.cap + it.key0) * a.c.stored;
        auto load = [&](int j, const uint8_t* src, uint8_t* dst, uint64_t* full, uint64_t* empty, uint32_t& n) -> bool {
          const uint32_t st = n % kRing;
          if (!mbar_wait(&empty[st], (n / kRing & 1) ^ 1, a.status, kTimeoutProducer, abort_flag)) return false;
          mbar_arrive_expect_tx(&full[st], bytes);
          bulk_load(dst + st * kTile8, src + at + static_cast<int64_t>(j) * bytes, bytes, &full[st]);
          ++n;
          return true;
        };
        if (it.tiles > 0) ok = load(0, a.c.k, rK, rk_full, rk_empty, nk);
        for (int j = 0; ok && j < it.tiles; ++j) {
          if (j + 1 < it.tiles) ok = load(j + 1, a.c.k, rK, rk_full, rk_empty, nk);
          if (ok) ok = load(j, a.c.v, rV, rv_full, rv_empty, nv);
        }
      }
      // own copies in flight (after an abort nobody else waits for them)
      for (uint32_t i = 0; i < kRing; ++i) {
        if (nk > i) mbar_wait(&rk_full[(nk - 1 - i) % kRing], (nk - 1 - i) / kRing & 1, a.status, kTimeoutProducer, nullptr);
        if (nv > i) mbar_wait(&rv_full[(nv - 1 - i) % kRing], (nv - 1 - i) / kRing & 1, a.status, kTimeoutProducer, nullptr);
      }
    }
  } else if (warp == 1) {
    setmaxnreg_dec<kRegsLow>();
    if (elect_one()) {
      constexpr uint32_t idesc_s = idesc_f16(kM, kN, false), idesc_o = idesc_f16(kM, kD, true);
      uint32_t nk = 0, nv = 0;         // ring positions
      uint32_t cnt[2] = {0, 0};        // tiles of a group whose P . V was issued
      uint32_t scnt[2] = {0, 0};       // tiles of a group whose scores were issued
      uint32_t qcnt[2] = {0, 0};       // items of a group
      bool ok = true;
      for (int64_t w = blockIdx.x; ok && w < items; w += gridDim.x) {
        const Item it = item_at(a, w);
        if (it.tiles == 0) continue;
        // scores of the next tile for one group; its K tile is freed behind the last group
        auto scores = [&](int g) -> bool {
          const uint32_t st = nk % kRing;
          if (!mbar_wait(&k_full[st], nk / kRing & 1, a.status, kTimeoutMma, abort_flag)) return false;
          if (scnt[g] > 0 && !mbar_wait(&s_free[g], (scnt[g] - 1) & 1, a.status, kTimeoutMma, abort_flag)) return false;
          tc_fence_after();
          const uint32_t q = smem_u32(sQ + g * kTile16), k = smem_u32(sK + st * kTile16);
#pragma unroll
          for (int i = 0; i < kD / 16; ++i)
            umma_bf16_ss(tmem + g * kN, umma_desc_kmajor_sw128(q + i * 32), umma_desc_kmajor_sw128(k + i * 32), idesc_s,
                         i > 0 ? 1u : 0u);
          umma_commit(&s_full[g]);
          ++scnt[g];
          if (g == it.groups - 1) {
            umma_commit(&k_empty[st]);
            ++nk;
          }
          return true;
        };
        for (int g = 0; ok && g < it.groups; ++g) {
          ok = mbar_wait(&q_full[g], qcnt[g] & 1, a.status, kTimeoutMma, abort_flag) && scores(g);
        }
        for (int j = 0; ok && j < it.tiles; ++j) {
          for (int g = 0; ok && g < it.groups; ++g) {
            if (j + 1 < it.tiles && !(ok = scores(g))) break;
            const uint32_t st = nv % kRing;
            ok = mbar_wait(&p_full[g], cnt[g] & 1, a.status, kTimeoutMma, abort_flag) &&
                 mbar_wait(&v_full[st], nv / kRing & 1, a.status, kTimeoutMma, abort_flag);
            // the accumulator of the group's previous item has been read
            if (ok && j == 0 && qcnt[g] > 0)
              ok = mbar_wait(&o_free[g], (qcnt[g] - 1) & 1, a.status, kTimeoutMma, abort_flag);
            if (!ok) break;
            tc_fence_after();
            const uint32_t v = smem_u32(sV + st * kTile16);
#pragma unroll
            for (int i = 0; i < kN / 16; ++i)
              umma_bf16_ts(tmem + kOcol + g * kD, tmem + kPcol + g * (kN / 2) + i * 8,
                           umma_smem_desc(v + i * 2048, 8192, 1024, 2), idesc_o, (i > 0 || j > 0) ? 1u : 0u);
            umma_commit(&o_full[g]);
            ++cnt[g];
            if (g == it.groups - 1) {
              umma_commit(&v_empty[st]);
              ++nv;
            }
          }
        }
        for (int g = 0; g < it.groups; ++g) ++qcnt[g];
      }
      umma_commit(done);
      mbar_wait(done, 0, a.status, kTimeoutMma, nullptr);
    }
  } else if (warp < 4) {
    setmaxnreg_dec<kRegsLow>();
  } else if (warp >= 12) {
    setmaxnreg_dec<kRegsLow>();
    // ------------------------------------------------------------ codes -> fp16 tiles
    const int tid = threadIdx.x - 12 * 32;
    const uint32_t units = static_cast<uint32_t>(a.c.stored / 8), inverse = 65536u / units + 1;
    uint32_t nk = 0, nv = 0;
    auto widen_tile = [&](const uint8_t* codes, uint8_t* tiles, uint64_t* cfull, uint64_t* cempty, uint64_t* full,
                          uint64_t* empty, uint32_t& n) -> bool {
      const uint32_t st = n % kRing, ph = n / kRing & 1;
      if (!mbar_wait_warp(&cfull[st], ph, a.status, kTimeoutEpilogue, abort_flag)) return false;
      if (!mbar_wait_warp(&empty[st], ph ^ 1, a.status, kTimeoutEpilogue, abort_flag)) return false;
      const uint2* src = reinterpret_cast<const uint2*>(codes + st * kTile8);
      uint8_t* dst = tiles + st * kTile16;
      // piece i: eight codes of row i / units; eight threads' pieces fill a row of 128 bytes
#pragma unroll 4
      for (uint32_t i = tid; i < kN * units; i += kConvertWarps * 32) {
        const uint32_t row = i * inverse >> 16, c = i - row * units;
        const uint2 x = src[i];
        uint4 y;
        widen<FP8>(biased<FP8>(x.x), y.x, y.y);
        widen<FP8>(biased<FP8>(x.y), y.z, y.w);
        *reinterpret_cast<uint4*>(dst + row * 128 + ((c ^ (row & 7)) << 4)) = y;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&cempty[st]);
        mbar_arrive(&full[st]);
      }
      ++n;
      return true;
    };
    bool ok = true;
    for (int64_t w = blockIdx.x; ok && w < items; w += gridDim.x) {
      const int tiles = item_at(a, w).tiles;
      if (tiles > 0) ok = widen_tile(rK, sK, rk_full, rk_empty, k_full, k_empty, nk);
      for (int j = 0; ok && j < tiles; ++j) {
        if (j + 1 < tiles) ok = widen_tile(rK, sK, rk_full, rk_empty, k_full, k_empty, nk);
        if (ok) ok = widen_tile(rV, sV, rv_full, rv_empty, v_full, v_empty, nv);
      }
    }
  } else {
    setmaxnreg_inc<kRegsSoftmax>();
    // ------------------------------------------------------------ softmax
    const int g = (warp - 4) / 4;
    const int r = (warp & 3) * 32 + lane;  // row of the tile == TMEM lane
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + g * kN + lane_off, tP = tmem + kPcol + g * (kN / 2) + lane_off,
                   tO = tmem + kOcol + g * kD + lane_off;
    uint8_t* q_row = sQ + g * kTile16 + r * 128;
    uint32_t cnt = 0;  // tiles of this group so far
    bool ok = true;
    for (int64_t w = blockIdx.x; ok && w < items; w += gridDim.x) {
      const Item it = item_at(a, w);
      if (g >= it.groups) continue;
      const int64_t row = it.row0 + g * kM + r;
      const bool there = row < a.rows;
      const int64_t n = there ? row / a.group : 0;
      const int head = it.h * a.group + static_cast<int>(there ? row % a.group : 0);
      float m = -INFINITY, l = 0.f;
      if (it.tiles > 0) {
        // ---- the query row as fp16, times a power of two (the group's last scores are done, so
        // nothing reads its Q any more)
        float fac;
        {
          uint32_t x[kD / 2];
          const uint16_t* src = static_cast<const uint16_t*>(a.q.p) + a.q.offset(it.b, n, head);
#pragma unroll
          for (int i = 0; i < kD / 2; ++i) x[i] = 0;
          if (there && q_vec) {
#pragma unroll
            for (int c = 0; c < kD / 8; ++c)
              if (c * 8 < a.c.width) {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(src) + c);
                x[4 * c] = v.x, x[4 * c + 1] = v.y, x[4 * c + 2] = v.z, x[4 * c + 3] = v.w;
              }
          } else if (there) {
#pragma unroll
            for (int i = 0; i < kD / 2; ++i) {
              if (2 * i < a.c.width) x[i] = __ldg(src + 2 * i);
              if (2 * i + 1 < a.c.width) x[i] |= static_cast<uint32_t>(__ldg(src + 2 * i + 1)) << 16;
            }
          }
          uint32_t top2 = 0;  // magnitudes order like their bits, infinities and NaN on top
#pragma unroll
          for (int i = 0; i < kD / 2; ++i) top2 = __vmaxu2(top2, x[i] & 0x7fff7fffu);
          const uint32_t t16 = max(top2 & 0xffffu, top2 >> 16);
          const bool bf = a.type == kBF16;
          const float top = bf ? __uint_as_float(t16 << 16) : __half2float(__ushort_as_half(static_cast<uint16_t>(t16)));
          float up, down;
          row_scale(top, up, down);
          fac = down * a.scale_log2 * kCodeScale<FP8>;
#pragma unroll
          for (int c = 0; c < kD / 8; ++c) {
            uint32_t y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t v = x[4 * c + i];
              float lo, hi;
              if (bf) {
                lo = __uint_as_float(v << 16), hi = __uint_as_float(v & 0xffff0000u);
              } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
                lo = f.x, hi = f.y;
              }
              y[i] = pack_half2(lo * up, hi * up);
            }
            *reinterpret_cast<uint4*>(q_row + ((c ^ (r & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&q_full[g]);
        }
        const float* ks = a.c.k_scale + it.bh * a.c.blocks();
        const float* vs = a.c.v_scale + it.bh * a.c.blocks();
        for (int j = 0; j < it.tiles; ++j, ++cnt) {
          const int64_t key = it.key0 + static_cast<int64_t>(j) * kN;
          const int valid = static_cast<int>(min(it.len - key, int64_t{kN}));
          // lane i holds the scales of keys 32 (i % 4) .. + 31 (a block is 32 keys or more)
          const int64_t blk = (key + 32 * (lane & 3)) >> a.c.block_log2;
          const float sk_l = __ldg(ks + blk) , sv_l = safe_scale(__ldg(vs + blk));
          const float lv_l = log2f(sv_l), inv_l = 1.f / sv_l;
          if (!(ok = mbar_wait_warp(&s_full[g], cnt & 1, a.status, kTimeoutEpilogue, abort_flag))) break;
          tc_fence_after();
          uint32_t s0[32], s1[32], s2[32], s3[32];
          tmem_ld32(tS, s0);
          tmem_ld32(tS + 32, s1);
          tmem_ld32(tS + 64, s2);
          tmem_ld32(tS + 96, s3);
          tmem_wait_ld();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_free[g]);
          float f[4], lv[4], inv[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            f[c] = fac * __shfl_sync(0xffffffffu, sk_l, c);
            lv[c] = __shfl_sync(0xffffffffu, lv_l, c);
            inv[c] = __shfl_sync(0xffffffffu, inv_l, c);
            if (valid <= 32 * c) inv[c] = 0.f;  // a block behind the last row counts for nothing, whatever its scale
          }
          float cand = fmaf(max32(s0, valid), f[0], lv[0]);
          if (valid > 32) cand = fmaxf(cand, fmaf(max32(s1, valid - 32), f[1], lv[1]));
          if (valid > 64) cand = fmaxf(cand, fmaf(max32(s2, valid - 64), f[2], lv[2]));
          if (valid > 96) cand = fmaxf(cand, fmaf(max32(s3, valid - 96), f[3], lv[3]));
          // the group's previous P . V is done: P and O may be written
          if (cnt > 0 && !(ok = mbar_wait_warp(&o_full[g], (cnt - 1) & 1, a.status, kTimeoutEpilogue, abort_flag))) break;
          float back = 1.f;
          bool grow = false;
          if (j == 0) {
            m = cand;
          } else if (cand > m + kLazy) {
            back = exp2_mufu(m - cand);
            m = cand;
            grow = true;
          }
          const float lift = kLift - m;
          float sum;
          {
            uint32_t pk[16];
            sum = weights32(s0, valid, f[0], lv[0] + lift, pk) * inv[0];
            tmem_st16(tP, pk);
            sum = fmaf(weights32(s1, valid - 32, f[1], lv[1] + lift, pk), inv[1], sum);
            tmem_st16(tP + 16, pk);
            sum = fmaf(weights32(s2, valid - 64, f[2], lv[2] + lift, pk), inv[2], sum);
            tmem_st16(tP + 32, pk);
            sum = fmaf(weights32(s3, valid - 96, f[3], lv[3] + lift, pk), inv[3], sum);
            tmem_st16(tP + 48, pk);
          }
          if (__any_sync(0xffffffffu, grow)) {
            tc_fence_after();
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              uint32_t o[32];
              tmem_ld32(tO + half * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * back);
              tmem_st32(tO + half * 32, o);
            }
          }
          l = fmaf(l, back, sum);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[g]);
        }
        if (!ok) break;
        if (!(ok = mbar_wait_warp(&o_full[g], (cnt - 1) & 1, a.status, kTimeoutEpilogue, abort_flag))) break;
        tc_fence_after();
      }
      // ---- O (64 columns) to memory
      uint32_t o0[32], o1[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) o0[i] = o1[i] = 0;
      if (it.tiles > 0) {
        tmem_ld32(tO, o0);
        tmem_ld32(tO + 32, o1);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free[g]);
        if (!(m < INFINITY)) l = __uint_as_float(0x7fc00000u);  // an infinite score (or a NaN) somewhere
      }
      if (!there) continue;
      if (a.splits > 1) {
        const int64_t cell = (it.bh * ((a.rows + kPairRows - 1) / kPairRows) + it.row0 / kPairRows) * a.splits + it.split;
        const int64_t pr = cell * kPairRows + g * kM + r;
        a.part_ml[pr] = make_float2(m, l);
        if (it.tiles > 0) {
          float4* dst = reinterpret_cast<float4*>(a.part_o + pr * kMaxWidth);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            dst[i] = make_float4(__uint_as_float(o0[4 * i]), __uint_as_float(o0[4 * i + 1]), __uint_as_float(o0[4 * i + 2]),
                                 __uint_as_float(o0[4 * i + 3]));
            dst[8 + i] = make_float4(__uint_as_float(o1[4 * i]), __uint_as_float(o1[4 * i + 1]),
                                     __uint_as_float(o1[4 * i + 2]), __uint_as_float(o1[4 * i + 3]));
          }
        }
        continue;
      }
      const float norm = l != 0.f ? kCodeScale<FP8> / l : 0.f;
      uint16_t* dst = static_cast<uint16_t*>(a.o.p) + a.o.offset(it.b, n, head);
      uint32_t y[kD / 2];
#pragma unroll
      for (int i = 0; i < kD / 2; ++i) {
        const float lo = __uint_as_float(i < 16 ? o0[2 * i] : o1[2 * i - 32]) * norm;
        const float hi = __uint_as_float(i < 16 ? o0[2 * i + 1] : o1[2 * i - 31]) * norm;
        y[i] = a.type == kBF16 ? pack_bf16x2(lo, hi) : pack_half2(lo, hi);
      }
      if (o_vec) {
#pragma unroll
        for (int c = 0; c < kD / 8; ++c)
          if (c * 8 < a.c.width)
            reinterpret_cast<uint4*>(dst)[c] = make_uint4(y[4 * c], y[4 * c + 1], y[4 * c + 2], y[4 * c + 3]);
      } else {
#pragma unroll
        for (int i = 0; i < kD / 2; ++i) {
          if (2 * i < a.c.width) dst[2 * i] = static_cast<uint16_t>(y[i]);
          if (2 * i + 1 < a.c.width) dst[2 * i + 1] = static_cast<uint16_t>(y[i] >> 16);
        }
      }
      if (a.lse != nullptr)
        a.lse[(static_cast<int64_t>(it.b) * a.c.heads * a.group + head) * a.n + n] = row_lse(m, l);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

bool vectors(const Rows& r, int width) {
  return width % 8 == 0 && reinterpret_cast<uintptr_t>(r.p) % 16 == 0 && r.s0 % 8 == 0 && r.s1 % 8 == 0 && r.sn % 8 == 0 &&
         r.sh % 8 == 0;
}

template <bool FP8>
cudaError_t tc_typed(const Attention& a, int ctas, cudaStream_t stream) {
  const int64_t items = (a.rows + kPairRows - 1) / kPairRows * a.splits * a.c.batch * a.c.heads;
  const cudaError_t e = cudaFuncSetAttribute(tc_kernel<FP8>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  tc_kernel<FP8><<<static_cast<unsigned>(items < ctas ? items : ctas), kThreads, kSmem, stream>>>(
      a, items, vectors(a.q, a.c.width), vectors(a.o, a.c.width));
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_tc(const Attention& a, int ctas, cudaStream_t stream) {
  return a.c.fp8 ? tc_typed<true>(a, ctas, stream) : tc_typed<false>(a, ctas, stream);
}

}  // namespace bc
}  // namespace nori
