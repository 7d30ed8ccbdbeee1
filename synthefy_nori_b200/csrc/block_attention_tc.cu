// Attention of many query rows over a context cache in 8 bits with block scales, on the 5th-generation
// tensor cores.
//
// Persistent, one CTA of 28 warps per SM; a work item is 256 query rows (two tiles of 128) against a
// range of the keys of one (sequence, K/V head).  Roles:
//   warp 0        copies the codes of 128-key tiles of K and V, each one contiguous piece of the
//                 cache, into two rings (untiled bulk copies: no stride rules, so any width);
//   warps 4..7    widen the codes of K to fp16, exactly, into the swizzled tiles that the products
//   warps 8..11   read, and those of V: once for 256 query rows;
//   warps 1, 2    issue the products of one query tile each: S = Q K^T (128 x 64 x 64) and O += P V;
//   warps 12..27  softmax, four groups: (query tile) x (half of the keys of every tile), each with its
//                 own maximum, sum and accumulator; thread = query row (its TMEM lane), 64 score columns
//                 in registers; P (fp16 pairs) goes over S in TMEM and is the A operand of P V.
// A group's tile is a chain (scores, maximum, weights, two products) whose latency is several times its
// arithmetic, so four of them share an SM: with one thread for all 128 columns of a row and two
// groups the same arithmetic took 1.3 times as long, with row maxima exchanged between the
// halves 1.2 times.  The two halves of a query tile are joined once per item.
//
// Scales cost nothing per value: with c = scale log2(e) s_k 2^-e (2^e brings the query row into
// fp16's range, exactly) and t = c (q . k) + log2 s_v,
//   w = 2^(t - max t),  O = sum w v_code,  l = sum over blocks of (sum of w) / s_v.
// The maximum is lazy (O is rescaled when it grows by more than 2^4); w is kept at up to 2^15 so
// that fp16 holds 11 bits down to 2^-25 of the largest weight.  Scores, sums and O are fp32.
// All exponentials run on the MUFU: a polynomial on the FMA pipe for a quarter of them made a tile
// slower (3634 cycles for 3180), since the warps' issue slots are as scarce as the MUFU.
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
constexpr int kThreads = 896;
constexpr int kRing = 3;                 // stages of each ring (codes and fp16 tiles, K and V)
constexpr int kTile16 = kN * kD * 2;     // bytes of an fp16 tile of 128 x 64 (Q, K or V)
constexpr int kTile8 = kN * kD;          // room for a tile of codes
constexpr int kSmem = kTile16 * (2 + 2 * kRing) + kTile8 * 2 * kRing + 512 + 1024;
constexpr int kHalf = kN / 2;            // keys of a group's tile
// S 0..255 (64 a group, P over its first 32), O 256..511 (64 a group)
constexpr uint32_t kTmemCols = 512, kOcol = 256;
constexpr int kConvertWarps = 4, kSoftmaxWarp0 = 12;
// registers of a thread: launch 72 (896 threads); the softmax warps take what the others give up
constexpr uint32_t kRegsLow = 40, kRegsSoftmax = 96;
static_assert(12 * 32 * kRegsLow + 16 * 32 * kRegsSoftmax <= kThreads * 72, "register split over the launch total");

constexpr uint32_t idesc_f16(int M, int N, bool b_mn_major) {  // fp16 A and B, fp32 D
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
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
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float max32(const uint32_t (&v)[32]) {
  float m[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    m[i] = max3(__uint_as_float(v[i]), __uint_as_float(v[i + 8]), __uint_as_float(v[i + 16]));
#pragma unroll
  for (int i = 0; i < 8; ++i) m[i] = fmaxf(m[i], __uint_as_float(v[i + 24]));
  return max3(max3(m[0], m[1], m[2]), max3(m[3], m[4], m[5]), fmaxf(m[6], m[7]));
}

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// w = 2^(s c + shift) for 32 columns as fp16 pairs, to TMEM; returns their sum in fp32.
__device__ __forceinline__ float weights32(const uint32_t (&v)[32], float c, float shift, uint32_t tP) {
  const uint64_t c2 = f2pack(c, c), s2 = f2pack(shift, shift);
  uint64_t ra = 0, rb = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t pk[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float e0, e1;
      f2unpack(f2fma(f2pack(__uint_as_float(v[16 * h + 2 * i]), __uint_as_float(v[16 * h + 2 * i + 1])), c2, s2), e0, e1);
      e0 = exp2_mufu(e0), e1 = exp2_mufu(e1);
      pk[i] = pack_half2(e0, e1);
      if (i % 2)
        rb = f2add(rb, f2pack(e0, e1));
      else
        ra = f2add(ra, f2pack(e0, e1));
    }
    tmem_st8(tP + 8 * h, pk);
  }
  float r0, r1;
  f2unpack(f2add(ra, rb), r0, r1);
  return r0 + r1;
}

// (everything below 2^31, checked on the host: 64-bit divisions would take a microsecond an item)
struct Item {
  uint32_t b, h, split, bh;
  uint32_t pair, row0;  // pair of query tiles, its first row
  uint32_t tile0;       // first key tile
  int len;              // keys of the sequence
  int tiles;            // key tiles of this item
  int groups;           // query tiles with rows in them (1 or 2)
};

__device__ __forceinline__ Item item_at(const Attention& a, uint32_t w) {
  Item it;
  const uint32_t pairs = (static_cast<uint32_t>(a.rows) + kPairRows - 1) / kPairRows;
  it.pair = w % pairs;
  it.row0 = it.pair * kPairRows;
  w /= pairs;
  it.split = w % static_cast<uint32_t>(a.splits);
  it.bh = w / static_cast<uint32_t>(a.splits);
  it.b = it.bh / static_cast<uint32_t>(a.c.heads);
  it.h = it.bh - it.b * static_cast<uint32_t>(a.c.heads);
  it.len = static_cast<int>(min(max(a.length.at(it.b), int64_t{0}), a.c.cap));
  const uint32_t all = (static_cast<uint32_t>(it.len) + kN - 1) / kN, each = (all + a.splits - 1) / static_cast<uint32_t>(a.splits);
  it.tile0 = min(it.split * each, all);
  it.tiles = static_cast<int>(min(it.tile0 + each, all) - it.tile0);
  it.groups = it.row0 + kM < static_cast<uint32_t>(a.rows) ? 2 : 1;
  return it;
}

template <bool FP8>
__global__ void __launch_bounds__(kThreads, 1)
    tc_kernel(const __grid_constant__ Attention a, uint32_t items, bool q_vec,
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
  uint64_t* q_full = v_empty + kRing;     // [query tile] per item
  uint64_t* o_free = q_full + 2;          // [query tile] per item: O is in registers
  uint64_t* s_full = o_free + 2;          // [group] per tile: scores (and the last P V), and once more per item
  uint64_t* p_full = s_full + 4;          // [group] per tile: P is in TMEM
  uint64_t* pair = p_full + 4;            // [query tile][lane quarter] the two halves have exchanged
  uint64_t* done = pair + 8;              // [query tile] every product of this CTA
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  __shared__ float2 swap[2][16][32];  // [parity of the exchange][softmax warp][row]
  static_assert((8 * kRing + 22) * 8 + 8 <= 512, "barriers fit their room");

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (*reinterpret_cast<volatile int*>(a.status) != 0) return;  // another CTA or kernel timed out

  asm volatile("griddepcontrol.launch_dependents;");  // (the join of parts may be set up now)
  if (threadIdx.x == 0) {
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&rk_full[i], 1);
      mbar_init(&rv_full[i], 1);
      mbar_init(&rk_empty[i], kConvertWarps);
      mbar_init(&rv_empty[i], kConvertWarps);
      mbar_init(&k_full[i], kConvertWarps);
      mbar_init(&v_full[i], kConvertWarps);
      mbar_init(&k_empty[i], 2);
      mbar_init(&v_empty[i], 2);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 8);
      mbar_init(&o_free[t], 8);
      mbar_init(&done[t], 1);
    }
    for (int g = 0; g < 4; ++g) {
      mbar_init(&s_full[g], 1);
      mbar_init(&p_full[g], 4);
    }
    for (int i = 0; i < 8; ++i) mbar_init(&pair[i], 2);
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
      for (uint32_t w = blockIdx.x; ok && w < items; w += gridDim.x) {
        const Item it = item_at(a, w);
        const int64_t at = (it.bh * a.c.cap + static_cast<int64_t>(it.tile0) * kN) * a.c.stored;
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
  } else if (warp <= 2) {
    setmaxnreg_dec<kRegsLow>();
    if (elect_one()) {
      constexpr uint32_t idesc_s = idesc_f16(kM, kHalf, false), idesc_o = idesc_f16(kM, kD, true);
      const int t = warp - 1;          // query tile
      // operands: 32 bytes further for each 16 columns of Q and K, 2048 for each 16 keys of V
      const uint64_t dq = umma_desc_kmajor_sw128(smem_u32(sQ + t * kTile16));
      const uint64_t dk = umma_desc_kmajor_sw128(smem_u32(sK)), dv = umma_smem_desc(smem_u32(sV), 8192, 1024, 2);
      constexpr uint32_t kStage = kTile16 >> 4, kHalfTile = kStage / 2;
      uint32_t nk = 0, nv = 0;         // ring positions
      uint32_t cnt = 0;                // tiles of this query tile so far
      uint32_t qcnt = 0;               // items of this query tile so far
      bool ok = true;
      auto wait = [&](uint64_t* b, uint32_t parity) -> bool {
        return mbar_wait(b, parity & 1, a.status, kTimeoutMma, abort_flag);
      };
      for (uint32_t w = blockIdx.x; ok && w < items; w += gridDim.x) {
        const Item it = item_at(a, w);
        if (it.tiles == 0) continue;
        if (t >= it.groups) {  // no rows: the tiles of K and V are the other issuer's
          for (int j = 0; ok && j < it.tiles; ++j) {
            if (!(ok = wait(&k_full[nk % kRing], nk / kRing))) break;
            mbar_arrive(&k_empty[nk++ % kRing]);
            if (!(ok = wait(&v_full[nv % kRing], nv / kRing))) break;
            mbar_arrive(&v_empty[nv++ % kRing]);
          }
          continue;
        }
        auto scores = [&](int p) {  // of K tile nk, for keys 64 p .. + 63
          const uint64_t k = dk + nk % kRing * kStage + p * kHalfTile;
#pragma unroll
          for (int i = 0; i < kD / 16; ++i)
            umma_bf16_ss(tmem + (2 * t + p) * kHalf, dq + 2 * i, k + 2 * i, idesc_s, i > 0 ? 1u : 0u);
        };
        if (!(ok = wait(&q_full[t], qcnt) && wait(&k_full[nk % kRing], nk / kRing))) break;
        tc_fence_after();
        for (int p = 0; p < 2; ++p) {
          scores(p);
          umma_commit(&s_full[2 * t + p]);
        }
        umma_commit(&k_empty[nk++ % kRing]);
        for (int j = 0; ok && j < it.tiles; ++j, ++cnt) {
          const bool more = j + 1 < it.tiles;
          // the accumulators of the previous item have been read
          if (j == 0 && qcnt > 0 && !(ok = wait(&o_free[t], qcnt - 1))) break;
          if (!(ok = wait(&v_full[nv % kRing], nv / kRing) && (!more || wait(&k_full[nk % kRing], nk / kRing)))) break;
          for (int p = 0; p < 2; ++p) {
            const int g = 2 * t + p;
            if (!(ok = wait(&p_full[g], cnt))) break;
            tc_fence_after();
            const uint64_t v = dv + nv % kRing * kStage + p * kHalfTile;
#pragma unroll
            for (int i = 0; i < kHalf / 16; ++i)
              umma_bf16_ts(tmem + kOcol + g * kD, tmem + g * kHalf + i * 8, v + i * 128, idesc_o, (i > 0 || j > 0) ? 1u : 0u);
            // P V reads the columns that the next scores overwrite: products of one thread run in order
            if (more) scores(p);
            umma_commit(&s_full[g]);
          }
          if (!ok) break;
          umma_commit(&v_empty[nv++ % kRing]);
          if (more) umma_commit(&k_empty[nk++ % kRing]);
        }
        ++qcnt;
      }
      umma_commit(&done[t]);
      mbar_wait(&done[t], 0, a.status, kTimeoutMma, nullptr);
    }
  } else if (warp < 4) {
    setmaxnreg_dec<kRegsLow>();
  } else if (warp < kSoftmaxWarp0) {
    setmaxnreg_dec<kRegsLow>();
    // ------------------------------------------------------------ codes -> fp16 tiles
    // Thread: eight codes (unit c) of rows row0, row0 + 16, ..: fixed steps in both tiles.  The codes
    // are in registers before the fp16 tile's last reader is waited for.
    const bool is_v = warp >= 8;
    const uint32_t units = static_cast<uint32_t>(a.c.stored / 8), tid = threadIdx.x % (kConvertWarps * 32);
    const uint32_t row0 = tid / units, c = tid - row0 * units;
    const bool works = row0 < 16;
    const uint8_t* src = (is_v ? rV : rK) + row0 * a.c.stored + c * 8;
    uint8_t* dst = (is_v ? sV : sK) + row0 * 128 + ((c ^ (row0 & 7)) << 4);
    const uint32_t step = 16 * a.c.stored;
    uint64_t* code_full = is_v ? rv_full : rk_full;
    uint64_t* code_empty = is_v ? rv_empty : rk_empty;
    uint64_t* full = is_v ? v_full : k_full;
    uint64_t* empty = is_v ? v_empty : k_empty;
    uint32_t st = 0, ph = 0;
    bool ok = true;
    for (uint32_t w = blockIdx.x; ok && w < items; w += gridDim.x) {
      const Item it = item_at(a, w);
      const int tiles = it.tiles;
#pragma unroll 1
      for (int j = 0; j < tiles; ++j) {
        if (!(ok = mbar_wait_warp(&code_full[st], ph, a.status, kTimeoutEpilogue, abort_flag))) break;
        uint2 x[kN / 16];
        const uint8_t* from = src + st * kTile8;
        if (works) {
#pragma unroll
          for (int e = 0; e < kN / 16; ++e) x[e] = *reinterpret_cast<const uint2*>(from + e * step);
        }
        if (!(ok = mbar_wait_warp(&empty[st], ph ^ 1, a.status, kTimeoutEpilogue, abort_flag))) break;
        uint8_t* to = dst + st * kTile16;
        if (works) {
#pragma unroll
          for (int e = 0; e < kN / 16; ++e) {
            uint4 y;
            widen<FP8>(biased<FP8>(x[e].x), y.x, y.y);
            widen<FP8>(biased<FP8>(x[e].y), y.z, y.w);
            // codes behind the last row may be NaN (0 x NaN is none of its business)
            if (FP8 && is_v && static_cast<int>((it.tile0 + j) * kN + row0 + 16 * e) >= it.len) y = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(to + e * 2048) = y;
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          // (only now: with the codes released as soon as their loads were issued, the next copy overtook them)
          mbar_arrive(&code_empty[st]);
          mbar_arrive(&full[st]);
        }
        if (++st == kRing) st = 0, ph ^= 1;
      }
    }
  } else {
    setmaxnreg_inc<kRegsSoftmax>();
    // ------------------------------------------------------------ softmax
    // Group (query tile qt, half): 64 key columns of every tile; of Q and the result, columns 32 half ..
    // + 31.  The two warps of the same 32 rows exchange magnitudes of Q and, at the end, (maximum, sum).
    const int sw = warp - kSoftmaxWarp0, g = sw / 4, qt = g / 2, half = g % 2, quarter = sw % 4;
    const int r = quarter * 32 + lane;  // row of the tile == TMEM lane
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tS = tmem + g * kHalf + lane_off, tO = tmem + kOcol + g * kD + lane_off,
                   tO2 = tmem + kOcol + 2 * qt * kD + half * 32 + lane_off;  // this half's columns, both accumulators
    uint8_t* q_row = sQ + qt * kTile16 + r * 128;
    uint64_t* bar = &pair[qt * 4 + quarter];
    uint32_t cnt = 0;  // completions of s_full so far
    uint32_t xc = 0;   // exchanges so far
    bool ok = true;
    auto exchange = [&](float2 x) -> float2 {  // the other half's x for this row (valid if ok)
      swap[xc & 1][sw][lane] = x;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
      ok = mbar_wait_warp(bar, xc & 1, a.status, kTimeoutEpilogue, abort_flag);
      return swap[xc++ & 1][sw ^ 4][lane];
    };
    auto scores_ready = [&]() -> bool {
      ok = mbar_wait_warp(&s_full[g], cnt++ & 1, a.status, kTimeoutEpilogue, abort_flag);
      tc_fence_after();
      return ok;
    };
    for (uint32_t w = blockIdx.x; ok && w < items; w += gridDim.x) {
      const Item it = item_at(a, w);
      if (qt >= it.groups) continue;
      const uint32_t row = it.row0 + qt * kM + r;
      const bool there = row < a.rows;
      const uint32_t n = there ? row / static_cast<uint32_t>(a.group) : 0;
      const int head = static_cast<int>(it.h * a.group + (there ? row - n * a.group : 0));
      float m = -INFINITY, l = 0.f;
      if (it.tiles > 0) {
        // ---- 32 columns of the query row as fp16, times a power of two (the group's last scores are
        // done, so nothing reads its Q any more)
        float fac;
        {
          uint32_t x[16];
          const uint16_t* src = static_cast<const uint16_t*>(a.q.p) + a.q.offset(it.b, n, head) + half * 32;
          const int have = there ? a.c.width - half * 32 : 0;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (q_vec && c * 8 < have) v = __ldg(reinterpret_cast<const uint4*>(src) + c);
            x[4 * c] = v.x, x[4 * c + 1] = v.y, x[4 * c + 2] = v.z, x[4 * c + 3] = v.w;
          }
          if (!q_vec) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if (2 * i < have) x[i] = __ldg(src + 2 * i);
              if (2 * i + 1 < have) x[i] |= static_cast<uint32_t>(__ldg(src + 2 * i + 1)) << 16;
            }
          }
          uint32_t top2 = 0;  // magnitudes order like their bits, infinities and NaN on top
#pragma unroll
          for (int i = 0; i < 16; ++i) top2 = __vmaxu2(top2, x[i] & 0x7fff7fffu);
          uint32_t t16 = max(top2 & 0xffffu, top2 >> 16);
          t16 = max(t16, __float_as_uint(exchange(make_float2(__uint_as_float(t16), 0.f)).x));
          if (!ok) break;
          const bool bf = a.type == kBF16;
          const float top = bf ? __uint_as_float(t16 << 16) : __half2float(__ushort_as_half(static_cast<uint16_t>(t16)));
          float up, down;
          row_scale(top, up, down);
          fac = down * a.scale_log2;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
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
            *reinterpret_cast<uint4*>(q_row + (((4 * half + c) ^ (r & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&q_full[qt]);
        }
        const float* ks = a.c.k_scale + it.bh * a.c.blocks();
        const float* vs = a.c.v_scale + it.bh * a.c.blocks();
        // scales of the next tile: lane i those of this half's keys 32 (i % 2) .. + 31 (a block is 32 keys or more)
        const uint32_t key = it.tile0 * kN + kHalf * half + 32 * (lane & 1);
        float sk = __ldg(ks + (key >> a.c.block_log2)), sv = __ldg(vs + (key >> a.c.block_log2));
        for (int j = 0; j < it.tiles; ++j) {
          const int valid = min(it.len - static_cast<int>(it.tile0 + j) * kN, kN) - kHalf * half;
          float f0, f1, lv0, lv1, inv0, inv1;
          {
            const bool none = valid <= 32 * (lane & 1);  // a block behind the last row counts for nothing
            const float svc = none ? 1.f : safe_scale(sv);
            const float lv = __log2f(svc), inv = none ? 0.f : __fdividef(1.f, svc);
            // (never 0: a masked key's -inf stays -inf)
            f0 = fac * __shfl_sync(0xffffffffu, sk, 0), f1 = fac * __shfl_sync(0xffffffffu, sk, 1);
            f0 = valid <= 0 ? 1.f : f0 < 1e-38f ? 1e-38f : f0;
            f1 = valid <= 32 ? 1.f : f1 < 1e-38f ? 1e-38f : f1;
            lv0 = __shfl_sync(0xffffffffu, lv, 0), lv1 = __shfl_sync(0xffffffffu, lv, 1);
            inv0 = __shfl_sync(0xffffffffu, inv, 0), inv1 = __shfl_sync(0xffffffffu, inv, 1);
          }
          if (j + 1 < it.tiles) {
            const uint32_t blk = (key + static_cast<uint32_t>(j + 1) * kN) >> a.c.block_log2;
            sk = __ldg(ks + blk), sv = __ldg(vs + blk);
          }
          if (!scores_ready()) break;
          uint32_t s0[32], s1[32];
          tmem_ld32(tS, s0);
          tmem_ld32(tS + 32, s1);
          tmem_wait_ld();
          if (valid < kHalf) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              if (i >= valid) s0[i] = 0xff800000u;
              if (32 + i >= valid) s1[i] = 0xff800000u;
            }
          }
          const float cand = fmaxf(fmaf(max32(s0), f0, lv0), fmaf(max32(s1), f1, lv1));
          float back = 1.f;
          bool grow = false;
          if (j == 0) {
            m = cand;
          } else if (cand > m + kLazy) {
            back = exp2_mufu(m - cand);
            m = cand;
            grow = true;
          }
          const float lift = m == -INFINITY ? 0.f : kLift - m;  // (no key of this half is there)
          float sum = weights32(s0, f0, lv0 + lift, tS) * inv0;
          sum = fmaf(weights32(s1, f1, lv1 + lift, tS + 16), inv1, sum);
          l = fmaf(l, back, sum);
          // (the products before these scores are done: O may be changed)
          if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint32_t o[16];
              tmem_ld16(tO + q * 16, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * back);
              tmem_st16(tO + q * 16, o);
            }
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[g]);
        }
        if (!ok || !scores_ready()) break;  // the last P V
      }
      // ---- the halves joined: 32 columns of O from both accumulators
      float o[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = 0.f;
      if (it.tiles > 0) {
        if (!(m < INFINITY)) l = __uint_as_float(0x7fc00000u);  // an infinite score (or a NaN) somewhere
        const float2 other = exchange(make_float2(m, l));
        if (!ok) break;
        const float top = fmaxf(m, other.x);
        const float f = m == -INFINITY ? 0.f : exp2f(m - top), f2 = other.x == -INFINITY ? 0.f : exp2f(other.x - top);
        l = l * f + other.y * f2;
        m = top;
        const float fa = half ? f2 : f, fb = half ? f : f2;  // of the first and the second half's accumulator
        tc_fence_after();
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t x[16], y[16];
          tmem_ld16(tO2 + 16 * q, x);
          tmem_ld16(tO2 + kD + 16 * q, y);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) o[16 * q + i] = __uint_as_float(x[i]) * fa + __uint_as_float(y[i]) * fb;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free[qt]);
      }
      if (!there) continue;
      if (a.splits > 1) {
        const int64_t pairs = (static_cast<uint32_t>(a.rows) + kPairRows - 1) / kPairRows;
        const int64_t cell = (it.bh * pairs + it.pair) * a.splits + it.split;
        const int64_t pr = cell * kPairRows + qt * kM + r;
        if (half == 0) a.part_ml[pr] = make_float2(m, l);
        if (it.tiles > 0) {
          float4* dst = reinterpret_cast<float4*>(a.part_o + pr * kMaxWidth + half * 32);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            dst[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
        continue;
      }
      const float norm = l != 0.f ? 1.f / l : 0.f;
      uint16_t* dst = static_cast<uint16_t*>(a.o.p) + a.o.offset(it.b, n, head) + half * 32;
      const int have = a.c.width - half * 32;
      uint32_t y[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float lo = o[2 * i] * norm, hi = o[2 * i + 1] * norm;
        y[i] = a.type == kBF16 ? pack_bf16x2(lo, hi) : pack_half2(lo, hi);
      }
      if (o_vec) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (c * 8 < have)
            reinterpret_cast<uint4*>(dst)[c] = make_uint4(y[4 * c], y[4 * c + 1], y[4 * c + 2], y[4 * c + 3]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (2 * i < have) dst[2 * i] = static_cast<uint16_t>(y[i]);
          if (2 * i + 1 < have) dst[2 * i + 1] = static_cast<uint16_t>(y[i] >> 16);
        }
      }
      if (a.lse != nullptr && half == 0)
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

template <bool FP8>
cudaError_t tc_typed(const Attention& a, int ctas, cudaStream_t stream) {
  if (a.rows > INT32_MAX - kPairRows) return cudaErrorInvalidConfiguration;
  const int64_t items = (a.rows + kPairRows - 1) / kPairRows * a.splits * a.c.batch * a.c.heads;
  if (items > INT32_MAX) return cudaErrorInvalidConfiguration;
  const cudaError_t e = cudaFuncSetAttribute(tc_kernel<FP8>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  tc_kernel<FP8><<<static_cast<unsigned>(items < ctas ? items : ctas), kThreads, kSmem, stream>>>(
      a, static_cast<uint32_t>(items), vectors(a.q, a.c.width), vectors(a.o, a.c.width));
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_tc(const Attention& a, int ctas, cudaStream_t stream) {
  return a.c.fp8 ? tc_typed<true>(a, ctas, stream) : tc_typed<false>(a, ctas, stream);
}

}  // namespace bc
}  // namespace nori
