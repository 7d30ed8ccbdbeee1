// Attention of few query rows (a single new row, rows of heads that share one K/V head) over a
// context cache in 8 bits with block scales; and the join of partial results.
//
// Bound: every stored byte is read once, 2 W bytes a key, for up to 16 rows.  So the work is split
// over the keys: a CTA takes a range of one (sequence, K/V head), its four warps every fourth piece
// of 32 keys, each with a running maximum, sum and output of its own; warps are joined in shared
// memory, up to eight ranges in their cluster's, and only more than eight through a workspace by a
// second kernel.
//
// Keys (of K) and values (of V, transposed) are the M side of m16n8k16 products, the query rows N, 8 or
// 16 of them.  The order of a summed index is free as long as both operands agree, so lanes take whole
// 8-byte units: in k . q lane (g, t) holds units t and t + 4 of keys g and g + 8; in v . w it holds unit g
// of four keys, and rows g, g + 8 of product j are values 8 g + 2 j and 8 g + 2 j + 1.  Weights go from the
// one product's result to the other's operand by 8 x 8 transposes.  Each warp keeps pieces of 32 keys in
// flight (contiguous bulk copies into a ring of its own; no warp waits for another), reads them in
// 8-byte units and widens them to fp16 in registers.
//
// Scales cost nothing per value.  With c = scale log2(e) s_k and t = c (q . k) + log2 s_v for the
// block of a key (one block per piece, since blocks are of 32 rows or more),
//   w = 2^(t - max t),  O = sum w v_code,  l = sum over blocks of (sum of w) / s_v,
//   out = O / l,  lse = ln 2 (max t + log2 l).
// Sums, maxima and outputs are fp32; w is rounded to fp16 (11 bits) for the product alone.
//
// One row x 168 x 50,000 keys x 56 int8 takes 185 us, 5.1 TB/s of codes (78% of the copy rate): 400
// instructions a piece keep the issue slots two thirds and the ALU (bytes put in place) 60% busy.
//
// Reference counterpart: attention over a quantised context cache (model/layer.py:747-934).
#include <cooperative_groups.h>

#include "block_cache.cuh"
#include "sm100.cuh"

namespace nori {
namespace bc {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kPiece = 32;  // keys of one step of a warp
constexpr int kStages = 2;  // pieces of a warp in flight
constexpr int resident(int row_tiles) { return row_tiles == 1 ? 5 : 4; }  // CTAs of an SM (registers)
constexpr int kPieceBytes = kPiece * kMaxWidth;

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float log2_fast(float x) {  // (of a normal number)
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 to_float2(uint32_t x, int type) {
  if (type == kBF16) return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}
__device__ __forceinline__ void put(void* p, int64_t i, float x, int type) {
  if (type == kBF16)
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else
    static_cast<__half*>(p)[i] = __float2half_rn(x);
}
// over the lanes that hold the same rows (t)
__device__ __forceinline__ float keys_max(float x) {
#pragma unroll
  for (int o = 4; o < 32; o *= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
__device__ __forceinline__ float keys_sum(float x) {
#pragma unroll
  for (int o = 4; o < 32; o *= 2) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {  // an 8 x 8 tile of 16-bit values
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

struct Row {  // where row r of a K/V head's query rows lies
  int64_t n;
  int head;
  __device__ __forceinline__ Row(const Attention& a, int kv_head, int64_t r)
      : n(r / a.group), head(kv_head * a.group + static_cast<int>(r % a.group)) {}
};

// NT: tiles of 8 query rows.  W: bytes of a stored row (with it known at compile time every load has a
// fixed offset: 171 us for 253 at 168 x 50,000 x 56).  Lanes whose unit lies past the row read what
// follows it in the ring: q is 0 there, and no result is taken from there (e4m3's NaN is cleared first).
// Which key of eight stands at place i of a product: lanes t of V's operand then read rows of both
// parities, which for rows of 64 bytes are different banks.
__device__ __forceinline__ constexpr int key_at(int i) { return (i & 4) | (i & 1) << 1 | (i >> 1 & 1); }

template <bool FP8, int NT, int W>
__global__ void __launch_bounds__(kThreads, resident(NT)) few_kernel(Attention a, bool q_vec) {
  constexpr int kHalf = W > 32 ? 2 : 1;  // units of a lane in k . q: t and t + 4, or 2 t and 2 t + 1 in one load
  constexpr bool kPairs = kHalf == 2 && W % 16 == 0;
  constexpr int kRows = 8 * NT;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
  const auto unit_of = [&](int i) { return kPairs ? 2 * t + i : t + 4 * i; };
  const int64_t tiles = (a.rows - a.first + kRows - 1) / kRows;
  const int split = static_cast<int>(blockIdx.x % a.splits);
  const int64_t cell = blockIdx.x / a.splits;
  const int64_t tile = cell % tiles, bh = cell / tiles;
  const int b = static_cast<int>(bh / a.c.heads), h = static_cast<int>(bh % a.c.heads);
  const int64_t row0 = a.first + tile * kRows;

  asm volatile("griddepcontrol.launch_dependents;");  // (the join of parts may be set up now)
  // this CTA's keys: whole pieces, the same number for every split
  const int64_t len = min(max(a.length.at(b), int64_t{0}), a.c.cap);
  const int64_t pieces = (len + kPiece - 1) / kPiece, each = (pieces + a.splits - 1) / a.splits;
  const int64_t p0 = split * each, p1 = min(p0 + each, pieces);

  const uint8_t* kbase = a.c.k + bh * a.c.cap * W;
  const uint8_t* vbase = a.c.v + bh * a.c.cap * W;
  const float* ks = a.c.k_scale + bh * a.c.blocks();
  const float* vs = a.c.v_scale + bh * a.c.blocks();
  constexpr uint32_t bytes = kPiece * W;
  static_assert((kPiece - 1) * W + kMaxWidth <= kPieceBytes);

  // this warp's ring of pieces (K, then V): contiguous copies that lane 0 asks for kStages ahead
  extern __shared__ __align__(128) uint8_t ring_all[];
  __shared__ uint64_t bars[kWarps][kStages];
  uint8_t* ring = ring_all + warp * (kStages * 2 * kPieceBytes);
  const int64_t first = p0 + warp;
  const int mine = static_cast<int>(first < p1 ? (p1 - first + kWarps - 1) / kWarps : 0);  // this warp's pieces
  const uint8_t *k_next = kbase + first * bytes, *v_next = vbase + first * bytes;
  auto ask = [&](int i) {  // (for every piece in turn)
    uint64_t* bar = &bars[warp][i % kStages];
    uint8_t* dst = ring + i % kStages * (2 * kPieceBytes);
    mbar_arrive_expect_tx(bar, 2 * bytes);
    bulk_load(dst, k_next, bytes, bar);
    bulk_load(dst + kPieceBytes, v_next, bytes, bar);
    k_next += kWarps * bytes, v_next += kWarps * bytes;
  };
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&bars[warp][i], 1);
    fence_barrier_init();
    for (int i = 0; i < min(mine, kStages); ++i) ask(i);
  }
  __syncwarp();

  // the query rows as operand B (lane: row g, its units) while the first pieces arrive; a power of two
  // brings each into fp16's range, exactly; fac[nt][i]: of row 8 nt + 2 t + i
  uint32_t qf[NT][2 * kHalf][2];
  float fac[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int64_t r = row0 + 8 * nt + g;
    const bool there = r < a.rows;
    float x[kHalf][8], top = 0.f;
    bool bad = false;
    const Row row(a, h, there ? r : 0);
    const int64_t at = a.q.offset(b, row.n, row.head);
#pragma unroll
    for (int i = 0; i < kHalf; ++i) {
      const int d = 8 * unit_of(i);
      uint32_t w[4] = {0, 0, 0, 0};
      const uint16_t* src = static_cast<const uint16_t*>(a.q.p) + at + d;
      if (q_vec) {
        if (there && d < a.c.width) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(src));
          w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (there && d + e < a.c.width) w[e / 2] |= static_cast<uint32_t>(__ldg(src + e)) << 16 * (e % 2);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = to_float2(w[e], a.type);
        x[i][2 * e] = f.x, x[i][2 * e + 1] = f.y;
        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        bad |= f.x != f.x || f.y != f.y;
      }
    }
    if (bad) top = INFINITY;
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    float up, down;
    row_scale(top, up, down);
    down *= a.scale_log2;
    fac[nt][0] = __shfl_sync(0xffffffffu, down, 8 * t);      // lane (2 t, 0)
    fac[nt][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);  // lane (2 t + 1, 0)
#pragma unroll
    for (int i = 0; i < kHalf; ++i)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        qf[nt][2 * i + s][0] = pack_half2(x[i][4 * s] * up, x[i][4 * s + 1] * up);
        qf[nt][2 * i + s][1] = pack_half2(x[i][4 * s + 2] * up, x[i][4 * s + 3] * up);
      }
  }

  float o[NT][4][4];  // [row tile][product j]: (value 8 g + 2 j, row 2 t), (.., 2 t + 1), (value + 1, 2 t), ..
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[nt][j][i] = 0.f;
    m[nt][0] = m[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.f;
  }
  float sk = 0.f, sv = 0.f, least = kLeastScale;
  // (a warp's pieces are 128 keys apart, a whole number of blocks)
  const int64_t blk = first * kPiece >> a.c.block_log2;
  const int blk_step = kWarps * kPiece >> a.c.block_log2;
  static_assert(kWarps * kPiece == 128);
  ks += blk, vs += blk;
  if (mine > 0) sk = __ldg(ks), sv = __ldg(vs);
  int rest = static_cast<int>(len - first * kPiece);  // keys from this piece's first on

  for (int i = 0; i < mine; ++i, rest -= kWarps * kPiece) {
    raise_floor(least, sv);
    const float sk_now = sk, svc = safe_scale(sv, least);
    if (i + 1 < mine) sk = __ldg(ks += blk_step), sv = __ldg(vs += blk_step);
    if (!mbar_wait_warp(&bars[warp][i % kStages], i / kStages & 1, a.status, kTimeoutEpilogue, nullptr)) {
      if (lane == 0)  // own copies in flight
        for (int k = i; k < min(mine, i + kStages); ++k)
          mbar_wait(&bars[warp][k % kStages], k / kStages & 1, a.status, kTimeoutEpilogue, nullptr);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) l[nt][0] = l[nt][1] = __uint_as_float(0x7fc00000u);  // no result of a part of the keys
      break;
    }
    const uint8_t* kp = ring + i % kStages * (2 * kPieceBytes) + key_at(g) * W + unit_of(0) * 8;
    const uint8_t* vp = ring + i % kStages * (2 * kPieceBytes) + kPieceBytes + key_at(2 * t) * W + g * 8;
    uint2 kq[4][kHalf], vq[2][4];
#pragma unroll
    for (int nt = 0; nt < 4; ++nt) {
      if constexpr (kPairs) {
        const uint4 x = *reinterpret_cast<const uint4*>(kp + nt * 8 * W);
        kq[nt][0] = make_uint2(x.x, x.y), kq[nt][1] = make_uint2(x.z, x.w);
      } else {
#pragma unroll
        for (int j = 0; j < kHalf; ++j) kq[nt][j] = *reinterpret_cast<const uint2*>(kp + nt * 8 * W + j * 32);
      }
      if constexpr (FP8 && W % 32 != 0) {
#pragma unroll
        for (int j = 0; j < kHalf; ++j) {
          const uint32_t in_row = unit_of(j) < W / 8 ? 0xffffffffu : 0u;
          kq[nt][j].x &= in_row, kq[nt][j].y &= in_row;
        }
      }
    }
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e)  // (key_at(2 t + 1) = key_at(2 t) + 2)
        vq[kt][e] = *reinterpret_cast<const uint2*>(vp + (kt * 16 + (e >> 1) * 8 + (e & 1) * 2) * W);
    const int left = min(rest, kPiece);  // keys of the piece that are there
    if (FP8 && left < kPiece) {  // codes behind the last row may be NaN (0 x NaN is none of its business)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (kt * 16 + (e >> 1) * 8 + (e & 1) * 2 + key_at(2 * t) >= left) vq[kt][e] = make_uint2(0, 0);
    }
    // scores of keys 16 kt + g (values 0, 1) and + 8 (2, 3), rows 2 t and 2 t + 1
    float s[NT][2][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][kt][e] = 0.f;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int j = 0; j < kHalf; ++j) {
        uint32_t af[4];
        widen<FP8>(biased<FP8>(kq[2 * kt][j].x), af[0], af[2]);
        widen<FP8>(biased<FP8>(kq[2 * kt + 1][j].x), af[1], af[3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816(s[nt][kt], af, qf[nt][2 * j][0], qf[nt][2 * j][1]);
        widen<FP8>(biased<FP8>(kq[2 * kt][j].y), af[0], af[2]);
        widen<FP8>(biased<FP8>(kq[2 * kt + 1][j].y), af[1], af[3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816(s[nt][kt], af, qf[nt][2 * j + 1][0], qf[nt][2 * j + 1][1]);
      }
    // (approximate: 2^-22 of a log2 that reaches -49 is 1e-5 of a weight, 1 / 30 of its rounding to fp16)
    const float lv = log2_fast(svc), inv = rcp_fast(svc);
    if (left < kPiece) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (16 * kt + 8 * (e >> 1) + key_at(g) >= left) s[nt][kt][e] = -INFINITY;
    }
    // the maximum moves only where a score is more than 2^kLazy above it: rarely, and only then do the
    // lanes of a row exchange theirs
    float cand[NT][2];
    bool grow = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i2 = 0; i2 < 2; ++i2) {
        const float mx = fmaxf(fmaxf(s[nt][0][i2], s[nt][0][2 + i2]), fmaxf(s[nt][1][i2], s[nt][1][2 + i2]));
        cand[nt][i2] = fmaf(mx, fac[nt][i2] * sk_now, lv);
        grow |= !(cand[nt][i2] <= m[nt][i2] + kLazy);  // (also the first piece, and a NaN)
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i2 = 0; i2 < 2; ++i2) {
          const float all = keys_max(cand[nt][i2]);
          if (all > m[nt][i2] + kLazy || m[nt][i2] == -INFINITY) {
            const float h = m[nt][i2] == -INFINITY ? 0.f : exp2_fast(0.5f * (m[nt][i2] - all)), back = h * h;
            m[nt][i2] = all;
            l[nt][i2] = lowered(l[nt][i2], h);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[nt][j][i2] *= back, o[nt][j][2 + i2] *= back;
          }
        }
    }
    uint32_t pf[NT][4];  // weights as operand B: [keys 8 i ..]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i2 = e & 1;
          float& x = s[nt][kt][e];
          x = exp2_fast(fmaf(x, fac[nt][i2] * sk_now, lv - m[nt][i2] + kLift));
          // (a masked key's weight is 0 whatever the scale)
          if (left < kPiece && 16 * kt + 8 * (e >> 1) + key_at(g) >= left) x = 0.f;
          sum[i2] += x;
        }
        pf[nt][2 * kt] = transposed(pack_half2(s[nt][kt][0], s[nt][kt][1]));
        pf[nt][2 * kt + 1] = transposed(pack_half2(s[nt][kt][2], s[nt][kt][3]));
      }
      l[nt][0] = fmaf(sum[0], inv, l[nt][0]);
      l[nt][1] = fmaf(sum[1], inv, l[nt][1]);
    }
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint32_t x0 = biased<FP8>(w ? vq[kt][0].y : vq[kt][0].x), x1 = biased<FP8>(w ? vq[kt][1].y : vq[kt][1].x);
        const uint32_t x2 = biased<FP8>(w ? vq[kt][2].y : vq[kt][2].x), x3 = biased<FP8>(w ? vq[kt][3].y : vq[kt][3].x);
#pragma unroll
        for (int u = 0; u < 2; ++u) {  // values 4 w + 2 u and + 1 of unit g: (key, next key)
          uint32_t af[4];
          widen<FP8>(__byte_perm(x0, x1, u ? 0x7362 : 0x5140), af[0], af[1]);
          widen<FP8>(__byte_perm(x2, x3, u ? 0x7362 : 0x5140), af[2], af[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][2 * w + u], af, pf[nt][2 * kt], pf[nt][2 * kt + 1]);
        }
      }
    // the codes have been used by every lane: their place may be filled again
    __syncwarp();
    if (lane == 0 && i + kStages < mine) ask(i + kStages);
  }

  // join the warps
  __shared__ float sm_m[kWarps][16], sm_l[kWarps][16];
  auto sm_o = reinterpret_cast<float(*)[kRows][kMaxWidth + 4]>(ring_all);  // (in place of the rings)
  static_assert(sizeof(float) * kWarps * kRows * (kMaxWidth + 4) <= kWarps * kStages * 2 * kPieceBytes);
  __syncthreads();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 8 * nt + 2 * t + i;
      const float sum = keys_sum(l[nt][i]);
      if (g == 0) sm_m[warp][r] = m[nt][i], sm_l[warp][r] = sum;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sm_o[warp][r][8 * g + 2 * j] = o[nt][j][i];
        sm_o[warp][r][8 * g + 2 * j + 1] = o[nt][j][2 + i];
      }
    }
  __syncthreads();
  const int64_t left_rows = a.rows - row0;
  const int rows = static_cast<int>(left_rows < kRows ? left_rows : kRows);
  __shared__ float2 fin_ml[kRows];
  float* fin_o = reinterpret_cast<float*>(ring_all) + kWarps * kRows * (kMaxWidth + 4);
  static_assert(sizeof(float) * kRows * (kWarps * (kMaxWidth + 4) + kMaxWidth) <= kWarps * kStages * 2 * kPieceBytes);
  // where value d of row r goes: the result, or a part of it
  auto put_row = [&](int r, int d, float top, float sum, float acc) {
    if (a.splits > a.cluster) {
      const int64_t at = (cell * (a.splits / a.cluster) + split / a.cluster) * kRows + r;
      a.part_o[at * kMaxWidth + d] = acc;
      if (d == 0) a.part_ml[at] = make_float2(top, sum);
      return;
    }
    const Row row(a, h, row0 + r);
    if (d < a.c.width) put(a.o.p, a.o.offset(b, row.n, row.head) + d, sum != 0.f ? acc / sum : 0.f, a.type);
    if (d == 0 && a.lse != nullptr)
      a.lse[(static_cast<int64_t>(b) * a.c.heads * a.group + row.head) * a.n + row.n] = row_lse(top, sum);
  };
  for (int i = threadIdx.x; i < rows * kMaxWidth; i += kThreads) {
    const int r = i / kMaxWidth, d = i % kMaxWidth;
    float top = sm_m[0][r];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sm_m[w][r]);
    float sum = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float h = sm_m[w][r] == -INFINITY && sm_l[w][r] == 0.f ? 0.f : exp2f(0.5f * (sm_m[w][r] - top));
      sum = fmaf(sm_l[w][r] * h, h, sum);
      acc = fmaf(sm_o[w][r][d], h * h, acc);
    }
    if (a.cluster == 1) {
      put_row(r, d, top, sum, acc);
    } else {
      fin_o[r * kMaxWidth + d] = acc;
      if (d == 0) fin_ml[r] = make_float2(top, sum);
    }
  }
  // where this kernel was launched beside one that still runs: what follows on the stream waits for this one
  // alone, so it ends no sooner
  const auto wait_beside = [] { asm volatile("griddepcontrol.wait;" ::: "memory"); };
  if (a.cluster == 1) return wait_beside();
  // join the cluster: every CTA has written its part; the threads of all share the values
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  for (int i = static_cast<int>(cluster.block_rank()) * kThreads + threadIdx.x; i < rows * kMaxWidth;
       i += a.cluster * kThreads) {
    const int r = i / kMaxWidth, d = i % kMaxWidth;
    float2 ml[8];
    float v[8], top = -INFINITY;
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < a.cluster) {
        ml[c] = cluster.map_shared_rank(fin_ml, c)[r];
        v[c] = cluster.map_shared_rank(fin_o, c)[i];
        top = fmaxf(top, ml[c].x);
      }
    float sum = 0.f, acc = 0.f;
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < a.cluster) {
        const float h = ml[c].x == -INFINITY && ml[c].y == 0.f ? 0.f : exp2f(0.5f * (ml[c].x - top));
        sum = fmaf(ml[c].y * h, h, sum);
        acc = fmaf(v[c], h * h, acc);
      }
    put_row(r, d, top, sum, acc);
  }
  cluster.sync();  // nobody leaves while its shared memory is read
  wait_beside();
}

// Joins the parts of a row: 16 lanes, four values each, take its parts four at a time (so that their loads
// do not wait for one another) under a running maximum.  Few parts: a CTA takes 16 rows; many: a CTA takes a
// row, its 16 groups of lanes every 16th part.  43,008 rows of 4 parts: a warp for a row, the maximum of all
// parts first, took 39 us for 14.  Started while the kernel before it still runs (its last CTAs leave the
// launch's latency free), it waits for it before the first read.
constexpr int kJoinThreads = 256, kJoinRows = kJoinThreads / 16;
__device__ __forceinline__ void fma4(float4& y, const float4& x, float f) {
  y.x = fmaf(x.x, f, y.x), y.y = fmaf(x.y, f, y.y), y.z = fmaf(x.z, f, y.z), y.w = fmaf(x.w, f, y.w);
}
struct Joined {
  float top = -INFINITY, sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  __device__ __forceinline__ void rescale(float t) {
    const float h = top == -INFINITY ? 0.f : exp2f(0.5f * (top - t)), back = h * h;
    top = t, sum = lowered(sum, h);
    acc.x *= back, acc.y *= back, acc.z *= back, acc.w *= back;
  }
};
template <bool MANY>
__global__ void __launch_bounds__(kJoinThreads) combine_kernel(Attention a, int tile_rows, int parts) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const bool written = read_status(a.status) == 0;  // (the parts may never have been, after a wait that ran out)
  const int lane = threadIdx.x % 16, group = threadIdx.x / 16;
  const uint32_t unit = MANY ? blockIdx.x : blockIdx.x * kJoinRows + group;  // rows of the cells that are split
  const uint32_t count = static_cast<uint32_t>(a.rows - a.first), tiles = (count + tile_rows - 1) / tile_rows;
  const uint32_t split_cell = unit / tile_rows, in_tile = unit - split_cell * tile_rows;
  const uint32_t cell = static_cast<uint32_t>(a.whole) + split_cell, bh = cell / tiles;
  const uint32_t r = (cell - bh * tiles) * tile_rows + in_tile;
  if (bh >= static_cast<uint32_t>(a.c.batch) * a.c.heads || r >= count) return;  // (a whole CTA where MANY)
  const int64_t at = static_cast<int64_t>(split_cell) * parts * tile_rows + in_tile;  // of part 0
  const float4* part_o = reinterpret_cast<const float4*>(a.part_o) + lane;
  constexpr int kStride = MANY ? kJoinRows : 1;
  Joined j;
  for (int s0 = MANY ? group : 0; s0 < parts; s0 += 4 * kStride) {
    float2 ml[4];
    float4 v[4];
    float t = j.top;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int s = s0 + k * kStride;
      ml[k] = make_float2(-INFINITY, 0.f);
      v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (s < parts) {
        const int64_t i = at + static_cast<int64_t>(s) * tile_rows;
        ml[k] = a.part_ml[i];
        v[k] = part_o[i * (kMaxWidth / 4)];
      }
      t = fmaxf(t, ml[k].x);
    }
    j.rescale(t);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (ml[k].x == -INFINITY && ml[k].y == 0.f) continue;  // no keys there (and perhaps no values written)
      const float h = exp2f(0.5f * (ml[k].x - t));
      j.sum = fmaf(ml[k].y * h, h, j.sum);
      fma4(j.acc, v[k], h * h);
    }
  }
  if constexpr (MANY) {
    __shared__ float4 sm_o[kJoinRows][16];
    __shared__ float2 sm_ml[kJoinRows];
    sm_o[group][lane] = j.acc;
    if (lane == 0) sm_ml[group] = make_float2(j.top, j.sum);
    __syncthreads();
    if (group > 0) return;
    float t = -INFINITY;
#pragma unroll
    for (int w = 0; w < kJoinRows; ++w) t = fmaxf(t, sm_ml[w].x);
    j = Joined();
    j.top = t;
#pragma unroll
    for (int w = 0; w < kJoinRows; ++w) {
      if (sm_ml[w].x == -INFINITY && sm_ml[w].y == 0.f) continue;
      const float h = exp2f(0.5f * (sm_ml[w].x - t));
      j.sum = fmaf(sm_ml[w].y * h, h, j.sum);
      fma4(j.acc, sm_o[w][lane], h * h);
    }
  }
  const int b = static_cast<int>(bh / a.c.heads), h = static_cast<int>(bh % a.c.heads);
  const Row row(a, h, a.first + r);
  const float norm = j.sum != 0.f ? 1.f / j.sum : 0.f;
  const int64_t out = a.o.offset(b, row.n, row.head) + 4 * lane;
  const float y[4] = {j.acc.x * norm, j.acc.y * norm, j.acc.z * norm, j.acc.w * norm};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (written && 4 * lane + i < a.c.width) put(a.o.p, out + i, y[i], a.type);
  if (written && lane == 0 && a.lse != nullptr)
    a.lse[(static_cast<int64_t>(b) * a.c.heads * a.group + row.head) * a.n + row.n] = row_lse(j.top, j.sum);
}

template <bool FP8, int NT, int W>
cudaError_t few_typed(const Attention& a, bool beside, cudaStream_t stream) {
  constexpr int kRows = 8 * NT;
  const int64_t grid = (a.rows - a.first + kRows - 1) / kRows * a.splits * a.c.batch * a.c.heads;
  if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
  constexpr int kSmem = kWarps * kStages * 2 * kPieceBytes;
  const cudaError_t e =
      cudaFuncSetAttribute(few_kernel<FP8, NT, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2]{};
  cfg.attrs = attr;
  if (a.cluster > 1) {
    cudaLaunchAttribute& x = attr[cfg.numAttrs++];
    x.id = cudaLaunchAttributeClusterDimension;
    x.val.clusterDim.x = static_cast<unsigned>(a.cluster);
    x.val.clusterDim.y = x.val.clusterDim.z = 1;
  }
  if (beside) {
    cudaLaunchAttribute& x = attr[cfg.numAttrs++];
    x.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    x.val.programmaticStreamSerializationAllowed = 1;
  }
  return cudaLaunchKernelEx(&cfg, few_kernel<FP8, NT, W>, a, access_bytes(a.q, a.c.width) == 16);
}

}  // namespace

int few_tile_rows(int64_t rows) { return rows > 8 ? 16 : 8; }
int few_resident(int64_t rows) { return resident(few_tile_rows(rows) / 8); }

cudaError_t launch_few(const Attention& a, bool beside, cudaStream_t stream) {
  const bool two = few_tile_rows(a.rows - a.first) == 16;
  auto go = [&](auto w) {
    constexpr int W = w.value;
    if (a.c.fp8) return two ? few_typed<true, 2, W>(a, beside, stream) : few_typed<true, 1, W>(a, beside, stream);
    return two ? few_typed<false, 2, W>(a, beside, stream) : few_typed<false, 1, W>(a, beside, stream);
  };
  switch (a.c.stored) {
    case 8: return go(std::integral_constant<int, 8>());
    case 16: return go(std::integral_constant<int, 16>());
    case 24: return go(std::integral_constant<int, 24>());
    case 32: return go(std::integral_constant<int, 32>());
    case 40: return go(std::integral_constant<int, 40>());
    case 48: return go(std::integral_constant<int, 48>());
    case 56: return go(std::integral_constant<int, 56>());
    case 64: return go(std::integral_constant<int, 64>());
  }
  return cudaErrorInvalidValue;
}

cudaError_t launch_combine(const Attention& a, int tile_rows, cudaStream_t stream) {
  const int parts = a.splits / a.cluster;
  const bool many = parts > 32;
  const int64_t cells = (a.rows - a.first + tile_rows - 1) / tile_rows * a.c.batch * a.c.heads - a.whole;
  const int64_t rows = cells * tile_rows, grid = many ? rows : (rows + kJoinRows - 1) / kJoinRows;
  if (rows > INT32_MAX) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return many ? cudaLaunchKernelEx(&cfg, combine_kernel<true>, a, tile_rows, parts)
              : cudaLaunchKernelEx(&cfg, combine_kernel<false>, a, tile_rows, parts);
}

}  // namespace bc
}  // namespace nori
