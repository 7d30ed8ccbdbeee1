// Attention of few query rows (a single new row, rows of heads that share one K/V head) over a
// context cache in 8 bits with block scales; and the join of partial results.
//
// Bound: every stored byte is read once, 2 W bytes a key, for up to 16 rows.  So the work is split
// over the keys: a CTA takes a range of one (sequence, K/V head), its four warps every fourth piece
// of 32 keys, each with a running maximum, sum and output of its own; warps are joined in shared
// memory, ranges through a workspace by a second kernel.
//
// The rows are the M side of m16n8k16 products.  The order of the summed index is free as long as
// both operands agree, so lanes take whole 8-byte units: in q . k lane (g, t) holds units t and
// t + 4 of key g; in w . v it holds unit g of four keys, and column c of product j is value
// 8 c + j.  Loads are 8 bytes, widened to fp16 in registers; nothing goes through shared memory.
//
// Scales cost nothing per value.  With c = scale log2(e) s_k and t = c (q . k) + log2 s_v for the
// block of a key (one block per piece, since blocks are of 32 rows or more),
//   w = 2^(t - max t),  O = sum w v_code,  l = sum over blocks of (sum of w) / s_v,
//   out = O / l,  lse = ln 2 (max t + log2 l).
// Sums, maxima and outputs are fp32; w is rounded to fp16 (11 bits) for the product alone.
//
// Reference counterpart: attention over a quantised context cache (model/layer.py:747-934).
#include "block_cache.cuh"

namespace nori {
namespace bc {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kPiece = 32;  // keys of one step of a warp

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
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float to_float(const void* p, int64_t i, int type) {
  if (type == kBF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void put(void* p, int64_t i, float x, int type) {
  if (type == kBF16)
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else
    static_cast<__half*>(p)[i] = __float2half_rn(x);
}
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 1);
  return x + __shfl_xor_sync(0xffffffffu, x, 2);
}

struct Row {  // where row r of a K/V head's query rows lies
  int64_t n;
  int head;
  __device__ __forceinline__ Row(const Attention& a, int kv_head, int64_t r)
      : n(r / a.group), head(kv_head * a.group + static_cast<int>(r % a.group)) {}
};

// TWO: rows g + 8 exist as well.  UNITS: 4 or 8 units of 8 columns.
template <bool FP8, bool TWO, int UNITS>
__global__ void __launch_bounds__(kThreads) few_kernel(Attention a) {
  constexpr int kHalf = UNITS / 4;   // units of a lane in q . k
  constexpr int kRows = TWO ? 16 : 8;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
  const int64_t tiles = (a.rows + kRows - 1) / kRows;
  int64_t unit = blockIdx.x;
  const int64_t tile = unit % tiles;
  unit /= tiles;
  const int split = static_cast<int>(unit % a.splits);
  const int64_t bh = unit / a.splits;
  const int b = static_cast<int>(bh / a.c.heads), h = static_cast<int>(bh % a.c.heads);
  const int64_t row0 = tile * kRows;
  const int units = a.c.stored / 8;

  // this CTA's keys: whole pieces, the same number for every split
  const int64_t len = min(max(a.length.at(b), int64_t{0}), a.c.cap);
  const int64_t pieces = (len + kPiece - 1) / kPiece, each = (pieces + a.splits - 1) / a.splits;
  const int64_t p0 = split * each, p1 = min(p0 + each, pieces);

  // query rows g and g + 8: a power of two brings them into fp16's range, exactly
  uint32_t qf[2 * kHalf][4];
  float fac[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int64_t r = row0 + g + 8 * half;
    const bool there = r < a.rows && (TWO || half == 0);
    float x[kHalf][8], top = 0.f;
    bool bad = false;
    const Row row(a, h, there ? r : 0);
    const int64_t at = a.q.offset(b, row.n, row.head);
#pragma unroll
    for (int i = 0; i < kHalf; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = 8 * (t + 4 * i) + e;
        x[i][e] = there && d < a.c.width ? to_float(a.q.p, at + d, a.type) : 0.f;
        top = fmaxf(top, fabsf(x[i][e]));
        bad |= x[i][e] != x[i][e];
      }
    top = quad_max(bad ? INFINITY : top);
    float up, down;
    row_scale(top, up, down);
    fac[half] = down * a.scale_log2 * kCodeScale<FP8>;
#pragma unroll
    for (int i = 0; i < kHalf; ++i)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        qf[2 * i + s][half] = pack_half2(x[i][4 * s] * up, x[i][4 * s + 1] * up);
        qf[2 * i + s][2 + half] = pack_half2(x[i][4 * s + 2] * up, x[i][4 * s + 3] * up);
      }
  }

  float o[8][4];
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[j][i] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  const uint8_t* kbase = a.c.k + bh * a.c.cap * a.c.stored;
  const uint8_t* vbase = a.c.v + bh * a.c.cap * a.c.stored;
  const float* ks = a.c.k_scale + bh * a.c.blocks();
  const float* vs = a.c.v_scale + bh * a.c.blocks();
  const int koff = g * a.c.stored + t * 8, voff = 2 * t * a.c.stored + g * 8;
  const bool kthere[2] = {t < units, t + 4 < units};
  const bool vthere = g < units;

  uint2 kq[4][kHalf], vq[2][4];
  float sk = 0.f, sv = 0.f;
  auto load = [&](int64_t p) {
    const uint8_t* kp = kbase + p * kPiece * a.c.stored + koff;
    const uint8_t* vp = vbase + p * kPiece * a.c.stored + voff;
#pragma unroll
    for (int nt = 0; nt < 4; ++nt)
#pragma unroll
      for (int i = 0; i < kHalf; ++i)
        kq[nt][i] = kthere[i] ? __ldg(reinterpret_cast<const uint2*>(kp + nt * 8 * a.c.stored + i * 32)) : make_uint2(0, 0);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        vq[kt][e] = vthere ? __ldg(reinterpret_cast<const uint2*>(vp + (kt * 16 + (e >> 1) * 8 + (e & 1)) * a.c.stored))
                           : make_uint2(0, 0);
    const int64_t blk = p * kPiece >> a.c.block_log2;
    sk = __ldg(ks + blk);
    sv = __ldg(vs + blk);
  };

  for (int64_t p = p0 + warp; p < p1; p += kWarps) {
    load(p);
    // scores: 4 tiles of 8 keys
    float s[4][4];
#pragma unroll
    for (int nt = 0; nt < 4; ++nt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[nt][i] = 0.f;
#pragma unroll
      for (int i = 0; i < kHalf; ++i) {
        uint32_t b0, b1;
        widen<FP8>(biased<FP8>(kq[nt][i].x), b0, b1);
        mma16816(s[nt], qf[2 * i], b0, b1);
        widen<FP8>(biased<FP8>(kq[nt][i].y), b0, b1);
        mma16816(s[nt], qf[2 * i + 1], b0, b1);
      }
    }
    const float svc = safe_scale(sv);
    const float lv = log2f(svc), inv = 1.f / svc;
    const int left = static_cast<int>(min(len - p * kPiece, int64_t{kPiece}));  // keys of the piece that are there
    if (left < kPiece) {
#pragma unroll
      for (int nt = 0; nt < 4; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (nt * 8 + 2 * t + (i & 1) >= left) s[nt][i] = -INFINITY;
    }
    float shift[2], back[2];
    bool grow = false;
#pragma unroll
    for (int half = 0; half < (TWO ? 2 : 1); ++half) {
      float mx = -INFINITY;
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) mx = fmaxf(mx, fmaxf(s[nt][2 * half], s[nt][2 * half + 1]));
      mx = quad_max(mx);
      const float cand = fmaf(mx, fac[half] * sk, lv);
      back[half] = 1.f;
      if (cand > m[half] + kLazy || m[half] == -INFINITY) {
        back[half] = m[half] == -INFINITY ? 0.f : exp2_fast(m[half] - cand);
        m[half] = cand;
        grow = true;
      }
      shift[half] = lv - m[half] + kLift;
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        o[j][0] *= back[0], o[j][1] *= back[0];
        if (TWO) o[j][2] *= back[1], o[j][3] *= back[1];
      }
      l[0] *= back[0];
      if (TWO) l[1] *= back[1];
    }
#pragma unroll
    for (int half = 0; half < (TWO ? 2 : 1); ++half) {
      const float c = fac[half] * sk;
      float sum = 0.f;
#pragma unroll
      for (int nt = 0; nt < 4; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float& x = s[nt][2 * half + i];
          // (a masked key's -inf stays 0 whatever the scale)
          x = left < kPiece && nt * 8 + 2 * t + i >= left ? 0.f : exp2_fast(fmaf(x, c, shift[half]));
          sum += x;
        }
      l[half] = fmaf(sum, inv, l[half]);
    }
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const uint32_t af[4] = {pack_half2(s[2 * kt][0], s[2 * kt][1]), TWO ? pack_half2(s[2 * kt][2], s[2 * kt][3]) : 0u,
                              pack_half2(s[2 * kt + 1][0], s[2 * kt + 1][1]),
                              TWO ? pack_half2(s[2 * kt + 1][2], s[2 * kt + 1][3]) : 0u};
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint32_t x0 = biased<FP8>(w ? vq[kt][0].y : vq[kt][0].x), x1 = biased<FP8>(w ? vq[kt][1].y : vq[kt][1].x);
        const uint32_t x2 = biased<FP8>(w ? vq[kt][2].y : vq[kt][2].x), x3 = biased<FP8>(w ? vq[kt][3].y : vq[kt][3].x);
        uint32_t b0[4], b1[4];  // columns 4w .. 4w + 3: (key, next key)
        widen<FP8>(__byte_perm(x0, x1, 0x5140), b0[0], b0[1]);
        widen<FP8>(__byte_perm(x0, x1, 0x7362), b0[2], b0[3]);
        widen<FP8>(__byte_perm(x2, x3, 0x5140), b1[0], b1[1]);
        widen<FP8>(__byte_perm(x2, x3, 0x7362), b1[2], b1[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) mma16816(o[4 * w + j], af, b0[j], b1[j]);
      }
    }
  }

  // join the warps
  __shared__ float sm_m[kWarps][16], sm_l[kWarps][16];
  __shared__ float sm_o[kWarps][kRows][kMaxWidth + 4];
#pragma unroll
  for (int half = 0; half < (TWO ? 2 : 1); ++half) {
    l[half] = quad_sum(l[half]);
    const int r = g + 8 * half;
    if (t == 0) sm_m[warp][r] = m[half], sm_l[warp][r] = l[half];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) sm_o[warp][r][8 * (2 * t + i) + j] = o[j][2 * half + i];
  }
  __syncthreads();
  const int64_t cell = (bh * tiles + tile) * a.splits + split;
  for (int i = threadIdx.x; i < kRows * kMaxWidth; i += kThreads) {
    const int r = i / kMaxWidth, d = i % kMaxWidth;
    if (row0 + r >= a.rows) break;
    float top = sm_m[0][r];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sm_m[w][r]);
    float sum = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = sm_m[w][r] == -INFINITY && sm_l[w][r] == 0.f ? 0.f : exp2f(sm_m[w][r] - top);
      sum = fmaf(sm_l[w][r], f, sum);
      acc = fmaf(sm_o[w][r][d], f, acc);
    }
    if (a.splits > 1) {
      a.part_o[(cell * kRows + r) * kMaxWidth + d] = acc;
      if (d == 0) a.part_ml[cell * kRows + r] = make_float2(top, sum);
      continue;
    }
    const Row row(a, h, row0 + r);
    if (d < a.c.width) put(a.o.p, a.o.offset(b, row.n, row.head) + d, sum != 0.f ? acc * kCodeScale<FP8> / sum : 0.f, a.type);
    if (d == 0 && a.lse != nullptr)
      a.lse[(static_cast<int64_t>(b) * a.c.heads * a.group + row.head) * a.n + row.n] = row_lse(top, sum);
  }
}

// One CTA joins the splits of one row: each warp a run of them, then the warps.
constexpr int kJoinThreads = 256;
__global__ void __launch_bounds__(kJoinThreads) combine_kernel(Attention a, int tile_rows, float code_scale) {
  const int64_t r = blockIdx.x % a.rows, bh = blockIdx.x / a.rows;
  const int64_t tiles = (a.rows + tile_rows - 1) / tile_rows;
  const int64_t cell0 = (bh * tiles + r / tile_rows) * a.splits;
  const int tr = static_cast<int>(r % tile_rows);
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  float top = -INFINITY;
  for (int s = lane; s < a.splits; s += 32) top = fmaxf(top, a.part_ml[(cell0 + s) * tile_rows + tr].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float sum = 0.f, a0 = 0.f, a1 = 0.f;
  for (int s = warp; s < a.splits; s += kJoinThreads / 32) {
    const float2 ml = a.part_ml[(cell0 + s) * tile_rows + tr];
    if (ml.x == -INFINITY && ml.y == 0.f) continue;  // no keys there (and perhaps no values written)
    const float f = exp2f(ml.x - top);
    const float2 v = *reinterpret_cast<const float2*>(a.part_o + ((cell0 + s) * tile_rows + tr) * kMaxWidth + 2 * lane);
    sum = fmaf(ml.y, f, sum);
    a0 = fmaf(v.x, f, a0);
    a1 = fmaf(v.y, f, a1);
  }
  __shared__ float sm[kJoinThreads / 32][kMaxWidth + 1];
  sm[warp][2 * lane] = a0;
  sm[warp][2 * lane + 1] = a1;
  if (lane == 0) sm[warp][kMaxWidth] = sum;
  __syncthreads();
  if (threadIdx.x >= kMaxWidth) return;
  const int d = threadIdx.x;
  float acc = 0.f;
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; ++w) acc += sm[w][d], sum += sm[w][kMaxWidth];
  const int b = static_cast<int>(bh / a.c.heads), h = static_cast<int>(bh % a.c.heads);
  const Row row(a, h, r);
  if (d < a.c.width) put(a.o.p, a.o.offset(b, row.n, row.head) + d, sum != 0.f ? acc * code_scale / sum : 0.f, a.type);
  if (d == 0 && a.lse != nullptr)
    a.lse[(static_cast<int64_t>(b) * a.c.heads * a.group + row.head) * a.n + row.n] = row_lse(top, sum);
}

template <bool FP8, bool TWO, int UNITS>
cudaError_t few_typed(const Attention& a, cudaStream_t stream) {
  constexpr int kRows = TWO ? 16 : 8;
  const int64_t grid = (a.rows + kRows - 1) / kRows * a.splits * a.c.batch * a.c.heads;
  if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
  few_kernel<FP8, TWO, UNITS><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace

int few_tile_rows(int64_t rows) { return rows > 8 ? 16 : 8; }

cudaError_t launch_few(const Attention& a, cudaStream_t stream) {
  const bool two = few_tile_rows(a.rows) == 16, wide = a.c.stored > 32;
  if (a.c.fp8) {
    if (wide) return two ? few_typed<true, true, 8>(a, stream) : few_typed<true, false, 8>(a, stream);
    return two ? few_typed<true, true, 4>(a, stream) : few_typed<true, false, 4>(a, stream);
  }
  if (wide) return two ? few_typed<false, true, 8>(a, stream) : few_typed<false, false, 8>(a, stream);
  return two ? few_typed<false, true, 4>(a, stream) : few_typed<false, false, 4>(a, stream);
}

cudaError_t launch_combine(const Attention& a, int tile_rows, cudaStream_t stream) {
  const int64_t grid = a.rows * a.c.batch * a.c.heads;
  if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
  combine_kernel<<<static_cast<unsigned>(grid), kJoinThreads, 0, stream>>>(a, tile_rows, a.c.fp8 ? kCodeScale<true> : kCodeScale<false>);
  return cudaGetLastError();
}

}  // namespace bc
}  // namespace nori
