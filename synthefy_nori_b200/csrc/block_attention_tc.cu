// Attention of many query rows over a context cache in 8 bits with block scales, on the 5th-generation
// tensor cores.
//
// Persistent, one CTA of 28 warps per SM; a work item is 256 query rows (two tiles of 128) against a
// range of the keys of one (sequence, K/V head).  Roles:
//   warp 0        takes the next work item (a CTA not yet started is cancelled and its item taken over,
//                 so sequences of different lengths even out) and tells the others; copies the
//                 codes of 128-key tiles of K and V, each one contiguous piece of the cache, into
//                 two rings (untiled bulk copies: no stride rules, so any width);
//   warps 4..7    widen the codes of K to fp16, exactly, into the swizzled tiles that the products
//   warps 8..11   read, and those of V: once for 256 query rows; before an item's first tile each
//                 warpgroup brings one of its query tiles to shared memory as fp16;
//   warps 1, 2    issue the products of one query tile each: S = Q K^T (128 x 64 x 64) and O += P V;
//   warps 12..27  softmax, four groups: (query tile) x (half of the keys of every tile), each with its
//                 own maximum, sum and accumulator; thread = query row (its TMEM lane), 32 scores of a chunk
//                 in registers; P (fp16 pairs) goes over S in TMEM and is the A operand of P V.  A group has
//                 two chunks: products of the one run while it works on the other (with one chunk of 64
//                 that was waited for, 1024 rows x 10,000 took 691 us for 680).
// A group's tile is a chain (scores, maximum, weights, two products) whose latency is several times its
// arithmetic, so four of them share an SM: with one thread for all 128 columns of a row and two
// groups the same arithmetic took 1.3 times as long, with row maxima exchanged between the
// halves 1.2 times.  The two halves of a query tile are joined once per item.
//
// Scales cost nothing per value: with c = scale log2(e) s_k 2^-e (2^e brings the query row into
// fp16's range, exactly) and t = c (q . k) + log2 s_v,
//   w = 2^(t - max t),  O = sum w v_code,  l = sum over blocks of (sum of w) / s_v.
// The maximum is lazy (O is rescaled when it grows by more than 2^8); w is kept at up to 2^15 so
// that fp16 holds 11 bits down to 2^-21 of the largest weight.  Scores, sums and O are fp32.
// All exponentials run on the MUFU: a polynomial on the FMA pipe for a quarter of them made a tile
// a seventh slower, since the warps' issue slots are as scarce as the MUFU.
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
constexpr int kSmem = kTile16 * (4 + 2 * kRing) + kTile8 * 2 * kRing + 1024 + 1024;
constexpr int kItems = 4;                // items that are known ahead
constexpr int kConsumers = 2 + 8 + 16;   // of an item: issuers, converter and softmax warps
constexpr int kHalf = kN / 2;            // keys of a group's tile
constexpr int kChunk = kHalf / 2;        // keys of a step of its softmax
// S 0..255 (64 a group, P of each 32 over its first 16), O 256..511 (64 a group)
constexpr uint32_t kTmemCols = 512, kOcol = 256;
constexpr int kConvertWarps = 4, kSoftmaxWarp0 = 12;
// registers of a thread: launch 72 (896 threads); the softmax warps take what the others give up
constexpr uint32_t kRegsLow = 56, kRegsSoftmax = 80;
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

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_st1(uint32_t taddr, uint32_t x) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(x) : "memory");
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

// 16 bytes (values 8 c .. 8 c + 7) of the query row at src, in pieces of 4 or 2 bytes; zeros where it ends.
__device__ __forceinline__ uint4 query_piece(const uint16_t* src, int c, int width, int bytes) {
  uint32_t v[4] = {0, 0, 0, 0};
  if (bytes == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c * 8 + 2 * e < width) v[e] = __ldg(reinterpret_cast<const uint32_t*>(src) + e);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c * 8 + e < width) v[e / 2] |= static_cast<uint32_t>(__ldg(src + e)) << 16 * (e % 2);
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// Four query rows, r0 and every fourth after it, to the tile as fp16 times each row's power of two, and the
// factors that their scores take.  Eight neighbouring lanes hold a row, 16 bytes (unit c) each.  The four go
// through every step side by side: one after the other they took a third longer (6,100 cycles a tile for 4,700).
__device__ __forceinline__ void query_rows(const Attention& a, int64_t begin, uint32_t row_first, int r0, int c, int bytes,
                                           uint8_t* tile, float* factors) {
  uint4 x[4];
  auto source = [&](int i) -> const uint16_t* {  // null where there is no such row or unit
    const uint32_t row = row_first + r0 + 4 * i;
    if (row >= static_cast<uint32_t>(a.rows) || c * 8 >= a.c.width) return nullptr;
    const uint32_t n = a.group == 1 ? row : row / static_cast<uint32_t>(a.group);
    return static_cast<const uint16_t*>(a.q.p) + begin + n * a.q.sn + (row - n * a.group) * a.q.sh + c * 8;
  };
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = make_uint4(0, 0, 0, 0);
  if (bytes == 16) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (const uint16_t* src = source(i)) x[i] = __ldg(reinterpret_cast<const uint4*>(src));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (const uint16_t* src = source(i)) x[i] = query_piece(src, c, a.c.width, bytes);
  }
  // magnitudes order like their bits, infinities and NaN on top
  uint32_t top[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    top[i] = __vmaxu2(__vmaxu2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu), __vmaxu2(x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu));
#pragma unroll
  for (int o = 1; o < 8; o *= 2)
#pragma unroll
    for (int i = 0; i < 4; ++i) top[i] = __vmaxu2(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
  const bool bf = a.type == kBF16;
  float mine = 0.f;  // lane c keeps the factor of row c
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t t16 = max(top[i] & 0xffffu, top[i] >> 16);
    float up, down;
    row_scale(bf ? __uint_as_float(t16 << 16) : __half2float(__ushort_as_half(static_cast<uint16_t>(t16))), up, down);
    mine = c == i ? down * a.scale_log2 : mine;
    const uint32_t v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    uint32_t y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float2 f = make_float2(__uint_as_float(v[k] << 16), __uint_as_float(v[k] & 0xffff0000u));
      if (!bf) f = __half22float2(*reinterpret_cast<const __half2*>(&v[k]));
      y[k] = pack_half2(f.x * up, f.y * up);
    }
    const int r = r0 + 4 * i;
    *reinterpret_cast<uint4*>(tile + r * 128 + ((c ^ (r & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
  }
  if (c < 4) factors[r0 + 4 * c] = mine;
}

// (everything below 2^31, checked on the host: 64-bit divisions would take a microsecond an item)
constexpr uint32_t kNoPart = 0xffffffffu;
struct alignas(16) Item {
  uint32_t b, h, bh, part;  // part: of the partial results, or kNoPart
  uint32_t row0;            // first query row
  uint32_t tile0;           // first key tile
  int len;                  // keys of the sequence
  int tiles;                // key tiles of this item
  int groups;               // query tiles with rows in them (1 or 2; 0: there is no item)
  int64_t in, out;          // where the query rows and the results of this (sequence, K/V head) begin
};

__device__ __forceinline__ Item item_at(const Attention& a, uint32_t w) {
  Item it;
  const uint32_t pairs = (static_cast<uint32_t>(a.rows - a.first) + kPairRows - 1) / kPairRows;
  const uint32_t whole = static_cast<uint32_t>(a.whole), n = w < whole ? 1u : static_cast<uint32_t>(a.splits);
  uint32_t cell = w, split = 0;  // cell: (sequence, K/V head) and pair of query tiles
  it.part = kNoPart;
  if (n > 1) {
    it.part = w - whole;
    split = it.part % n;
    cell = whole + it.part / n;
  }
  it.bh = cell / pairs;
  it.row0 = static_cast<uint32_t>(a.first) + (cell - it.bh * pairs) * kPairRows;
  it.b = it.bh / static_cast<uint32_t>(a.c.heads);
  it.h = it.bh - it.b * static_cast<uint32_t>(a.c.heads);
  it.len = static_cast<int>(min(max(a.length.at(it.b), int64_t{0}), a.c.cap));
  const uint32_t all = (static_cast<uint32_t>(it.len) + kN - 1) / kN, each = n > 1 ? (all + n - 1) / n : all;
  it.tile0 = min(split * each, all);
  it.tiles = static_cast<int>(min(it.tile0 + each, all) - it.tile0);
  it.groups = it.row0 + kM < static_cast<uint32_t>(a.rows) ? 2 : 1;
  it.in = a.q.offset(static_cast<int>(it.b), 0, static_cast<int>(it.h * a.group));
  it.out = a.o.offset(static_cast<int>(it.b), 0, static_cast<int>(it.h * a.group));
  return it;
}

template <bool FP8>
__global__ void __launch_bounds__(kThreads, 1)
    tc_kernel(const __grid_constant__ Attention a, uint32_t items, int q_bytes, int o_bytes) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                     // [item parity][query tile]
  uint8_t* sK = sQ + 4 * kTile16;         // [kRing] fp16, swizzled
  uint8_t* sV = sK + kRing * kTile16;     // [kRing]
  uint8_t* rK = sV + kRing * kTile16;     // [kRing] codes
  uint8_t* rV = rK + kRing * kTile8;      // [kRing]
  uint64_t* bars = reinterpret_cast<uint64_t*>(rV + kRing * kTile8);
  uint64_t* rk_full = bars;               // codes have arrived
  uint64_t* rk_empty = rk_full + kRing;   // codes are widened
  uint64_t* k_full = rk_empty + kRing;    // fp16 tile is there
  uint64_t* k_empty = k_full + kRing;     // the products that read it are done
  uint64_t* rv_full = k_empty + kRing;    // the same four for V
  uint64_t* rv_empty = rv_full + kRing;
  uint64_t* v_full = rv_empty + kRing;
  uint64_t* v_empty = v_full + kRing;
  uint64_t* item_full = v_empty + kRing;  // [kItems]
  uint64_t* item_empty = item_full + kItems;
  uint64_t* q_full = item_empty + kItems; // [item parity][query tile]
  uint64_t* q_empty = q_full + 4;         // the item's scores are done, its factors read and its results on their way
  uint64_t* o_free = q_empty + 4;         // [query tile] per item: O is in registers
  uint64_t* s_full = o_free + 2;          // [group][chunk] per tile: scores are there, the P V before them done
  uint64_t* p_full = s_full + 8;          // [group][chunk] per tile: P is in TMEM
  uint64_t* o_full = p_full + 8;          // [group][chunk] per item: the last P V is done (not another phase of
                                          // s_full: the next item's scores do not wait for the warps that wait for it)
  uint64_t* pair = o_full + 8;            // [query tile][lane quarter] the two halves have exchanged
  uint64_t* done = pair + 8;              // [query tile] every product of this CTA
  uint64_t* taken = done + 2;             // the answer to a request for an item
  uint64_t* answer = taken + 2;           // (16 bytes, 16-byte aligned)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(answer + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  __shared__ float2 swap[2][16][32];  // [parity of the exchange][softmax warp][row]
  __shared__ Item known[kItems];
  __shared__ float factors[2][2 * kM];  // [item parity][row]: of the row's scores
  // (s_k, log2 s_v, 1 / s_v) of each 32 keys of a tile, written with its K; a slot is used again four tiles
  // on, when the scores three tiles before that are done and so the weights of this tile
  __shared__ float4 scales[4][4];
  static_assert((8 * kRing + 2 * kItems + 48) * 8 + 8 <= 1024, "barriers fit their room");
  static_assert((8 * kRing + 2 * kItems + 46) % 2 == 0, "the answer is 16-byte aligned");

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int failed = read_status(a.status);  // (looked at below)

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
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], kConsumers);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&q_full[i], kConvertWarps);
      mbar_init(&q_empty[i], 1 + 8);
    }
    mbar_init(taken, 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&o_free[t], 8);
      mbar_init(&done[t], 1);
    }
    for (int i = 0; i < 8; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < 8; ++i) mbar_init(&pair[i], 2);
    *abort_flag = 0;
    fence_barrier_init();
  }
  // columns of K and V past the width are never written: zero (finite; Q is 0 there)
  const int unit0 = a.c.stored / 8, units = 8 - unit0;
  for (int i = threadIdx.x; i < 2 * kRing * kN * units; i += kThreads) {
    const int row = i / units, c = unit0 + i - row * units;
    *reinterpret_cast<uint4*>(sK + row * 128 + ((c ^ (row & 7)) << 4)) = make_uint4(0, 0, 0, 0);
  }
  if (threadIdx.x == 0) known[0] = item_at(a, blockIdx.x);  // (while the others write)
  fence_proxy_async_smem();
  if (warp == 1) tmem_alloc(tmem_slot, kTmemCols);
  tc_fence_before();
  const bool stop = __syncthreads_or(failed) != 0;  // another CTA or kernel timed out: nothing is written
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (stop) {
    if (warp == 1) tmem_dealloc(tmem, kTmemCols);
    return;
  }

  // The next item, for one thread or a whole warp (`all`): null past the last one or after a timeout.  It
  // stays in shared memory (registers are scarce) until `done_with`.
  uint32_t seen = 0;
  auto next_item = [&](bool all) -> const Item* {
    const uint32_t i = seen % kItems, ph = seen / kItems & 1;
    const bool ok = all ? mbar_wait_warp(&item_full[i], ph, a.status, kTimeoutEpilogue, abort_flag)
                        : mbar_wait(&item_full[i], ph, a.status, kTimeoutMma, abort_flag);
    return ok && known[i].groups > 0 ? &known[i] : nullptr;
  };
  auto done_with = [&](bool all) {
    if (all) __syncwarp();
    if (!all || lane == 0) mbar_arrive(&item_empty[seen % kItems]);
    ++seen;
  };

  if (warp == 0) {
    setmaxnreg_dec<kRegsLow>();
    if (elect_one()) {
      const uint32_t bytes = static_cast<uint32_t>(kN * a.c.stored);
      uint32_t nk = 0, nv = 0;  // tiles asked for so far
      uint32_t told = 0, asked = 0;
      bool ok = true;
      auto tell = [&](uint32_t w) -> bool {  // (`items`: there is none left)
        const uint32_t i = told % kItems;
        if (!mbar_wait(&item_empty[i], (told / kItems & 1) ^ 1, a.status, kTimeoutProducer, abort_flag)) return false;
        if (told > 0) known[i] = item_at(a, w < items ? w : 0);  // (the first is there)
        if (w >= items) known[i].groups = 0;
        mbar_arrive(&item_full[i]);
        ++told;
        return true;
      };
      auto ask = [&] {  // for a CTA that has not started
        mbar_arrive_expect_tx(taken, 16);
        asm volatile(
            "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                smem_u32(answer)),
            "r"(smem_u32(taken))
            : "memory");
        ++asked;
      };
      auto answered = [&](uint32_t& w) -> bool {  // the item taken over, `items` where there is none left
        if (!mbar_wait(taken, (asked - 1) & 1, a.status, kTimeoutProducer, abort_flag)) return false;
        uint32_t got, id;
        asm volatile(
            "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\t"
            "ld.shared.b128 h, [%2];\n\t"
            "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t"
            "mov.u32 %1, 0;\n\t"
            "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
            : "=r"(got), "=r"(id)
            : "r"(smem_u32(answer))
            : "memory");
        fence_proxy_async_smem();
        w = got ? id : items;
        return true;
      };
      uint32_t cur = blockIdx.x, nxt = items;
      ok = tell(cur);
      while (ok && cur < items) {
        const Item& it = known[(told - 1) % kItems];  // (told only now: its slot is not reused before this item is done)
        const int tiles = it.tiles;
        const int64_t at = (it.bh * a.c.cap + static_cast<int64_t>(it.tile0) * kN) * a.c.stored;
        auto load = [&](int j, const uint8_t* src, uint8_t* dst, uint64_t* full, uint64_t* empty, uint32_t& n) -> bool {
          const uint32_t st = n % kRing;
          if (!mbar_wait(&empty[st], (n / kRing & 1) ^ 1, a.status, kTimeoutProducer, abort_flag)) return false;
          mbar_arrive_expect_tx(&full[st], bytes);
          bulk_load(dst + st * kTile8, src + at + static_cast<int64_t>(j) * bytes, bytes, &full[st]);
          ++n;
          return true;
        };
        if (tiles > 0 && !(ok = load(0, a.c.k, rK, rk_full, rk_empty, nk))) break;
        // the next item is asked for two tiles before it is needed and no sooner: it would be held back from
        // a CTA that is done earlier (never again after a refusal: the loop ends there)
        if (tiles == 0) ask();
        for (int j = 0; ok && j < tiles; ++j) {
          if (j == max(tiles - 2, 0)) ask();
          if (j + 1 < tiles) ok = load(j + 1, a.c.k, rK, rk_full, rk_empty, nk);
          if (ok) ok = load(j, a.c.v, rV, rv_full, rv_empty, nv);
        }
        if (!ok || !(ok = answered(nxt) && tell(nxt))) break;
        cur = nxt;
      }
      // own copies and requests in flight (after an abort nobody else waits for them)
      if (asked > 0) mbar_wait(taken, (asked - 1) & 1, a.status, kTimeoutProducer, nullptr);
      for (uint32_t i = 0; i < kRing; ++i) {
        if (nk > i) mbar_wait(&rk_full[(nk - 1 - i) % kRing], (nk - 1 - i) / kRing & 1, a.status, kTimeoutProducer, nullptr);
        if (nv > i) mbar_wait(&rv_full[(nv - 1 - i) % kRing], (nv - 1 - i) / kRing & 1, a.status, kTimeoutProducer, nullptr);
      }
    }
  } else if (warp <= 2) {
    setmaxnreg_dec<kRegsLow>();
    if (elect_one()) {
      constexpr uint32_t idesc_s = idesc_f16(kM, kChunk, false), idesc_o = idesc_f16(kM, kD, true);
      const int t = warp - 1;          // query tile
      // operands: 32 bytes further for each 16 columns of Q and K, 2048 for each 16 keys of V
      const uint64_t dq = umma_desc_kmajor_sw128(smem_u32(sQ + t * kTile16));
      const uint64_t dk = umma_desc_kmajor_sw128(smem_u32(sK)), dv = umma_smem_desc(smem_u32(sV), 8192, 1024, 2);
      constexpr uint32_t kStage = kTile16 >> 4, kHalfTile = kStage / 2, kChunkTile = kStage / 4;
      uint32_t nk = 0, nv = 0;         // ring positions
      uint32_t cnt = 0;                // tiles of this query tile so far
      uint32_t qcnt = 0;               // items of this query tile so far
      bool ok = true;
      auto wait = [&](uint64_t* b, uint32_t parity) -> bool {
        return mbar_wait(b, parity & 1, a.status, kTimeoutMma, abort_flag);
      };
      while (const Item* it = ok ? next_item(false) : nullptr) {
        const int tiles = it->tiles;
        const bool mine = t < it->groups;
        done_with(false);
        if (tiles == 0) continue;
        if (!mine) {  // no rows: the tiles of K and V are the other issuer's
          for (int j = 0; ok && j < tiles; ++j) {
            if (!(ok = wait(&k_full[nk % kRing], nk / kRing))) break;
            mbar_arrive(&k_empty[nk++ % kRing]);
            if (!(ok = wait(&v_full[nv % kRing], nv / kRing))) break;
            mbar_arrive(&v_empty[nv++ % kRing]);
          }
          continue;
        }
        const uint32_t buf = qcnt & 1;
        const uint64_t q = dq + buf * (2 * kStage);
        auto scores = [&](int p, int u) {  // of K tile nk, for keys 64 p + 32 u .. + 31
          const uint64_t k = dk + nk % kRing * kStage + p * kHalfTile + u * kChunkTile;
#pragma unroll
          for (int i = 0; i < kD / 16; ++i)
            umma_bf16_ss(tmem + (2 * t + p) * kHalf + u * kChunk, q + 2 * i, k + 2 * i, idesc_s, i > 0 ? 1u : 0u);
        };
        if (!(ok = wait(&q_full[2 * buf + t], qcnt / 2) && wait(&k_full[nk % kRing], nk / kRing))) break;
        tc_fence_after();
        for (int u = 0; u < 2; ++u)
          for (int p = 0; p < 2; ++p) {
            scores(p, u);
            umma_commit(&s_full[2 * (2 * t + p) + u]);
          }
        umma_commit(&k_empty[nk++ % kRing]);
        if (tiles == 1) umma_commit(&q_empty[2 * buf + t]);
        for (int j = 0; ok && j < tiles; ++j, ++cnt) {
          const bool more = j + 1 < tiles;
          // the accumulators of the previous item have been read
          if (j == 0 && qcnt > 0 && !(ok = wait(&o_free[t], qcnt - 1))) break;
          if (!(ok = wait(&v_full[nv % kRing], nv / kRing) && (!more || wait(&k_full[nk % kRing], nk / kRing)))) break;
          for (int i = 0; ok && i < 4; ++i) {
            const int u = i / 2, p = i % 2, g = 2 * t + p;
            if (!(ok = wait(&p_full[2 * g + u], cnt))) break;
            tc_fence_after();
            const uint64_t v = dv + nv % kRing * kStage + p * kHalfTile + u * kChunkTile;
#pragma unroll
            for (int k = 0; k < kChunk / 16; ++k)
              umma_bf16_ts(tmem + kOcol + g * kD, tmem + g * kHalf + u * kChunk + k * 8, v + k * 128, idesc_o,
                           (k > 0 || u > 0 || j > 0) ? 1u : 0u);
            // P V reads the columns that the next scores overwrite: products of one thread run in order
            if (more) scores(p, u);
            umma_commit(more ? &s_full[2 * g + u] : &o_full[2 * g + u]);
          }
          if (!ok) break;
          umma_commit(&v_empty[nv++ % kRing]);
          if (more) umma_commit(&k_empty[nk++ % kRing]);
          if (j + 2 == tiles) umma_commit(&q_empty[2 * buf + t]);  // the item's scores are all issued
        }
        ++qcnt;
      }
      umma_commit(&done[t]);
      mbar_wait(&done[t], 0, a.status, kTimeoutMma, nullptr);
    }
  } else if (warp == 3) {
    setmaxnreg_dec<kRegsLow>();  // (its warpgroup's share)
  } else if (warp < kSoftmaxWarp0) {
    setmaxnreg_dec<kRegsLow>();
    // ------------------------------------------------------------ codes -> fp16 tiles
    // Thread: eight codes (unit c) of rows row0, row0 + 16, ..: fixed steps in both tiles, and eight threads
    // a row whatever its width, so that their 16-byte pieces never meet in a bank.  The codes are in
    // registers before the fp16 tile's last reader is waited for.
    const bool is_v = warp >= 8;
    const uint32_t tid = threadIdx.x % (kConvertWarps * 32), row0 = tid / 8, c = tid % 8;
    const bool works = static_cast<int>(c * 8) < a.c.stored;
    const uint8_t* src = (is_v ? rV : rK) + row0 * a.c.stored + c * 8;
    uint8_t* dst = (is_v ? sV : sK) + row0 * 128 + ((c ^ (row0 & 7)) << 4);
    const uint32_t step = 16 * a.c.stored;
    uint64_t* bar = is_v ? rv_full : rk_full;  // then code_empty, full, empty, kRing each
    uint32_t st = 0, ph = 0, n = 0;
    const int qt = is_v;  // the query tile that this warpgroup brings
    uint32_t qcnt = 0;
    bool ok = true;
    while (const Item* it = ok ? next_item(true) : nullptr) {
      const int tiles = it->tiles;
      // keys of the item from this thread's first row on (warp 4: from chunk lane % 4 on)
      int left = it->len - static_cast<int>(it->tile0 * kN + (warp == 4 ? 32 * (lane & 3) : row0));
      const int64_t blk = it->bh * a.c.blocks() + ((it->tile0 * kN + 32 * (lane & 3)) >> a.c.block_log2);
      const float *ks = a.c.k_scale + blk, *vs = a.c.v_scale + blk;
      const bool has_rows = tiles > 0 && qt < it->groups;
      const uint32_t row_first = it->row0 + qt * kM;
      const int64_t begin = it->in;
      done_with(true);
      if (has_rows) {
        // ---- query rows: eight lanes a row, 16 bytes each; a power of two brings the row into fp16's
        // range, exactly
        const uint32_t buf = 2 * (qcnt & 1) + qt;
        if (!(ok = mbar_wait_warp(&q_empty[buf], (qcnt / 2 & 1) ^ 1, a.status, kTimeoutProducer, abort_flag))) break;
        uint8_t* tile = sQ + buf * kTile16;
#pragma unroll 1
        for (int r1 = warp % 4 * 32 + lane / 8; r1 < warp % 4 * 32 + 32; r1 += 16)
          query_rows(a, begin, row_first, r1, lane % 8, q_bytes, tile, &factors[qcnt & 1][qt * kM]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[buf]);
        ++qcnt;
      }
      float sk = 0.f, sv = 0.f, least = kLeastScale;
      if (warp == 4 && tiles > 0) sk = __ldg(ks), sv = __ldg(vs);
#pragma unroll 1
      for (int j = 0; j < tiles; ++j, ++n, left -= kN) {
        if (!(ok = mbar_wait_warp(bar + st, ph, a.status, kTimeoutEpilogue, abort_flag))) break;
        uint2 x[kN / 16];
        const uint8_t* from = src + st * kTile8;
        if (works) {
#pragma unroll
          for (int e = 0; e < kN / 16; ++e) x[e] = *reinterpret_cast<const uint2*>(from + e * step);
        }
        if (!(ok = mbar_wait_warp(bar + 3 * kRing + st, ph ^ 1, a.status, kTimeoutEpilogue, abort_flag))) break;
        uint8_t* to = dst + st * kTile16;
        if (works) {
#pragma unroll
          for (int e = 0; e < kN / 16; ++e) {
            uint4 y;
            widen<FP8>(biased<FP8>(x[e].x), y.x, y.y);
            widen<FP8>(biased<FP8>(x[e].y), y.z, y.w);
            // codes behind the last row may be NaN (0 x NaN is none of its business)
            if (FP8 && is_v && 16 * e >= left) y = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(to + e * 2048) = y;
          }
        }
        if (warp == 4) {
          const float there = left > 0 ? sv : 0.f;  // (the other chunk of a group is the next lane's)
          raise_floor(least, fmaxf(there, __shfl_xor_sync(0xffffffffu, there, 1)));
          const float svc = safe_scale(sv, least);
          // (a block behind the last row counts for nothing, whatever its scale; log2 and reciprocal approximate, 1e-5 of
          // a weight at most: 1 / 30 of its rounding to fp16)
          const float4 y = left > 0 ? make_float4(sk, __log2f(svc), __fdividef(1.f, svc), 0.f) : make_float4(0.f, 0.f, 0.f, 0.f);
          if (lane < 4) scales[n & 3][lane] = y;
          if (j + 1 < tiles) sk = __ldg(ks += kN >> a.c.block_log2), sv = __ldg(vs += kN >> a.c.block_log2);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          // (only now: with the codes released as soon as their loads were issued, the next copy overtook them)
          mbar_arrive(bar + kRing + st);
          mbar_arrive(bar + 2 * kRing + st);
        }
        if (++st == kRing) st = 0, ph ^= 1;
      }
    }
  } else {
    setmaxnreg_inc<kRegsSoftmax>();
    // ------------------------------------------------------------ softmax
    // Group (query tile qt, half): 64 key columns of every tile, and columns 32 half .. + 31 of the
    // result.  The two warps of the same 32 rows exchange (maximum, sum) at the end.
    const int sw = warp - kSoftmaxWarp0, g = sw / 4, qt = g / 2, half = g % 2, quarter = sw % 4;
    const int r = quarter * 32 + lane;  // row of the tile == TMEM lane
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tS = tmem + g * kHalf + lane_off, tO = tmem + kOcol + g * kD + lane_off,
                   tO2 = tmem + kOcol + 2 * qt * kD + half * 32 + lane_off;  // this half's columns, both accumulators
    uint64_t* pair_bar = &pair[qt * 4 + quarter];
    uint32_t cnt = 0;  // completions of each s_full so far
    uint32_t nt = 0;   // tiles of all items so far
    uint32_t xc = 0;   // exchanges, and so items, so far
    bool ok = true;
    auto exchange = [&](float2 x) -> float2 {  // the other half's x for this row (valid if ok)
      swap[xc & 1][sw][lane] = x;
      __syncwarp();
      if (lane == 0) mbar_arrive(pair_bar);
      ok = mbar_wait_warp(pair_bar, xc & 1, a.status, kTimeoutEpilogue, abort_flag);
      return swap[xc++ & 1][sw ^ 4][lane];
    };
    while (const Item* it = ok ? next_item(true) : nullptr) {
      if (qt >= it->groups) {
        nt += it->tiles;
        done_with(true);
        continue;
      }
      const int tiles = it->tiles;
      float m = -INFINITY, l = 0.f;
      if (tiles > 0) {
        if (!(ok = mbar_wait_warp(&q_full[2 * (xc & 1) + qt], xc / 2 & 1, a.status, kTimeoutEpilogue, abort_flag))) break;
        const float fac = factors[xc & 1][qt * kM + r];
        int valid = it->len - static_cast<int>(it->tile0 * kN) - kHalf * half;  // keys from this half's first on
        uint64_t* bar = &s_full[2 * g];
#pragma unroll 2
        for (int step = 0; step < 2 * tiles; ++step) {  // (tile, chunk)
          const int u = step & 1;
          if (!(ok = mbar_wait_warp(bar + u, cnt + step / 2 & 1, a.status, kTimeoutEpilogue, abort_flag))) break;
          tc_fence_after();
          const uint32_t tC = tS + u * kChunk;
          if (valid < kChunk) {  // keys behind the last row
#pragma unroll 1
            for (int i = max(valid, 0); i < kChunk; ++i) tmem_st1(tC + i, 0xff800000u);
            tmem_wait_st();
          }
          valid -= u ? kN - kChunk : kChunk;
          uint32_t x[32];
          tmem_ld32(tC, x);
          const float4 sc = scales[(nt + step / 2) & 3][2 * half + u];
          const float f0 = fac * sc.x, f = f0 < 1e-38f ? 1e-38f : f0;  // (never 0: a masked key's -inf stays -inf)
          tmem_wait_ld();
          const float cand = fmaf(max32(x), f, sc.y);
          float h = 1.f;  // its square rescales the sums (lowered())
          bool grow = false;
          if (step == 0) {
            m = cand;
          } else if (cand > m + kLazy) {
            h = exp2_mufu(0.5f * (m - cand));
            l *= h;
            m = cand;
            grow = true;
          }
          const float lift = m == -INFINITY ? 0.f : kLift - m;  // (no key of this half is there)
          l = fmaf(weights32(x, f, sc.y + lift, tC), sc.z, l * h);
          if (__any_sync(0xffffffffu, grow)) {
            // the other chunk's product may still be under way: its next scores, if there are any, come behind it
            const bool last = step == 2 * tiles - 1;
            if (!(ok = mbar_wait_warp(last ? &o_full[2 * g] : bar + (u ^ 1), (last ? xc : cnt + (step + 1) / 2) & 1, a.status,
                                      kTimeoutEpilogue, abort_flag)))
              break;
            tc_fence_after();
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {
              uint32_t o[16];
              tmem_ld16(tO + q * 16, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * (h * h));
              tmem_st16(tO + q * 16, o);
            }
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[2 * g + u]);
        }
        nt += tiles;
        cnt += tiles;
        for (int u = 0; u < 2 && ok; ++u)  // the last P V
          ok = mbar_wait_warp(&o_full[2 * g + u], xc & 1, a.status, kTimeoutEpilogue, abort_flag);
        if (!ok) break;
        tc_fence_after();
      }
      // ---- the halves joined: 32 columns of O from both accumulators, to memory.  (Once an item, so its
      // instructions come from far: a loop over 8 columns.)
      const uint32_t row = it->row0 + qt * kM + r;
      const bool there = row < static_cast<uint32_t>(a.rows);
      const uint32_t n = a.group == 1 ? row : row / static_cast<uint32_t>(a.group), in_group = row - n * a.group;
      const int64_t out = it->out + n * a.o.sn + in_group * a.o.sh;
      const bool part = it->part != kNoPart;
      const int64_t pr = static_cast<int64_t>(it->part) * kPairRows + qt * kM + r;
      const int64_t lse_row = static_cast<int64_t>(it->bh) * a.group + in_group;
      done_with(true);
      float fa = 0.f, fb = 0.f;  // of the first and the second half's accumulator
      if (tiles > 0) {
        if (!(m < INFINITY)) l = __uint_as_float(0x7fc00000u);  // an infinite score (or a NaN) somewhere
        const float2 other = exchange(make_float2(m, l));
        if (!ok) break;
        const float top = fmaxf(m, other.x);
        const float h1 = m == -INFINITY ? 0.f : exp2f(0.5f * (m - top));
        const float h2 = other.x == -INFINITY ? 0.f : exp2f(0.5f * (other.x - top));
        l = lowered(l, h1) + lowered(other.y, h2);
        m = top;
        fa = half ? h2 * h2 : h1 * h1, fb = half ? h1 * h1 : h2 * h2;
        tc_fence_after();
      }
      if (!part) {
        const float norm = l != 0.f ? 1.f / l : 0.f;
        fa *= norm, fb *= norm;
      }
      uint16_t* dst = static_cast<uint16_t*>(a.o.p) + half * 32;
      float* part_dst = a.part_o + pr * kMaxWidth + half * 32;
      const int have = a.c.width - half * 32;
      // the item's query tile becomes the tile of results (nothing reads it any more): a row in pieces of 16 bytes
      uint8_t* stage = sQ + (2 * ((xc ^ (tiles > 0)) & 1) + qt) * kTile16 + quarter * 32 * 128;
#pragma unroll 2
      for (int c = 0; c < 4; ++c) {
        float o[8];
        if (tiles > 0) {
          uint32_t x[8], y[8];
          tmem_ld8(tO2 + 8 * c, x);
          tmem_ld8(tO2 + kD + 8 * c, y);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = __uint_as_float(x[i]) * fa + __uint_as_float(y[i]) * fb;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = 0.f;
        }
        if (part) {
          if (there) {
            reinterpret_cast<float4*>(part_dst + 8 * c)[0] = make_float4(o[0], o[1], o[2], o[3]);
            reinterpret_cast<float4*>(part_dst + 8 * c)[1] = make_float4(o[4], o[5], o[6], o[7]);
          }
          continue;
        }
        uint32_t y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          y[i] = a.type == kBF16 ? pack_bf16x2(o[2 * i], o[2 * i + 1]) : pack_half2(o[2 * i], o[2 * i + 1]);
        if (tiles > 0) {
          *reinterpret_cast<uint4*>(stage + lane * 128 + ((4 * half + c) ^ (lane & 7)) * 16) = make_uint4(y[0], y[1], y[2], y[3]);
        } else if (there) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (8 * c + i < have) dst[out + 8 * c + i] = static_cast<uint16_t>(y[i / 2] >> 16 * (i % 2));
        }
      }
      if (tiles > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free[qt]);
        if (!part) {
          // 4 lanes a row (or 16, or 32 where rows are not aligned): a store of the warp meets 8 lines or
          // fewer (32 with a lane for each row)
          const int lanes = 64 / o_bytes < 32 ? 64 / o_bytes : 32, col = lane % lanes * (o_bytes / 2);
#pragma unroll 1
          for (int i = 0; i < lanes; ++i) {
            const int rr = i * (32 / lanes) + lane / lanes;
            const int64_t to = __shfl_sync(0xffffffffu, out, rr) + col;
            const uint8_t* from = stage + rr * 128 + ((4 * half + col / 8) ^ (rr & 7)) * 16 + col % 8 * 2;
            if (row - lane + rr >= static_cast<uint32_t>(a.rows) || col >= have) continue;
            if (o_bytes == 16)
              *reinterpret_cast<uint4*>(dst + to) = *reinterpret_cast<const uint4*>(from);
            else if (o_bytes == 4)
              *reinterpret_cast<uint32_t*>(dst + to) = *reinterpret_cast<const uint32_t*>(from);
            else
              dst[to] = *reinterpret_cast<const uint16_t*>(from);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(&q_empty[2 * (~xc & 1) + qt]);
      }
      if (there && half == 0) {
        if (part)
          a.part_ml[pr] = make_float2(m, l);
        else if (a.lse != nullptr)
          a.lse[lse_row * a.n + n] = row_lse(m, l);
      }
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
cudaError_t tc_typed(const Attention& a, cudaStream_t stream) {
  if (a.rows > INT32_MAX - kPairRows) return cudaErrorInvalidConfiguration;
  const int64_t cells = (a.rows - a.first + kPairRows - 1) / kPairRows * a.c.batch * a.c.heads;
  const int64_t items = a.whole + (cells - a.whole) * a.splits;
  if (items > INT32_MAX) return cudaErrorInvalidConfiguration;
  const cudaError_t e = cudaFuncSetAttribute(tc_kernel<FP8>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  tc_kernel<FP8><<<static_cast<unsigned>(items), kThreads, kSmem, stream>>>(
      a, static_cast<uint32_t>(items), access_bytes(a.q, a.c.width), access_bytes(a.o, a.c.width));
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_tc(const Attention& a, cudaStream_t stream) {
  return a.c.fp8 ? tc_typed<true>(a, stream) : tc_typed<false>(a, stream);
}

}  // namespace bc
}  // namespace nori
