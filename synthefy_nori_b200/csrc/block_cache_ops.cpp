// Entry points of the context cache in 8 bits with block scales: checks of the arguments, the
// choice of kernel and of how far the keys are split.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <string>

#include "block_cache.cuh"
#include "plain.h"

namespace nori {
namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

// Numbers in messages as text: streamed as numbers they end the process where the module and torch were
// linked with different copies of the C++ library's locale facets.
std::string num(int64_t x) { return std::to_string(x); }

bc::View view_of(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, int64_t width, const char* who) {
  for (const Tensor* t : {&k, &v, &ks, &vs}) {
    check_plain(*t, who);
    TORCH_CHECK(t->is_contiguous(), who, ": contiguous cache tensors expected");
  }
  TORCH_CHECK(k.scalar_type() == v.scalar_type() &&
                  (k.scalar_type() == at::kChar || k.scalar_type() == at::kFloat8_e4m3fn),
              who, ": the cache's k and v must both be int8 or float8_e4m3fn");
  TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes(), who, ": k and v [batch, heads, capacity, width] expected");
  TORCH_CHECK(ks.scalar_type() == at::kFloat && vs.scalar_type() == at::kFloat && ks.dim() == 3 &&
                  ks.sizes() == vs.sizes() && ks.size(0) == k.size(0) && ks.size(1) == k.size(1),
              who, ": fp32 scales [batch, heads, capacity / block] expected");
  const int64_t cap = k.size(2), blocks = ks.size(2);
  TORCH_CHECK(width >= 1 && width <= bc::kMaxWidth && k.size(3) == (width + 7) / 8 * 8, who,
              ": head widths of 1 to 64 in rows of the next multiple of 8 expected");
  TORCH_CHECK(cap >= bc::kTile && cap % bc::kTile == 0 && cap < (int64_t{1} << 31), who,
              ": the capacity must be a multiple of 128 below 2^31");
  int log2 = 0;
  for (int l : {5, 6, 7})
    if (blocks << l == cap) log2 = l;
  TORCH_CHECK(log2 != 0, who, ": one scale for each 32, 64 or 128 rows expected");
  TORCH_CHECK(k.size(0) <= INT32_MAX && k.size(1) <= INT32_MAX, who, ": too many sequences or heads");
  for (const Tensor* t : {&k, &v, &ks, &vs})
    TORCH_CHECK(t->is_cuda() && t->device() == k.device(), who, ": cache tensors on one CUDA device expected");
  for (const Tensor* t : {&k, &v})
    TORCH_CHECK(reinterpret_cast<uintptr_t>(t->const_data_ptr()) % 16 == 0, who, ": a cache 16-byte aligned expected");
  bc::View c{};
  c.k = static_cast<uint8_t*>(const_cast<void*>(k.const_data_ptr()));
  c.v = static_cast<uint8_t*>(const_cast<void*>(v.const_data_ptr()));
  c.k_scale = const_cast<float*>(ks.const_data_ptr<float>());
  c.v_scale = const_cast<float*>(vs.const_data_ptr<float>());
  c.batch = static_cast<int>(k.size(0));
  c.heads = static_cast<int>(k.size(1));
  c.cap = cap;
  c.width = static_cast<int>(width);
  c.stored = static_cast<int>(k.size(3));
  c.block_log2 = log2;
  c.fp8 = k.scalar_type() == at::kFloat8_e4m3fn;
  return c;
}

int float_type(const Tensor& t, bool fp32, const char* who, const char* what) {
  const auto s = t.scalar_type();
  TORCH_CHECK(s == at::kBFloat16 || s == at::kHalf || (fp32 && s == at::kFloat), who, ": ", what, " must be ",
              fp32 ? "fp32, bf16 or fp16" : "bf16 or fp16", ", got ", s);
  return s == at::kFloat ? bc::kF32 : s == at::kBFloat16 ? bc::kBF16 : bc::kF16;
}

// [batch, n, heads, width] or [b0, b1, n, heads, width] (b0 * b1 = batch), columns contiguous
bc::Rows rows_of(const Tensor& t, const bc::View& c, int64_t n, int64_t heads, const torch::Device& dev, const char* who,
                 const char* what) {
  check_plain(t, who);
  TORCH_CHECK(t.is_cuda() && t.device() == dev, who, ": ", what, " must be on the cache's device");
  const int64_t d = t.dim();
  TORCH_CHECK((d == 4 || d == 5) && t.size(d - 1) == c.width && t.size(d - 2) == heads && t.size(d - 3) == n &&
                  (d == 4 ? t.size(0) : t.size(0) * t.size(1)) == c.batch,
              who, ": ", what, " must be [batch, n, heads, width] (or two batch dimensions), batch ", num(c.batch), ", n ",
              num(n), ", heads ", num(heads), ", width ", num(c.width));
  TORCH_CHECK(c.width == 1 || t.stride(d - 1) == 1, who, ": the columns of ", what, " must be contiguous");
  bc::Rows r{};
  r.p = const_cast<void*>(t.const_data_ptr());
  r.s0 = t.stride(0);
  r.s1 = d == 5 ? t.stride(1) : 0;
  r.n1 = d == 5 ? static_cast<int>(std::max<int64_t>(t.size(1), 1)) : 1;
  r.sn = t.stride(d - 3);
  r.sh = t.stride(d - 2);
  return r;
}

bc::PerSequence per_sequence(const OptTensor& dev, int64_t all, const bc::View& c, const torch::Device& device,
                             const char* who, const char* what) {
  bc::PerSequence p{nullptr, all};
  if (dev.has_value() && dev->defined()) {
    check_plain(*dev, who);
    TORCH_CHECK(dev->device() == device && dev->scalar_type() == at::kInt && dev->is_contiguous() && dev->numel() == c.batch,
                who, ": ", what, " must be an int or int32 [batch] on the cache's device");
    p.dev = dev->const_data_ptr<int>();
  }
  return p;
}

int sm_count(int dev) { return at::cuda::getDeviceProperties(dev)->multiProcessorCount; }

// Up to this many rows of one K/V head run on the kernel that streams the cache through registers, 16 of them a
// pass: 168 heads x 10,000 keys take 84 us with 16 rows, 119 with 32 and 147 with 33, where the kernel for many rows
// takes 147 with any number up to 64; 21 x 6001 keys of 56: 22 for 29, and 27 with 33.  Few heads with a long
// context, which that one splits over all SMs, meet earlier (2 x 100,003 keys of 64: 33 for 35 with 16 rows, 43 for
// 35 with 32).
constexpr int64_t kFewRows = 32;

// Splits of the keys of each cell for few rows, joined in clusters of up to 8.  A CTA's time goes with its
// keys and a start and end worth some 400 more (measured), whatever else its SM runs, up to the 5 or
// 4 CTAs that an SM holds: so the fewest waves of the shortest CTAs, each of 256 keys or more.
int few_splits(int64_t cells, int64_t longest, int resident) {
  const int64_t most = std::max<int64_t>((longest + 255) / 256, 1);
  if (cells * 8 <= resident && most > 8) return static_cast<int>(std::min(resident / cells, most) / 8 * 8);
  int best = 1;
  int64_t least = INT64_MAX;
  for (int64_t s = 1; s <= std::min<int64_t>(most, 8); ++s) {
    const int64_t cost = (cells * s + resident - 1) / resident * ((longest + s - 1) / s + 400);
    if (cost < least) least = cost, best = static_cast<int>(s);
  }
  return best;
}

// Cells that the persistent kernel takes whole, and splits of the keys of the others: as many whole ones as
// fill every SM some number of times, so that only a last, partial wave is split.  The time is the waves of
// items, each as long as its key tiles and the start and end of an item; partial results cost a second
// kernel and their traffic (and a workspace, held to 16 items an SM: 155 MB).  A split has to promise 3%, since
// long runs of items even out by themselves (4096 rows x 1000 of 168 cells: 378 us whole, 395 split for 1%;
// 256 rows x 10,000: 234 us with every cell split, 196 with the last 20).
struct Split {
  int64_t whole;
  int splits;
};
Split tc_splits(int64_t cells, int64_t longest, int ctas) {
  const int64_t tiles = std::max<int64_t>((longest + bc::kTile - 1) / bc::kTile, 1);
  Split best{cells, 1};
  double least = 0.97 * static_cast<double>((cells + ctas - 1) / ctas) * (static_cast<double>(tiles) + 4.0);
  for (int64_t waves = cells / ctas, tried = 0; waves >= 0 && tried < 3; --waves, ++tried) {
    const int64_t whole = waves * ctas, rest = cells - whole;
    for (int64_t s = 2; rest > 0 && s <= std::min<int64_t>(tiles, 64) && rest * s <= 16 * ctas; ++s) {
      const double cost = waves * (static_cast<double>(tiles) + 4.0) +
                          static_cast<double>((rest * s + ctas - 1) / ctas) * (static_cast<double>((tiles + s - 1) / s) + 4.0) +
                          4.0 + 0.012 * rest * s;
      if (cost < least) least = cost, best = Split{whole, static_cast<int>(s)};
    }
  }
  return best;
}

}  // namespace

void block_cache_write(const Tensor& ck, const Tensor& cv, const Tensor& cks, const Tensor& cvs, int64_t width,
                       const Tensor& k, const Tensor& v, int64_t start_all, const OptTensor& start_dev,
                       const OptTensor& count_dev) {
  const char* who = "block_cache_write";
  const bc::View c = view_of(ck, cv, cks, cvs, width, who);
  TORCH_CHECK(k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type(), who, ": k and v of one shape and type expected");
  const int type = float_type(k, true, who, "k");
  TORCH_CHECK(k.dim() >= 4, who, ": k [batch, n, heads, width] expected");
  const int64_t n = k.size(-3);
  const bc::Rows rk = rows_of(k, c, n, c.heads, ck.device(), who, "k"), rv = rows_of(v, c, n, c.heads, ck.device(), who, "v");
  const bc::PerSequence start = per_sequence(start_dev, start_all, c, ck.device(), who, "start");
  const bc::PerSequence count = per_sequence(count_dev, n, c, ck.device(), who, "counts");
  if (start.dev == nullptr)
    TORCH_CHECK(start_all >= 0 && n <= c.cap && start_all <= c.cap - n, who, ": ", num(n), " rows from ", num(start_all),
                " on of a cache of ", num(c.cap));
  if (n == 0 || c.batch == 0 || c.heads == 0) return;
  const Tensor* parts[] = {&ck, &cv, &cks, &cvs};
  for (int i = 0; i < 4; ++i) {
    for (int j = 0; j < i; ++j) TORCH_CHECK(!overlap(*parts[i], *parts[j]), who, ": the cache's tensors share memory");
    TORCH_CHECK(!shares_memory(*parts[i], k) && !shares_memory(*parts[i], v), who, ": k or v shares memory with the cache");
  }
  const at::cuda::CUDAGuard guard(ck.device());
  C10_CUDA_CHECK(bc::launch_write(c, rk, rv, type, start, count, n, at::cuda::getCurrentCUDAStream()));
}

std::vector<Tensor> block_cache_read(const Tensor& ck, const Tensor& cv, const Tensor& cks, const Tensor& cvs,
                                     int64_t width, int64_t start, int64_t n, c10::ScalarType out_type) {
  const char* who = "block_cache_read";
  const bc::View c = view_of(ck, cv, cks, cvs, width, who);
  TORCH_CHECK(start >= 0 && n >= 0 && start <= c.cap && n <= c.cap - start, who, ": ", num(n), " rows from ",
              num(start), " on of a cache of ", num(c.cap));
  const at::cuda::CUDAGuard guard(ck.device());
  std::vector<Tensor> out;
  for (int i = 0; i < 2; ++i)
    out.push_back(torch::empty({c.batch, c.heads, n, width}, ck.options().dtype(out_type)));
  const int type = float_type(out[0], true, who, "the result");
  if (out[0].numel() > 0)
    C10_CUDA_CHECK(bc::launch_read(c, out[0].data_ptr(), out[1].data_ptr(), type, start, n, at::cuda::getCurrentCUDAStream()));
  for (auto& t : out) t = t.transpose(1, 2);
  return out;
}

// (result, log-sum-exp [batch, heads, n] or an undefined tensor)
std::tuple<Tensor, OptTensor> block_cache_attention(const Tensor& q, const Tensor& ck, const Tensor& cv, const Tensor& cks,
                                                    const Tensor& cvs, int64_t width, int64_t length_all,
                                                    const OptTensor& length_dev, double scale, const OptTensor& out,
                                                    bool want_lse, const Tensor& status) {
  const char* who = "block_cache_attention";
  bc::Attention a{};
  a.c = view_of(ck, cv, cks, cvs, width, who);
  TORCH_CHECK(q.dim() >= 4, who, ": q [batch, n, heads, width] expected");
  a.n = q.size(-3);
  const int64_t heads = q.size(-2);
  TORCH_CHECK(a.c.heads > 0 ? heads % a.c.heads == 0 : heads == 0, who, ": ", num(heads),
              " query heads do not share ", num(a.c.heads), " K/V heads evenly");
  a.type = float_type(q, false, who, "q");
  a.q = rows_of(q, a.c, a.n, heads, ck.device(), who, "q");
  const at::cuda::CUDAGuard guard(ck.device());
  const bool given = out.has_value() && out->defined();
  const Tensor o = given ? *out : torch::empty(q.sizes(), q.options());
  TORCH_CHECK(o.scalar_type() == q.scalar_type() && o.sizes() == q.sizes(), who, ": out of q's shape and type expected");
  a.o = rows_of(o, a.c, a.n, heads, ck.device(), who, "out");
  a.length = per_sequence(length_dev, length_all, a.c, ck.device(), who, "lengths");
  if (given) {
    TORCH_CHECK(!shares_memory(o, o, true), who, ": rows of out share memory");
    for (const Tensor* t : {&q, &ck, &cv, &cks, &cvs})
      TORCH_CHECK(!shares_memory(o, *t), who, ": out shares memory with q or the cache");
    TORCH_CHECK(a.length.dev == nullptr || !shares_memory(o, *length_dev), who, ": out shares memory with the lengths");
  }
  if (a.length.dev == nullptr)
    TORCH_CHECK(length_all >= 0 && length_all <= a.c.cap, who, ": length ", num(length_all), " of a cache of ", num(a.c.cap));
  TORCH_CHECK(scale > 0.0 && scale < 1e30, who, ": a positive finite scale expected");
  a.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  OptTensor lse;
  if (want_lse) lse = torch::empty({a.c.batch, heads, a.n}, cks.options());
  if (q.numel() == 0) return {o, lse};
  a.lse = want_lse ? lse->data_ptr<float>() : nullptr;
  a.group = static_cast<int>(heads / a.c.heads);
  a.rows = a.n * a.group;
  TORCH_CHECK(a.rows < INT32_MAX - bc::kPairRows, who, ": 2^31 or more query rows of one K/V head");
  a.status = status.data_ptr<int>();
  // the longest a sequence can be (lengths on the device are not read here)
  const int64_t longest = a.length.dev != nullptr ? a.c.cap : length_all;
  const int sms = sm_count(ck.get_device());
  const auto stream = at::cuda::getCurrentCUDAStream();
  Tensor part_o[2], part_ml[2];
  auto plan = [&](int64_t first, int64_t end, bool few) {  // rows first .. end - 1 on one of the kernels
    bc::Attention p = a;
    p.first = first;
    p.rows = end;
    const int tile = few ? bc::few_tile_rows(end - first) : bc::kPairRows;
    const int64_t cells = (end - first + tile - 1) / tile * a.c.batch * a.c.heads;
    const Split by = few ? Split{0, few_splits(cells, longest, sms * bc::few_resident(end - first))} : tc_splits(cells, longest, sms);
    p.whole = by.whole;
    p.splits = by.splits;
    p.cluster = few ? std::min(p.splits, 8) : 1;
    const int parts = p.splits / p.cluster;
    if (parts > 1) {
      const int64_t part_rows = (cells - by.whole) * parts * tile;
      part_o[few] = torch::empty({part_rows * bc::kMaxWidth}, cks.options());
      part_ml[few] = torch::empty({part_rows * 2}, cks.options());
      p.part_o = part_o[few].data_ptr<float>();
      p.part_ml = reinterpret_cast<float2*>(part_ml[few].data_ptr<float>());
    }
    return p;
  };
  auto join = [&](const bc::Attention& p, bool few) {
    if (p.splits > p.cluster)
      C10_CUDA_CHECK(bc::launch_combine(p, few ? bc::few_tile_rows(p.rows - p.first) : bc::kPairRows, stream));
  };
  // a few rows behind the last whole pair of tiles would cost a pair's time on the tensor cores
  const int64_t rows = a.rows, whole = rows / bc::kPairRows * bc::kPairRows;
  const int64_t many = rows - whole > kFewRows ? rows : whole;
  bc::Attention tc{}, few{};
  if (many > 0) {
    tc = plan(0, many, false);
    C10_CUDA_CHECK(bc::launch_tc(tc, stream));
  }
  if (many < rows) {
    few = plan(many, rows, true);
    C10_CUDA_CHECK(bc::launch_few(few, many > 0, stream));
  }
  join(tc, false);
  join(few, true);
  return {o, lse};
}

}  // namespace nori
