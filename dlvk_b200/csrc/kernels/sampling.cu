// Choice of the next word from its logits and a given uniform number.
//
// In descending order, equal logits in that of their words' numbers: the first
// top_k words; of these the fewest whose share of their weights' sum reaches
// top_p; of these the ones at least min_p times as likely as the first.  Of what
// is left, in the order of the numbers, the first word whose running sum of
// weights passes uniform times their total.  weight = exp((z - max) / temperature).
//
// Weights are summed as whole numbers, in steps of 2^-44 of the largest weight:
// the word does not depend on the order of the additions.  The three cuts each
// keep a beginning of the descending order, so all of them together are one
// word: the last one kept.
#include "dlvk/common.h"
#include "dlvk/kernels.h"

namespace dlvk {
namespace {

constexpr int THREADS = 1024;
constexpr double ONE = 17592186044416.0;  // 2^44
using u64 = unsigned long long;

// Logits as whole numbers in the same order; NaN as -infinity, -0 as 0.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) x = -INFINITY;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// exp((x - top) / temperature) in steps of 2^-44; words as good as the top weigh 1.
__device__ __forceinline__ u64 weight_of(float x, float top, double inv) {
  if (x == top) return (u64)ONE;
  if (!(x > -INFINITY) || top == INFINITY) return 0;
  return __double2ull_rn(exp(((double)x - (double)top) * inv) * ONE);
}

// A beginning of the descending order: all above `key`, and the first `ties` with it.
struct Cut {
  uint32_t key;
  u64 ties;
};
__device__ __forceinline__ Cut shorter(Cut a, Cut b) {
  if (a.key != b.key) return a.key > b.key ? a : b;
  return a.ties < b.ties ? a : b;
}

template <typename T>
struct Row {
  const T* p;
  int words;
  float top;
  double inv;
  __device__ __forceinline__ uint32_t key(int i) const { return key_of(to_f32(p[i])); }
  __device__ __forceinline__ u64 weight(uint32_t key) const { return weight_of(value_of(key), top, inv); }
};

struct Shared {
  u64 sums[256];
  unsigned counts[256];
  u64 scan[32];
  u64 picked[3];
};

// The last word whose running amount before it is below `want` (> 0), in
// descending order; amounts are 1 (by_count) or the weights.  Four passes over
// the digits of the keys.
template <typename T>
__device__ Cut cut_at(const Row<T>& r, u64 want, bool by_count, Shared& sh) {
  uint32_t prefix = 0, mask = 0;
  u64 before = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += THREADS) sh.sums[i] = 0, sh.counts[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < r.words; i += THREADS) {
      const uint32_t k = r.key(i);
      if ((k & mask) != prefix) continue;
      const int d = k >> shift & 255;
      atomicAdd(&sh.counts[d], 1u);
      if (!by_count) atomicAdd(&sh.sums[d], r.weight(k));
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      u64 acc = before, last = before;
      int pick = 255;
      for (int d = 255; d >= 0 && acc < want; --d) {
        if (!sh.counts[d]) continue;
        pick = d;
        last = acc;
        acc += by_count ? sh.counts[d] : sh.sums[d];
      }
      sh.picked[0] = pick;
      sh.picked[1] = last;
      sh.picked[2] = sh.counts[pick];
    }
    __syncthreads();
    prefix |= (uint32_t)sh.picked[0] << shift;
    mask |= 255u << shift;
    before = sh.picked[1];
  }
  const u64 one = by_count ? 1 : r.weight(prefix), count = sh.picked[2];
  __syncthreads();
  Cut c{prefix, count};
  if (one > 0) c.ties = min(count, (want - before + one - 1) / one);
  return c;
}

// Sum over the block; exclusive prefix in `before`.
__device__ u64 block_scan(u64 v, u64& before, Shared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  __syncthreads();
  if (lane == 31) sh.scan[warp] = s;
  __syncthreads();
  u64 base = 0, total = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) base += sh.scan[w];
    total += sh.scan[w];
  }
  before = base + s - v;
  return total;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) sample_kernel(Sampling a, int32_t* __restrict__ tokens) {
  __shared__ Shared sh;
  const int64_t row = blockIdx.x;
  Row<T> r{static_cast<const T*>(a.logits) + row * a.ld, (int)a.words, 0.f, 1.0};
  const double temperature = a.temperature.rows ? (double)a.temperature.rows[row] : a.temperature.one;
  const double top_p = a.top_p.rows ? (double)a.top_p.rows[row] : a.top_p.one;
  const double min_p = a.min_p.rows ? (double)a.min_p.rows[row] : a.min_p.one;
  const int64_t top_k = a.top_k.rows ? a.top_k.rows[row] : a.top_k.one;
  // the largest key, the lowest word with it
  u64 best = 0;
  for (int i = threadIdx.x; i < r.words; i += THREADS) {
    const u64 v = (u64)r.key(i) << 32 | (0xffffffffu - (unsigned)i);
    best = v > best ? v : best;
  }
  for (int o = 16; o > 0; o >>= 1) {
    const u64 v = __shfl_xor_sync(0xffffffffu, best, o);
    best = v > best ? v : best;
  }
  if ((threadIdx.x & 31) == 0) sh.scan[threadIdx.x >> 5] = best;
  __syncthreads();
  for (int w = 0; w < THREADS / 32; ++w) best = sh.scan[w] > best ? sh.scan[w] : best;
  __syncthreads();
  r.top = value_of((uint32_t)(best >> 32));
  const int first = (int)(0xffffffffu - (uint32_t)best);
  if (!(r.top > -INFINITY) || !(temperature > 0)) {
    if (threadIdx.x == 0) tokens[row] = r.top > -INFINITY ? first : -1;
    return;
  }
  r.inv = 1.0 / temperature;
  Cut cut{0, (u64)r.words};
  if (top_k > 0 && top_k < r.words) cut = cut_at(r, (u64)top_k, true, sh);
  // a thread's words: neighbours, so that sums in their order are sums over threads
  const int per = (r.words + THREADS - 1) / THREADS;
  const int lo = min(r.words, (int)threadIdx.x * per), hi = min(r.words, lo + per);
  const auto kept = [&](uint32_t k, u64& ties) { return k > cut.key || (k == cut.key && ties++ < cut.ties); };
  const auto ties_before = [&]() {
    u64 mine = 0, before;
    for (int i = lo; i < hi; ++i) mine += r.key(i) == cut.key;
    block_scan(mine, before, sh);
    return before;
  };
  if (top_p < 1) {
    u64 ties = ties_before(), sum = 0, before;
    for (int i = lo; i < hi; ++i) {
      const uint32_t k = r.key(i);
      if (kept(k, ties)) sum += r.weight(k);
    }
    const u64 total = block_scan(sum, before, sh);
    const double want = top_p > 0 ? ceil(top_p * (double)total) : 1.0;
    __syncthreads();
    cut = shorter(cut, cut_at(r, want >= 1.0 ? (u64)want : 1, false, sh));
  }
  const u64 least = min_p > 0 ? (u64)ceil(fmin(min_p, 1.0) * ONE) : 0;
  u64 ties = ties_before(), sum = 0, before;
  const u64 ties0 = ties;
  for (int i = lo; i < hi; ++i) {
    const uint32_t k = r.key(i);
    if (!kept(k, ties)) continue;
    const u64 w = r.weight(k);
    if (w >= least) sum += w;
  }
  const u64 total = block_scan(sum, before, sh);
  const double u = (double)a.uniform[row];
  u64 want = u > 0 ? (u64)(u * (double)total) : 0;  // running sums above u total: above its whole part
  want = want < total ? want : total - 1;
  if (before <= want && want < before + sum) {
    ties = ties0;
    u64 upto = before;
    for (int i = lo; i < hi; ++i) {
      const uint32_t k = r.key(i);
      if (!kept(k, ties)) continue;
      const u64 w = r.weight(k);
      if (w >= least) upto += w;
      if (upto > want) {
        tokens[row] = i;
        break;
      }
    }
  }
}

}  // namespace

void sample_tokens(const Sampling& a, int32_t* tokens, cudaStream_t s) {
  if (a.rows == 0) return;
  DLVK_CHECK(a.words >= 1 && a.words <= SAMPLING_WORDS, "sample_tokens: 1 to 2^18 words");
  DLVK_CHECK(a.rows < (1LL << 31), "sample_tokens: too many rows for one launch");
  DLVK_CHECK(a.dt == DType::BF16 || a.dt == DType::F32, "sample_tokens: fp32 or bf16");
  if (a.dt == DType::BF16) sample_kernel<__nv_bfloat16><<<(unsigned)a.rows, THREADS, 0, s>>>(a, tokens);
  else sample_kernel<float><<<(unsigned)a.rows, THREADS, 0, s>>>(a, tokens);
  DLVK_POST_LAUNCH();
}

}  // namespace dlvk
