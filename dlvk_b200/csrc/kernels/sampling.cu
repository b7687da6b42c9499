// Choice of the next word from its logits and a given uniform number.
//
// In descending order, equal logits in that of their words' numbers: the first
// top_k words; of these the fewest whose share of their weights' sum reaches
// top_p; of these the ones at least min_p times as likely as the first.  Of what
// is left, in the order of the numbers, the first word whose running sum of
// weights passes uniform times their total.  weight = exp((z - max) / temperature).
//
// Weights are summed as whole numbers, in steps of 2^-44 of the largest weight:
// the word does not depend on the order of the additions.  An element is one
// 64-bit number, its logit's bits in ascending order above its inverted word
// number, so that the descending order is that of these numbers, no two are
// alike, and a cut is one of them: the last element kept.
//
// A row is read once, into the shared memory of a cluster of up to eight blocks
// that pass sums to each other.  Where the cut lies among the first thousand or
// so, it is found in a list: the n-th largest of the threads' largest elements is
// a bound that at least n elements reach, those that do are sorted by one block.
// Otherwise histograms narrow the range down to as few elements.
#include <cooperative_groups.h>

#include <algorithm>

#include "dlvk/common.h"
#include "dlvk/kernels.h"

namespace cg = cooperative_groups;

namespace dlvk {
namespace {

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int MOST_BLOCKS = 8;     // of a cluster
constexpr int LIST = 2048;         // elements that one block sorts
constexpr int NUCLEUS = 512;       // elements of a list for top_p alone
constexpr int BINS = 2048;
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

struct Shared {
  double powers[128];                   // 2^(i / 128)
  u64 best[MOST_BLOCKS];                // of each block: its largest element
  u64 sums[MOST_BLOCKS];                // and its sum of weights
  unsigned listed[MOST_BLOCKS];         // and its elements in the list
  uint32_t maxima[MOST_BLOCKS * THREADS];  // block 0: every thread's largest key
  u64 scan[WARPS];
  unsigned count[33];
  unsigned members;
  u64 lowest, highest;
  u64 found[3];
  union {
    u64 list[LIST];
    struct {
      u64 mass[BINS];
      unsigned amount[BINS];
    } bins;
  };
};

// exp(d), d <= 0, in steps of 2^-44, with the table of 2^(i/128) and the
// exponential's series to the fourth power (P. T. P. Tang, "Table-driven
// implementation of the exponential function", 1989): relative error 2^-48.
struct Weights {
  float top;
  double scale;  // 128 / (ln 2 temperature)
  const double* powers;
  __device__ __forceinline__ u64 operator()(uint32_t key) const {
    const float x = value_of(key);
    if (x == top) return (u64)ONE;
    if (top == INFINITY) return 0;
    const double y = ((double)x - (double)top) * scale;  // -infinity where x is
    if (!(y > -5800.0)) return 0;                        // below 2^-45
    const double magic = 6755399441055744.0;             // 1.5 2^52: adding it rounds to whole numbers
    const double z = y + magic;
    const int k = __double2loint(z);
    const double r = (y - (z - magic)) * 0.0054152123481245727;  // ln 2 / 128
    const double p = fma(r, fma(r, fma(r, fma(r, 1.0 / 24, 1.0 / 6), 0.5), 1.0), 1.0) * powers[k & 127];
    const double v = __hiloint2double(__double2hiint(p) + ((44 + (k >> 7)) << 20), __double2loint(p));
    return __double_as_longlong(v + 4503599627370496.0) & 0xfffffffffffffull;  // + 2^52: rounds to whole numbers
  }
};

__device__ __forceinline__ u64 warp_add(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sum over the block, and the sum of the threads before this one.
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
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) base += sh.scan[w];
    total += sh.scan[w];
  }
  before = base + s - v;
  return total;
}

// The n-th largest of `count` keys (all, where there are no more), up to its last 12 bits.
__device__ uint32_t nth_largest(const uint32_t* keys, int count, int n, Shared& sh) {
  uint32_t mine[MOST_BLOCKS];
#pragma unroll
  for (int i = 0; i < MOST_BLOCKS; ++i) mine[i] = i * THREADS + threadIdx.x < count ? keys[i * THREADS + threadIdx.x] : 0;
  if (threadIdx.x < 33) sh.count[threadIdx.x] = 0;
  __syncthreads();
  uint32_t bound = 0;
  for (int bit = 31; bit >= 12; --bit) {
    const uint32_t trial = bound | 1u << bit;
    unsigned c = 0;
#pragma unroll
    for (int i = 0; i < MOST_BLOCKS; ++i) c += mine[i] >= trial;
    c = __reduce_add_sync(0xffffffffu, c);
    if ((threadIdx.x & 31) == 0 && c) atomicAdd(&sh.count[bit], c);
    __syncthreads();
    if (sh.count[bit] >= (unsigned)n) bound = trial;
  }
  return bound;
}

// Descending order of sh.list[0, n); n <= LIST.
__device__ void sort_list(int n, Shared& sh) {
  int size = 32;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += THREADS) sh.list[i] = 0;
  __syncthreads();
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = threadIdx.x; i < size / 2; i += THREADS) {
        const int a = (i / j) * 2 * j + i % j, b = a + j;
        const u64 x = sh.list[a], y = sh.list[b];
        if ((x < y) == ((a & k) == 0)) sh.list[a] = y, sh.list[b] = x;
      }
      __syncthreads();
    }
}

// One row's elements, dealt out to the blocks of a cluster in runs of `run` words.
struct Row {
  cg::cluster_group cluster;
  int blocks, rank, first, n;  // this block's words: first.., n of them
  const uint32_t* keys;
  Weights weight;
  Shared& sh;
  __device__ __forceinline__ u64 element(int i) const { return (u64)keys[i] << 32 | ~(uint32_t)(first + i); }

  // Everything for the whole cluster to see; ends with a barrier of all.
  __device__ u64 total_weight(u64 cut, u64 least) {
    u64 s = 0, before;
    for (int i = threadIdx.x; i < n; i += THREADS)
      if (element(i) >= cut) {
        const u64 w = weight(keys[i]);
        if (w >= least) s += w;
      }
    s = block_scan(s, before, sh);
    if (threadIdx.x < blocks) *cluster.map_shared_rank(&sh.sums[rank], threadIdx.x) = s;
    cluster.sync();
    s = 0;
    for (int b = 0; b < blocks; ++b) s += sh.sums[b];
    return s;
  }

  // Lists the elements that `member` picks, at most LIST of a block; their number,
  // smallest and largest in sh.members, sh.lowest, sh.highest.
  template <typename F>
  __device__ void gather(F&& member) {
    __syncthreads();
    if (threadIdx.x == 0) sh.members = 0, sh.lowest = ~0ull, sh.highest = 0;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    u64 lo = ~0ull, hi = 0;
    for (int i0 = threadIdx.x & ~31; i0 < n; i0 += THREADS) {
      const int i = i0 + lane;
      const bool in = i < n && member(i);
      const unsigned who = __ballot_sync(0xffffffffu, in);
      if (!who) continue;
      unsigned base = 0;
      if (lane == 0) base = atomicAdd(&sh.members, __popc(who));
      base = __shfl_sync(0xffffffffu, base, 0);
      if (in) {
        const u64 e = element(i);
        const unsigned at = base + __popc(who & ((1u << lane) - 1));
        if (at < LIST) sh.list[at] = e;
        lo = e < lo ? e : lo;
        hi = e > hi ? e : hi;
      }
    }
    if (hi) {
      atomicMin(&sh.lowest, lo);
      atomicMax(&sh.highest, hi);
    }
    __syncthreads();
  }

  // Block 0: the lists of all blocks one after the other; their length, or -1 where there is no room.
  __device__ int join_lists() {
    int total = 0;
    for (int b = 0; b < blocks; ++b) total += sh.listed[b];
    if (total > LIST) return -1;
    int at = sh.listed[0];
    for (int b = 1; b < blocks; ++b) {
      const u64* from = cluster.map_shared_rank(sh.list, b);
      for (int i = threadIdx.x; i < (int)sh.listed[b]; i += THREADS) sh.list[at + i] = from[i];
      at += sh.listed[b];
    }
    return total;
  }

  // Block 0, list sorted, `acc` the amount before its first element: the last
  // element with less than `want` before it, and in sh.found[1] whether the
  // list's amounts reach `want`.  by_count: amounts are 1, else weights; only the
  // first `most` elements are looked at.
  __device__ u64 cut_of_list(int total, int most, u64 acc, u64 want, bool by_count) {
    const int per = (min(total, most) + THREADS - 1) / THREADS;
    const int lo = min(min(total, most), (int)threadIdx.x * per), hi = min(min(total, most), lo + per);
    u64 mine = 0, before;
    for (int i = lo; i < hi; ++i) mine += by_count ? 1 : weight((uint32_t)(sh.list[i] >> 32));
    const u64 sum = block_scan(mine, before, sh);
    if (threadIdx.x == 0) sh.found[0] = 0;
    __syncthreads();
    u64 upto = acc + before;
    int last = -1;
    for (int i = lo; i < hi && upto < want; ++i) {
      last = i;
      upto += by_count ? 1 : weight((uint32_t)(sh.list[i] >> 32));
    }
    if (last >= 0) atomicMax(&sh.found[0], (u64)last + 1);
    if (threadIdx.x == 0) sh.found[1] = acc + sum >= want;
    __syncthreads();
    return sh.found[0] ? sh.list[sh.found[0] - 1] : ~0ull;
  }

  // The sum of the weights of the first `most` elements of the list.
  __device__ u64 weight_of_list(int most) {
    u64 s = 0, before;
    for (int i = threadIdx.x; i < most; i += THREADS) s += weight((uint32_t)(sh.list[i] >> 32));
    return block_scan(s, before, sh);
  }

  // sh.found[..] of block 0 to all; ends with a barrier of all.
  __device__ void tell(u64 a, u64 b, u64 c) {
    if (rank == 0 && threadIdx.x < blocks) {
      u64* to = cluster.map_shared_rank(sh.found, threadIdx.x);
      to[0] = a, to[1] = b, to[2] = c;
    }
    cluster.sync();
  }

  // The cut where less than `want` comes before its element, wherever it lies:
  // the range of elements is narrowed down by histograms, first over the logit's
  // distance from the largest, then over the elements as numbers.
  __device__ u64 search(u64 want, bool by_count, float per_unit) {
    u64 acc = 0, lowest = 0, highest = ~0ull;
    int shift = -1;  // -1: by distance
    const auto bin_of = [&](int i) {
      if (shift >= 0) return (int)((highest - element(i)) >> shift);
      const float x = value_of(keys[i]), q = (weight.top - x) * per_unit;
      return x == weight.top ? 0 : q < BINS - 1 ? (int)q : BINS - 1;
    };
    while (true) {
      cluster.sync();  // the lists and bins of before have been read
      for (int i = threadIdx.x; i < BINS; i += THREADS) sh.bins.mass[i] = 0, sh.bins.amount[i] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < n; i += THREADS) {
        const u64 e = element(i);
        if (e < lowest || e > highest) continue;
        const int b = bin_of(i);
        atomicAdd(&sh.bins.amount[b], 1u);
        if (!by_count) {
          const u64 w = weight(keys[i]);
          if (w) atomicAdd(&sh.bins.mass[b], w);
        }
      }
      cluster.sync();
      if (rank == 0) {
        constexpr int PER = BINS / THREADS;
        u64 mass[PER], mine = 0, before;
        unsigned amount[PER];
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          mass[k] = 0, amount[k] = 0;
          const int i = threadIdx.x * PER + k;
          for (int b = 0; b < blocks; ++b) {
            amount[k] += cluster.map_shared_rank(sh.bins.amount, b)[i];
            if (!by_count) mass[k] += cluster.map_shared_rank(sh.bins.mass, b)[i];
          }
          if (by_count) mass[k] = amount[k];
          mine += mass[k];
        }
        block_scan(mine, before, sh);
        if (threadIdx.x == 0) sh.lowest = 0;
        __syncthreads();
        u64 upto = acc + before;
        int last = -1;
        u64 at = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          if (amount[k] && upto < want) last = threadIdx.x * PER + k, at = upto;
          upto += mass[k];
        }
        if (last >= 0) atomicMax(&sh.lowest, (u64)last + 1);
        __syncthreads();
        if (last >= 0 && sh.lowest == (u64)last + 1) sh.highest = at;
        __syncthreads();
      }
      tell(sh.lowest - 1, sh.highest, 0);
      const int pick = (int)sh.found[0];
      acc = sh.found[1];
      __syncthreads();
      const u64 lo = lowest, hi = highest;
      gather([&](int i) {
        const u64 e = element(i);
        return e >= lo && e <= hi && bin_of(i) == pick;
      });
      if (threadIdx.x < blocks) {
        Shared* to = cluster.map_shared_rank(&sh, threadIdx.x);
        to->listed[rank] = sh.members;
        to->best[rank] = sh.lowest;
        to->sums[rank] = sh.highest;
      }
      cluster.sync();
      unsigned total = 0;
      lowest = ~0ull, highest = 0;
      for (int b = 0; b < blocks; ++b) {
        total += sh.listed[b];
        lowest = min(lowest, sh.best[b]);
        highest = max(highest, sh.sums[b]);
      }
      if (total <= LIST) {
        u64 cut = 0;
        if (rank == 0) {
          sort_list(join_lists(), sh);
          cut = cut_of_list((int)total, (int)total, acc, want, by_count);
        }
        tell(cut, 0, 0);
        return sh.found[0];
      }
      shift = max(0, 64 - __clzll(highest - lowest) - 11);
    }
  }
};

template <typename T, int VEC>
__global__ void __launch_bounds__(THREADS) sample_kernel(Sampling a, int run, int32_t* __restrict__ tokens) {
  extern __shared__ __align__(16) char raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  uint32_t* keys = reinterpret_cast<uint32_t*>(raw + sizeof(Shared));
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), words = (int)a.words;
  const int64_t row = blockIdx.x / blocks;
  const int first = min(words, rank * run), n = min(words, first + run) - first;
  const T* p = static_cast<const T*>(a.logits) + row * a.ld + first;
  const double temperature = a.temperature.rows ? (double)a.temperature.rows[row] : a.temperature.one;
  const double top_p = a.top_p.rows ? (double)a.top_p.rows[row] : a.top_p.one;
  const double min_p = a.min_p.rows ? (double)a.min_p.rows[row] : a.min_p.one;
  const int64_t top_k = a.top_k.rows ? a.top_k.rows[row] : a.top_k.one;
  // no block writes to another one before that has begun
  cg::cluster_group::arrival_token begun = cluster.barrier_arrive();
  if (threadIdx.x < 128) sh.powers[threadIdx.x] = exp2(threadIdx.x / 128.0);

  // the row, the largest element
  uint32_t high = 0;
  int where = 0;
  if constexpr (VEC > 1) {
#pragma unroll 4
    for (int i = threadIdx.x * VEC; i < n; i += THREADS * VEC) {
      const uint4 u = *reinterpret_cast<const uint4*>(p + i);
      const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const uint32_t k = key_of(to_f32(e[j]));
        keys[i + j] = k;
        if (k > high) high = k, where = i + j;
      }
    }
  } else {
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += THREADS) {
      const uint32_t k = key_of(to_f32(p[i]));
      keys[i] = k;
      if (k > high) high = k, where = i;
    }
  }
  u64 best = high ? (u64)high << 32 | ~(uint32_t)(first + where) : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((threadIdx.x & 31) == 0) sh.scan[threadIdx.x >> 5] = best;
  cluster.barrier_wait(std::move(begun));
  cluster.map_shared_rank(sh.maxima, 0)[rank * THREADS + threadIdx.x] = high;
  __syncthreads();
  if (threadIdx.x < blocks) {
    for (int w = 0; w < WARPS; ++w) best = max(best, sh.scan[w]);
    *cluster.map_shared_rank(&sh.best[rank], threadIdx.x) = best;
  }
  cluster.sync();
  best = 0;
  for (int b = 0; b < blocks; ++b) best = max(best, sh.best[b]);
  const float top = value_of((uint32_t)(best >> 32));
  if (!(top > -INFINITY) || !(temperature > 0)) {
    if (rank == 0 && threadIdx.x == 0) tokens[row] = top > -INFINITY ? (int32_t)~(uint32_t)best : -1;
    return;
  }
  Row r{cluster, blocks, rank, first, n, keys, {top, 184.66496523378731 / temperature, sh.powers}, sh};  // 128 / ln 2

  const bool cut_k = top_k > 0 && top_k < words, cut_p = top_p < 1;
  const auto wanted = [&](u64 total) {  // the whole number that a running sum below top_p total is below
    const double w = top_p > 0 ? ceil(top_p * (double)total) : 1.0;
    return w >= 1.0 ? (u64)w : 1;
  };
  u64 cut = 0;
  if (cut_k || cut_p) {
    const int64_t ask = cut_k ? top_k : NUCLEUS;
    u64 total = 0;
    if (!cut_k) total = r.total_weight(0, 0);
    bool done = false;
    if (ask <= (int64_t)blocks * THREADS) {
      uint32_t bound = 0;
      if (rank == 0) bound = nth_largest(sh.maxima, blocks * THREADS, (int)ask, sh);
      r.tell(bound, 0, 0);
      bound = (uint32_t)sh.found[0];
      r.gather([&](int i) { return keys[i] >= bound; });
      if (threadIdx.x == 0) cluster.map_shared_rank(&sh, 0)->listed[rank] = sh.members;
      cluster.sync();
      u64 mine = 0, ok = 0;
      if (rank == 0) {
        const int count = r.join_lists();
        if (count >= 0) {
          sort_list(count, sh);
          const int most = cut_k ? min(count, (int)top_k) : count;  // at least top_k elements reach the bound
          ok = 1;
          if (cut_k) {
            mine = sh.list[most - 1];
            if (cut_p) total = r.weight_of_list(most);
          }
          if (cut_p) {
            mine = r.cut_of_list(count, most, 0, wanted(total), false);
            ok = sh.found[1];
          }
        }
        __syncthreads();
      }
      r.tell(mine, ok, 0);
      cut = sh.found[0];
      done = sh.found[1];
    }
    if (!done) {
      const float per_unit = (float)(BINS / (32.0 * temperature));
      cut = 0;
      if (cut_k) cut = r.search((u64)top_k, true, per_unit);
      if (cut_p) {
        if (cut_k) total = r.total_weight(cut, 0);
        cut = max(cut, r.search(wanted(total), false, per_unit));
      }
    }
  }

  // sums of what is left, by warps that each own neighbouring words
  const u64 least = min_p > 0 ? (u64)ceil(fmin(min_p, 1.0) * ONE) : 0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per = ((n + WARPS - 1) / WARPS + 31) / 32 * 32;
  const int lo = min(n, warp * per), hi = min(n, lo + per);
  const auto kept = [&](int i) -> u64 {
    if (i >= hi || r.element(i) < cut) return 0;
    const u64 w = r.weight(keys[i]);
    return w >= least ? w : 0;
  };
  u64 mine = 0;
  for (int i = lo + lane; i < hi; i += 32) mine += kept(i);
  mine = warp_add(mine);
  __syncthreads();
  if (lane == 0) sh.scan[warp] = mine;
  __syncthreads();
  u64 before = 0, all = 0;
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += sh.scan[w];
    all += sh.scan[w];
  }
  if (threadIdx.x < blocks) *cluster.map_shared_rank(&sh.sums[rank], threadIdx.x) = all;
  cluster.sync();
  u64 total = 0;
  for (int b = 0; b < blocks; ++b) {
    if (b < rank) before += sh.sums[b];
    total += sh.sums[b];
  }
  const double u = (double)a.uniform[row];
  u64 want = u > 0 ? (u64)(fmin(u, 1.0) * (double)total) : 0;  // a running sum above u total is above its whole part
  want = want < total ? want : total - 1;
  if (want < before || want >= before + mine) return;
  for (int i0 = lo; i0 < hi; i0 += 32) {
    u64 s = kept(i0 + lane);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 t = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += t;
    }
    const unsigned past = __ballot_sync(0xffffffffu, before + s > want);
    if (past) {
      if (lane == 0) tokens[row] = first + i0 + __ffs(past) - 1;
      return;
    }
    before += __shfl_sync(0xffffffffu, s, 31);
  }
}

template <typename T, int VEC>
void launch(const Sampling& a, int32_t* tokens, int blocks, int run, cudaStream_t s) {
  const size_t smem = sizeof(Shared) + (size_t)run * 4;
  const auto kernel = sample_kernel<T, VEC>;
  static std::atomic<size_t> allowed[kMaxDevices];
  std::atomic<size_t>& here = allowed[current_device_slot()];
  if (here.load() < smem) {
    DLVK_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    here.store(227 * 1024);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * blocks));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)blocks, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  DLVK_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, a, run, tokens));
  DLVK_POST_LAUNCH();
}

}  // namespace

void sample_tokens(const Sampling& a, int32_t* tokens, cudaStream_t s) {
  if (a.rows == 0) return;
  DLVK_CHECK(a.words >= 1 && a.words <= SAMPLING_WORDS, "sample_tokens: 1 to 2^18 words");
  DLVK_CHECK(a.rows < (1LL << 31) / MOST_BLOCKS, "sample_tokens: too many rows for one launch");
  DLVK_CHECK(a.dt == DType::BF16 || a.dt == DType::F32, "sample_tokens: fp32 or bf16");
  // blocks of a row: enough that a block has at most 16384 words, and that the rows fill the GPU as long as a
  // block has some thousands
  int blocks = 1;
  const auto run_of = [&](int b) { return (int)(((a.words + b - 1) / b + 7) / 8 * 8); };
  while (blocks < MOST_BLOCKS && (run_of(blocks) > 16384 || (a.rows * blocks < 148 && run_of(blocks) > 2048))) blocks *= 2;
  const int run = run_of(blocks);
  const int64_t bytes = a.dt == DType::BF16 ? 2 : 4;
  const bool wide = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && a.ld * bytes % 16 == 0 && a.words * bytes % 16 == 0;
  if (a.dt == DType::BF16) {
    if (wide) launch<__nv_bfloat16, 8>(a, tokens, blocks, run, s);
    else launch<__nv_bfloat16, 1>(a, tokens, blocks, run, s);
  } else {
    if (wide) launch<float, 4>(a, tokens, blocks, run, s);
    else launch<float, 1>(a, tokens, blocks, run, s);
  }
}

}  // namespace dlvk
