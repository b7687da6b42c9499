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
// so, one block finds it and the word in a list: what the n-th largest of
// the threads' largest elements reaches, at least n elements do, and those that
// do are the list.  Otherwise histograms of the elements' numbers narrow the
// range down to as few: a bin's weights lie between those of its ends, which
// brackets the cut, so that sums are made in registers and not in the bins.
//
// One read of the logits is the floor (20 us for 256 x 128000 fp32, less than a launch
// for what a server usually asks).  Small calls are a chain of barriers: 64 x 32000 bf16
// with top_k 50 and top_p takes 16.4 us, some 21000 cycles: 5000 reading, 4000 the bound,
// 5000 the list, 5000 the word, the rest the cluster's five barriers.  Large ones are bound
// by the weights, 64-bit arithmetic of some 50 issue slots a warp and word and pass: 256 x
// 128000 take 58 us for the largest word alone, 118 with top_k 40, 165 from all words
// (one pass), 740-750 with a nucleus of thousands of words (four), of mixed settings 231-241.
#include <cooperative_groups.h>

#include <algorithm>
#include <cstddef>

#include "dlvk/common.h"
#include "dlvk/kernels.h"

namespace cg = cooperative_groups;

namespace dlvk {
namespace {

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int MOST_BLOCKS = 8;     // of a cluster
constexpr int LIST = 3 * THREADS;  // elements that one block cuts by itself
constexpr int ASK = 1152;          // most elements that a list is made for: it may have some more
constexpr int SHORT = 128;         // elements of a list that all see all
constexpr int NUCLEUS = 96, NUCLEUS_MORE = 900;  // elements of a list for top_p alone, first and second try
constexpr int BINS = 2048;         // that a range of elements is cut into
constexpr int PARTS = 1024;        // where they hold exact weights
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

struct Settings {
  int64_t top_k;
  double top_p;
  u64 least;      // smallest weight that min_p lets stand
  double uniform;
  bool cut_k, cut_p;
};
// What the functions below work on lies in shared memory, the row's keys behind
// it: arguments of functions that are not inlined would pass through local memory,
// which the row's loads push out of the first cache.
struct Shared {
  Settings set;
  float top;                               // the largest logit
  double scale;                            // 128 / (ln 2 temperature)
  int blocks, rank, first, n;              // the cluster; this block's words: first.., n of them
  double powers[128];                      // 2^(i / 128)
  u64 best[MOST_BLOCKS];                   // of each block: its largest element,
  u64 sums[MOST_BLOCKS];                   // a sum of weights,
  u64 lowest[MOST_BLOCKS], highest[MOST_BLOCKS];  // its elements' ends in a range
  uint32_t maxima[MOST_BLOCKS * THREADS];  // block 0: every thread's largest key
  u64 scan[2][WARPS], scan2[2 * WARPS];
  unsigned count[8];
  unsigned members;                        // block 0: elements of the list
  unsigned owned;                          // elements of this block's own list
  u64 told[6];                             // by block 0, by Told
  union {
    struct {
      u64 list[LIST], weights[LIST];
    };
    struct {
      alignas(16) unsigned amount[BINS];  // read by fours
      unsigned mass[3][PARTS];
    } bins;
  };
};
static_assert(offsetof(Shared, bins.amount) % 16 == 0 && sizeof(Shared) % 16 == 0, "");

enum Told { BOUND, IN_LIST, FIRST_BIN, LAST_BIN, IN_BINS, CUT };

extern __shared__ __align__(16) char raw_shared[];
__device__ __forceinline__ Shared& shared() { return *reinterpret_cast<Shared*>(raw_shared); }
__device__ __forceinline__ uint32_t* row_keys() { return reinterpret_cast<uint32_t*>(raw_shared + sizeof(Shared)); }

// exp(d), d <= 0, in steps of 2^-44, with the table of 2^(i/128) and the
// exponential's series to the fourth power (P. T. P. Tang, "Table-driven
// implementation of the exponential function", 1989): relative error 2^-48.
struct Weights {
  float top;
  double scale;  // 128 / (ln 2 temperature)
  const double* powers;
  // No branches: the loops over words have several of these under way.
  __device__ __forceinline__ u64 operator()(uint32_t key) const {
    const float x = value_of(key);
    const u64 w = at(((double)x - (double)top) * scale);
    return x == top ? (u64)ONE : w;
  }
  // exp(y ln 2 / 128); nothing below 2^-45, nor where y is no number
  __device__ __forceinline__ u64 at(double y) const {
    y = fmax(y, -5888.0);
    const double magic = 6755399441055744.0;  // 1.5 2^52: adding it rounds to whole numbers
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

// The sums of the threads before this one, and those of the block.
template <int M>
struct Scans {
  u64 before[M], total[M];
};
template <int M>
__device__ __forceinline__ Scans<M> block_scans(const u64 (&v)[M]) {
  Shared& sh = shared();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 s[M], w[M];
#pragma unroll
  for (int m = 0; m < M; ++m) s[m] = v[m];
#pragma unroll 1
  for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const u64 t = __shfl_up_sync(0xffffffffu, s[m], o);
      if (lane >= o) s[m] += t;
    }
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < M; ++m)
    if (lane == 31) sh.scan[m][warp] = s[m];
  __syncthreads();
#pragma unroll
  for (int m = 0; m < M; ++m) w[m] = lane < WARPS ? sh.scan[m][lane] : 0;
#pragma unroll 1
  for (int o = 1; o < WARPS; o <<= 1) {
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const u64 t = __shfl_up_sync(0xffffffffu, w[m], o);
      if (lane >= o) w[m] += t;
    }
  }
  Scans<M> r;
#pragma unroll
  for (int m = 0; m < M; ++m) {
    const u64 base = __shfl_sync(0xffffffffu, w[m], warp ? warp - 1 : 0);
    r.before[m] = (warp ? base : 0) + s[m] - v[m];
    r.total[m] = __shfl_sync(0xffffffffu, w[m], WARPS - 1);
  }
  return r;
}
struct Scan {
  u64 before, total;
};
__device__ __forceinline__ Scan block_scan(u64 v) {
  const u64 one[1] = {v};
  const Scans<1> s = block_scans(one);
  return {s.before[0], s.total[0]};
}

// A weight into a bin, in three numbers of 15 bits each: additions of 64 bits to
// shared memory are loops, and equal logits meet in them.  2^17 weights fit.
__device__ __forceinline__ void add_mass(unsigned (*mass)[PARTS], int bin, u64 w) {
  atomicAdd(&mass[0][bin], (unsigned)w & 0x7fffu);
  atomicAdd(&mass[1][bin], (unsigned)(w >> 15) & 0x7fffu);
  atomicAdd(&mass[2][bin], (unsigned)(w >> 30));
}
__device__ __forceinline__ u64 mass_of(const unsigned (*mass)[PARTS], int bin) {
  return mass[0][bin] + ((u64)mass[1][bin] << 15) + ((u64)mass[2][bin] << 30);
}

// A bound that at least n of the first `count` maxima reach, and few more: the
// smallest of those whose distances from `top`, in 64 bins an octave, lie in the
// n-th largest's bin or above.  0 where fewer than n are no zeros.
__device__ __forceinline__ uint32_t bound_of(int count, int n) {
  Shared& sh = shared();
  const float top = sh.top;
  const uint32_t* keys = sh.maxima;
  const auto bin_of = [&](uint32_t k) {
    const int b = (int)(__float_as_uint(top - value_of(k)) >> 17) - ((127 - 12) << 6);
    return max(0, min(b, BINS - 1));  // (the largest of infinities: infinity - infinity is not a number, and far)
  };
  uint32_t mine[MOST_BLOCKS];
#pragma unroll
  for (int i = 0; i < MOST_BLOCKS; ++i) mine[i] = i * THREADS + threadIdx.x < count ? keys[i * THREADS + threadIdx.x] : 0;
  for (int i = threadIdx.x; i < BINS; i += THREADS) sh.bins.amount[i] = 0;
  if (threadIdx.x == 0) sh.count[0] = BINS, sh.count[1] = 0xffffffffu;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MOST_BLOCKS; ++i)
    if (mine[i]) atomicAdd(&sh.bins.amount[bin_of(mine[i])], 1u);
  __syncthreads();
  constexpr int PER = BINS / THREADS;
  const uint4 a = *reinterpret_cast<const uint4*>(&sh.bins.amount[threadIdx.x * PER]);
  static_assert(PER == 4, "");
  const u64 upto = block_scan(a.x + a.y + a.z + a.w).before;
  int first = BINS;
#pragma unroll
  for (int k = PER - 1; k >= 0; --k) {
    u64 sum = upto;
#pragma unroll
    for (int j = 0; j <= k; ++j) sum += (&a.x)[j];
    if (sum >= (u64)n) first = threadIdx.x * PER + k;
  }
  const unsigned lowest = __reduce_min_sync(0xffffffffu, first);
  if ((threadIdx.x & 31) == 0) atomicMin(&sh.count[0], lowest);
  __syncthreads();
  const int bin = sh.count[0];
  uint32_t bound = 0xffffffffu;
#pragma unroll
  for (int i = 0; i < MOST_BLOCKS; ++i)
    if (mine[i] && bin_of(mine[i]) <= bin) bound = min(bound, mine[i]);
  bound = __reduce_min_sync(0xffffffffu, bound);
  if ((threadIdx.x & 31) == 0) atomicMin(&sh.count[1], bound);
  __syncthreads();
  return bin < BINS ? sh.count[1] : 0;
}

// The last element, in descending order, with less than `want` before it, of
// `count` in sh.list, all above lo and none above hi.  What comes before is
// counted, or weighed by sh.weights (BY_WORD: of the elements' lower halves alone,
// whose descending order is the words' ascending one).  The range is cut into 1024
// parts until the one that holds it has no other element: two or three rounds of
// some 1500 cycles, where a bisection takes 50 of a thousand.
enum Order { COUNTED, WEIGHED, BY_WORD };
__device__ __forceinline__ u64 last_below(int count, u64 lo, u64 hi, u64 want, Order order) {
  Shared& sh = shared();
  constexpr int PER = LIST / THREADS;
  static_assert(PARTS == 2 * THREADS && 4 * PARTS * sizeof(unsigned) <= sizeof(sh.maxima), "");
  unsigned(*mass)[PARTS] = reinterpret_cast<unsigned(*)[PARTS]>(sh.maxima);  // no longer needed
  unsigned* amount = mass[3];
  u64 e[PER], w[PER], acc = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = i * THREADS + threadIdx.x;
    e[i] = at < count ? sh.list[at] : 0;
    if (order == BY_WORD) e[i] &= 0xffffffffull;
    w[i] = at >= count || order == COUNTED ? 0 : sh.weights[at];
    if (at >= count) e[i] = 0;
  }
#pragma unroll 1
  while (true) {
    const int shift = max(0, 64 - __clzll(hi - lo - 1) - 10);
#pragma unroll
    for (int i = threadIdx.x; i < 4 * PARTS; i += THREADS) mass[0][i] = 0;
    if (threadIdx.x == 0) sh.count[0] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (e[i] > lo && e[i] <= hi) {
        const int part = (int)((hi - e[i]) >> shift);
        atomicAdd(&amount[part], 1u);
        if (order != COUNTED) add_mass(mass, part, w[i]);
      }
    __syncthreads();
    const int mine = 2 * threadIdx.x;
    const u64 first = order == COUNTED ? amount[mine] : mass_of(mass, mine),
              second = order == COUNTED ? amount[mine + 1] : mass_of(mass, mine + 1);
    const u64 before = acc + block_scan(first + second).before;
    const bool in0 = amount[mine] && before < want, in1 = amount[mine + 1] && before + first < want;
    const unsigned last = __reduce_max_sync(0xffffffffu, in1 ? mine + 2 : in0 ? mine + 1 : 0);
    if ((threadIdx.x & 31) == 0 && last) atomicMax(&sh.count[0], last);
    __syncthreads();
    const int part = (int)sh.count[0] - 1;
    if (part >> 1 == threadIdx.x) sh.scan2[1] = part & 1 ? before + first : before;
    __syncthreads();
    if (part < 0) return hi;  // not reached: the first element has nothing before it
    acc = sh.scan2[1];
    hi -= (u64)part << shift;
    if (shift < 64) lo = max(lo, hi - min(hi, (u64)1 << shift));
    if (amount[part] == 1 || shift == 0) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (e[i] > lo && e[i] <= hi) sh.scan2[2] = e[i];
      __syncthreads();
      return sh.scan2[2];
    }
    __syncthreads();
  }
}

// The whole number that a sum is below where it is below top_p total.
__device__ __forceinline__ u64 wanted(double top_p, u64 total) {
  const double w = top_p > 0 ? ceil(top_p * (double)total) : 1.0;
  return w >= 1.0 ? (u64)w : 1;
}
// Running sums above uniform total are above this.
__device__ __forceinline__ u64 passed(double uniform, u64 total) {
  const u64 want = uniform > 0 ? (u64)(fmin(uniform, 1.0) * (double)total) : 0;
  return want < total ? want : total - 1;
}

// The word, from a list of `count` elements that begins the descending order and
// holds the cut.  total: the weights of all words (top_p alone).  A row runs this
// once, so most of its time is the fetching of its instructions: loops are short
// and not unrolled (a sort in unrolled steps took 122000 cycles for 40 elements,
// these loops take 5000).
//
// Short lists: four threads an element add up what is larger (64 x 32000 with top_k 50 and
// top_p 20.5 us, by the other way 28.7; at 110 elements 22.5 and 26.6).
__device__ __forceinline__ void word_of_short_list(int count, u64 total, int32_t* token) {
  Shared& sh = shared();
  const Settings& set = sh.set;
  u64* weights = sh.weights;
  __syncthreads();
  if (threadIdx.x < count) weights[threadIdx.x] = Weights{sh.top, sh.scale, sh.powers}((uint32_t)(sh.list[threadIdx.x] >> 32));
  __syncthreads();
  const int me = threadIdx.x / 4, part = threadIdx.x % 4;
  const u64 e = me < count ? sh.list[me] : 0, w = me < count ? weights[me] : 0;
  const auto add_parts = [](u64 v) {
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v + __shfl_xor_sync(0xffffffffu, v, 2);
  };
  u64 before = 0, rank = 0;
#pragma unroll 1
  for (int j = part; j < count; j += 4)
    if (sh.list[j] > e) before += weights[j], ++rank;
  before = add_parts(before);
  rank = add_parts(rank);
  if (set.cut_k && me < count && rank + 1 == (u64)set.top_k) sh.scan2[0] = before + w;  // of the first top_k
  __syncthreads();
  if (set.cut_k) total = sh.scan2[0];
  const bool keep = me < count && (!set.cut_k || rank < (u64)set.top_k) && (!set.cut_p || before < wanted(set.top_p, total)) &&
                    w >= set.least;
  if (part == 0 && me < count && !keep) weights[me] = 0;
  __syncthreads();
  u64 upto = 0, all = 0;
#pragma unroll 1
  for (int j = part; j < count; j += 4) {
    all += weights[j];
    if ((uint32_t)sh.list[j] > (uint32_t)e) upto += weights[j];  // words with smaller numbers
  }
  upto = add_parts(upto);
  all = add_parts(all);
  const u64 want = passed(set.uniform, all);
  if (keep && part == 0 && upto <= want && want < upto + w) *token = (int32_t)~(uint32_t)e;
}
__device__ __forceinline__ void word_of_list(int count, u64 total, u64 lo, u64 hi, int words, int32_t* token) {
  Shared& sh = shared();
  const Settings& set = sh.set;
  u64 cut = 0;
#pragma unroll 1
  for (int stage = set.cut_k ? COUNTED : WEIGHED; stage <= BY_WORD; ++stage) {
    u64 want = (u64)set.top_k, from = lo, to = hi;
    if (stage != COUNTED) {
      const Weights weight{sh.top, sh.scale, sh.powers};
      u64 mine = 0;
#pragma unroll 1
      for (int i = threadIdx.x; i < count; i += THREADS) {
        const u64 e = sh.list[i], w = e >= cut ? weight((uint32_t)(e >> 32)) : 0;
        mine += sh.weights[i] = stage == BY_WORD && w < set.least ? 0 : w;
      }
      const u64 sum = block_scan(mine).total;
      if (stage == WEIGHED) {
        if (!set.cut_p) continue;
        want = wanted(set.top_p, set.cut_k ? sum : total);
      } else {  // the last word, in ascending order, with no more than this before it
        want = passed(set.uniform, sum) + 1;
        from = ~(uint32_t)words, to = ~0u;
      }
    }
    cut = last_below(count, from, to, want, (Order)stage);
  }
  if (threadIdx.x == 0) *token = (int32_t)~(uint32_t)cut;
}

// One row's elements, dealt out to the blocks of a cluster in runs of words.
struct Row {
  Shared& sh;
  uint32_t* keys;
  int blocks, rank, first, n;
  Weights weight;
  __device__ __forceinline__ Row()
      : sh(shared()), keys(row_keys()), blocks(sh.blocks), rank(sh.rank), first(sh.first), n(sh.n),
        weight{sh.top, sh.scale, sh.powers} {}
  __device__ __forceinline__ static cg::cluster_group cluster() { return cg::this_cluster(); }
  __device__ __forceinline__ u64 element(int i) const { return (u64)keys[i] << 32 | ~(uint32_t)(first + i); }

  // A number of each block to all; ends with a barrier of all.
  __device__ __forceinline__ u64 add_up(u64 mine) {
    if (threadIdx.x < blocks) *cluster().map_shared_rank(&sh.sums[rank], threadIdx.x) = mine;
    cluster().sync();
    u64 s = 0;
    for (int b = 0; b < blocks; ++b) s += sh.sums[b];
    return s;
  }
  // The weights of the elements from `cut` on, of the whole row.
  __device__ __forceinline__ u64 total_weight(u64 cut) {
    u64 s = 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += THREADS)
      if (element(i) >= cut) s += weight(keys[i]);
    return add_up(block_scan(s).total);
  }
  // Block 0's number to all, to be read behind the next barrier of the cluster.
  // A kind of number has a place of its own: a thread may read it as late as
  // before the barrier after that, when block 0 is at its next number already.
  __device__ __forceinline__ void tell(int place, u64 v) {
    if (rank == 0 && threadIdx.x < blocks) cluster().map_shared_rank(sh.told, threadIdx.x)[place] = v;
  }
  // Elements to block 0's list (its length counts those that found no room).
  __device__ __forceinline__ void list(u64 e) {
    Shared* to = cluster().map_shared_rank(&sh, 0);
    const unsigned at = atomicAdd(&to->members, 1u);
    if (at < LIST) to->list[at] = e;
  }

  // The last element with less than `want` before it (by_count: elements, else
  // weights), wherever it lies.  Histograms narrow the range of elements down,
  // first over the logit's distance from the largest, then over the elements as
  // numbers, until the elements that may be it fit a list.  The first two rounds
  // bracket it by the weights of the bins' ends; where that leaves too many (very
  // small weights, many equal ones) they hold their exact weights, and each round
  // leaves one of 2^10 parts of the numbers.  What the first round leaves of a
  // block's elements makes a list of its own, where it has room, so that later
  // rounds do not go through the whole row again.
  __device__ __forceinline__ u64 search(u64 want, bool by_count, float per_unit) {
    u64 acc = 0, lowest = 0, highest = ~0ull;  // acc: amount above `highest`
    int shift = -1;                            // -1: by distance
    bool exact = by_count;
    u64* own = reinterpret_cast<u64*>(sh.maxima);  // no longer needed
    constexpr unsigned ROOM = sizeof(sh.maxima) / sizeof(u64);
    bool listed = false;  // own has all elements of the range
    // by distance: halves, as a difference of two numbers may be none of fp32; all that is far, or not a number, in the last
    const float half_top = 0.5f * weight.top;
    const auto distance_bin = [&](uint32_t key) {
      const float x = value_of(key), q = fmaf(x, -0.5f, half_top) * (2.f * per_unit);
      return x == weight.top ? 0 : (int)fminf(q, BINS - 1);
    };
    const auto bin_of = [&](u64 e) { return shift >= 0 ? (int)((highest - e) >> shift) : distance_bin((uint32_t)(e >> 32)); };
    // The smallest number, up to the largest logit's, in a bin (by distance) before `bin`, which is none of the
    // first: the bins fall as the numbers rise, and 32 lanes look at once.
    const auto edge = [&](int bin) {
      u64 lo = key_of(-INFINITY) - 1, hi = key_of(weight.top);
#pragma unroll 1
      while (hi - lo > 1) {
        const u64 step = (hi - lo + 31) / 32, k = min(hi, lo + ((threadIdx.x & 31) + 1) * step);
        const int first = __ffs(__ballot_sync(0xffffffffu, distance_bin((uint32_t)k) < bin)) - 1;
        hi = min(hi, lo + (first + 1) * step);
        lo += first * step;
      }
      return hi;
    };
    // f of every element that may lie in the range.  (Two loops: a choice of where from would be a branch around each load.)
    const auto each = [&](auto&& f) {
      if (listed) {
        const int m = (int)sh.owned;
#pragma unroll 1
        for (int i = threadIdx.x; i < m; i += THREADS) f(own[i]);
      } else {
#pragma unroll 4
        for (int i = threadIdx.x; i < n; i += THREADS) f(element(i));
      }
    };
    for (int round = 0; round < 10; ++round) {  // 2, and 10 of 64 bits in each of at most 7 more
      exact = by_count || round >= 2;
      cluster().sync();  // the list and bins of before have been read
      for (int i = threadIdx.x; i < BINS; i += THREADS) sh.bins.amount[i] = 0;
      if (exact) for (int i = threadIdx.x; i < 3 * PARTS; i += THREADS) sh.bins.mass[0][i] = 0;
      __syncthreads();
      each([&](u64 e) {
        if (e < lowest || e > highest) return;
        const int b = bin_of(e);
        // words that weigh nothing are no cut of weights
        if (shift >= 0 || by_count || b < BINS - 1) atomicAdd(&sh.bins.amount[b], 1u);
        if (exact && !by_count) add_mass(sh.bins.mass, b, weight((uint32_t)(e >> 32)));
      });
      cluster().sync();
      if (rank == 0) {
        constexpr int PER = BINS / THREADS;
        u64 low[PER], high[PER];
        unsigned amount[PER];
        static_assert(PER == 4, "");
        uint4 a[MOST_BLOCKS];
#pragma unroll
        for (int b = 0; b < MOST_BLOCKS; ++b)  // all blocks' loads at once
          a[b] = b < blocks ? *reinterpret_cast<const uint4*>(&cluster().map_shared_rank(sh.bins.amount, b)[threadIdx.x * PER])
                            : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          amount[k] = 0;
#pragma unroll
          for (int b = 0; b < MOST_BLOCKS; ++b) amount[k] += (&a[b].x)[k];
          low[k] = high[k] = amount[k];
        }
        if (!by_count && exact) {
#pragma unroll
          for (int k = 0; k < PER; ++k) {
            const int i = threadIdx.x * PER + k;
            low[k] = 0;
            if (i < PARTS)
              for (int b = 0; b < blocks; ++b) low[k] += mass_of(cluster().map_shared_rank(sh.bins.mass, b), i);
            high[k] = low[k];
          }
        } else if (!by_count) {
          // the weights of a bin's ends, a step (of 2^-44) or 2^-12 of a bin's width to the safe side; those of empty
          // bins too, as a branch would keep them from being under way together
          u64 most[PER], least[PER];
          if (shift >= 0) {
#pragma unroll
            for (int k = 0; k < PER; ++k) {
              const u64 top = highest - ((u64)(threadIdx.x * PER + k) << shift), bottom = top - (((u64)1 << shift) - 1);
              most[k] = weight((uint32_t)(top >> 32)) + 1;
              least[k] = weight((uint32_t)((bottom > top ? 0 : bottom) >> 32));
            }
          } else {
            const double unit = weight.scale / (double)per_unit;  // a bin's width; no number where the temperature is infinite
#pragma unroll
            for (int k = 0; k < PER; ++k) {
              const double i = threadIdx.x * PER + k;
              most[k] = unit >= 0 ? weight.at(fmin(0.0, -(i - 1.0 / 4096) * unit)) + 1 : (u64)ONE;
              least[k] = unit >= 0 ? weight.at(-(i + 1 + 1.0 / 4096) * unit) : 0;
            }
          }
#pragma unroll
          for (int k = 0; k < PER; ++k) {
            low[k] = amount[k] * (least[k] ? least[k] - 1 : 0);
            high[k] = amount[k] * min(most[k], (u64)ONE);
          }
        }
        const u64 sums[2] = {low[0] + low[1] + low[2] + low[3], high[0] + high[1] + high[2] + high[3]};
        const Scans<2> scans = block_scans(sums);
        u64 low_before = scans.before[0], high_before = scans.before[1];
        if (threadIdx.x == 0) sh.count[0] = BINS, sh.count[1] = 0, sh.count[2] = 0, sh.count[3] = 0, sh.members = 0;
        __syncthreads();
        low_before += acc, high_before += acc;
        // the first bin that the cut may lie in, the last that it may, the last of all
        unsigned from = BINS, to = 0, last = 0, in = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const unsigned i = threadIdx.x * PER + k;
          if (amount[k]) {
            last = i;
            if (from == BINS && high_before + high[k] >= want) from = i;
            if (low_before < want) to = i;
          }
          low_before += low[k], high_before += high[k];
        }
        from = __reduce_min_sync(0xffffffffu, from);
        to = __reduce_max_sync(0xffffffffu, to);
        last = __reduce_max_sync(0xffffffffu, last);
        if ((threadIdx.x & 31) == 0) atomicMin(&sh.count[0], from), atomicMax(&sh.count[1], to), atomicMax(&sh.count[2], last);
        __syncthreads();
        from = min(sh.count[0], sh.count[2]), to = sh.count[1];
#pragma unroll
        for (int k = 0; k < PER; ++k) in += threadIdx.x * PER + k >= from && threadIdx.x * PER + k <= to ? amount[k] : 0;
        in = __reduce_add_sync(0xffffffffu, in);
        if ((threadIdx.x & 31) == 0 && in) atomicAdd(&sh.count[3], in);
        __syncthreads();
      }
      tell(FIRST_BIN, min(sh.count[0], sh.count[2]));
      tell(LAST_BIN, sh.count[1]);
      tell(IN_BINS, sh.count[3]);
      cluster().sync();
      const int from = (int)sh.told[FIRST_BIN], to = (int)sh.told[LAST_BIN];
      const bool fits = sh.told[IN_BINS] <= LIST;
      // the bins' ends
      u64 hi, lo;
      if (shift >= 0) {
        hi = highest - ((u64)from << shift);
        lo = max(lowest, highest - min(highest, ((u64)(to + 1) << shift) - 1));
      } else {
        hi = from ? (edge(from) << 32) - 1 : ~0ull;
        lo = edge(to + 1) << 32;
      }
      u64 sums[2] = {0, 0};  // above the range, and how many lie in it
      each([&](u64 e) {
        const u64 w = by_count ? 1 : weight((uint32_t)(e >> 32));
        sums[0] += e > hi && e <= highest ? w : 0;
        sums[1] += e >= lo && e <= hi;
      });
      const Scans<2> scans = block_scans(sums);
      const bool keep = !listed && scans.total[1] <= ROOM;
      if (keep || fits) {
        u64* put = own + scans.before[1];
        each([&](u64 e) {  // (apart: its branches would keep the weights from each other)
          if (e < lo || e > hi) return;
          if (keep) *put++ = e;
          if (fits) list(e);
        });
      }
      if (keep) sh.owned = (unsigned)scans.total[1];
      listed = listed || keep;
      __syncthreads();
      // the ends of what is left
      u64 least = ~0ull, most = 0;
      each([&](u64 e) {
        if (e >= lo && e <= hi) least = min(least, e), most = max(most, e);
      });
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
      }
      if ((threadIdx.x & 31) == 0) sh.scan2[threadIdx.x >> 5] = least, sh.scan2[WARPS + (threadIdx.x >> 5)] = most;
      __syncthreads();
#pragma unroll 4
      for (int w = 0; w < WARPS; ++w) least = min(least, sh.scan2[w]), most = max(most, sh.scan2[WARPS + w]);
      if (threadIdx.x < blocks) {
        Shared* there = cluster().map_shared_rank(&sh, threadIdx.x);
        there->lowest[rank] = least, there->highest[rank] = most;
      }
      acc += add_up(scans.total[0]);
      lowest = ~0ull, highest = 0;
      for (int b = 0; b < blocks; ++b) lowest = min(lowest, sh.lowest[b]), highest = max(highest, sh.highest[b]);
      if (fits) {
        u64 cut = 0;
        if (rank == 0) {
          const int count = (int)sh.members;
          if (!by_count)
            for (int i = threadIdx.x; i < count; i += THREADS) sh.weights[i] = weight((uint32_t)(sh.list[i] >> 32));
          cut = last_below(count, lowest - 1, highest, want - acc, by_count ? COUNTED : WEIGHED);
        }
        tell(CUT, cut);
        cluster().sync();
        return sh.told[CUT];
      }
      if (lowest > highest) break;
      shift = max(0, 64 - __clzll(highest - lowest) - (by_count || round == 0 ? 11 : 10));  // into BINS, or PARTS
    }
    return lowest;  // not reached
  }
};

template <typename T, int VEC>
__global__ void __launch_bounds__(THREADS, 2) sample_kernel(Sampling a, int run, int32_t* __restrict__ tokens) {
  Shared& sh = shared();
  uint32_t* keys = row_keys();
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

  // the row, the largest element; every thread's words in ascending order
  uint32_t high = 0;
  int where = 0;
  const auto note = [&](int i, uint32_t k) {
    keys[i] = k;
    if (k > high) high = k, where = i;
  };
  const int whole = n / VEC * VEC;
#pragma unroll 4
  for (int i = threadIdx.x * VEC; i < whole; i += THREADS * VEC) {
    if constexpr (VEC > 1) {
      const uint4 u = *reinterpret_cast<const uint4*>(p + i);
#pragma unroll
      for (int j = 0; j < VEC; ++j) note(i + j, key_of(to_f32(reinterpret_cast<const T*>(&u)[j])));
    } else {
      note(i, key_of(to_f32(p[i])));
    }
  }
  if (whole + (int)threadIdx.x < n) note(whole + threadIdx.x, key_of(to_f32(p[whole + threadIdx.x])));
  u64 best = high ? (u64)high << 32 | ~(uint32_t)(first + where) : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((threadIdx.x & 31) == 0) sh.scan[0][threadIdx.x >> 5] = best;
  cluster.barrier_wait(std::move(begun));
  cluster.map_shared_rank(sh.maxima, 0)[rank * THREADS + threadIdx.x] = high;
  __syncthreads();
  if (threadIdx.x < blocks) {
    for (int w = 0; w < WARPS; ++w) best = max(best, sh.scan[0][w]);
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
  if (threadIdx.x == 0) {
    sh.set = {top_k, top_p, min_p > 0 ? (u64)ceil(fmin(min_p, 1.0) * ONE) : 0, (double)a.uniform[row],
              top_k > 0 && top_k < words, top_p < 1};
    sh.top = top, sh.scale = 184.66496523378731 / temperature;  // 128 / ln 2
    sh.blocks = blocks, sh.rank = rank, sh.first = first, sh.n = n;
  }
  __syncthreads();
  const Settings& set = sh.set;
  Row r;
  u64 cut = 0;
  if (set.cut_k || set.cut_p) {
    u64 total = 0;
    if (!set.cut_k) total = r.total_weight(0);
    // no word weighs more than one, most weigh far less: the nucleus is likely to have some sixteen
    // times as many words as its weight
    const u64 likely = set.cut_k ? 0 : 16 * (wanted(top_p, total) >> 44);
    for (int64_t ask = set.cut_k ? top_k : likely > NUCLEUS ? NUCLEUS_MORE : NUCLEUS;
         ask <= ASK && likely <= (u64)NUCLEUS_MORE; ask = NUCLEUS_MORE) {
      uint32_t bound = 0;
      if (rank == 0) bound = bound_of(blocks * THREADS, (int)ask);
      if (threadIdx.x == 0) sh.members = 0;
      r.tell(BOUND, bound);
      cluster.sync();
      bound = (uint32_t)sh.told[BOUND];
      // (a bound of 0, where fewer threads than asked for have words, lists every word)
      if (high >= bound && (bound || words <= LIST)) {
#pragma unroll 2
        for (int i = threadIdx.x * VEC; i < whole; i += THREADS * VEC) {
          if constexpr (VEC >= 4) {
#pragma unroll
            for (int j = i; j < i + VEC; j += 4) {
              const uint4 k = *reinterpret_cast<const uint4*>(keys + j);
              if (max(max(k.x, k.y), max(k.z, k.w)) >= bound)
#pragma unroll 1
                for (int l = j; l < j + 4; ++l)
                  if (keys[l] >= bound) r.list(r.element(l));
            }
          } else if (keys[i] >= bound) {
            r.list(r.element(i));
          }
        }
        if (whole + (int)threadIdx.x < n && keys[whole + threadIdx.x] >= bound) r.list(r.element(whole + threadIdx.x));
      }
      cluster.sync();
      u64 ok = 0;
      if (rank == 0 && sh.members <= LIST && (bound || words <= LIST)) {
        ok = 1;
        if (!set.cut_k) {  // does the cut lie in the list?
          u64 sum = 0;
#pragma unroll 1
          for (int i = threadIdx.x; i < (int)sh.members; i += THREADS) sum += r.weight((uint32_t)(sh.list[i] >> 32));
          ok = block_scan(sum).total >= wanted(top_p, total);
        }
      }
      r.tell(IN_LIST, ok);
      // Block 0 finds the word: it need not wait for the others, which wait for its number to leave (staying
      // until it is done would take issue slots from other rows).
      if (ok) (void)cluster.barrier_arrive();
      else cluster.sync();
      if (ok || sh.told[IN_LIST]) {
        if (rank) return;
        const int count = (int)sh.members;
        if (count <= SHORT) word_of_short_list(count, total, tokens + row);
        else word_of_list(count, total, ((u64)bound << 32) - (bound ? 1 : 0), best, words, tokens + row);
        return;
      }
      if (set.cut_k || ask == NUCLEUS_MORE) break;
    }
    const float per_unit = (float)fmin(BINS / (32.0 * temperature), 1.7e38);
#pragma unroll 1
    for (int pass = set.cut_k ? 0 : 1; pass < (set.cut_p ? 2 : 1); ++pass) {
      if (pass == 1 && set.cut_k) total = r.total_weight(cut);
      cut = max(cut, r.search(pass ? wanted(set.top_p, total) : (u64)set.top_k, !pass, per_unit));
    }
  }

  // sums of what is left, by warps that each own neighbouring words
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per = ((n + WARPS - 1) / WARPS + 31) / 32 * 32;
  const int lo = min(n, warp * per), hi = min(n, lo + per);
  const auto kept = [&](int i) -> u64 {
    if (i >= hi || r.element(i) < cut) return 0;
    const u64 w = r.weight(keys[i]);
    return w >= set.least ? w : 0;
  };
  u64 mine = 0;
#pragma unroll 4
  for (int i = lo + lane; i < hi; i += 32) mine += kept(i);
  mine = warp_add(mine);
  __syncthreads();
  if (lane == 0) sh.scan[0][warp] = mine;
  __syncthreads();
  u64 before = 0, all = 0;
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += sh.scan[0][w];
    all += sh.scan[0][w];
  }
  if (threadIdx.x < blocks) *cluster.map_shared_rank(&sh.sums[rank], threadIdx.x) = all;
  cluster.sync();
  u64 total = 0;
  for (int b = 0; b < blocks; ++b) {
    if (b < rank) before += sh.sums[b];
    total += sh.sums[b];
  }
  const u64 want = passed(set.uniform, total);
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
  static std::atomic<bool> allowed[kMaxDevices];
  std::atomic<bool>& here = allowed[current_device_slot()];
  if (!here.load()) {
    DLVK_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    here.store(true);
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
  // block has some thousands (8 x 8000 with blocks of 2000 12.3 us, of 4000 14.3; below that no difference)
  int blocks = 1;
  const auto run_of = [&](int b) { return (int)(((a.words + b - 1) / b + 7) / 8 * 8); };
  while (blocks < MOST_BLOCKS && (run_of(blocks) > 16384 || (a.rows * blocks < 148 && run_of(blocks) > 2048))) blocks *= 2;
  const int run = run_of(blocks);
  const int64_t bytes = a.dt == DType::BF16 ? 2 : 4;
  const bool wide = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && (a.ld * bytes % 16 == 0 || a.rows == 1);
  if (a.dt == DType::BF16) {
    if (wide) launch<__nv_bfloat16, 8>(a, tokens, blocks, run, s);
    else launch<__nv_bfloat16, 1>(a, tokens, blocks, run, s);
  } else {
    if (wide) launch<float, 4>(a, tokens, blocks, run, s);
    else launch<float, 1>(a, tokens, blocks, run, s);
  }
}

}  // namespace dlvk
