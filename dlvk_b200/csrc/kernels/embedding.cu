// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   y[i, :]  = scale * table[id_i, :]              (zeros for ids outside [0, V))
//   dT[v, :] = scale * sum over i with id_i = v, in ascending i, of dy[i, :]
//
// The reference's lookup (shaders/embedding_lookup.comp:24-55) has no scale
// and returns no gradient.  Here the gradient has no floating-point atomics:
// the tokens are sorted by word, stably, and every row of dT is written once
// by a sum whose order depends on nothing but the ids, so two runs agree bit
// for bit, and rows without a token get their zeros in the same pass.
//
// What bounds them: the lookup moves n D elements in and out; the gradient
// reads dy once and writes V D fp32 once (8192 x 1024 bf16 tokens over 32000
// words: 17 MB in, 131 MB out, 22.6 us at the measured copy rate), so the
// sort has to be short.  Measured: that lookup 6.1 us, that gradient 35.3 (sort
// 6.2, sums 21.0, joins 10.0, each starting up while the one before it ends).
// The same bits on every run have a price where the sort is most of the work.
// Against float atomics after a memset, cold caches, one call: 40.0 us (39.7
// with atomics) at that size, 17 (11) for 512 tokens x 256 over 5000 words, 52 (30)
// for 65536 x 64 over 100000, 517 (503) for 524288 x 1024 over 32000.
#include <algorithm>
#include <type_traits>

#include "dlvk/common.h"
#include "dlvk/kernels.h"

namespace dlvk {
namespace {

constexpr int SORT_THREADS = 1024;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int SORT_WORDS = 1024;  // most words of one block: a count per warp and word in shared memory
constexpr int RED_THREADS = 256;

template <typename T> struct Vec { static constexpr int N = 16 / (int)sizeof(T); };

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float* v) {
  if constexpr (VEC == 1) {
    v[0] = to_f32(*p);
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = to_f32(e[k]);
  }
}

// ---------------------------------------------------------------- lookup
// A warp copies a row; a lane has up to four 16-byte loads in flight.
template <typename T, typename ID, int VEC>
__global__ void __launch_bounds__(256) lookup_kernel(const ID* __restrict__ ids, const T* __restrict__ table,
                                                     T* __restrict__ out, int64_t n, int64_t V, int D, int64_t ld,
                                                     float scale) {
  const int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= n) return;
  const int lane = threadIdx.x & 31;
  const int64_t id = (int64_t)ids[i];
  const bool ok = id >= 0 && id < V;
  const T* src = table + (ok ? id : 0) * ld;
  T* dst = out + i * D;
  for (int c = lane * VEC; c < D; c += 4 * 32 * VEC) {
    float v[4][VEC];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[k][j] = 0.f;
      if (ok && c + k * 32 * VEC < D) load_vec<T, VEC>(src + c + k * 32 * VEC, v[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int at = c + k * 32 * VEC;
      if (at >= D) break;
      if constexpr (VEC == 1) {
        dst[at] = from_f32<T>(v[k][0] * scale);
      } else {
        uint4 u;
        T* e = reinterpret_cast<T*>(&u);
#pragma unroll
        for (int j = 0; j < VEC; ++j) e[j] = from_f32<T>(v[k][j] * scale);
        *reinterpret_cast<uint4*>(dst + at) = u;
      }
    }
  }
}

// ---------------------------------------------------------------- sort
// Writing the zero rows is most of the gradient's traffic (32000 words of
// 1024: 131 MB, of which 8192 tokens touch a quarter), and the last joining
// pass is bound by latency.  So [0, Z) are cleared beside the sums and [Z, V)
// beside the joins.
// A warp clears `floats` consecutive floats from p on: up to the first line of
// 128 bytes, 16 bytes a lane (whole lines: at any other offset each store of a
// warp touches five), the rest.
__device__ __forceinline__ void clear_span(float* p, int64_t floats) {
  const int lane = threadIdx.x & 31;
  const int head = (int)min(floats, (int64_t)((128 - reinterpret_cast<uintptr_t>(p) % 128) / 4 % 32));
  const int64_t body = (floats - head) / 4 * 4;
  if (lane < head) p[lane] = 0.f;
  for (int64_t c = lane * 4; c < body; c += 128)
    *reinterpret_cast<float4*>(p + head + c) = make_float4(0.f, 0.f, 0.f, 0.f);
  if (head + body + lane < floats) p[head + body + lane] = 0.f;
}
// The order of the words in the sort: word v is the (v >> log)-th of block
// v mod 2^log's `per` places.  Tokenizers number their words by frequency; blocks
// of neighbouring words would leave the first one most of the tokens (65536
// tokens x 1024 over 32000 words, word k as common as 1 / (k + 2.7): the sort 57 us,
// dealt out 27).
struct WordOrder {
  int log, per;
  __device__ __forceinline__ int at(int v) const { return (v & ((1 << log) - 1)) * per + (v >> log); }
  __host__ __device__ __forceinline__ int places() const { return per << log; }
};

// A warp of `warps` takes every warps-th group of consecutive rows (about 4 KB,
// at most 32) of [v0, v1) and clears the runs of rows without a token in it.
__device__ __forceinline__ void clear_rows(const int* start, WordOrder words, float* dtable, int v0, int v1, int D,
                                           int warp, int warps) {
  const int lane = threadIdx.x & 31, per = max(1, min(32, 1024 / D));
  for (int64_t v = v0 + (int64_t)warp * per; v < v1; v += (int64_t)warps * per) {
    const int rows = (int)min((int64_t)per, v1 - v);
    bool empty = false;
    if (lane < rows) {
      const int at = words.at((int)v + lane);
      empty = start[at] == start[at + 1];
    }
    unsigned left = __ballot_sync(0xffffffffu, empty);
    while (left) {
      const int first = __ffs(left) - 1, run = __ffs(~(left >> first)) - 1;  // run 32: ~0 has no bit, __ffs gives 0
      const int count = run < 0 ? 32 : run;
      clear_span(dtable + (v + first) * D, (int64_t)count * D);
      left = first + count >= 32 ? 0u : left & ~((2u << (first + count - 1)) - 1u);
    }
  }
}

// The word of token i < hi, -1 for none: past the end, padding, or an id that
// no int holds (negative ones are kept negative).
template <typename ID>
__device__ __forceinline__ int word_at(const ID* ids, int i, int hi, int padding) {
  if (i >= hi) return -1;
  const ID raw = ids[i];
  int w = (int)raw;
  if (sizeof(ID) == 8 && (ID)w != raw) w = -1;
  return w == padding ? -1 : w;
}

// Stable sort of the tokens by word in one launch, without a word between
// blocks.  Block b of B = 2^log owns the words b, b + B, b + 2 B, ... and reads all
// ids twice: once to count its own words (per warp: warp w has the w-th part of
// the ids) and the tokens of the blocks before it, which is where its part of
// the order begins; once more to place its tokens.  Rotated right by log, an id has
// its block in the upper bits and its place there in the lower ones, so that one
// subtraction and comparison tell both.  A token's place is its word's
// start + the counts of earlier warps + its rank among the warp's tokens so
// far, so equal words stay in ascending position.  Every block reading all
// ids costs 128 x 4 n bytes from L2 (8192 tokens: 4 MB), far less than the
// passes over memory of a radix sort of so few keys.
//   start[words.at(v)]: first place of word v, start[that + 1]: of what follows it;
//   order[place]: the token.
template <typename ID>
__global__ void __launch_bounds__(SORT_THREADS) sort_tokens_kernel(const ID* __restrict__ ids, int n, int V,
                                                                   WordOrder words, int padding, int* __restrict__ start,
                                                                   int* __restrict__ order, int* __restrict__ word) {
  pdl_wait();
  extern __shared__ int cnt[];  // [SORT_WARPS][R], then [R]: a word's first place
  __shared__ int warp_part[SORT_WARPS];
  __shared__ int before_sm;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int R = words.per, B = 1 << words.log, b = blockIdx.x;
  const unsigned base0 = words.log > 0 ? (unsigned)b << (32 - words.log) : 0u;
  int* first = cnt + SORT_WARPS * R;
  const int per = (max(n, 1) + SORT_THREADS - 1) / SORT_THREADS * 32;  // ids of a warp, whole groups of 32
  const int used = (int)(((unsigned)n + per - 1) / per);               // warps that have any
  for (int i = tid; i < used * R; i += SORT_THREADS) cnt[i] = 0;
  if (tid == 0) before_sm = 0;
  __syncthreads();

  const int lo = min((int64_t)n, (int64_t)warp * per), hi = min((int64_t)n, (int64_t)(warp + 1) * per);
  int* mine = cnt + warp * R;
  const unsigned range = (unsigned)((V - b + B - 1) >> words.log);  // words of this block
  int before = 0;
  unsigned key[8];  // places of the warp's last 256 ids in this block: below `range` for its words
  for (int base = lo; base < hi; base += 256) {
    int id[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) id[k] = word_at(ids, base + k * 32 + lane, hi, padding);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const unsigned turned = __funnelshift_r((unsigned)id[k], (unsigned)id[k], words.log);
      before += turned < base0 && (unsigned)id[k] < (unsigned)V;
      key[k] = turned - base0;
      if (key[k] < range) atomicAdd(&mine[key[k]], 1);
    }
  }
  before = __reduce_add_sync(0xffffffffu, before);
  if (lane == 0 && before) atomicAdd(&before_sm, before);
  __syncthreads();

  // Thread r scans its word's counts over the warps that have tokens, eight
  // loads at a time (a warp to a word, with shuffles, took 16.6 us instead of
  // 6.4 for 200000 words, 6.0 instead of 5.2 for 2048 tokens over 32000), ...
  int total = 0;
  if (tid < R) {
    for (int w0 = 0; w0 < used; w0 += 8) {
      int c[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) c[u] = w0 + u < used ? cnt[(w0 + u) * R + tid] : 0;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (w0 + u < used) cnt[(w0 + u) * R + tid] = total;
        total += c[u];
      }
    }
  }
  // ... the block the words' totals.
  int incl = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += t;
  }
  if (lane == 31) warp_part[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int p = warp_part[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, p, o);
      if (lane >= o) p += t;
    }
    warp_part[lane] = p;
  }
  __syncthreads();
  const int at = before_sm + incl - total + (warp > 0 ? warp_part[warp - 1] : 0);
  if (tid < R) {  // places without a word have none of the tokens
    start[b * R + tid] = at;
    if (b == B - 1 && tid == R - 1) start[words.places()] = at + total;
  }
  if (tid < R) first[tid] = at;
  __syncthreads();

  const bool held = hi - lo <= 256;  // one batch: still in registers
  for (int base = lo; base < hi; base += 256) {
    if (!held) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const unsigned id = (unsigned)word_at(ids, base + k * 32 + lane, hi, padding);
        key[k] = __funnelshift_r(id, id, words.log) - base0;
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const bool hit = key[k] < range;
      if (!__any_sync(0xffffffffu, hit)) continue;
      const unsigned peers = __match_any_sync(0xffffffffu, hit ? key[k] : range);
      if (hit) {
        const int place = first[key[k]] + mine[key[k]] + __popc(peers & ((1u << lane) - 1u));
        order[place] = base + k * 32 + lane;
        word[place] = (int)(key[k] << words.log) + b;
      }
      __syncwarp();
      if (hit && lane == __ffs(peers) - 1) mine[key[k]] += __popc(peers);
      __syncwarp();
    }
  }
}

// ---------------------------------------------------------------- sums
template <int VEC>
__device__ __forceinline__ void put_row(float* dst, const float* acc, float scale, bool accumulate) {
  if constexpr (VEC == 1) {
    *dst = accumulate ? fmaf(acc[0], scale, *dst) : acc[0] * scale;
  } else {
#pragma unroll
    for (int k = 0; k < VEC; k += 4) {
      float4 o = accumulate ? *reinterpret_cast<const float4*>(dst + k) : make_float4(0.f, 0.f, 0.f, 0.f);
      o.x = fmaf(acc[k], scale, o.x);
      o.y = fmaf(acc[k + 1], scale, o.y);
      o.z = fmaf(acc[k + 2], scale, o.z);
      o.w = fmaf(acc[k + 3], scale, o.w);
      *reinterpret_cast<float4*>(dst + k) = o;
    }
  }
}

// The first blocks sum chunks of C consecutive places of the order; the rest
// write zero rows.  TX threads go across a row, 256 / TX chunks to a
// block.  A word whose tokens lie in one chunk is finished here; what a chunk
// has of a word that continues from the chunk before goes to part[2 chunk],
// of one that begins here and continues to part[2 chunk + 1] (join_kernel).
template <typename T, int VEC>
__global__ void __launch_bounds__(RED_THREADS) sum_chunks_kernel(
    const T* __restrict__ dy, int64_t ld, const int* __restrict__ start, const int* __restrict__ order,
    const int* __restrict__ word, float* __restrict__ dtable, float* __restrict__ part, WordOrder words, int D, int C,
    int TX, int chunk_blocks, float scale, int accumulate, int clear_to) {
  pdl_wait();
  if ((int)blockIdx.x >= chunk_blocks) {
    clear_rows(start, words, dtable, 0, clear_to, D,
               (blockIdx.x - chunk_blocks) * (RED_THREADS / 32) + (threadIdx.x >> 5),
               (gridDim.x - chunk_blocks) * (RED_THREADS / 32));
    return;
  }
  const int tx = threadIdx.x % TX;
  const int chunk = blockIdx.x * (RED_THREADS / TX) + threadIdx.x / TX;
  const int total = start[words.places()];
  const int c0 = chunk * C, c1 = min(total, c0 + C);
  // the words beside the chunk (-1: none): one that goes on there is not finished here
  const int before = c0 > 0 && c0 < c1 ? word[c0 - 1] : -1, after = c0 < c1 && c1 < total ? word[c1] : -1;
  for (int col = tx * VEC; col < D && c0 < c1; col += TX * VEC) {
    float acc[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
    for (int j = c0; j < c1; j += 8) {
      float v[8][VEC];
      int w[9];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = min(j + u, c1 - 1);
        w[u] = word[i];
        load_vec<T, VEC>(dy + (int64_t)order[i] * ld + col, v[u]);
      }
      w[8] = j + 8 < c1 ? word[j + 8] : -1;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (j + u < c1) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) acc[k] += v[u][k];
          if (j + u + 1 == c1 || w[u + 1] != w[u]) {  // the last of its word in this chunk
            if (w[u] != before && w[u] != after) {
              put_row<VEC>(dtable + (int64_t)w[u] * D + col, acc, scale, accumulate);
            } else {
              put_row<VEC>(part + ((int64_t)chunk * 2 + (w[u] != before)) * D + col, acc, 1.f, false);
            }
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
          }
        }
      }
    }
  }
}

// Joins the parts of a word that spans chunks, in their order: the block row
// of the chunk where it begins.
template <int VEC>
__global__ void __launch_bounds__(RED_THREADS) join_kernel(const int* __restrict__ start, const int* __restrict__ word,
                                                           const float* __restrict__ part, float* __restrict__ dtable,
                                                           WordOrder words, int V, int D, int C, int TX, int chunks,
                                                           float scale, int accumulate, int join_blocks,
                                                           int clear_from) {
  pdl_wait();
  if ((int)blockIdx.x >= join_blocks) {
    clear_rows(start, words, dtable, clear_from, V, D,
               (blockIdx.x - join_blocks) * (RED_THREADS / 32) + (threadIdx.x >> 5),
               (gridDim.x - join_blocks) * (RED_THREADS / 32));
    return;
  }
  const int chunk = blockIdx.x * (RED_THREADS / TX) + threadIdx.x / TX;
  const int total = start[words.places()];
  const int64_t c1 = (int64_t)(chunk + 1) * C;
  if (chunk >= chunks || c1 >= total) return;
  const int w = word[c1 - 1];
  const int at = words.at(w), end = start[at + 1];
  if (end <= c1 || start[at] < c1 - C) return;
  const int last = (end - 1) / C;  // the chunk that holds its last token
  for (int col = (threadIdx.x % TX) * VEC; col < D; col += TX * VEC) {
    float acc[VEC];
    load_vec<float, VEC>(part + ((int64_t)chunk * 2 + 1) * D + col, acc);
    int c = chunk + 1;
    for (; c + 7 <= last; c += 8) {
      float v[8][VEC];
#pragma unroll
      for (int u = 0; u < 8; ++u) load_vec<float, VEC>(part + (int64_t)(c + u) * 2 * D + col, v[u]);
#pragma unroll
      for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] += v[u][k];
    }
    for (; c <= last; ++c) {
      float v[VEC];
      load_vec<float, VEC>(part + (int64_t)c * 2 * D + col, v);
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] += v[k];
    }
    put_row<VEC>(dtable + (int64_t)w * D + col, acc, scale, accumulate);
  }
}

// Places of one chunk: more for long inputs, where there are chunks enough.
int chunk_of(int64_t n) { return n <= 16384 ? 16 : (n <= 65536 ? 32 : 64); }

// Threads across a row of D elements, VEC each: a power of two up to a block.
int across(int D, int vec) {
  int tx = 1;
  while (tx < RED_THREADS && tx * vec < D) tx *= 2;
  return tx;
}

// Blocks of `warps` warps that clear `rows` rows of D (clear_rows' groups).
int clear_blocks(int64_t rows, int D, int warps) {
  const int64_t groups = (rows + std::max(1, std::min(32, 1024 / D)) - 1) / std::max(1, std::min(32, 1024 / D));
  return (int)std::min<int64_t>((groups + warps - 1) / warps, 148 * 8);
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T, typename ID>
void lookup_t(const ID* ids, const T* table, T* out, int64_t n, int64_t V, int D, int64_t ld, float scale,
              cudaStream_t s) {
  constexpr int VEC = Vec<T>::N;
  const unsigned grid = (unsigned)((n + 7) / 8);
  if (D % VEC == 0 && ld % VEC == 0 && al16(table) && al16(out))
    lookup_kernel<T, ID, VEC><<<grid, 256, 0, s>>>(ids, table, out, n, V, D, ld, scale);
  else
    lookup_kernel<T, ID, 1><<<grid, 256, 0, s>>>(ids, table, out, n, V, D, ld, scale);
  DLVK_POST_LAUNCH();
}

template <typename T, int VEC>
void sums(const T* dy, int64_t ld, const int* start, const int* order, const int* word, float* dtable, float* part,
          int64_t n, WordOrder words, int V, int D, float scale, bool accumulate, cudaStream_t s) {
  const int C = chunk_of(n);
  const int chunks = (int)((n + C - 1) / C);
  const int tx = across(D, VEC), per = RED_THREADS / tx;
  const int chunk_blocks = (chunks + per - 1) / per;
  // The share of the zero rows beside the joins (see clear_rows), none when
  // adding: 3 in 10 where both are long (8192 tokens x 1024 over 32000 words:
  // 40.0 -> 37.9 us, 2048 x 1024: 35.9 -> 33.8); for few tokens or a small
  // table it gains nothing (103 x 624 over 52597: 31.8 and 31.8), and where
  // most words have tokens there is little to clear.  Clearing a share beside
  // the sort as well, before it is known which rows have tokens, gained
  // nothing either (37.9) and cost 2 to 60 us for few tokens.
  const bool shared = n >= 1024 && n < V && (int64_t)V * D >= (1 << 23);
  const int z = accumulate ? 0 : (shared ? V - (int)((int64_t)V * 3 / 10) : V);
  const int zero_blocks = clear_blocks(z, D, RED_THREADS / 32);
  if (chunk_blocks + zero_blocks > 0) {
    launch_pdl(sum_chunks_kernel<T, VEC>, dim3(chunk_blocks + zero_blocks), dim3(RED_THREADS), 0, s, dy, ld, start,
               order, word, dtable, part, words, D, C, tx, chunk_blocks, scale, accumulate ? 1 : 0, z);
    DLVK_POST_LAUNCH();
  }
  const int last_blocks = accumulate ? 0 : clear_blocks(V - z, D, RED_THREADS / 32);
  if (chunks > 1 || last_blocks > 0) {
    constexpr int JV = VEC > 1 ? 4 : 1;
    const int jx = across(D, JV), jper = RED_THREADS / jx;
    const int join_blocks = chunks > 1 ? (chunks + jper - 1) / jper : 0;
    launch_pdl(join_kernel<JV>, dim3(join_blocks + last_blocks), dim3(RED_THREADS), 0, s, start, word, part, dtable,
               words, V, D, C, jx, chunks, scale, accumulate ? 1 : 0, join_blocks, z);
    DLVK_POST_LAUNCH();
  }
}

}  // namespace

void embedding_lookup(DType dt, bool ids64, const void* ids, const void* table, void* out, int64_t n, int64_t V, int D,
                      int64_t ld, float scale, cudaStream_t s) {
  if (n == 0 || D == 0) return;
  DLVK_CHECK(n < (1LL << 34), "embedding_lookup: too many tokens for one launch");
  const int32_t* i32 = reinterpret_cast<const int32_t*>(ids);
  const int64_t* i64 = reinterpret_cast<const int64_t*>(ids);
  if (dt == DType::F32) {
    const float* t = reinterpret_cast<const float*>(table);
    float* o = reinterpret_cast<float*>(out);
    if (ids64) lookup_t(i64, t, o, n, V, D, ld, scale, s);
    else lookup_t(i32, t, o, n, V, D, ld, scale, s);
  } else {
    DLVK_CHECK(dt == DType::BF16, "embedding_lookup: the table is fp32 or bf16");
    const __nv_bfloat16* t = reinterpret_cast<const __nv_bfloat16*>(table);
    __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(out);
    if (ids64) lookup_t(i64, t, o, n, V, D, ld, scale, s);
    else lookup_t(i32, t, o, n, V, D, ld, scale, s);
  }
}

// Blocks of the sort: a power of two near the number of SMs with at least 8 words
// each, more where the counts of a block's words have no room.
static WordOrder word_order(int64_t V) {
  int log = 0;
  while (log < 7 && V >> (log + 1) >= 8) ++log;
  while ((V + (1LL << log) - 1) >> log > SORT_WORDS) ++log;
  return {log, (int)((V + (1LL << log) - 1) >> log)};
}

int64_t embedding_grad_start_ints(int64_t V) { return word_order(V).places() + 1; }

int64_t embedding_grad_part_floats(int64_t n, int D) {
  const int C = chunk_of(n);
  return (n + C - 1) / C * 2 * D;
}

void embedding_grad(DType dt, bool ids64, const void* ids, const void* dy, int64_t ld, float* dtable, int64_t n,
                    int64_t V, int D, float scale, int64_t padding, bool accumulate, int* start, int* order, int* word,
                    float* part, cudaStream_t s) {
  if (V == 0 || D == 0) return;
  DLVK_CHECK(n < EMBEDDING_GRAD_TOKENS && V < EMBEDDING_GRAD_WORDS, "embedding_grad: more than 2^31 tokens or words");
  const WordOrder words = word_order(V);
  const auto room = [](int per) { return (SORT_WARPS + 1) * per * (int)sizeof(int); };
  const size_t smem = (size_t)room(words.per);
  static bool attr_set[kMaxDevices] = {false};
  const int dev = current_device_slot();
  if (!attr_set[dev]) {
    const int most = room(SORT_WORDS);
    const auto attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
    DLVK_CUDA_CHECK(cudaFuncSetAttribute(sort_tokens_kernel<int32_t>, attr, most));
    DLVK_CUDA_CHECK(cudaFuncSetAttribute(sort_tokens_kernel<int64_t>, attr, most));
    attr_set[dev] = true;
  }
  const int pad = padding >= 0 && padding < V ? (int)padding : -1;
  const bool f32 = dt == DType::F32;
  DLVK_CHECK(f32 || dt == DType::BF16, "embedding_grad: dy is fp32 or bf16");
  const int step = f32 ? 4 : 8;
  const bool vec = D % step == 0 && ld % step == 0 && al16(dy) && al16(dtable) && al16(part);
  const auto sort = [&](const auto* p) {
    using ID = std::remove_cv_t<std::remove_reference_t<decltype(*p)>>;
    launch_pdl(sort_tokens_kernel<ID>, dim3(1u << words.log), dim3(SORT_THREADS), smem, s, p, (int)n, (int)V, words,
               pad, start, order, word);
  };
  if (ids64) sort(reinterpret_cast<const int64_t*>(ids));
  else sort(reinterpret_cast<const int32_t*>(ids));
  DLVK_POST_LAUNCH();
  const float* gf = reinterpret_cast<const float*>(dy);
  const __nv_bfloat16* gb = reinterpret_cast<const __nv_bfloat16*>(dy);
  if (f32 && vec) sums<float, 4>(gf, ld, start, order, word, dtable, part, n, words, (int)V, D, scale, accumulate, s);
  else if (f32) sums<float, 1>(gf, ld, start, order, word, dtable, part, n, words, (int)V, D, scale, accumulate, s);
  else if (vec)
    sums<__nv_bfloat16, 8>(gb, ld, start, order, word, dtable, part, n, words, (int)V, D, scale, accumulate, s);
  else sums<__nv_bfloat16, 1>(gb, ld, start, order, word, dtable, part, n, words, (int)V, D, scale, accumulate, s);
}

}  // namespace dlvk
