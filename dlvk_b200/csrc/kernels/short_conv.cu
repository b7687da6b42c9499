// Causal depthwise convolution over a few tokens, channels last, with SiLU:
// forward from a state (the tokens before the first), the state after the last
// token, and the backward pass.
//
//   p[t, d] = bias[d] + sum_j w[d, j] x[t - K + 1 + j, d]        y = silu(p) = p / (1 + e^-p)
//   g = dy silu'(p)     dx[t] = sum_j w[j] g[t + K - 1 - j]      dw[j] = sum_t g[t] x[t - K + 1 + j]
//
// A thread walks a run of tokens of some neighbouring channels with the last
// K - 1 tokens in registers, so each element is read once and the K - 1 tokens
// before a run again.  The backward pass makes p again from x (cheaper than
// keeping it: K multiplications against a read and a write) and walks K - 1
// tokens past its run for the g that its dx needs.  dw and db are summed by
// thread, by block and over the blocks in a fixed order, without atomics.
//
// Their floor is the bytes of x, y, dy and dx (16 x 512 x 2048 bf16: 10 us forward, 15
// backward at the copy rate).  They take 20-22 and 32 us: a thread's own part of a
// token, address, copy, wait and store, is half of the instructions, issue slots are
// 55-60% busy, and the registers of longer runs or wider threads (eight channels: the
// taps alone are 32) leave too few warps to hide the memory's latency.
#include <algorithm>
#include <type_traits>

#include "dlvk/seq.h"

namespace dlvk {
namespace {

constexpr int RUNS = 8;    // runs of a block, a warp each

template <typename T, int V> struct Pack;  // V elements as loaded
template <> struct Pack<float, 4> { using type = float4; };
template <> struct Pack<float, 1> { using type = float; };
template <> struct Pack<__nv_bfloat16, 4> { using type = uint2; };
template <> struct Pack<__nv_bfloat16, 1> { using type = __nv_bfloat16; };

// V neighbouring channels of a token, in pairs (a single one is half a pair).
template <typename T, int V>
struct Vec {
  static constexpr int PAIRS = (V + 1) / 2;
  typename Pack<T, V>::type raw;
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const typename Pack<T, V>::type*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<typename Pack<T, V>::type*>(p) = raw; }
  __device__ __forceinline__ f2 get(int i) const {
    const T* e = reinterpret_cast<const T*>(&raw);
    if constexpr (V == 1) return pack(to_f32(e[0]), 0.f);
    else return pack(to_f32(e[2 * i]), to_f32(e[2 * i + 1]));
  }
  __device__ __forceinline__ void set(int i, f2 v) {
    const float2 f = unpack(v);
    T* e = reinterpret_cast<T*>(&raw);
    if constexpr (V == 1) e[0] = from_f32<T>(f.x);
    else if constexpr (sizeof(T) == 2) reinterpret_cast<__nv_bfloat162*>(&raw)[i] = __floats2bfloat162_rn(f.x, f.y);
    else e[2 * i] = f.x, e[2 * i + 1] = f.y;
  }
};

template <int V, int K>
__device__ __forceinline__ void load_taps(const ShortConv& a, int c, f2 (&w)[(V + 1) / 2][K], f2 (&bias)[(V + 1) / 2]) {
  float flat[2 * K * ((V + 1) / 2)], b[V + V % 2];
  if constexpr (V > 1) {  // whole aligned fours
#pragma unroll
    for (int i = 0; i < V * K; i += 4)
      *reinterpret_cast<float4*>(&flat[i]) = *reinterpret_cast<const float4*>(a.weight + (int64_t)c * K + i);
  } else {
#pragma unroll
    for (int i = 0; i < K; ++i) flat[i] = a.weight[(int64_t)c * K + i], flat[K + i] = 0.f;
    b[1] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) b[i] = a.bias ? a.bias[c + i] : 0.f;
#pragma unroll
  for (int i = 0; i < (V + 1) / 2; ++i) {
#pragma unroll
    for (int j = 0; j < K; ++j) w[i][j] = pack(flat[2 * i * K + j], flat[(2 * i + 1) * K + j]);
    bias[i] = pack(b[2 * i], b[2 * i + 1]);
  }
}

// The work's division: `run` tokens of a sequence and 32 V channels a warp.
struct Grid {
  int64_t runs, run, rows;  // runs of a sequence; rows of blocks
  int blocks;               // blocks of a row
};
struct Place {  // of a thread: sequence, tokens [t, end), first channel
  int64_t b, t, end;
  int c;
  bool ok;
};
template <int V>
__device__ __forceinline__ Place place(const ShortConv& a, const Grid& g) {
  const int64_t q = (int64_t)(blockIdx.x / g.blocks) * RUNS + threadIdx.y;
  Place p;
  p.b = q / g.runs;
  p.t = q % g.runs * g.run;
  p.end = min(p.t + g.run, a.T);
  p.c = ((int)(blockIdx.x % g.blocks) * 32 + threadIdx.x) * V;
  p.ok = p.b < a.B && p.c < a.D;
  return p;
}

__device__ __forceinline__ int64_t length_of(const ShortConv& a, int64_t b) {
  return a.lengths ? min(max((int64_t)a.lengths[b], (int64_t)0), a.T) : a.T;
}

// Token t of a sequence of n that counts, or of the tokens before it, or zeros:
// always one load, of the taps where there is no such token (a branch around a
// load would make the next one wait for it).
template <typename T, int V, int K>
__device__ __forceinline__ void token(const ShortConv& a, const Place& p, int64_t t, int64_t n, f2 (&x)[(V + 1) / 2]) {
  const bool here = t >= 0 ? t < n : a.state.p != nullptr;
  Vec<T, V> v;
  v.load(!here ? reinterpret_cast<const T*>(a.weight) : t >= 0 ? at<T>(a.x, p.b, t, p.c) : at<T>(a.state, p.b, t + K - 1, p.c));
#pragma unroll
  for (int i = 0; i < (V + 1) / 2; ++i) x[i] = here ? v.get(i) : 0;
}

// Tokens t to t + COUNT of r, zeros past the sequence's n: copied to a place in
// shared memory that this thread alone reads; single elements are loaded.
template <typename T, int V, int COUNT>
struct Ahead {
  Vec<T, V> v[COUNT][32 * RUNS];
  __device__ __forceinline__ void fetch(const SeqRef& r, const Place& p, int64_t t, int64_t n) {
    const int me = threadIdx.y * 32 + threadIdx.x;
#pragma unroll
    for (int k = 0; k < COUNT; ++k) {
      const bool here = t + k < n;
      if constexpr (V * sizeof(T) >= 4) copy_async<V * sizeof(T)>(&v[k][me], here ? at<T>(r, p.b, t + k, p.c) : r.p, here);
      else v[k][me].raw = here ? *at<T>(r, p.b, t + k, p.c) : from_f32<T>(0.f);
    }
  }
  __device__ __forceinline__ const Vec<T, V>& operator[](int k) const { return v[k][threadIdx.y * 32 + threadIdx.x]; }
};

template <typename T, int V>
struct FwdShared {
  static constexpr int AHEAD = 8;
  Ahead<T, V, AHEAD> x[2];
};

// Two batches of eight tokens on their way to a thread at a time.  Loads into registers ahead of use, without
// shared memory between, took 30 us for the above.
template <typename T, int V, int K>
__global__ void __launch_bounds__(32 * RUNS, 3) conv_fwd_kernel(ShortConv a, SeqRef y, SeqRef out_state, Grid grid) {
  constexpr int AHEAD = FwdShared<T, V>::AHEAD;
  extern __shared__ __align__(16) char raw[];
  auto& sh = *reinterpret_cast<FwdShared<T, V>*>(raw);
  const Place p = place<V>(a, grid);
  if (!p.ok) return;
  const int64_t n = length_of(a, p.b), stop = min(p.end, n);  // tokens of the run that count
  if (p.t < stop) sh.x[0].fetch(a.x, p, p.t, stop);
  copies_issued();
  constexpr int P = Vec<T, V>::PAIRS;
  f2 w[P][K], bias[P], last[K - 1][P];
  load_taps<V, K>(a, p.c, w, bias);
#pragma unroll
  for (int j = 0; j < K - 1; ++j) token<T, V, K>(a, p, p.t - (K - 1) + j, n, last[j]);
  if (out_state.p && p.t == 0) {
    // read before any of it is written: out_state may be the state
    f2 keep[K - 1][P];
#pragma unroll
    for (int j = 0; j < K - 1; ++j) token<T, V, K>(a, p, n - (K - 1) + j, n, keep[j]);
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      Vec<T, V> o;
#pragma unroll
      for (int i = 0; i < P; ++i) o.set(i, keep[j][i]);
      o.store(at<T>(out_state, p.b, j, p.c));
    }
  }
  int now = 0;
  T* to = at<T>(y, p.b, p.t, p.c);
  for (int64_t t0 = p.t; t0 < p.end; t0 += AHEAD, now ^= 1) {
    if (t0 + AHEAD < stop) sh.x[now ^ 1].fetch(a.x, p, t0 + AHEAD, stop);
    copies_issued();
    wait_copies<1>();
    const int count = (int)min((int64_t)AHEAD, p.end - t0), real = (int)max((int64_t)0, min((int64_t)AHEAD, n - t0));
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (k >= count) break;
      const Vec<T, V> v = sh.x[now][k];
      Vec<T, V> out;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const f2 x = v.get(i);
        f2 s = fma2(w[i][K - 1], x, bias[i]);
#pragma unroll
        for (int j = 0; j < K - 1; ++j) s = fma2(w[i][j], last[j][i], s);
#pragma unroll
        for (int j = 0; j < K - 2; ++j) last[j][i] = last[j + 1][i];
        last[K - 2][i] = x;
        if (a.silu) s = mul2(s, sigmoid_2(s));
        out.set(i, k < real ? s : 0);
      }
      out.store(to);
      to += y.token;
    }
  }
}

template <typename T, int V>
struct BwdShared {
  static constexpr int AHEAD = 4, STAGES = 3;
  Ahead<T, V, AHEAD> x[STAGES], g[STAGES];
  float sums[RUNS][32 * V + 1];
};

// part [block rows][K + 1][D]: the sums of a block's runs, bias last.
template <typename T, int V, int K>
__global__ void __launch_bounds__(32 * RUNS, 2) conv_bwd_kernel(ShortConv a, SeqRef dy, SeqRef dx, float* __restrict__ part,
                                                                Grid grid) {
  constexpr int AHEAD = BwdShared<T, V>::AHEAD, STAGES = BwdShared<T, V>::STAGES;
  extern __shared__ __align__(16) char raw[];
  auto& sh = *reinterpret_cast<BwdShared<T, V>*>(raw);
  constexpr int P = Vec<T, V>::PAIRS;
  const Place p = place<V>(a, grid);
  f2 dw[P][K + 1];
#pragma unroll
  for (int i = 0; i < P; ++i)
#pragma unroll
    for (int j = 0; j <= K; ++j) dw[i][j] = 0;
  if (p.ok) {
    const int64_t n = length_of(a, p.b);
    const int64_t past = p.end + K - 1, stop = min(past, n);  // the tokens behind the run for their g alone
    const auto fetch = [&](int64_t t, int stage) {
      if (t < stop) {
        sh.x[stage].fetch(a.x, p, t, stop);
        sh.g[stage].fetch(dy, p, t, stop);
      }
      copies_issued();
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) fetch(p.t + i * AHEAD, i);
    f2 w[P][K], bias[P], x[K - 1 + AHEAD][P], g[K - 1 + AHEAD][P];  // the last K - 1 tokens first
    load_taps<V, K>(a, p.c, w, bias);
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      token<T, V, K>(a, p, p.t - (K - 1) + j, n, x[j]);
#pragma unroll
      for (int i = 0; i < P; ++i) g[j][i] = 0;
    }
    const f2 one = pack(1.f, 1.f), minus = pack(-1.f, -1.f);
    int now = 0;
    T* to = at<T>(dx, p.b, p.t - (K - 1), p.c);
    // AHEAD tokens from t0 on; EDGE: not all of them are the run's own, count, and lie behind its first K - 1
    const auto walk = [&](int64_t t0, auto edge) {
      constexpr bool EDGE = decltype(edge)::value;
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int64_t t = t0 + k;
        const Vec<T, V> vx = sh.x[now][k], vg = sh.g[now][k];
        const bool here = !EDGE || t < stop;
        Vec<T, V> out;
#pragma unroll
        for (int i = 0; i < P; ++i) {
          x[K - 1 + k][i] = here ? vx.get(i) : 0;
          f2 gi = vg.get(i);
          if (a.silu) {
            f2 s = bias[i];
#pragma unroll
            for (int j = 0; j < K; ++j) s = fma2(w[i][j], x[k + j][i], s);
            const f2 q = sigmoid_2(s);
            gi = mul2(gi, mul2(q, fma2(s, fma2(q, minus, one), one)));
          }
          gi = here ? gi : 0;
          g[K - 1 + k][i] = gi;
          const f2 own = !EDGE || t < p.end ? gi : 0;
#pragma unroll
          for (int j = 0; j < K; ++j) dw[i][j] = fma2(own, x[k + j][i], dw[i][j]);
          dw[i][K] = add2(dw[i][K], own);
          f2 d = mul2(w[i][0], g[K - 1 + k][i]);  // dx[t - K + 1] = sum_j w[j] g[t - j]
#pragma unroll
          for (int j = 1; j < K; ++j) d = fma2(w[i][j], g[K - 1 + k - j][i], d);
          out.set(i, d);
        }
        if (!EDGE || (t - (K - 1) >= p.t && t < past)) out.store(to);
        to += dx.token;
      }
    };
    for (int64_t t0 = p.t; t0 < past; t0 += AHEAD) {
      fetch(t0 + (STAGES - 1) * AHEAD, now == 0 ? STAGES - 1 : now - 1);
      wait_copies<STAGES - 1>();
      if (t0 > p.t && t0 + AHEAD <= min(stop, p.end)) walk(t0, std::false_type());
      else walk(t0, std::true_type());
#pragma unroll
      for (int j = 0; j < K - 1; ++j)
#pragma unroll
        for (int i = 0; i < P; ++i) x[j][i] = x[AHEAD + j][i], g[j][i] = g[AHEAD + j][i];
      now = now + 1 == STAGES ? 0 : now + 1;
    }
  }
  const int64_t row = blockIdx.x / grid.blocks;
#pragma unroll
  for (int j = 0; j <= K; ++j) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 d = unpack(dw[i / 2][j]);
      sh.sums[threadIdx.y][threadIdx.x * V + i] = i % 2 ? d.y : d.x;
    }
    __syncthreads();
    for (int c = threadIdx.y * 32 + threadIdx.x; c < 32 * V; c += 32 * RUNS) {
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < RUNS; ++r) s += sh.sums[r][c];
      const int d = (int)(blockIdx.x % grid.blocks) * 32 * V + c;
      if (d < a.D) part[(row * (K + 1) + j) * a.D + d] = s;
    }
  }
}

// dweight[d, j] (and dbias) = the sum of part[:, j, d] in ascending rows, eight threads a sum.
__global__ void __launch_bounds__(256) conv_join_kernel(const float* __restrict__ part, int64_t rows, int D, int taps,
                                                        float* __restrict__ dweight, float* __restrict__ dbias,
                                                        bool accumulate) {
  __shared__ float sums[8][33];
  const int64_t total = (int64_t)(taps + 1) * D, e = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (e < total)
    for (int64_t r = threadIdx.y; r < rows; r += 8) s += part[r * total + e];
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y || e >= total) return;
  s = 0.f;
#pragma unroll
  for (int r = 0; r < 8; ++r) s += sums[r][threadIdx.x];
  const int j = (int)(e / D), d = (int)(e % D);
  float* out = j < taps ? (dweight ? dweight + (int64_t)d * taps + j : nullptr) : (dbias ? dbias + d : nullptr);
  if (out) *out = accumulate ? *out + s : s;
}

// Whether `v` neighbouring elements are one load.
bool aligned(const SeqRef& r, int v, int64_t bytes) {
  return !r.p || (reinterpret_cast<uintptr_t>(r.p) % (v * bytes) == 0 && r.batch % v == 0 && r.token % v == 0);
}
bool aligned(const ShortConv& a, int v) {
  const int64_t bytes = a.dt == DType::BF16 ? 2 : 4;
  return a.D % v == 0 && reinterpret_cast<uintptr_t>(a.weight) % 16 == 0 && aligned(a.x, v, bytes) &&
         aligned(a.state, v, bytes);
}

// As many runs as there are warps on the GPU at once, each of at least eight
// tokens: a run reads K - 1 tokens again, and the taps.
Grid grid_of(const ShortConv& a, int v, int blocks_an_sm) {
  Grid g;
  g.blocks = (a.D + 32 * v - 1) / (32 * v);
  const int64_t fit = std::max<int64_t>(1, 148 * blocks_an_sm * RUNS / std::max<int64_t>(1, a.B * g.blocks));
  g.run = std::max<int64_t>(8, (a.T + fit - 1) / fit);
  g.runs = std::max<int64_t>(1, (a.T + g.run - 1) / g.run);
  g.rows = (a.B * g.runs + RUNS - 1) / RUNS;
  DLVK_CHECK(g.rows * g.blocks < (1LL << 31), "short_conv: too many elements for one launch");
  return g;
}
template <typename Kernel, typename... Args>
void launch(Kernel kernel, size_t smem, const Grid& g, cudaStream_t s, Args... args) {
  if (smem > 48 * 1024)
    DLVK_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  kernel<<<(unsigned)(g.rows * g.blocks), dim3(32, RUNS), smem, s>>>(args..., g);
  DLVK_POST_LAUNCH();
}
constexpr int FWD_BLOCKS = 3, BWD_BLOCKS = 2;  // an SM holds; of bf16 too a thread has only four channels, and more registers
constexpr int VEC = 4;

template <typename F>
void by_taps(int taps, F&& f) {
  switch (taps) {
    case 2: f(std::integral_constant<int, 2>()); break;
    case 3: f(std::integral_constant<int, 3>()); break;
    case 4: f(std::integral_constant<int, 4>()); break;
    default: DLVK_CHECK(false, "short_conv: 2 to 4 taps");
  }
}

}  // namespace

void short_conv_fwd(const ShortConv& a, SeqRef y, SeqRef out_state, cudaStream_t s) {
  DLVK_CHECK(a.dt == DType::BF16 || a.dt == DType::F32, "short_conv: fp32 or bf16");
  // without tokens there is a state to copy, or nothing to do
  if (a.B == 0 || a.D == 0 || (a.T == 0 && !out_state.p)) return;
  const int64_t bytes = a.dt == DType::BF16 ? 2 : 4;
  const bool wide = aligned(a, VEC) && aligned(y, VEC, bytes) && aligned(out_state, VEC, bytes);
  const Grid g = grid_of(a, wide ? VEC : 1, FWD_BLOCKS);
  by_taps(a.taps, [&](auto taps) {
    constexpr int K = decltype(taps)::value;
    using bf16 = __nv_bfloat16;
    if (a.dt == DType::BF16) {
      if (wide) launch(conv_fwd_kernel<bf16, VEC, K>, sizeof(FwdShared<bf16, VEC>), g, s, a, y, out_state);
      else launch(conv_fwd_kernel<bf16, 1, K>, sizeof(FwdShared<bf16, 1>), g, s, a, y, out_state);
    } else {
      if (wide) launch(conv_fwd_kernel<float, VEC, K>, sizeof(FwdShared<float, VEC>), g, s, a, y, out_state);
      else launch(conv_fwd_kernel<float, 1, K>, sizeof(FwdShared<float, 1>), g, s, a, y, out_state);
    }
  });
}

namespace {
bool wide_bwd(const ShortConv& a, const SeqRef& dy, const SeqRef& dx) {
  const int64_t bytes = a.dt == DType::BF16 ? 2 : 4;
  return aligned(a, VEC) && aligned(dy, VEC, bytes) && aligned(dx, VEC, bytes);
}
}  // namespace

// The larger of the two ways to divide the channels.
int64_t short_conv_part_floats(const ShortConv& a) {
  return std::max(grid_of(a, VEC, BWD_BLOCKS).rows, grid_of(a, 1, BWD_BLOCKS).rows) * (a.taps + 1) * a.D;
}

void short_conv_bwd(const ShortConv& a, SeqRef dy, SeqRef dx, float* dweight, float* dbias, bool accumulate, float* part,
                    cudaStream_t s) {
  DLVK_CHECK(a.dt == DType::BF16 || a.dt == DType::F32, "short_conv: fp32 or bf16");
  if (a.D == 0) return;
  int64_t rows = 0;
  if (a.B > 0 && a.T > 0) {
    const bool wide = wide_bwd(a, dy, dx);
    const Grid g = grid_of(a, wide ? VEC : 1, BWD_BLOCKS);
    rows = g.rows;
    by_taps(a.taps, [&](auto taps) {
      constexpr int K = decltype(taps)::value;
      using bf16 = __nv_bfloat16;
      if (a.dt == DType::BF16) {
        if (wide) launch(conv_bwd_kernel<bf16, VEC, K>, sizeof(BwdShared<bf16, VEC>), g, s, a, dy, dx, part);
        else launch(conv_bwd_kernel<bf16, 1, K>, sizeof(BwdShared<bf16, 1>), g, s, a, dy, dx, part);
      } else {
        if (wide) launch(conv_bwd_kernel<float, VEC, K>, sizeof(BwdShared<float, VEC>), g, s, a, dy, dx, part);
        else launch(conv_bwd_kernel<float, 1, K>, sizeof(BwdShared<float, 1>), g, s, a, dy, dx, part);
      }
    });
  }
  conv_join_kernel<<<(unsigned)(((int64_t)(a.taps + 1) * a.D + 31) / 32), dim3(32, 8), 0, s>>>(
      part, rows, a.D, a.taps, dweight, dbias, accumulate);
  DLVK_POST_LAUNCH();
}

}  // namespace dlvk
