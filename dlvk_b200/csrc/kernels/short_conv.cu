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
// What bounds both: the bytes of x, y, dy and dx.
#include <algorithm>
#include <type_traits>

#include "dlvk/common.h"
#include "dlvk/kernels.h"

namespace dlvk {
namespace {

constexpr int RUN = 16;    // tokens of a thread: 3 of 19 reads come twice (K = 4)
constexpr int RUNS = 8;    // runs of a block, a warp each
constexpr int AHEAD = 8;   // tokens whose loads are in flight

template <typename T, int V> struct Pack;  // V elements as loaded
template <> struct Pack<float, 4> { using type = float4; };
template <> struct Pack<float, 1> { using type = float; };
template <> struct Pack<__nv_bfloat16, 8> { using type = uint4; };
template <> struct Pack<__nv_bfloat16, 1> { using type = __nv_bfloat16; };

template <typename T, int V>
struct Vec {
  typename Pack<T, V>::type raw;
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const typename Pack<T, V>::type*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<typename Pack<T, V>::type*>(p) = raw; }
  __device__ __forceinline__ void zero() {
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = from_f32<T>(0.f);
  }
  __device__ __forceinline__ float get(int i) const { return to_f32(reinterpret_cast<const T*>(&raw)[i]); }
  __device__ __forceinline__ void set(int i, float v) { reinterpret_cast<T*>(&raw)[i] = from_f32<T>(v); }
};

__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

template <typename T>
__device__ __forceinline__ T* at(const SeqRef& r, int64_t b, int64_t t, int c) {
  return static_cast<T*>(r.p) + b * r.batch + t * r.token + c;
}

template <int V, int K>
__device__ __forceinline__ void load_taps(const ShortConv& a, int c, float (&w)[V][K], float (&bias)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int j = 0; j < K; ++j) w[i][j] = a.weight[(int64_t)(c + i) * K + j];
    bias[i] = a.bias ? a.bias[c + i] : 0.f;
  }
}

// The place of a thread: sequence, first token and first channel of its run.
struct Place {
  int64_t b, t;
  int c;
  bool ok;
};
template <int V>
__device__ __forceinline__ Place place(const ShortConv& a, int64_t runs, int64_t row) {
  const int blocks = (a.D + 32 * V - 1) / (32 * V);
  const int64_t q = row * RUNS + threadIdx.y;
  Place p;
  p.b = q / runs;
  p.t = (q % runs) * RUN;
  p.c = ((int)(blockIdx.x % blocks) * 32 + threadIdx.x) * V;
  p.ok = p.b < a.B && p.c < a.D;
  return p;
}

__device__ __forceinline__ int64_t length_of(const ShortConv& a, int64_t b) {
  return a.lengths ? min(max((int64_t)a.lengths[b], (int64_t)0), a.T) : a.T;
}

// Token t of a sequence of n that counts, or of the tokens before it, or zeros.
template <typename T, int V, int K>
__device__ __forceinline__ Vec<T, V> token(const ShortConv& a, const Place& p, int64_t t, int64_t n) {
  Vec<T, V> v;
  if (t >= 0 && t < n) v.load(at<T>(a.x, p.b, t, p.c));
  else if (t < 0 && a.state.p) v.load(at<T>(a.state, p.b, t + K - 1, p.c));
  else v.zero();
  return v;
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(32 * RUNS) conv_fwd_kernel(ShortConv a, SeqRef y, SeqRef out_state, int64_t runs) {
  const int blocks = (a.D + 32 * V - 1) / (32 * V);
  const Place p = place<V>(a, runs, blockIdx.x / blocks);
  if (!p.ok) return;
  const int64_t n = length_of(a, p.b);
  float w[V][K], bias[V], last[K - 1][V];
  load_taps<V, K>(a, p.c, w, bias);
#pragma unroll
  for (int j = 0; j < K - 1; ++j) {
    const Vec<T, V> v = token<T, V, K>(a, p, p.t - (K - 1) + j, n);
#pragma unroll
    for (int i = 0; i < V; ++i) last[j][i] = v.get(i);
  }
  if (out_state.p && p.t == 0) {
    // read before any of it is written: out_state may be the state
    Vec<T, V> keep[K - 1];
#pragma unroll
    for (int j = 0; j < K - 1; ++j) keep[j] = token<T, V, K>(a, p, n - (K - 1) + j, n);
#pragma unroll
    for (int j = 0; j < K - 1; ++j) keep[j].store(at<T>(out_state, p.b, j, p.c));
  }
  for (int64_t t0 = p.t; t0 < min(p.t + RUN, a.T); t0 += AHEAD) {
    Vec<T, V> v[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      v[k].zero();
      if (t0 + k < n) v[k].load(at<T>(a.x, p.b, t0 + k, p.c));
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (t0 + k >= a.T) break;
      Vec<T, V> out;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float x = v[k].get(i);
        float s = fmaf(w[i][K - 1], x, bias[i]);
#pragma unroll
        for (int j = 0; j < K - 1; ++j) s = fmaf(w[i][j], last[j][i], s);
#pragma unroll
        for (int j = 0; j < K - 2; ++j) last[j][i] = last[j + 1][i];
        last[K - 2][i] = x;
        if (a.silu) s *= sigmoid(s);
        out.set(i, t0 + k < n ? s : 0.f);
      }
      out.store(at<T>(y, p.b, t0 + k, p.c));
    }
  }
}

// part [block rows][K + 1][D]: the sums of a block's runs, bias last.
template <typename T, int V, int K>
__global__ void __launch_bounds__(32 * RUNS) conv_bwd_kernel(ShortConv a, SeqRef dy, SeqRef dx, float* __restrict__ part,
                                                             int64_t runs) {
  const int blocks = (a.D + 32 * V - 1) / (32 * V);
  const int64_t row = blockIdx.x / blocks;
  const Place p = place<V>(a, runs, row);
  float dw[V][K + 1];
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j <= K; ++j) dw[i][j] = 0.f;
  if (p.ok) {
    const int64_t n = length_of(a, p.b);
    float w[V][K], bias[V], x[K][V], g[K][V];  // the last K tokens of each, the current one at K - 1
    load_taps<V, K>(a, p.c, w, bias);
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      const Vec<T, V> v = token<T, V, K>(a, p, p.t - (K - 1) + j, n);
#pragma unroll
      for (int i = 0; i < V; ++i) x[j + 1][i] = v.get(i), g[j + 1][i] = 0.f;
    }
    const int64_t end = min(p.t + RUN, a.T);
    for (int64_t t = p.t; t < end + K - 1; ++t) {
      Vec<T, V> vx, vg;
      vx.zero();
      vg.zero();
      if (t < n) {
        vx.load(at<T>(a.x, p.b, t, p.c));
        vg.load(at<T>(dy, p.b, t, p.c));
      }
      Vec<T, V> out;
#pragma unroll
      for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int j = 0; j < K - 1; ++j) x[j][i] = x[j + 1][i], g[j][i] = g[j + 1][i];
        x[K - 1][i] = vx.get(i);
        float gi = vg.get(i);
        if (a.silu) {
          float s = bias[i];
#pragma unroll
          for (int j = 0; j < K; ++j) s = fmaf(w[i][j], x[j][i], s);
          const float q = sigmoid(s);
          gi *= t < n ? q * fmaf(s, 1.f - q, 1.f) : 0.f;
        }
        g[K - 1][i] = gi;
        if (t < end) {
#pragma unroll
          for (int j = 0; j < K; ++j) dw[i][j] = fmaf(gi, x[j][i], dw[i][j]);
          dw[i][K] += gi;
        }
        float d = 0.f;  // dx[t - K + 1] = sum_j w[j] g[t - j]
#pragma unroll
        for (int j = 0; j < K; ++j) d = fmaf(w[i][j], g[K - 1 - j][i], d);
        out.set(i, d);
      }
      if (t - (K - 1) >= p.t) out.store(at<T>(dx, p.b, t - (K - 1), p.c));
    }
  }
  __shared__ float sums[RUNS][32 * V + 1];
#pragma unroll
  for (int j = 0; j <= K; ++j) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) sums[threadIdx.y][threadIdx.x * V + i] = dw[i][j];
    __syncthreads();
    for (int c = threadIdx.y * 32 + threadIdx.x; c < 32 * V; c += 32 * RUNS) {
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < RUNS; ++r) s += sums[r][c];
      const int d = (int)(blockIdx.x % blocks) * 32 * V + c;
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

bool aligned(const SeqRef& r, int64_t bytes) {
  return !r.p || (reinterpret_cast<uintptr_t>(r.p) % 16 == 0 && r.batch * bytes % 16 == 0 && r.token * bytes % 16 == 0);
}

int64_t run_rows(const ShortConv& a) {  // rows of blocks
  return (a.B * ((a.T + RUN - 1) / RUN) + RUNS - 1) / RUNS;
}

template <typename F>
void by_taps(int taps, F&& f) {
  switch (taps) {
    case 2: f(std::integral_constant<int, 2>()); break;
    case 3: f(std::integral_constant<int, 3>()); break;
    case 4: f(std::integral_constant<int, 4>()); break;
    default: DLVK_CHECK(false, "short_conv: 2 to 4 taps");
  }
}

// f(element type, channels of a thread): 16 bytes, or one element where the rows do not allow it.
template <typename F>
void by_type(DType dt, bool wide, F&& f) {
  if (dt == DType::BF16) {
    if (wide) f(__nv_bfloat16(), std::integral_constant<int, 8>());
    else f(__nv_bfloat16(), std::integral_constant<int, 1>());
  } else {
    DLVK_CHECK(dt == DType::F32, "short_conv: fp32 or bf16");
    if (wide) f(float(), std::integral_constant<int, 4>());
    else f(float(), std::integral_constant<int, 1>());
  }
}

unsigned grid_of(const ShortConv& a, int v) {
  const int64_t g = run_rows(a) * ((a.D + 32 * v - 1) / (32 * v));
  DLVK_CHECK(g < (1LL << 31), "short_conv: too many elements for one launch");
  return (unsigned)g;
}

}  // namespace

void short_conv_fwd(const ShortConv& a, SeqRef y, SeqRef out_state, cudaStream_t s) {
  if (a.B == 0 || a.D == 0) return;
  // a state without tokens is copied by the same kernel: one run
  const int64_t bytes = a.dt == DType::BF16 ? 2 : 4, runs = std::max<int64_t>(1, (a.T + RUN - 1) / RUN);
  if (a.T == 0 && !out_state.p) return;
  const bool wide = a.D % (16 / bytes) == 0 && aligned(a.x, bytes) && aligned(a.state, bytes) && aligned(y, bytes) &&
                    aligned(out_state, bytes);
  ShortConv k = a;
  if (a.T == 0) k.x = a.state;  // never read
  by_type(a.dt, wide, [&](auto type, auto vec) {
    by_taps(a.taps, [&](auto taps) {
      const int64_t rows = (a.B * runs + RUNS - 1) / RUNS, g = rows * ((a.D + 32 * vec - 1) / (32 * vec));
      DLVK_CHECK(g < (1LL << 31), "short_conv: too many elements for one launch");
      conv_fwd_kernel<decltype(type), decltype(vec)::value, decltype(taps)::value>
          <<<(unsigned)g, dim3(32, RUNS), 0, s>>>(k, y, out_state, runs);
    });
  });
  DLVK_POST_LAUNCH();
}

int64_t short_conv_part_floats(const ShortConv& a) { return run_rows(a) * (a.taps + 1) * a.D; }

void short_conv_bwd(const ShortConv& a, SeqRef dy, SeqRef dx, float* dweight, float* dbias, bool accumulate, float* part,
                    cudaStream_t s) {
  if (a.D == 0) return;
  const int64_t bytes = a.dt == DType::BF16 ? 2 : 4, rows = run_rows(a);
  if (rows > 0) {
    const bool wide = a.D % (16 / bytes) == 0 && aligned(a.x, bytes) && aligned(a.state, bytes) && aligned(dy, bytes) &&
                      aligned(dx, bytes);
    by_type(a.dt, wide, [&](auto type, auto vec) {
      by_taps(a.taps, [&](auto taps) {
        conv_bwd_kernel<decltype(type), decltype(vec)::value, decltype(taps)::value>
            <<<grid_of(a, vec), dim3(32, RUNS), 0, s>>>(a, dy, dx, part, (a.T + RUN - 1) / RUN);
      });
    });
    DLVK_POST_LAUNCH();
  }
  conv_join_kernel<<<(unsigned)(((int64_t)(a.taps + 1) * a.D + 31) / 32), dim3(32, 8), 0, s>>>(
      part, rows, a.D, a.taps, dweight, dbias, accumulate);
  DLVK_POST_LAUNCH();
}

}  // namespace dlvk
