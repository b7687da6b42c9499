// Selective state space scan, channels last: forward from a state, the state
// after the last token, single tokens, and the backward pass.
//
//   s = softplus(dt + dt_bias)    A = -exp(a_log)    a[t, n] = exp(s A)
//   h[t] = a[t] h[t-1] + s u b[t]                    p = sum_n c[t] h[t] + skip u
//   y = p silu(z)
// Backward, q = dy silu(z):
//   g[t] = c[t] q + a[t+1] g[t+1]                    dc[t] = sum_d q h[t]     db[t] = sum_d g s u
//   v = sum_n g b                                    du = v s + q skip        dz = dy p silu'(z)
//   ds = sum_n g a[t] h[t-1] A + v u                 ddt = ds sigmoid(dt + dt_bias)
//   da_log = A sum_t g a[t] h[t-1] s                 dskip = sum q u          ddt_bias = sum ddt
//
// A block owns some channels of one sequence and walks its tokens span by
// span.  What is one value a token and channel (softplus, gates) is made by all
// threads together before a span and after it; the scan between them gives each
// thread four states of a channel, which stay in its registers, so a channel of
// N states has N / 4 lanes and sums over states cross lanes by shuffles.
#include <algorithm>
#include <type_traits>

#include "dlvk/common.h"
#include "dlvk/kernels.h"

namespace dlvk {
namespace {

constexpr int THREADS = 128;
constexpr int NS = 4;  // states of a thread
constexpr int SPAN = STATE_SCAN_SPAN;
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }
// steps are small, so log1p of a small number has to keep its relative precision
__device__ __forceinline__ float softplus(float x) { return x > 20.f ? x : log1pf(expf(x)); }

template <typename T, int V> struct Pack;
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

template <typename T>
__device__ __forceinline__ T* at(const SeqRef& r, int64_t b, int64_t t, int64_t c) {
  return static_cast<T*>(r.p) + b * r.batch + t * r.token + c;
}
__device__ __forceinline__ int64_t length_of(const StateScan& a, int64_t b) {
  return a.lengths ? min(max((int64_t)a.lengths[b], (int64_t)0), a.T) : a.T;
}

// The channels of a block: CH = THREADS / L of one group of one sequence.
template <int L>
struct Tile {
  static constexpr int CH = THREADS / L;
  int64_t b;
  int group, c0, count;  // first channel, channels of the tile that exist
  __device__ __forceinline__ explicit Tile(const StateScan& a) {
    const int per = a.D / a.G, tiles = (per + CH - 1) / CH;
    const int64_t i = blockIdx.x;
    const int k = (int)(i % ((int64_t)tiles * a.G));
    b = i / ((int64_t)tiles * a.G);
    group = k / tiles;
    c0 = group * per + k % tiles * CH;
    count = min(CH, per - k % tiles * CH);
  }
};

// Sums of v[0..M) over the lanes that differ in the bits FROM, 2 FROM, ... < TO,
// dealt out to them: on return v[0..dealt(M, FROM, TO)) are the sums of the values
// first.. of all M, and `mine` says whether this lane is the one to write them.
constexpr int dealt(int m, int from, int to) { return from >= to ? m : dealt(m > 1 ? m / 2 : 1, from * 2, to); }
template <int M, int FROM, int TO>
__device__ __forceinline__ void deal(float* v, int lane, int& first, bool& mine) {
  if constexpr (FROM < TO) {
    const bool up = lane & FROM;
    if constexpr (M > 1) {
#pragma unroll
      for (int i = 0; i < M / 2; ++i) {
        const float send = up ? v[i] : v[i + M / 2], keep = up ? v[i + M / 2] : v[i];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, send, FROM);
      }
      first += up ? M / 2 : 0;
      deal<M / 2, FROM * 2, TO>(v, lane, first, mine);
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], FROM);
      mine = mine && !up;
      deal<1, FROM * 2, TO>(v, lane, first, mine);
    }
  }
}

// b or c of a span to shared memory, rows of NS L states, zeros past N and past the tokens.
template <typename T, int L>
__device__ __forceinline__ void load_states(float (*dst)[NS * L], const SeqRef& r, int64_t b, int64_t t0, int64_t n,
                                            int group, int N) {
  for (int i = threadIdx.x; i < SPAN * NS * L; i += THREADS) {
    const int t = i / (NS * L), k = i % (NS * L);
    dst[t][k] = t0 + t < n && k < N ? to_f32(*at<T>(r, b, t0 + t, (int64_t)group * N + k)) : 0.f;
  }
}

__device__ __forceinline__ void load4(float (&h)[NS], const float* p, int n0, int N) {
#pragma unroll
  for (int i = 0; i < NS; ++i) h[i] = n0 + i < N ? p[i] : 0.f;
}
__device__ __forceinline__ void store4(const float (&h)[NS], float* p, int n0, int N) {
#pragma unroll
  for (int i = 0; i < NS; ++i)
    if (n0 + i < N) p[i] = h[i];
}

// ---------------------------------------------------------------- forward
template <typename T, int L, int V>
__global__ void __launch_bounds__(THREADS) scan_fwd_kernel(StateScan a, SeqRef y, float* out_state, float* saved) {
  using Tl = Tile<L>;
  constexpr int CH = Tl::CH, PER = (SPAN * CH / V + THREADS - 1) / THREADS;
  __shared__ float2 sx[SPAN][CH];   // s, s u
  __shared__ float sy[SPAN][CH];
  __shared__ float sb[SPAN][NS * L], sc[SPAN][NS * L];
  const Tl tile(a);
  const int lane = threadIdx.x % L, ch = threadIdx.x / L, n0 = lane * NS;
  const bool real = ch < tile.count;
  const int64_t n = length_of(a, tile.b);
  const int64_t row = (tile.b * a.D + tile.c0 + ch) * a.N + n0;  // of this thread's states
  float h[NS], rate[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) h[i] = rate[i] = 0.f;
  if (real) {
    if (a.state) load4(h, a.state + row, n0, a.N);
    load4(rate, a.a_log + (int64_t)(tile.c0 + ch) * a.N + n0, n0, a.N);
#pragma unroll
    for (int i = 0; i < NS; ++i) rate[i] = n0 + i < a.N ? -expf(rate[i]) * LOG2E : 0.f;
  }
  const int64_t spans = (a.T + SPAN - 1) / SPAN;
  for (int64_t k = 0; k < spans; ++k) {
    const int64_t t0 = k * SPAN;
    Vec<T, V> u[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = (threadIdx.x + i * THREADS) * V, t = e / CH, c = e % CH;
      if (t >= SPAN) break;
      Vec<T, V> dt;
      u[i].zero();
      const bool here = t0 + t < n && c < tile.count;
      if (here) {
        u[i].load(at<T>(a.u, tile.b, t0 + t, tile.c0 + c));
        dt.load(at<T>(a.dt, tile.b, t0 + t, tile.c0 + c));
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float s = here ? softplus(dt.get(j) + (a.dt_bias ? a.dt_bias[tile.c0 + c + j] : 0.f)) : 0.f;
        sx[t][c + j] = make_float2(s, s * u[i].get(j));
      }
    }
    load_states<T, L>(sb, a.b, tile.b, t0, n, tile.group, a.N);
    load_states<T, L>(sc, a.c, tile.b, t0, n, tile.group, a.N);
    __syncthreads();
    if (saved && real) store4(h, saved + ((tile.b * spans + k) * a.D + tile.c0 + ch) * a.N + n0, n0, a.N);
#pragma unroll
    for (int t = 0; t < SPAN; t += 4) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 x = sx[t + j][ch];
        const float4 bb = *reinterpret_cast<const float4*>(&sb[t + j][n0]);
        const float4 cc = *reinterpret_cast<const float4*>(&sc[t + j][n0]);
        h[0] = fmaf(ex2(x.x * rate[0]), h[0], x.y * bb.x);
        h[1] = fmaf(ex2(x.x * rate[1]), h[1], x.y * bb.y);
        h[2] = fmaf(ex2(x.x * rate[2]), h[2], x.y * bb.z);
        h[3] = fmaf(ex2(x.x * rate[3]), h[3], x.y * bb.w);
        v[j] = fmaf(cc.x, h[0], fmaf(cc.y, h[1], fmaf(cc.z, h[2], cc.w * h[3])));
      }
      int first = 0;
      bool mine = true;
      deal<4, 1, L>(v, threadIdx.x & 31, first, mine);
      if (mine) {
#pragma unroll
        for (int j = 0; j < dealt(4, 1, L); ++j) sy[t + first + j][ch] = v[j];
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = (threadIdx.x + i * THREADS) * V, t = e / CH, c = e % CH;
      if (t >= SPAN || t0 + t >= a.T || c >= tile.count) break;
      Vec<T, V> z, out;
      z.zero();
      if (a.z.p && t0 + t < n) z.load(at<T>(a.z, tile.b, t0 + t, tile.c0 + c));
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float p = sy[t][c + j];
        if (a.skip) p = fmaf(a.skip[tile.c0 + c + j], u[i].get(j), p);
        if (a.z.p) p *= z.get(j) * sigmoid(z.get(j));
        out.set(j, t0 + t < n ? p : 0.f);
      }
      out.store(at<T>(y, tile.b, t0 + t, tile.c0 + c));
    }
  }
  if (out_state && real) store4(h, out_state + row, n0, a.N);
}

// ---------------------------------------------------------------- backward
// part_bc [tiles of a group][B][T][G][2][N]; part_d [B][D][N + 2]: da, dskip, ddt_bias.
template <typename T, int L, int V>
__global__ void __launch_bounds__(THREADS) scan_bwd_kernel(StateScan a, const float* __restrict__ saved, SeqRef dy,
                                                           StateScanGrads g, float* __restrict__ part_bc,
                                                           float* __restrict__ part_d) {
  using Tl = Tile<L>;
  constexpr int CH = Tl::CH, PER = (SPAN * CH / V + THREADS - 1) / THREADS, WARPS = THREADS / 32;
  __shared__ float2 sx[SPAN][CH];         // s, s u
  __shared__ float sq[SPAN][CH];          // q
  __shared__ float sy[SPAN][CH];          // sum_n c h
  __shared__ float sv[SPAN][CH], sd[SPAN][CH];  // sum_n g b, sum_n g a h' A
  __shared__ float sb[SPAN][NS * L], sc[SPAN][NS * L];
  __shared__ float red[WARPS][SPAN][2 * NS * L];
  const Tl tile(a);
  const int lane = threadIdx.x % L, ch = threadIdx.x / L, n0 = lane * NS, warp = threadIdx.x / 32;
  const bool real = ch < tile.count;
  const int64_t n = length_of(a, tile.b), spans = (a.T + SPAN - 1) / SPAN;
  const int per = a.D / a.G, tile_of_group = (tile.c0 - tile.group * per) / CH;
  float rate[NS], ga[NS], da[NS], dskip[V], dbias[V];
#pragma unroll
  for (int i = 0; i < NS; ++i) rate[i] = ga[i] = da[i] = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) dskip[j] = dbias[j] = 0.f;
  if (real) {
    load4(rate, a.a_log + (int64_t)(tile.c0 + ch) * a.N + n0, n0, a.N);
#pragma unroll
    for (int i = 0; i < NS; ++i) rate[i] = n0 + i < a.N ? -expf(rate[i]) : 0.f;
  }
  for (int64_t k = spans - 1; k >= 0; --k) {
    const int64_t t0 = k * SPAN;
    Vec<T, V> u[PER], dt[PER], z[PER], go[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = (threadIdx.x + i * THREADS) * V, t = e / CH, c = e % CH;
      u[i].zero();
      dt[i].zero();
      z[i].zero();
      go[i].zero();
      if (t >= SPAN) break;
      const bool here = t0 + t < n && c < tile.count;
      if (here) {
        u[i].load(at<T>(a.u, tile.b, t0 + t, tile.c0 + c));
        dt[i].load(at<T>(a.dt, tile.b, t0 + t, tile.c0 + c));
        if (a.z.p) z[i].load(at<T>(a.z, tile.b, t0 + t, tile.c0 + c));
        go[i].load(at<T>(dy, tile.b, t0 + t, tile.c0 + c));
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float s = here ? softplus(dt[i].get(j) + (a.dt_bias ? a.dt_bias[tile.c0 + c + j] : 0.f)) : 0.f;
        sx[t][c + j] = make_float2(s, s * u[i].get(j));
        sq[t][c + j] = go[i].get(j) * (a.z.p ? z[i].get(j) * sigmoid(z[i].get(j)) : 1.f);
      }
    }
    load_states<T, L>(sb, a.b, tile.b, t0, n, tile.group, a.N);
    load_states<T, L>(sc, a.c, tile.b, t0, n, tile.group, a.N);
    float h[SPAN + 1][NS];  // h[t]: before token t of the span
#pragma unroll
    for (int i = 0; i < NS; ++i) h[0][i] = 0.f;
    if (real) load4(h[0], saved + ((tile.b * spans + k) * a.D + tile.c0 + ch) * a.N + n0, n0, a.N);
    __syncthreads();
#pragma unroll
    for (int t = 0; t < SPAN; t += 4) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 x = sx[t + j][ch];
        const float4 bb = *reinterpret_cast<const float4*>(&sb[t + j][n0]);
        const float4 cc = *reinterpret_cast<const float4*>(&sc[t + j][n0]);
        const float sl = x.x * LOG2E;
        h[t + j + 1][0] = fmaf(ex2(sl * rate[0]), h[t + j][0], x.y * bb.x);
        h[t + j + 1][1] = fmaf(ex2(sl * rate[1]), h[t + j][1], x.y * bb.y);
        h[t + j + 1][2] = fmaf(ex2(sl * rate[2]), h[t + j][2], x.y * bb.z);
        h[t + j + 1][3] = fmaf(ex2(sl * rate[3]), h[t + j][3], x.y * bb.w);
        v[j] = cc.x * h[t + j + 1][0] + cc.y * h[t + j + 1][1] + cc.z * h[t + j + 1][2] + cc.w * h[t + j + 1][3];
      }
      int first = 0;
      bool mine = true;
      deal<4, 1, L>(v, threadIdx.x & 31, first, mine);
      if (mine) {
#pragma unroll
        for (int j = 0; j < dealt(4, 1, L); ++j) sy[t + first + j][ch] = v[j];
      }
    }
#pragma unroll
    for (int t4 = SPAN - 4; t4 >= 0; t4 -= 4) {
      float sums[8];  // of four tokens: sum_n g b, sum_n g a h' A
#pragma unroll
      for (int j = 3; j >= 0; --j) {
        const int t = t4 + j;
        const float2 x = sx[t][ch];
        const float q = sq[t][ch], sl = x.x * LOG2E;
        float w[8];  // db and dc of this channel
        sums[2 * j] = sums[2 * j + 1] = 0.f;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          const float gi = fmaf(q, sc[t][n0 + i], ga[i]);
          w[i] = gi * x.y;
          w[NS + i] = q * h[t + 1][i];
          sums[2 * j] = fmaf(gi, sb[t][n0 + i], sums[2 * j]);
          ga[i] = gi * ex2(sl * rate[i]);
          const float through = ga[i] * h[t][i];
          sums[2 * j + 1] = fmaf(through, rate[i], sums[2 * j + 1]);
          da[i] = fmaf(through, x.x, da[i]);
        }
        int first = 0;
        bool mine = true;
        deal<8, L, 32>(w, threadIdx.x & 31, first, mine);
        if (mine) {
#pragma unroll
          for (int i = 0; i < dealt(8, L, 32); ++i) {
            const int e = first + i;  // < NS: db of state n0 + e
            red[warp][t][(e / NS) * NS * L + n0 + e % NS] = w[i];
          }
        }
      }
      int first = 0;
      bool mine = true;
      deal<8, 1, L>(sums, threadIdx.x & 31, first, mine);
      if (mine) {
#pragma unroll
        for (int i = 0; i < dealt(8, 1, L); ++i) {
          const int e = first + i;
          (e % 2 ? sd : sv)[t4 + e / 2][ch] = sums[i];
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = (threadIdx.x + i * THREADS) * V, t = e / CH, c = e % CH;
      if (t >= SPAN || t0 + t >= a.T || c >= tile.count) break;
      const bool here = t0 + t < n;
      Vec<T, V> du, ddt, dz;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int d = tile.c0 + c + j;
        const float uj = u[i].get(j), zj = z[i].get(j), sk = a.skip ? a.skip[d] : 0.f, q = sq[t][c + j];
        const float raw = dt[i].get(j) + (a.dt_bias ? a.dt_bias[d] : 0.f), v = sv[t][c + j];
        du.set(j, here ? fmaf(v, sx[t][c + j].x, q * sk) : 0.f);
        const float dr = here ? fmaf(v, uj, sd[t][c + j]) * sigmoid(raw) : 0.f;
        ddt.set(j, dr);
        dbias[j] += dr;
        dskip[j] = fmaf(q, uj, dskip[j]);
        if (a.z.p) {
          const float sz = sigmoid(zj);
          dz.set(j, here ? go[i].get(j) * fmaf(sk, uj, sy[t][c + j]) * sz * fmaf(zj, 1.f - sz, 1.f) : 0.f);
        }
      }
      du.store(at<T>(g.du, tile.b, t0 + t, tile.c0 + c));
      ddt.store(at<T>(g.ddt, tile.b, t0 + t, tile.c0 + c));
      if (a.z.p) dz.store(at<T>(g.dz, tile.b, t0 + t, tile.c0 + c));
    }
    for (int i = threadIdx.x; i < SPAN * 2 * NS * L; i += THREADS) {
      const int t = i / (2 * NS * L), e = i % (2 * NS * L), half = e / (NS * L), st = e % (NS * L);
      if (t0 + t >= a.T || st >= a.N) continue;
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) s += red[w][t][e];
      part_bc[((((tile_of_group * a.B + tile.b) * a.T + t0 + t) * a.G + tile.group) * 2 + half) * a.N + st] = s;
    }
    __syncthreads();
  }
  if (real) {
    float* out = part_d + (tile.b * a.D + tile.c0 + ch) * (a.N + 2);
#pragma unroll
    for (int i = 0; i < NS; ++i)
      if (n0 + i < a.N) out[n0 + i] = da[i] * rate[i];
  }
  // dskip and ddt_bias: threads CH / V apart hold the same channels
  constexpr int SAME = CH / V < THREADS ? CH / V : THREADS;
  float* buf = &sv[0][0];
  const int c = threadIdx.x * V % CH, rows = SPAN * CH / V < THREADS ? SPAN * CH / V : THREADS;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    __syncthreads();
    if (threadIdx.x < rows) {
#pragma unroll
      for (int j = 0; j < V; ++j) buf[threadIdx.x * V + j] = half ? dbias[j] : dskip[j];
    }
    __syncthreads();
    if (threadIdx.x < SAME) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float s = 0.f;
        for (int r = threadIdx.x; r < rows; r += SAME) s += buf[r * V + j];
        if (c + j < tile.count) part_d[(tile.b * a.D + tile.c0 + c + j) * (a.N + 2) + a.N + half] = s;
      }
    }
  }
}

// db and dc: the sums over a group's tiles, in their order.
template <typename T>
__global__ void __launch_bounds__(256) join_bc_kernel(const float* __restrict__ part, int tiles, int64_t B, int64_t T_,
                                                      int G, int N, SeqRef db, SeqRef dc) {
  const int64_t row = (int64_t)G * 2 * N, total = B * T_ * row;
  for (int64_t i = blockIdx.x * 256LL + threadIdx.x; i < total; i += 256LL * gridDim.x) {
    float s = 0.f;
    for (int k = 0; k < tiles; ++k) s += part[k * total + i];
    const int e = (int)(i % row), group = e / (2 * N), half = e / N % 2, n = e % N;
    const int64_t t = i / row % T_, b = i / row / T_;
    *at<T>(half ? dc : db, b, t, (int64_t)group * N + n) = from_f32<T>(s);
  }
}
// da_log, dskip and ddt_bias: the sums over the sequences.
__global__ void __launch_bounds__(256) join_d_kernel(const float* __restrict__ part, int64_t B, int D, int N,
                                                     StateScanGrads g) {
  const int64_t total = (int64_t)D * (N + 2), i = blockIdx.x * 256LL + threadIdx.x;
  if (i >= total) return;
  float s = 0.f;
  for (int64_t b = 0; b < B; ++b) s += part[b * total + i];
  const int64_t d = i / (N + 2);
  const int k = (int)(i % (N + 2));
  float* out = k < N ? (g.da_log ? g.da_log + d * N + k : nullptr)
                     : k == N ? (g.dskip ? g.dskip + d : nullptr) : (g.ddt_bias ? g.ddt_bias + d : nullptr);
  if (out) *out = g.accumulate ? *out + s : s;
}

bool aligned(const SeqRef& r, int64_t bytes) {
  return !r.p || (reinterpret_cast<uintptr_t>(r.p) % 16 == 0 && r.batch * bytes % 16 == 0 && r.token * bytes % 16 == 0);
}
int lanes_of(int N) { return N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }
int tiles_of(const StateScan& a) {  // of a group
  const int ch = THREADS / lanes_of(a.N);
  return (a.D / a.G + ch - 1) / ch;
}
template <typename F>
void by_lanes(int N, F&& f) {
  switch (lanes_of(N)) {
    case 2: f(std::integral_constant<int, 2>()); break;
    case 4: f(std::integral_constant<int, 4>()); break;
    case 8: f(std::integral_constant<int, 8>()); break;
    default: f(std::integral_constant<int, 16>());
  }
}
template <typename F>
void by_type(DType dt, bool wide, F&& f) {
  if (dt == DType::BF16) {
    if (wide) f(__nv_bfloat16(), std::integral_constant<int, 8>());
    else f(__nv_bfloat16(), std::integral_constant<int, 1>());
  } else {
    if (wide) f(float(), std::integral_constant<int, 4>());
    else f(float(), std::integral_constant<int, 1>());
  }
}
unsigned grid_of(const StateScan& a) {
  const int64_t g = a.B * a.G * tiles_of(a);
  DLVK_CHECK(g < (1LL << 31), "state_scan: too many channels for one launch");
  return (unsigned)g;
}
void check(const StateScan& a) {
  DLVK_CHECK(a.type == DType::BF16 || a.type == DType::F32, "state_scan: fp32 or bf16");
  DLVK_CHECK(a.N >= 1 && a.N <= STATE_SCAN_STATES, "state_scan: 1 to 64 states");
  DLVK_CHECK(a.G >= 1 && a.D % a.G == 0, "state_scan: channels of equal groups");
}

}  // namespace

void state_scan_fwd(const StateScan& a, SeqRef y, float* out_state, float* saved, cudaStream_t s) {
  check(a);
  if (a.B == 0 || a.D == 0) return;
  const int64_t bytes = a.type == DType::BF16 ? 2 : 4;
  const bool wide = a.D / a.G % (16 / bytes) == 0 && aligned(a.u, bytes) && aligned(a.dt, bytes) &&
                    aligned(a.z, bytes) && aligned(y, bytes);
  by_type(a.type, wide, [&](auto type, auto vec) {
    by_lanes(a.N, [&](auto lanes) {
      scan_fwd_kernel<decltype(type), decltype(lanes)::value, decltype(vec)::value>
          <<<grid_of(a), THREADS, 0, s>>>(a, y, out_state, saved);
    });
  });
  DLVK_POST_LAUNCH();
}

int64_t state_scan_scratch_floats(const StateScan& a) {
  check(a);
  return (int64_t)tiles_of(a) * a.B * a.T * a.G * 2 * a.N + a.B * a.D * (a.N + 2);
}

void state_scan_bwd(const StateScan& a, const float* saved, SeqRef dy, const StateScanGrads& g, float* scratch,
                    cudaStream_t s) {
  check(a);
  if (a.D == 0) return;
  const int64_t bytes = a.type == DType::BF16 ? 2 : 4;
  float* part_bc = scratch;
  float* part_d = scratch + (int64_t)tiles_of(a) * a.B * a.T * a.G * 2 * a.N;
  if (a.B > 0) {
    const bool wide = a.D / a.G % (16 / bytes) == 0 && aligned(a.u, bytes) && aligned(a.dt, bytes) &&
                      aligned(a.z, bytes) && aligned(dy, bytes) && aligned(g.du, bytes) && aligned(g.ddt, bytes) &&
                      aligned(g.dz, bytes);
    by_type(a.type, wide, [&](auto type, auto vec) {
      by_lanes(a.N, [&](auto lanes) {
        scan_bwd_kernel<decltype(type), decltype(lanes)::value, decltype(vec)::value>
            <<<grid_of(a), THREADS, 0, s>>>(a, saved, dy, g, part_bc, part_d);
      });
    });
    DLVK_POST_LAUNCH();
    const int64_t total = a.B * a.T * a.G * 2 * a.N;
    if (total > 0) {
      const unsigned blocks = (unsigned)std::min<int64_t>((total + 255) / 256, 148 * 16);
      if (a.type == DType::BF16)
        join_bc_kernel<__nv_bfloat16><<<blocks, 256, 0, s>>>(part_bc, tiles_of(a), a.B, a.T, a.G, a.N, g.db, g.dc);
      else
        join_bc_kernel<float><<<blocks, 256, 0, s>>>(part_bc, tiles_of(a), a.B, a.T, a.G, a.N, g.db, g.dc);
      DLVK_POST_LAUNCH();
    }
  }
  join_d_kernel<<<(unsigned)(((int64_t)a.D * (a.N + 2) + 255) / 256), 256, 0, s>>>(part_d, a.B, a.D, a.N, g);
  DLVK_POST_LAUNCH();
}

}  // namespace dlvk
