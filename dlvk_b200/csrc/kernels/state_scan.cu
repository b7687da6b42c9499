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
// N states has N / 4 lanes, and sums over states and channels cross lanes by
// shuffles.  The next span's elements are on their way to shared memory
// meanwhile, each to a place that only the thread that asked for it reads.
//
// What bounds it is the exponentials, one a token, channel and state (the special
// function units make 16 a clock and SM: 60 us for the 268 M of 16 x 512 tokens x
// 2048 channels x 16 states), and the issue slots and shared memory around them;
// the bytes are less (41 us of forward and backward together).  A thread has four
// states because fewer share a channel's step and input among too many lanes, and
// more leave too few warps: two channels a thread, whose loads of b and c are
// shared, and blocks of 64 threads were both slower.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "dlvk/seq.h"

namespace dlvk {
namespace {

constexpr int THREADS = 128, WARPS = THREADS / 32;
constexpr int NS = 4;  // states of a thread
constexpr int V = 4;   // elements of a thread's load
constexpr int PAD = 8;  // behind rows of sums, which a warp writes for several tokens at once: other banks
constexpr int SPAN = STATE_SCAN_SPAN;

// softplus(x) = max(x, 0) + log(1 + e), e = exp(-|x|).  Steps are small, so log(1 + e) has to
// keep its relative precision: 2 atanh(r), r = e / (2 + e) <= 1/3, by its series (to r^17: 2^-25);
// the exponent's rounding is made good by its remainder.  Below -200 e is 0 (an infinity would leave
// no remainder); NaN passes through the first term.
__device__ __forceinline__ f2 two(float x) { return pack(x, x); }
__device__ __forceinline__ f2 softplus_2(float x0, float x1) {
  const f2 m = pack(fmaxf(-fabsf(x0), -200.f), fmaxf(-fabsf(x1), -200.f)), t = mul2(m, two(-LOG2E));
  const f2 rest = fma2(m, two(1.925963033500e-8f), fma2(m, two(LOG2E), t));
  const float2 tv = unpack(t);
  f2 e = pack(ex2(-tv.x), ex2(-tv.y));
  e = fma2(mul2(e, rest), two(0.6931472f), e);
  const f2 r = mul2(e, rcp_2(add2(e, two(2.f)))), r2 = mul2(r, r);
  f2 p = fma2(r2, two(2.f / 17), two(2.f / 15));
  p = fma2(r2, p, two(2.f / 13));
  p = fma2(r2, p, two(2.f / 11));
  p = fma2(r2, p, two(2.f / 9));
  p = fma2(r2, p, two(2.f / 7));
  p = fma2(r2, p, two(2.f / 5));
  p = fma2(r2, p, two(2.f / 3));
  return add2(pack(x0 < 0.f ? 0.f : x0, x1 < 0.f ? 0.f : x1), fma2(mul2(r, r2), p, add2(r, r)));
}
__device__ __forceinline__ float softplus(float x) { return unpack(softplus_2(x, x)).x; }

__device__ __forceinline__ float both(f2 a) {
  const float2 v = unpack(a);
  return v.x + v.y;
}
// ex2_2, never taken from a register that an equal one has filled before: the
// backward pass's decays of a span would fill 64.
__device__ __forceinline__ f2 ex2_2_again(f2 x) {
  float2 v = unpack(x);
  asm volatile("ex2.approx.ftz.f32 %0, %0;" : "+f"(v.x));
  asm volatile("ex2.approx.ftz.f32 %0, %0;" : "+f"(v.y));
  return pack(v.x, v.y);
}
struct Quad {  // a thread's four states
  f2 v[2];
};
__device__ __forceinline__ Quad load_quad(const float* p) {
  const ulonglong2 u = *reinterpret_cast<const ulonglong2*>(p);
  return {{u.x, u.y}};
}

// Four neighbouring elements of a row.
template <typename T> struct Raw;
template <> struct Raw<float> { using type = float4; };
template <> struct Raw<__nv_bfloat16> { using type = uint2; };
template <typename T>
struct Four {
  typename Raw<T>::type raw;
  __device__ __forceinline__ float get(int i) const { return to_f32(reinterpret_cast<const T*>(&raw)[i]); }
  __device__ __forceinline__ void set(int i, float v) { reinterpret_cast<T*>(&raw)[i] = from_f32<T>(v); }
  __device__ __forceinline__ static Four zeros() {
    Four f;
#pragma unroll
    for (int i = 0; i < V; ++i) f.set(i, 0.f);
    return f;
  }
  // `count` of them
  template <bool WIDE>
  __device__ __forceinline__ void store(T* p, int count) const {
    if constexpr (WIDE) {
      *reinterpret_cast<typename Raw<T>::type*>(p) = raw;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < count) p[i] = reinterpret_cast<const T*>(&raw)[i];
    }
  }
};

// Four elements from p on, `count` of them (0: none) from memory, the others zeros.
// WIDE: rows of whole aligned fours, one copy.  Else fp32 is copied element by
// element, bf16 (2 bytes are too few for a copy) loaded.
template <typename T, bool WIDE>
__device__ __forceinline__ void fetch_four(Four<T>* dst, const T* p, const void* valid, int count) {
  if constexpr (WIDE) {
    copy_async<V * sizeof(T)>(dst, count > 0 ? (const void*)p : valid, count > 0);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      copy_async<4>(reinterpret_cast<T*>(dst) + i, i < count ? (const void*)(p + i) : valid, i < count);
  } else {
    Four<T> f;
#pragma unroll
    for (int i = 0; i < V; ++i) f.set(i, i < count ? to_f32(p[i]) : 0.f);
    *dst = f;
  }
}

// first: tokens before these, which lengths count too
__device__ __forceinline__ int64_t length_of(const StateScan& a, int64_t b, int64_t first = 0) {
  return a.lengths ? min(max((int64_t)a.lengths[b] - first, (int64_t)0), a.T) : a.T;
}

// The channels of a block, CH of one group of one sequence.
template <int CH>
struct Tile {
  int64_t b;
  int group, k, c0, count;  // tile of the group; first channel, channels of the tile that exist
  __device__ __forceinline__ explicit Tile(const StateScan& a) {
    const int per = a.D / a.G, tiles = (per + CH - 1) / CH;
    const int64_t i = blockIdx.x;
    const int j = (int)(i % ((int64_t)tiles * a.G));
    b = i / ((int64_t)tiles * a.G);
    group = j / tiles;
    k = j % tiles;
    c0 = group * per + k * CH;
    count = min(CH, per - k * CH);
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
      for (int i = 0; i < M / 2; i += 2) {
        if constexpr (M > 2) {
          const f2 low = pack(v[i], v[i + 1]), high = pack(v[i + M / 2], v[i + M / 2 + 1]);
          const float2 send = unpack(up ? low : high), got = unpack(add2(up ? high : low, pack(
              __shfl_xor_sync(0xffffffffu, send.x, FROM), __shfl_xor_sync(0xffffffffu, send.y, FROM))));
          v[i] = got.x, v[i + 1] = got.y;
        } else {
          const float send = up ? v[0] : v[1], keep = up ? v[1] : v[0];
          v[0] = keep + __shfl_xor_sync(0xffffffffu, send, FROM);
        }
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

// Rows of NS L states of a span, of b and behind them of c (or of one of them),
// zeros past N; a thread has four neighbouring states at a time.
template <typename T, int L, bool WIDE, int COUNT>
struct SpanStates {
  static constexpr int PER = (COUNT * SPAN * L + THREADS - 1) / THREADS;
  using Stage = Four<T>[PER][THREADS];
  __device__ __forceinline__ static void fetch(Stage& to, const SeqRef& first, const SeqRef& second, int64_t seq,
                                               int group, int N, int64_t t0, int64_t n) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = threadIdx.x + i * THREADS, t = e / L % SPAN, k = e % L * NS;
      const SeqRef& r = COUNT == 1 || e < SPAN * L ? first : second;
      if (e < COUNT * SPAN * L)
        fetch_four<T, WIDE>(&to[i][threadIdx.x], at<T>(r, seq, t0 + t, (int64_t)group * N + k), r.p, t0 + t < n ? N - k : 0);
    }
  }
  __device__ __forceinline__ static void widen(const Stage& from, float* sb) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = threadIdx.x + i * THREADS;
      if (e < COUNT * SPAN * L) {
        const Four<T> f = from[i][threadIdx.x];
        *reinterpret_cast<float4*>(sb + e * NS) = make_float4(f.get(0), f.get(1), f.get(2), f.get(3));
      }
    }
  }
};

// WIDE: four aligned states, or none (past N).
template <bool WIDE>
__device__ __forceinline__ Quad load_states(const float* p, int n0, int N) {
  if constexpr (WIDE) {
    return n0 < N ? load_quad(p) : Quad{};
  } else {
    float h[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) h[i] = n0 + i < N ? p[i] : 0.f;
    return {{pack(h[0], h[1]), pack(h[2], h[3])}};
  }
}
template <bool WIDE>
__device__ __forceinline__ void store_states(const Quad& q, float* p, int n0, int N) {
  if constexpr (WIDE) {
    if (n0 < N) *reinterpret_cast<ulonglong2*>(p) = make_ulonglong2(q.v[0], q.v[1]);
  } else {
    const float2 a = unpack(q.v[0]), b = unpack(q.v[1]);
    const float h[NS] = {a.x, a.y, b.x, b.y};
#pragma unroll
    for (int i = 0; i < NS; ++i)
      if (n0 + i < N) p[i] = h[i];
  }
}
// -exp(a_log), no further than fp32's lowest value: an infinity times a step of 0, which
// tokens that do not count have, is not a number.  Steps past 2^-120 see no difference.
__device__ __forceinline__ float rate_of(float a_log, float scale) {
  const float r = expf(a_log) * scale;
  return r > FLT_MAX ? -FLT_MAX : -r;
}
// Those of a thread's states, 0 past N.
__device__ __forceinline__ Quad load_rates(const StateScan& a, int d, int n0, float scale) {
  float r[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) r[i] = n0 + i < a.N ? rate_of(a.a_log[(int64_t)d * a.N + n0 + i], scale) : 0.f;
  return {{pack(r[0], r[1]), pack(r[2], r[3])}};
}

// A thread's channel of the block and first state.  The lanes of one state group
// are neighbours: eight lanes that read the same sixteen bytes of b or c take half
// the shared memory's cycles of eight that read different ones (measured: 2.1 and 4.0).
template <int L>
struct Place {
  static constexpr int LANES = 32 / L;  // of a state group
  int lane, ch, n0;
  __device__ __forceinline__ Place()
      : lane(threadIdx.x % 32), ch(threadIdx.x / 32 * LANES + threadIdx.x % LANES),
        n0(threadIdx.x % 32 / LANES * NS) {}
};
__device__ __forceinline__ float4 four(const float* p) { return *reinterpret_cast<const float4*>(p); }
// The steps of four elements, 0 where they do not count.
template <typename T>
__device__ __forceinline__ void steps_of(float (&s)[V], const Four<T>& dt, const float4& bias, bool here, int left) {
#pragma unroll
  for (int j = 0; j < V; j += 2) {
    const float2 v = unpack(softplus_2(dt.get(j) + (&bias.x)[j], dt.get(j + 1) + (&bias.x)[j + 1]));
    s[j] = here && j < left ? v.x : 0.f;
    s[j + 1] = here && j + 1 < left ? v.y : 0.f;
  }
}
__device__ __forceinline__ void put_four(float* p, const float (&v)[V]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}

// A thread's elements of a span: four neighbouring channels from c on, tokens t, t + STEP, ...
template <int CH>
struct Mine {
  static constexpr int PER = (SPAN * CH / V + THREADS - 1) / THREADS, STEP = THREADS * V / CH;
  int c, t, left;  // left: channels from c on that exist
  __device__ __forceinline__ explicit Mine(int count)
      : c(threadIdx.x * V % CH), t(threadIdx.x * V / CH), left(count - (int)(threadIdx.x * V % CH)) {}
};

// ---------------------------------------------------------------- pieces of the tokens
// Few channels leave most of the GPU idle, so long sequences are cut into pieces
// that run side by side: one pass takes each piece from a state of zeros to its
// end, the ends are joined in order (a piece's decays are exp(A sum s)), and the
// pass proper starts every piece from the state before it.  That makes the
// exponentials twice; where the channels fill the GPU there is one piece.
struct Pieces {
  int count = 1;
  int64_t spans = 0;        // of a piece
  float* ends = nullptr;    // [B][count][D][N]: the state after a piece of its own; joined: before it
  float* steps = nullptr;   // [B][count][D]: sum of s
};

// A part of the tokens of a backward pass that goes through them part by part, from the last on.
struct Part {
  int64_t first = 0;          // tokens before it, which lengths count too
  int64_t kept = 0;           // spans of a sequence, of all its tokens, whose states are kept
  const float* in = nullptr;  // [B][D][N]: what the part behind passes on; null: zeros
  float* out = nullptr;       // what this one passes on (may be `in`); null: not wanted
};

template <typename T, int L, bool WIDE>
struct EndsShared {
  static constexpr int CH = THREADS / L, PER = Mine<CH>::PER;
  float ss[SPAN][CH], sx[SPAN][CH];  // s; s u, or q
  float sb[SPAN * NS * L];           // b, or c
  float bias[CH];
  float4 sums[THREADS];              // of a thread's steps
  struct {
    Four<T> dt[PER][THREADS], x[PER][THREADS], z[PER][THREADS];
    typename SpanStates<T, L, WIDE, 1>::Stage bc;
  } stage[2];
};

// One sequence of 16384 tokens x 2048 channels, 16 pieces: 170-179 us, joining them 7,
// the pass proper 241-256, where one piece a sequence took 4871 in all.
//
// The end of a piece.  Forward: h[t] = a[t] h[t-1] + s u b[t].  BACK (what
// reaches the token before the piece): g[t] = c[t] q + a[t+1] g[t+1], times a[t].
template <typename T, int L, bool WIDE, bool BACK>
__global__ void __launch_bounds__(THREADS) scan_ends_kernel(StateScan a, SeqRef dy, Pieces pieces, int64_t first) {
  using States = SpanStates<T, L, WIDE, 1>;
  constexpr int CH = THREADS / L;
  extern __shared__ __align__(16) char raw[];
  auto& sh = *reinterpret_cast<EndsShared<T, L, WIDE>*>(raw);
  const Tile<CH> tile(a);
  const Mine<CH> my(tile.count);
  const Place<L> me;
  const int64_t n = length_of(a, tile.b, BACK ? first : 0), spans = (a.T + SPAN - 1) / SPAN;
  const int64_t from = blockIdx.y * pieces.spans;
  const int64_t to = min(min(spans, from + pieces.spans), (n + SPAN - 1) / SPAN);  // spans with a token that counts
  const bool real = me.ch < tile.count;
  Quad h{}, rate{};
  if (real) rate = load_rates(a, tile.c0 + me.ch, me.n0, LOG2E);
  for (int j = threadIdx.x; j < CH; j += THREADS) sh.bias[j] = a.dt_bias && j < tile.count ? a.dt_bias[tile.c0 + j] : 0.f;
  float total[V] = {0.f, 0.f, 0.f, 0.f};
  const auto fetch = [&](int64_t k) {
    auto& st = sh.stage[k % 2];
    const int64_t t0 = k * SPAN;
#pragma unroll
    for (int i = 0; i < my.PER; ++i) {
      const int t = my.t + i * my.STEP;
      if (t >= SPAN) break;
      const int count = t0 + t < n ? my.left : 0;
      const SeqRef& x = BACK ? dy : a.u;
      fetch_four<T, WIDE>(&st.dt[i][threadIdx.x], at<T>(a.dt, tile.b, t0 + t, tile.c0 + my.c), a.dt.p, count);
      fetch_four<T, WIDE>(&st.x[i][threadIdx.x], at<T>(x, tile.b, t0 + t, tile.c0 + my.c), x.p, count);
      if (BACK && a.z.p)
        fetch_four<T, WIDE>(&st.z[i][threadIdx.x], at<T>(a.z, tile.b, t0 + t, tile.c0 + my.c), a.z.p, count);
    }
    States::fetch(st.bc, BACK ? a.c : a.b, a.b, tile.b, tile.group, a.N, t0, n);
  };
  const int64_t count = to - from;
  const auto span_of = [&](int64_t i) { return BACK ? to - 1 - i : from + i; };
  if (count > 0) fetch(span_of(0));
  copies_issued();
  __syncthreads();
  for (int64_t i = 0; i < count; ++i) {
    const int64_t k = span_of(i), t0 = k * SPAN;
    auto& now = sh.stage[k % 2];
    if (i + 1 < count) fetch(span_of(i + 1));
    copies_issued();
    wait_copies<1>();
#pragma unroll
    for (int e = 0; e < my.PER; ++e) {
      const int t = my.t + e * my.STEP;
      if (t >= SPAN) break;
      const Four<T> dt = now.dt[e][threadIdx.x], x = now.x[e][threadIdx.x], z = now.z[e][threadIdx.x];
      const float4 bias = four(&sh.bias[my.c]);
      float s[V], sx[V];
      steps_of(s, dt, bias, t0 + t < n, my.left);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        total[j] += s[j];
        sx[j] = !BACK ? s[j] * x.get(j) : a.z.p ? x.get(j) * z.get(j) * sigmoid(z.get(j)) : x.get(j);
      }
      put_four(&sh.ss[t][my.c], s);
      put_four(&sh.sx[t][my.c], sx);
    }
    States::widen(now.bc, sh.sb);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SPAN; ++j) {
      const int t = BACK ? SPAN - 1 - j : j;
      const Quad q = load_quad(&sh.sb[t * NS * L + me.n0]);
      const f2 s = two(sh.ss[t][me.ch]), x = two(sh.sx[t][me.ch]);
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const f2 decay = ex2_2(mul2(s, rate.v[v]));
        h.v[v] = BACK ? mul2(fma2(x, q.v[v], h.v[v]), decay) : fma2(decay, h.v[v], mul2(x, q.v[v]));
      }
    }
    __syncthreads();
  }
  const int64_t piece = tile.b * pieces.count + blockIdx.y;
  if (real) store_states<WIDE>(h, pieces.ends + (piece * a.D + tile.c0 + me.ch) * a.N + me.n0, me.n0, a.N);
  put_four(&sh.sums[threadIdx.x].x, total);
  __syncthreads();
  constexpr int SAME = CH / V, ROWS = SPAN * SAME < THREADS ? SPAN * SAME : THREADS;
  for (int j = threadIdx.x; j < tile.count; j += THREADS) {
    float s = 0.f;
    for (int r = j / V; r < ROWS; r += SAME) s += (&sh.sums[r].x)[j % V];
    pieces.steps[piece * a.D + tile.c0 + j] = s;
  }
}

// ends: from what a piece ends with to what the one before it (BACK: behind it) passes on to it.
template <bool BACK>
__global__ void __launch_bounds__(256) scan_join_kernel(StateScan a, Pieces pieces, Part part) {
  const int64_t dn = (int64_t)a.D * a.N, i = blockIdx.x * 256LL + threadIdx.x;
  if (i >= a.B * dn) return;
  const int64_t b = i / dn, e = i % dn, d = e / a.N;
  const float rate = rate_of(a.a_log[e], 1.f);
  float carry = BACK ? (part.in ? part.in[i] : 0.f) : a.state ? a.state[i] : 0.f;
  // eight pieces' loads ahead of the stores, which might be to the same place for all that the compiler knows
  constexpr int AHEAD = 8;
  for (int j0 = 0; j0 < pieces.count; j0 += AHEAD) {
    float own[AHEAD], steps[AHEAD];
    int64_t piece[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int k = min(j0 + j, pieces.count - 1);
      piece[j] = b * pieces.count + (BACK ? pieces.count - 1 - k : k);
      own[j] = pieces.ends[piece[j] * dn + e];
      steps[j] = pieces.steps[piece[j] * a.D + d];
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (j0 + j >= pieces.count) break;
      pieces.ends[piece[j] * dn + e] = carry;
      carry = fmaf(expf(rate * steps[j]), carry, own[j]);
    }
  }
  if (BACK && part.out) part.out[i] = carry;
}

// ---------------------------------------------------------------- forward
template <typename T, int L, bool WIDE>
struct FwdShared {
  static constexpr int CH = THREADS / L, PER = Mine<CH>::PER;
  float ss[SPAN][CH], su[SPAN][CH];  // s, s u
  float sy[SPAN][CH + PAD];          // sum_n c h
  float sb[2 * SPAN * NS * L];
  float bias[CH], skip[CH];
  struct {
    Four<T> u[PER][THREADS], dt[PER][THREADS], z[PER][THREADS];
    typename SpanStates<T, L, WIDE, 2>::Stage bc;
  } stage[2];
};

// 16 x 512 x 2048, 16 states, bf16 with gates: 133 us, 45% of the special function units' rate.
// Issue slots 62%, shared memory 70%, special functions 60% busy on average; warps compete for all
// three until the blocks that an SM began with end one by one.  62 registers: seven blocks an SM.
// (Steps as pairs of equals in shared memory, which spares moves: 10% slower.)
template <typename T, int L, bool WIDE>
__global__ void __launch_bounds__(THREADS) scan_fwd_kernel(StateScan a, SeqRef y, float* out_state, float* saved,
                                                           Pieces pieces) {
  using States = SpanStates<T, L, WIDE, 2>;
  constexpr int CH = THREADS / L;
  extern __shared__ __align__(16) char raw[];
  auto& sh = *reinterpret_cast<FwdShared<T, L, WIDE>*>(raw);
  const Tile<CH> tile(a);
  const Mine<CH> my(tile.count);
  const Place<L> me;
  const int lane = me.lane, n0 = me.n0, ch = me.ch;
  const int64_t n = length_of(a, tile.b), spans = (a.T + SPAN - 1) / SPAN;
  const int64_t from = blockIdx.y * pieces.spans, end = min(spans, from + pieces.spans);
  const int64_t to = max(from, min(end, (n + SPAN - 1) / SPAN));  // spans with a token that counts
  const bool real = ch < tile.count;
  const int64_t states = (int64_t)(tile.c0 + ch) * a.N + n0;  // of this thread, in a [D][N]
  const int64_t dn = (int64_t)a.D * a.N;
  Quad h{}, rate{};
  if (real) {
    if (pieces.ends)
      h = load_states<WIDE>(pieces.ends + (tile.b * pieces.count + blockIdx.y) * dn + states, n0, a.N);
    else if (a.state)
      h = load_states<WIDE>(a.state + tile.b * dn + states, n0, a.N);
    rate = load_rates(a, tile.c0 + ch, n0, LOG2E);
  }
  for (int j = threadIdx.x; j < CH; j += THREADS) {
    sh.bias[j] = a.dt_bias && j < tile.count ? a.dt_bias[tile.c0 + j] : 0.f;
    sh.skip[j] = a.skip && j < tile.count ? a.skip[tile.c0 + j] : 0.f;
  }
  const auto fetch = [&](int64_t k) {
    auto& st = sh.stage[k % 2];
    const int64_t t0 = k * SPAN;
#pragma unroll
    for (int i = 0; i < my.PER; ++i) {
      const int t = my.t + i * my.STEP;
      if (t >= SPAN) break;
      const int count = t0 + t < n ? my.left : 0;
      fetch_four<T, WIDE>(&st.u[i][threadIdx.x], at<T>(a.u, tile.b, t0 + t, tile.c0 + my.c), a.u.p, count);
      fetch_four<T, WIDE>(&st.dt[i][threadIdx.x], at<T>(a.dt, tile.b, t0 + t, tile.c0 + my.c), a.dt.p, count);
      if (a.z.p) fetch_four<T, WIDE>(&st.z[i][threadIdx.x], at<T>(a.z, tile.b, t0 + t, tile.c0 + my.c), a.z.p, count);
    }
    States::fetch(st.bc, a.b, a.c, tile.b, tile.group, a.N, t0, n);
  };
  if (from < to) fetch(from);
  copies_issued();
  __syncthreads();
  for (int64_t k = from; k < to; ++k) {
    const int64_t t0 = k * SPAN;
    auto& now = sh.stage[k % 2];
    if (k + 1 < to) fetch(k + 1);
    copies_issued();
    wait_copies<1>();
#pragma unroll
    for (int i = 0; i < my.PER; ++i) {
      const int t = my.t + i * my.STEP;
      if (t >= SPAN) break;
      const Four<T> u = now.u[i][threadIdx.x], dt = now.dt[i][threadIdx.x];
      const float4 bias = four(&sh.bias[my.c]);
      float s[V], su[V];
      steps_of(s, dt, bias, t0 + t < n, my.left);
#pragma unroll
      for (int j = 0; j < V; ++j) su[j] = s[j] * u.get(j);
      put_four(&sh.ss[t][my.c], s);
      put_four(&sh.su[t][my.c], su);
    }
    States::widen(now.bc, sh.sb);
    __syncthreads();
    if (saved && real) store_states<WIDE>(h, saved + (tile.b * spans + k) * dn + states, n0, a.N);
#pragma unroll
    for (int t = 0; t < SPAN; t += 4) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f2 s = two(sh.ss[t + j][ch]), su = two(sh.su[t + j][ch]);
        const Quad qb = load_quad(&sh.sb[(t + j) * NS * L + n0]), qc = load_quad(&sh.sb[(SPAN + t + j) * NS * L + n0]);
        h.v[0] = fma2(ex2_2(mul2(s, rate.v[0])), h.v[0], mul2(su, qb.v[0]));
        h.v[1] = fma2(ex2_2(mul2(s, rate.v[1])), h.v[1], mul2(su, qb.v[1]));
        v[j] = both(fma2(qc.v[0], h.v[0], mul2(qc.v[1], h.v[1])));
      }
      int first = 0;
      bool mine = true;
      deal<4, me.LANES, 32>(v, lane, first, mine);
      if (mine) {
#pragma unroll
        for (int j = 0; j < dealt(4, me.LANES, 32); ++j) sh.sy[t + first + j][ch] = v[j];
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < my.PER; ++i) {
      const int t = my.t + i * my.STEP;
      if (t >= SPAN || t0 + t >= a.T || my.left <= 0) break;
      const Four<T> u = now.u[i][threadIdx.x], z = now.z[i][threadIdx.x];
      const float4 skip = four(&sh.skip[my.c]), sum = four(&sh.sy[t][my.c]);
      Four<T> out;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float p = fmaf((&skip.x)[j], u.get(j), (&sum.x)[j]);
        if (a.z.p) p *= z.get(j) * sigmoid(z.get(j));
        out.set(j, t0 + t < n ? p : 0.f);
      }
      out.template store<WIDE>(at<T>(y, tile.b, t0 + t, tile.c0 + my.c), my.left);
    }
  }
  for (int64_t k = to; k < end; ++k) {  // behind the sequence
    if (saved && real) store_states<WIDE>(h, saved + (tile.b * spans + k) * dn + states, n0, a.N);
#pragma unroll
    for (int i = 0; i < my.PER; ++i) {
      const int t = my.t + i * my.STEP;
      if (t < SPAN && k * SPAN + t < a.T && my.left > 0)
        Four<T>::zeros().template store<WIDE>(at<T>(y, tile.b, k * SPAN + t, tile.c0 + my.c), my.left);
    }
  }
  if (out_state && real && blockIdx.y + 1 == pieces.count) store_states<WIDE>(h, out_state + tile.b * dn + states, n0, a.N);
}

// One token of each sequence.  A thread has four states of a channel in R sequences,
// which share the channel's rates; what it reads is asked for before anything is
// computed.  Steps and gates, one value a channel and sequence, are dealt out to the
// channel's lanes: lane by lane they were most of the instructions, which bound this
// kernel before the memory did.  130 sequences x 1600 channels of 64 states (106 MB of
// states read and written): 27 us, 60% of the copy rate; 64 x 2048 of 16: 6.5 us, a
// launch and one round to the memory.
template <typename T, int L, bool WIDE, int R>
__global__ void __launch_bounds__(THREADS) scan_step_kernel(StateScan a, SeqRef y, float* out_state, float* saved) {
  constexpr int CH = THREADS / L, OWN = dealt(R, 1, L);
  const unsigned tiles = ((unsigned)a.D + CH - 1) / CH;
  const int64_t b0 = (int64_t)(blockIdx.x / tiles) * R, left = a.B - b0;
  const int channel = (int)(blockIdx.x % tiles) * CH + threadIdx.x / L, k = threadIdx.x % L, n0 = k * NS;
  const bool real = channel < a.D;
  const int d = real ? channel : 0, count = real ? a.N - n0 : 0;
  const int64_t dn = (int64_t)a.D * a.N, row = b0 * dn + (int64_t)d * a.N + n0;
  const int64_t state0 = (int64_t)(d / (a.D / a.G)) * a.N + n0;
  Quad h[R], rate;
  Four<T> fb[R], fc[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool in = r < left;
    const T *pb = at<T>(a.b, b0 + r, 0, state0), *pc = at<T>(a.c, b0 + r, 0, state0);
    h[r] = Quad{};
    if (a.state && in) h[r] = load_states<WIDE>(a.state + row + r * dn, 0, count);
    fb[r] = fc[r] = Four<T>::zeros();
    if constexpr (WIDE) {
      if (in && count > 0) {
        fb[r].raw = *reinterpret_cast<const typename Raw<T>::type*>(pb);
        fc[r].raw = *reinterpret_cast<const typename Raw<T>::type*>(pc);
      }
    } else {
#pragma unroll
      for (int j = 0; j < NS; ++j)
        if (in && j < count) fb[r].set(j, to_f32(pb[j])), fc[r].set(j, to_f32(pc[j]));
    }
  }
  // the sequences of this lane's sums
  int first = 0;
  bool mine = true;
  {
    float none[R] = {};
    deal<R, 1, L>(none, k, first, mine);
  }
  const float bias = a.dt_bias ? a.dt_bias[d] : 0.f, skip = a.skip ? a.skip[d] : 0.f;
  float u[OWN], z[OWN], s[OWN];
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    const int64_t b = min(b0 + first + i, a.B - 1);
    u[i] = to_f32(*at<T>(a.u, b, 0, d));
    s[i] = to_f32(*at<T>(a.dt, b, 0, d));
    z[i] = a.z.p ? to_f32(*at<T>(a.z, b, 0, d)) : 0.f;
    s[i] = length_of(a, b) > 0 ? softplus(s[i] + bias) : -1.f;  // -1: none
  }
  rate = load_rates(a, d, n0, LOG2E);
  float p[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (saved && r < left) store_states<false>(h[r], saved + row + r * dn, 0, count);
    int from = 0;  // the lane of this sequence
#pragma unroll
    for (int m = R / 2, bit = 1, e = r; m > 0 && bit < L; m /= 2, bit *= 2) from |= e / m ? bit : 0, e %= m;
    const float s1 = __shfl_sync(0xffffffffu, s[r % OWN], from, L), u1 = __shfl_sync(0xffffffffu, u[r % OWN], from, L);
    if (!(s1 < 0.f)) {
      const f2 s2 = two(s1), su = two(s1 * u1);
#pragma unroll
      for (int v = 0; v < 2; ++v)
        h[r].v[v] = fma2(ex2_2(mul2(s2, rate.v[v])), h[r].v[v], mul2(su, pack(fb[r].get(2 * v), fb[r].get(2 * v + 1))));
    }
    p[r] = both(fma2(pack(fc[r].get(0), fc[r].get(1)), h[r].v[0], mul2(pack(fc[r].get(2), fc[r].get(3)), h[r].v[1])));
    if (out_state && r < left) store_states<WIDE>(h[r], out_state + row + r * dn, 0, count);
  }
  int at_first = 0;
  deal<R, 1, L>(p, k, at_first, mine);
  if (!real || !mine) return;
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    if (first + i >= left) continue;
    float out = fmaf(skip, u[i], p[i]);
    if (a.z.p) out *= z[i] * sigmoid(z[i]);
    *at<T>(y, b0 + first + i, 0, d) = from_f32<T>(s[i] < 0.f ? 0.f : out);
  }
}

// ---------------------------------------------------------------- backward
template <typename T, int L, bool WIDE>
struct BwdShared {
  static constexpr int CH = THREADS / L, PER = Mine<CH>::PER;
  float ss[SPAN][CH], su[SPAN][CH];   // s, s u
  float sq[SPAN][CH];                 // q
  float sy[SPAN][CH + PAD];           // sum_n c h
  float sv[SPAN][CH + PAD], sd[SPAN][CH + PAD];  // sum_n g b, sum_n g a h' A
  float sb[2 * SPAN * NS * L];
  float red[WARPS][SPAN][2 * NS * L]; // db and dc of a warp's channels
  float4 sums[2][THREADS];            // dskip and ddt_bias of a thread's elements
  float4 da[THREADS];                 // da_log of its states
  float bias[CH], skip[CH];
  struct {
    Four<T> u[PER][THREADS], dt[PER][THREADS], z[PER][THREADS], go[PER][THREADS];
    typename SpanStates<T, L, WIDE, 2>::Stage bc;
    float4 h[THREADS];
  } stage[2];
};

// A span's states are made again from the one saved before it and stay in registers
// (68 of 128) while the tokens go back.  16 x 512 x 2048, 16 states, bf16 with gates:
// 386 us and 19 joining the sums, 120 instructions a warp and token: the exponentials
// twice, sums of db and dc over channels (7 shuffles, each of which halves the values
// that a lane still adds up), of du and ds over states.  Issue slots 62%, shared memory
// 67% busy; 16 warps an SM.  Sums over channels as tf32 products of ones and the values
// took longer (some 9 cycles a product of 16 x 8 x 4) and needed two for fp32.
//
// ALONG: a part of the tokens (pieces.ends has what reaches its last one).  An instance of its own: the
// registers of the others stay as they are, 358 us and not 380 at 16 x 512 x 2048 with 8 states.
// part_bc [tiles of a group][B][T][G][2][NS L]; part_d [B][pieces][D][N + 2]: da, dskip, ddt_bias.
template <typename T, int L, bool WIDE, bool ALONG>
__global__ void __launch_bounds__(THREADS, 4) scan_bwd_kernel(StateScan a, const float* __restrict__ saved, SeqRef dy,
                                                              StateScanGrads g, float* __restrict__ part_bc,
                                                              float* __restrict__ part_d, Pieces pieces, Part part) {
  using States = SpanStates<T, L, WIDE, 2>;
  constexpr int CH = THREADS / L, ROW = 2 * NS * L;
  extern __shared__ __align__(16) char raw[];
  auto& sh = *reinterpret_cast<BwdShared<T, L, WIDE>*>(raw);
  const Tile<CH> tile(a);
  const Mine<CH> my(tile.count);
  const Place<L> me;
  const int lane = me.lane, warp = threadIdx.x / 32, n0 = me.n0, ch = me.ch;
  const bool real = ch < tile.count;
  const int64_t n = length_of(a, tile.b, ALONG ? part.first : 0), spans = (a.T + SPAN - 1) / SPAN;
  Quad rate{}, ga{};
  const int64_t from = blockIdx.y * pieces.spans, end = min(spans, from + pieces.spans);
  const int64_t to = max(from, min(end, (n + SPAN - 1) / SPAN));  // spans with a token that counts
  const int64_t piece = tile.b * pieces.count + blockIdx.y;
  if (real) {
    rate = load_rates(a, tile.c0 + ch, n0, 1.f);
    if (pieces.ends) ga = load_states<WIDE>(pieces.ends + (piece * a.D + tile.c0 + ch) * a.N + n0, n0, a.N);
  }
  for (int j = threadIdx.x; j < CH; j += THREADS) {
    sh.bias[j] = a.dt_bias && j < tile.count ? a.dt_bias[tile.c0 + j] : 0.f;
    sh.skip[j] = a.skip && j < tile.count ? a.skip[tile.c0 + j] : 0.f;
  }
  sh.da[threadIdx.x] = sh.sums[0][threadIdx.x] = sh.sums[1][threadIdx.x] = make_float4(0.f, 0.f, 0.f, 0.f);
  const auto fetch = [&](int64_t k) {
    auto& st = sh.stage[k % 2];
    const int64_t t0 = k * SPAN;
#pragma unroll
    for (int i = 0; i < my.PER; ++i) {
      const int t = my.t + i * my.STEP;
      if (t >= SPAN) break;
      const int count = t0 + t < n ? my.left : 0;
      fetch_four<T, WIDE>(&st.u[i][threadIdx.x], at<T>(a.u, tile.b, t0 + t, tile.c0 + my.c), a.u.p, count);
      fetch_four<T, WIDE>(&st.dt[i][threadIdx.x], at<T>(a.dt, tile.b, t0 + t, tile.c0 + my.c), a.dt.p, count);
      if (a.z.p) fetch_four<T, WIDE>(&st.z[i][threadIdx.x], at<T>(a.z, tile.b, t0 + t, tile.c0 + my.c), a.z.p, count);
      fetch_four<T, WIDE>(&st.go[i][threadIdx.x], at<T>(dy, tile.b, t0 + t, tile.c0 + my.c), dy.p, count);
    }
    States::fetch(st.bc, a.b, a.c, tile.b, tile.group, a.N, t0, n);
    fetch_four<float, WIDE>(reinterpret_cast<Four<float>*>(&st.h[threadIdx.x]),
                            saved + ((tile.b * (ALONG ? part.kept : spans) + k) * a.D + tile.c0 + ch) * a.N + n0, saved, real ? a.N - n0 : 0);
  };
  for (int64_t k = to; k < end; ++k) {  // behind the sequence
    const int64_t t0 = k * SPAN;
#pragma unroll
    for (int i = 0; i < my.PER; ++i) {
      const int t = my.t + i * my.STEP;
      if (t < SPAN && t0 + t < a.T && my.left > 0) {
        Four<T>::zeros().template store<WIDE>(at<T>(g.du, tile.b, t0 + t, tile.c0 + my.c), my.left);
        Four<T>::zeros().template store<WIDE>(at<T>(g.ddt, tile.b, t0 + t, tile.c0 + my.c), my.left);
        if (a.z.p) Four<T>::zeros().template store<WIDE>(at<T>(g.dz, tile.b, t0 + t, tile.c0 + my.c), my.left);
      }
    }
    float* part = part_bc + (((tile.k * a.B + tile.b) * a.T + t0) * a.G + tile.group) * ROW;
    for (int i = threadIdx.x * 4; i < SPAN * ROW; i += THREADS * 4)
      if (t0 + i / ROW < a.T)
        *reinterpret_cast<float4*>(part + (int64_t)(i / ROW) * a.G * ROW + i % ROW) = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  if (from < to) fetch(to - 1);
  copies_issued();
  __syncthreads();
  for (int64_t k = to - 1; k >= from; --k) {
    const int64_t t0 = k * SPAN;
    auto& now = sh.stage[k % 2];
    if (k > from) fetch(k - 1);
    copies_issued();
    wait_copies<1>();
#pragma unroll
    for (int i = 0; i < my.PER; ++i) {
      const int t = my.t + i * my.STEP;
      if (t >= SPAN) break;
      const Four<T> u = now.u[i][threadIdx.x], dt = now.dt[i][threadIdx.x], z = now.z[i][threadIdx.x],
                    go = now.go[i][threadIdx.x];
      const float4 bias = four(&sh.bias[my.c]);
      float s[V], su[V], q[V];
      steps_of(s, dt, bias, t0 + t < n, my.left);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        su[j] = s[j] * u.get(j);
        q[j] = go.get(j) * (a.z.p ? z.get(j) * sigmoid(z.get(j)) : 1.f);
      }
      put_four(&sh.ss[t][my.c], s);
      put_four(&sh.su[t][my.c], su);
      put_four(&sh.sq[t][my.c], q);
    }
    States::widen(now.bc, sh.sb);
    Quad h[SPAN + 1];  // h[t]: before token t of the span
    h[0] = load_quad(reinterpret_cast<const float*>(&now.h[threadIdx.x]));
    __syncthreads();
#pragma unroll
    for (int t = 0; t < SPAN; t += 4) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float s1 = sh.ss[t + j][ch] * LOG2E, su1 = sh.su[t + j][ch];
        const Quad qb = load_quad(&sh.sb[(t + j) * NS * L + n0]), qc = load_quad(&sh.sb[(SPAN + t + j) * NS * L + n0]);
        const f2 s = pack(s1, s1), su = pack(su1, su1);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          h[t + j + 1].v[i] = fma2(ex2_2(mul2(s, rate.v[i])), h[t + j].v[i], mul2(su, qb.v[i]));
        v[j] = both(fma2(qc.v[0], h[t + j + 1].v[0], mul2(qc.v[1], h[t + j + 1].v[1])));
      }
      int first = 0;
      bool mine = true;
      deal<4, me.LANES, 32>(v, lane, first, mine);
      if (mine) {
#pragma unroll
        for (int j = 0; j < dealt(4, me.LANES, 32); ++j) sh.sy[t + first + j][ch] = v[j];
      }
    }
    Quad da{};
#pragma unroll
    for (int t4 = SPAN - 4; t4 >= 0; t4 -= 4) {
      float sums[8];  // of four tokens: sum_n g b, sum_n g a h' A
#pragma unroll
      for (int j = 3; j >= 0; --j) {
        const int t = t4 + j;
        const float s1 = sh.ss[t][ch], su1 = sh.su[t][ch], q1 = sh.sq[t][ch], sl1 = s1 * LOG2E;
        const Quad qb = load_quad(&sh.sb[t * NS * L + n0]), qc = load_quad(&sh.sb[(SPAN + t) * NS * L + n0]);
        const f2 q = pack(q1, q1), s = pack(s1, s1), su = pack(su1, su1), sl = pack(sl1, sl1);
        f2 into = 0, through_a = 0;  // two zeros
        float w[8];                  // db and dc of this channel
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const f2 gi = fma2(q, qc.v[i], ga.v[i]);
          const float2 wb = unpack(mul2(gi, su)), wc = unpack(mul2(q, h[t + 1].v[i]));
          w[2 * i] = wb.x, w[2 * i + 1] = wb.y, w[NS + 2 * i] = wc.x, w[NS + 2 * i + 1] = wc.y;
          into = fma2(gi, qb.v[i], into);
          ga.v[i] = mul2(gi, ex2_2_again(mul2(sl, rate.v[i])));
          const f2 through = mul2(ga.v[i], h[t].v[i]);
          through_a = fma2(through, rate.v[i], through_a);
          da.v[i] = fma2(through, s, da.v[i]);
        }
        sums[2 * j] = both(into);
        sums[2 * j + 1] = both(through_a);
        int first = 0;
        bool mine = true;
        deal<8, 1, me.LANES>(w, lane, first, mine);
        if (mine) {
#pragma unroll
          for (int i = 0; i < dealt(8, 1, me.LANES); ++i) {
            const int e = first + i;  // < NS: db of state n0 + e
            sh.red[warp][t][(e / NS) * NS * L + n0 + e % NS] = w[i];
          }
        }
      }
      int first = 0;
      bool mine = true;
      deal<8, me.LANES, 32>(sums, lane, first, mine);
      if (mine) {
#pragma unroll
        for (int i = 0; i < dealt(8, me.LANES, 32); ++i) {
          const int e = first + i;
          (e % 2 ? sh.sd : sh.sv)[t4 + e / 2][ch] = sums[i];
        }
      }
    }
    {  // (span by span, so that the sum over all tokens rounds once a span)
      const Quad before = load_quad(&sh.da[threadIdx.x].x);
      store_states<true>({{add2(before.v[0], da.v[0]), add2(before.v[1], da.v[1])}}, &sh.da[threadIdx.x].x, 0, 1);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < my.PER; ++i) {
      const int t = my.t + i * my.STEP;
      if (t >= SPAN || t0 + t >= a.T || my.left <= 0) break;
      const bool here = t0 + t < n;
      const Four<T> u = now.u[i][threadIdx.x], dt = now.dt[i][threadIdx.x], z = now.z[i][threadIdx.x],
                    go = now.go[i][threadIdx.x];
      Four<T> du, ddt, dz;
      float4 ds = sh.sums[0][threadIdx.x], db = sh.sums[1][threadIdx.x];
      const float4 q4 = four(&sh.sq[t][my.c]), v4 = four(&sh.sv[t][my.c]), d4 = four(&sh.sd[t][my.c]),
                   y4 = four(&sh.sy[t][my.c]), s4 = four(&sh.ss[t][my.c]), skip4 = four(&sh.skip[my.c]),
                   bias4 = four(&sh.bias[my.c]);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float uj = u.get(j), zj = z.get(j), q = (&q4.x)[j], v = (&v4.x)[j], skip = (&skip4.x)[j];
        du.set(j, here ? fmaf(v, (&s4.x)[j], q * skip) : 0.f);
        // a step of 0 has no slope, however large the rates are (an infinite sum times it is not a number)
        const float slope = sigmoid(dt.get(j) + (&bias4.x)[j]);
        const float dr = here && slope != 0.f ? fmaf(v, uj, (&d4.x)[j]) * slope : 0.f;
        ddt.set(j, dr);
        (&ds.x)[j] = fmaf(q, uj, (&ds.x)[j]);
        (&db.x)[j] += dr;
        const float sz = sigmoid(zj);
        dz.set(j, here ? go.get(j) * fmaf(skip, uj, (&y4.x)[j]) * sz * fmaf(zj, 1.f - sz, 1.f) : 0.f);
      }
      sh.sums[0][threadIdx.x] = ds;
      sh.sums[1][threadIdx.x] = db;
      du.template store<WIDE>(at<T>(g.du, tile.b, t0 + t, tile.c0 + my.c), my.left);
      ddt.template store<WIDE>(at<T>(g.ddt, tile.b, t0 + t, tile.c0 + my.c), my.left);
      if (a.z.p) dz.template store<WIDE>(at<T>(g.dz, tile.b, t0 + t, tile.c0 + my.c), my.left);
    }
    float* part = part_bc + (((tile.k * a.B + tile.b) * a.T + t0) * a.G + tile.group) * ROW;
    for (int i = threadIdx.x * 4; i < SPAN * ROW; i += THREADS * 4) {
      const int t = i / ROW, e = i % ROW;
      if (t0 + t >= a.T) break;
      float4 s = *reinterpret_cast<const float4*>(&sh.red[0][t][e]);
#pragma unroll
      for (int w = 1; w < WARPS; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(&sh.red[w][t][e]);
        s.x += x.x, s.y += x.y, s.z += x.z, s.w += x.w;
      }
      *reinterpret_cast<float4*>(part + (int64_t)t * a.G * ROW + e) = s;
    }
    // (the barrier after the next span's elements is between these reads and what comes to their places)
  }
  if (ALONG && real && part.out) store_states<WIDE>(ga, part.out + (piece * a.D + tile.c0 + ch) * a.N + n0, n0, a.N);
  const Quad da = load_quad(&sh.da[threadIdx.x].x);
  if (real) store_states<false>({{mul2(da.v[0], rate.v[0]), mul2(da.v[1], rate.v[1])}},
                         part_d + (piece * a.D + tile.c0 + ch) * (a.N + 2) + n0, n0, a.N);
  // dskip and ddt_bias: threads CH / V apart hold the same channels
  constexpr int SAME = CH / V, ROWS = SPAN * SAME < THREADS ? SPAN * SAME : THREADS;
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * CH; i += THREADS) {
    const int half = i / CH, at_ch = i % CH;
    float s = 0.f;
    for (int r = at_ch / V; r < ROWS; r += SAME) s += (&sh.sums[half][r].x)[at_ch % V];
    if (at_ch < tile.count) part_d[(piece * a.D + tile.c0 + at_ch) * (a.N + 2) + a.N + half] = s;
  }
}

// db and dc: the sums over a group's tiles, in their order; rows of 2 `states`, of which N are real.
template <typename T>
__global__ void __launch_bounds__(256) join_bc_kernel(const float* __restrict__ part, int tiles, int64_t B, int64_t T_,
                                                      int G, int N, int states, SeqRef db, SeqRef dc) {
  const int64_t row = (int64_t)G * 2 * states, total = B * T_ * row;
  for (int64_t i = blockIdx.x * 256LL + threadIdx.x; i < total; i += 256LL * gridDim.x) {
    const int e = (int)(i % row), group = e / (2 * states), half = e / states % 2, n = e % states;
    if (n >= N) continue;
    float s = 0.f;
    for (int k = 0; k < tiles; ++k) s += part[k * total + i];
    const int64_t t = i / row % T_, b = i / row / T_;
    *at<T>(half ? dc : db, b, t, (int64_t)group * N + n) = from_f32<T>(s);
  }
}
// da_log, dskip and ddt_bias: the sums over the sequences and their pieces, in 64 bits (there are few).
__global__ void __launch_bounds__(256) join_d_kernel(const float* __restrict__ part, int64_t B, int D, int N,
                                                     StateScanGrads g) {
  const int64_t total = (int64_t)D * (N + 2), i = blockIdx.x * 256LL + threadIdx.x;
  if (i >= total) return;
  double sum = 0.0;
#pragma unroll 4
  for (int64_t b = 0; b < B; ++b) sum += part[b * total + i];
  const float s = (float)sum;
  const int64_t d = i / (N + 2);
  const int k = (int)(i % (N + 2));
  float* out = k < N ? (g.da_log ? g.da_log + d * N + k : nullptr)
                     : k == N ? (g.dskip ? g.dskip + d : nullptr) : (g.ddt_bias ? g.ddt_bias + d : nullptr);
  if (out) *out = g.accumulate ? *out + s : s;
}

// Whether four neighbouring elements are one load.
bool aligned(const SeqRef& r, DType type) {
  const int64_t bytes = type == DType::BF16 ? 2 : 4;
  return !r.p || (reinterpret_cast<uintptr_t>(r.p) % (V * bytes) == 0 && r.batch % V == 0 && r.token % V == 0);
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

namespace {
template <typename Kernel, typename... Args>
void launch(Kernel kernel, size_t smem, const StateScan& a, int pieces, cudaStream_t s, Args... args) {
  if (smem > 48 * 1024)
    DLVK_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  kernel<<<dim3(grid_of(a), pieces), THREADS, smem, s>>>(a, args...);
  DLVK_POST_LAUNCH();
}
// f(element type, lanes of a channel, whether rows are of whole aligned fours)
template <typename F>
void by_kind(const StateScan& a, bool wide, F&& f) {
  by_lanes(a.N, [&](auto lanes) {
    if (a.type == DType::BF16) {
      if (wide) f(__nv_bfloat16(), lanes, std::true_type());
      else f(__nv_bfloat16(), lanes, std::false_type());
    } else {
      if (wide) f(float(), lanes, std::true_type());
      else f(float(), lanes, std::false_type());
    }
  });
}
bool wide_operands(const StateScan& a) {
  return a.D / a.G % V == 0 && a.N % V == 0 && aligned(a.u, a.type) && aligned(a.dt, a.type) && aligned(a.z, a.type) &&
         aligned(a.b, a.type) && aligned(a.c, a.type) && reinterpret_cast<uintptr_t>(a.state) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(a.a_log) % 16 == 0;
}
bool aligned16(const float* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
int64_t part_bc_floats(const StateScan& a) { return (int64_t)tiles_of(a) * a.B * a.T * a.G * 2 * NS * lanes_of(a.N); }

// Pieces as long as the GPU has room for their blocks at once, of at least four spans each
// (1 x 4096 x 64 channels of 16 states, forward and backward: 30 and 48 us; of eight 33 and 57,
// of two 32 and 54; one piece 334 and 795).  The pass for the ends costs two thirds of the pass
// proper, so few pieces are worse than one: forward, 3 x 1024 x 2048, five take 99 us and one 106,
// but of 4 x 1024 four take 122; backward, three of the former take 210 and one 277, two of the
// latter 300.
// These times, and the blocks that an SM is taken to have room for, are those of 9 to 16 states.  By
// shared memory fp32 has room for 5 (forward) at 8 states or fewer and past 32, for 2 or 3 (backward)
// there and at 17 to 32, bf16 for 3 (backward) there: pieces of such calls may take two rounds.
constexpr int FWD_BLOCKS = 7, BWD_BLOCKS = 4;
constexpr int FWD_PIECES = 5, BWD_PIECES = 3, PIECE_SPANS = 4;
Pieces pieces_of(const StateScan& a, int blocks_an_sm, int least) {
  Pieces p;
  const int64_t spans = (a.T + SPAN - 1) / SPAN, blocks = std::max<int64_t>(1, a.B * a.G * tiles_of(a));
  const int64_t most = std::min<int64_t>(148 * blocks_an_sm / blocks, spans / PIECE_SPANS);
  p.spans = most >= least ? (spans + most - 1) / most : std::max<int64_t>(spans, 1);
  p.count = (int)((spans + p.spans - 1) / p.spans);
  if (p.count < 1) p.count = 1;
  return p;
}
int64_t pieces_floats(const StateScan& a, const Pieces& p) { return p.count > 1 ? a.B * p.count * a.D * (a.N + 1) : 0; }
int64_t part_d_floats(const StateScan& a, const Pieces& p) { return a.B * p.count * a.D * (a.N + 2); }

template <typename T, int L, bool W, bool BACK>
void join_pieces(const StateScan& a, SeqRef dy, Pieces& p, const Part& part, float* scratch, cudaStream_t s) {
  if (p.count == 1) return;  // (what is carried is its end)
  p.ends = scratch;
  p.steps = scratch + a.B * p.count * a.D * a.N;
  launch(scan_ends_kernel<T, L, W, BACK>, sizeof(EndsShared<T, L, W>), a, p.count, s, dy, p, part.first);
  scan_join_kernel<BACK><<<(unsigned)((a.B * a.D * a.N + 255) / 256), 256, 0, s>>>(a, p, part);
  DLVK_POST_LAUNCH();
}

// The sums by tile (part_bc) have a row of 8 L floats a tile and token: at 64 states 32 times
// bf16 operands, 17 GB for 65536 tokens x 4096 channels.  So a backward pass goes in parts whose
// sums fit the room of the states that the forward pass kept, or 1 GB.  Of bf16 and 64 states
// 64 x 512 x 2048 takes 7073 us whole and 7178 in parts of whole sequences (7252 of some spans of all
// of them; 256 x 128 x 2048 7206, 7228 and 8030).  Parts of fewer blocks than PART_BLOCKS leave SMs
// without work at their ends: below it they are some spans of all sequences, from the last on
// (32 x 4096 x 512 7240 whole, 7300 so, 9546 in whole sequences).
struct Parts {
  int64_t sequences, spans;  // of a part
  bool along = false;        // the tokens: what crosses a border is carried
};
constexpr int64_t PART_FLOATS = 256LL << 20, PART_BLOCKS = 148 * 8;
Parts parts_of(const StateScan& a) {
  const int64_t spans = (a.T + SPAN - 1) / SPAN, tiles = a.G * tiles_of(a), span = (int64_t)SPAN * 2 * NS * lanes_of(a.N);
  const int64_t room = std::max(PART_FLOATS, a.B * spans * a.D * a.N);
  Parts p{std::max<int64_t>(a.B, 1), std::max<int64_t>(spans, 1)};
  if (a.B * tiles * spans * span <= room) return p;
  const auto equal = [](int64_t all, int64_t most) {
    const int64_t n = (all + most - 1) / most;
    return (all + n - 1) / n;
  };
  const int64_t whole = room / (spans * span);  // blocks whose sums of all tokens fit
  if (whole >= std::max(PART_BLOCKS, tiles)) {
    p.sequences = equal(a.B, whole / tiles);
  } else {
    p.spans = equal(spans, std::max<int64_t>(1, room / (a.B * tiles * span)));
    p.along = p.spans < spans;
  }
  return p;
}
SeqRef from(SeqRef r, DType type, int64_t b, int64_t t) {
  if (r.p) r.p = static_cast<char*>(r.p) + (b * r.batch + t * r.token) * (type == DType::BF16 ? 2 : 4);
  return r;
}
// f(the part's operands, its first sequence and span), the last tokens first.
template <typename F>
void each_part(const StateScan& a, const Parts& p, F&& f) {
  const int64_t spans = std::max<int64_t>(1, (a.T + SPAN - 1) / SPAN);
  for (int64_t b = 0; b < a.B; b += p.sequences)
    for (int64_t k = (spans - 1) / p.spans * p.spans; k >= 0; k -= p.spans) {
      StateScan v = a;
      const int64_t t = k * SPAN;
      v.B = std::min(p.sequences, a.B - b);
      v.T = std::min(p.spans * SPAN, a.T - t);
      for (SeqRef* r : {&v.u, &v.dt, &v.z, &v.b, &v.c}) *r = from(*r, a.type, b, t);
      if (v.lengths) v.lengths += b;
      f(v, b, k);
    }
}
// Scratch of a backward pass, in floats: sums by tile of one part, rows of sums for the
// parameters of all parts, what is carried, ends of one part's pieces.
struct BwdScratch {
  int64_t bc = 0, d = 0, carry = 0, ends = 0;
  int64_t all() const { return bc + d + carry + ends; }
};
}  // namespace

// Four sequences a thread where that still makes this many blocks: 64 x 1536 channels of 16
// states 12.3 -> 10.2 us, 130 x 1600 of 64 53 -> 33; below it four are as fast as one, or slower.
constexpr int64_t STEP_BLOCKS = 148 * 4;

int64_t state_scan_fwd_scratch_floats(const StateScan& a) {
  check(a);
  return pieces_floats(a, pieces_of(a, FWD_BLOCKS, FWD_PIECES));
}

void state_scan_fwd(const StateScan& a, SeqRef y, float* out_state, float* saved, float* scratch, cudaStream_t s) {
  check(a);
  if (a.B == 0 || a.D == 0) return;
  by_kind(a, wide_operands(a) && aligned(y, a.type) && aligned16(out_state), [&](auto type, auto lanes, auto wide) {
    using T = decltype(type);
    constexpr int L = decltype(lanes)::value;
    constexpr bool W = decltype(wide)::value;
    if (a.T == 1) {
      constexpr int CH = THREADS / L, R = 4;
      const int64_t tiles = (a.D + CH - 1) / CH, many = tiles * ((a.B + R - 1) / R);
      DLVK_CHECK(tiles * a.B < (1LL << 31), "state_scan: too many channels for one launch");
      if (many >= STEP_BLOCKS)
        scan_step_kernel<T, L, W, R><<<(unsigned)many, THREADS, 0, s>>>(a, y, out_state, saved);
      else
        scan_step_kernel<T, L, W, 1><<<(unsigned)(tiles * a.B), THREADS, 0, s>>>(a, y, out_state, saved);
      DLVK_POST_LAUNCH();
      return;
    }
    Pieces p = pieces_of(a, FWD_BLOCKS, FWD_PIECES);
    join_pieces<T, L, W, false>(a, {}, p, {}, scratch, s);
    launch(scan_fwd_kernel<T, L, W>, sizeof(FwdShared<T, L, W>), a, p.count, s, y, out_state, saved, p);
  });
}

namespace {
BwdScratch bwd_scratch(const StateScan& a, const Parts& parts) {
  const auto fours = [](int64_t n) { return (n + 3) / 4 * 4; };
  BwdScratch r;
  each_part(a, parts, [&](const StateScan& v, int64_t, int64_t) {
    const Pieces p = pieces_of(v, BWD_BLOCKS, BWD_PIECES);
    r.bc = std::max(r.bc, part_bc_floats(v));
    r.d += part_d_floats(v, p);
    r.ends = std::max(r.ends, pieces_floats(v, p));
  });
  r.d = fours(r.d);
  if (parts.along) r.carry = fours(a.B * a.D * a.N);
  return r;
}
void join_bc(const StateScan& a, const float* part_bc, const StateScanGrads& g, cudaStream_t s) {
  const int states = NS * lanes_of(a.N);
  const int64_t total = a.B * a.T * a.G * 2 * states;
  if (total == 0) return;
  const unsigned blocks = (unsigned)std::min<int64_t>((total + 255) / 256, 148 * 16);
  if (a.type == DType::BF16)
    join_bc_kernel<__nv_bfloat16><<<blocks, 256, 0, s>>>(part_bc, tiles_of(a), a.B, a.T, a.G, a.N, states, g.db, g.dc);
  else
    join_bc_kernel<float><<<blocks, 256, 0, s>>>(part_bc, tiles_of(a), a.B, a.T, a.G, a.N, states, g.db, g.dc);
  DLVK_POST_LAUNCH();
}
}  // namespace

int64_t state_scan_bwd_scratch_floats(const StateScan& a) {
  check(a);
  return bwd_scratch(a, parts_of(a)).all();
}

void state_scan_bwd(const StateScan& a, const float* saved, SeqRef dy, const StateScanGrads& g, float* scratch,
                    cudaStream_t s) {
  check(a);
  if (a.D == 0) return join_bc(a, nullptr, g, s);  // sums of no tiles
  const Parts parts = parts_of(a);
  const BwdScratch room = bwd_scratch(a, parts);
  float* part_bc = scratch;
  float* part_d = part_bc + room.bc;
  float* carry = part_d + room.d;
  float* ends = carry + room.carry;
  const int64_t spans = (a.T + SPAN - 1) / SPAN;
  int64_t rows = 0;
  each_part(a, parts, [&](const StateScan& v, int64_t b, int64_t k) {
    Pieces p = pieces_of(v, BWD_BLOCKS, BWD_PIECES);
    Part part{k * SPAN, spans};
    if (parts.along && k + parts.spans < spans) part.in = p.ends = carry;
    if (parts.along && k > 0) part.out = carry;
    const auto of = [&](const SeqRef& r) { return from(r, a.type, b, k * SPAN); };
    StateScanGrads h = g;
    for (SeqRef* r : {&h.du, &h.ddt, &h.dz, &h.db, &h.dc}) *r = of(*r);
    const SeqRef go = of(dy);
    const float* kept = saved + (b * spans + k) * a.D * a.N;
    const bool w = wide_operands(v) && aligned(go, a.type) && aligned(h.du, a.type) && aligned(h.ddt, a.type) &&
                   aligned(h.dz, a.type) && aligned16(kept);
    by_kind(v, w, [&](auto type, auto lanes, auto wide) {
      using T = decltype(type);
      constexpr int L = decltype(lanes)::value;
      constexpr bool W = decltype(wide)::value;
      join_pieces<T, L, W, true>(v, go, p, part, ends, s);
      if (p.count > 1) part.out = nullptr;  // joining the pieces has passed it on
      launch(parts.along ? scan_bwd_kernel<T, L, W, true> : scan_bwd_kernel<T, L, W, false>, sizeof(BwdShared<T, L, W>), v,
             p.count, s, kept, go, h, part_bc, part_d + rows * a.D * (a.N + 2), p, part);
    });
    join_bc(v, part_bc, h, s);
    rows += v.B * p.count;
  });
  join_d_kernel<<<(unsigned)(((int64_t)a.D * (a.N + 2) + 255) / 256), 256, 0, s>>>(part_d, rows, a.D, a.N, g);
  DLVK_POST_LAUNCH();
}

}  // namespace dlvk
