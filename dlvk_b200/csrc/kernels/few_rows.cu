// fp32 products with a dimension of at most 16: x W, dz W^T and x^T dz of a
// vocabulary projection for a handful of tokens.
//
// A tensor-core tile would be mostly padding, and splitting the weight into
// bf16 parts would write and read 6 bytes for each 4 of a weight that is needed
// once.  Here every weight element is read (or, for x^T dz, every output
// written) once, straight from memory.  8 x 520 x 58220, 121 MB of weight: loss
// and gradients 142 us, of which x W 44 + 5 joining its parts, dz W^T 47 + 12,
// x^T dz 22, passes over the logits 13; the weight's two reads and dW's write are
// 55 at the copy rate, so the two products that read are bound by their loads in
// flight and their sums, not by HBM (in parts on the tensor cores the call took
// 353).  Sums are fp32 fused multiply-adds in a fixed order.
#include <algorithm>
#include <type_traits>

#include "dlvk/common.h"
#include "dlvk/kernels.h"

namespace dlvk {
namespace {

constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr int KC = 512;  // columns of A staged at a time

template <int VEC>
__device__ __forceinline__ void load_cols(const float* p, int64_t c, int64_t cols, float* v) {
  if constexpr (VEC == 4) {
    const float4 u = c < cols ? *reinterpret_cast<const float4*>(p + c) : make_float4(0.f, 0.f, 0.f, 0.f);
    v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
  } else {
    v[0] = c < cols ? p[c] : 0.f;
  }
}

// A[n, k0 + j] for n < NR, j < KC into shared memory; zeros outside.
template <int NR>
__device__ __forceinline__ void stage(float (*As)[KC], const float* A, int64_t lda, int rows, int64_t k0, int64_t k1) {
  for (int i = threadIdx.x; i < NR * KC; i += THREADS) {
    const int n = i / KC, j = i % KC;
    As[n][j] = (n < rows && k0 + j < k1) ? A[n * lda + k0 + j] : 0.f;
  }
}

// out[n, c] = sum_k A[n, k] B[k, c], B's rows contiguous.  A block has 32 VEC
// columns and a part of k, whose rows its warps take in turn; the warps' sums
// are added in their order.  Several parts: out is [part][rows][cols].
template <int NR, int VEC>
__global__ void __launch_bounds__(THREADS) few_nn_kernel(const float* __restrict__ A, int64_t lda,
                                                         const float* __restrict__ B, int64_t ldb,
                                                         const float* __restrict__ bias, float* __restrict__ out,
                                                         int64_t ldo, int rows, int64_t K, int64_t cols, int64_t per,
                                                         int64_t part_stride) {
  pdl_wait();
  __shared__ __align__(16) float As[NR][KC];
  __shared__ float red[NR][32 * VEC];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = ((int64_t)blockIdx.x * 32 + lane) * VEC;
  const int64_t lo = blockIdx.y * per, hi = min(K, lo + per);
  float acc[NR][VEC];
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[n][j] = 0.f;
  for (int64_t k0 = lo; k0 < hi; k0 += KC) {
    __syncthreads();
    stage<NR>(As, A, lda, rows, k0, hi);
    __syncthreads();
    const int n_k = (int)min((int64_t)KC, hi - k0);
    // a warp takes four consecutive k at a time, twice: 16 bytes of A each
    for (int k = 4 * warp; k < n_k; k += 2 * 4 * WARPS) {
      float b[8][VEC];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int kk = k + (u >> 2) * 4 * WARPS + (u & 3);
        if (kk < n_k) {
          load_cols<VEC>(B + (k0 + kk) * ldb, c, cols, b[u]);
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) b[u][j] = 0.f;
        }
      }
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int kk = k + g * 4 * WARPS;
        if (kk >= n_k) break;
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          const float4 a = *reinterpret_cast<const float4*>(&As[n][kk]);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            acc[n][j] = fmaf(a.x, b[4 * g][j], acc[n][j]);
            acc[n][j] = fmaf(a.y, b[4 * g + 1][j], acc[n][j]);
            acc[n][j] = fmaf(a.z, b[4 * g + 2][j], acc[n][j]);
            acc[n][j] = fmaf(a.w, b[4 * g + 3][j], acc[n][j]);
          }
        }
      }
    }
  }
  for (int w = 0; w < WARPS; ++w) {
    if (warp == w) {
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          float* r = &red[n][lane * VEC + j];
          *r = w == 0 ? acc[n][j] : *r + acc[n][j];
        }
    }
    __syncthreads();
  }
  float* o = out + blockIdx.y * part_stride;
  for (int i = threadIdx.x; i < NR * 32 * VEC; i += THREADS) {
    const int n = i / (32 * VEC), j = i % (32 * VEC);
    const int64_t col = (int64_t)blockIdx.x * 32 * VEC + j;
    if (n < rows && col < cols) o[n * ldo + col] = red[n][j] + (bias != nullptr ? bias[col] : 0.f);
  }
}

// Sum over the 32 lanes of COUNT values each (a power of two), by halving:
// lane l ends with the values l * COUNT / 32 onwards (COUNT >= 32), or value
// l * COUNT / 32 (COUNT < 32), in v[0..].
template <int COUNT, int H = 16>
__device__ __forceinline__ void lane_sums(float* v, int lane) {
  if constexpr (H >= 1) {
    if constexpr (COUNT > 1) {
      constexpr int M = COUNT / 2;
      const bool up = (lane & H) != 0;
#pragma unroll
      for (int j = 0; j < M; ++j) {
        const float send = up ? v[j] : v[j + M];
        const float keep = up ? v[j + M] : v[j];
        v[j] = keep + __shfl_xor_sync(0xffffffffu, send, H);
      }
      lane_sums<M, H / 2>(v, lane);
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], H);
      lane_sums<1, H / 2>(v, lane);
    }
  }
}

// out[n, r] = sum_k A[n, k] B[r, k], B's rows contiguous.  A block has a part
// of k, at most KT, whose columns of A it stages once, and goes through groups
// of 32 rows of B; a warp has four of them, its lanes share k (so that what is
// read of A serves four rows).
constexpr int RR = 4, KT = 1024;
template <int NR, int VEC>
__global__ void __launch_bounds__(THREADS) few_nt_kernel(const float* __restrict__ A, int64_t lda,
                                                         const float* __restrict__ B, int64_t ldb,
                                                         const float* __restrict__ bias, float* __restrict__ out,
                                                         int64_t ldo, int rows, int64_t K, int64_t brows, int64_t per,
                                                         int64_t part_stride) {
  pdl_wait();
  extern __shared__ __align__(16) float At[];  // [NR][width]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t lo = blockIdx.y * per, hi = min(K, lo + per);
  const int steps = (int)((hi - lo + 32 * VEC - 1) / (32 * VEC)), width = steps * 32 * VEC;
  for (int n = 0; n < NR; ++n)
    for (int j = threadIdx.x; j < width; j += THREADS)
      At[n * width + j] = (n < rows && lo + j < hi) ? A[n * lda + lo + j] : 0.f;
  __syncthreads();
  for (int64_t group = blockIdx.x; group * (WARPS * RR) < brows; group += gridDim.x) {
    const int64_t r0 = (group * WARPS + warp) * RR;
    float acc[NR * RR];  // [n][row]
#pragma unroll
    for (int i = 0; i < NR * RR; ++i) acc[i] = 0.f;
#pragma unroll 2
    for (int s = 0; s < steps; ++s) {
      const int j0 = (s * 32 + lane) * VEC;
      float b[RR][VEC];
#pragma unroll
      for (int r = 0; r < RR; ++r) {
        if (r0 + r < brows) {
          load_cols<VEC>(B + (r0 + r) * ldb, lo + j0, hi, b[r]);
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) b[r][j] = 0.f;
        }
      }
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        float a[VEC];
        if constexpr (VEC == 4) {
          const float4 u = *reinterpret_cast<const float4*>(At + n * width + j0);
          a[0] = u.x; a[1] = u.y; a[2] = u.z; a[3] = u.w;
        } else {
          a[0] = At[n * width + j0];
        }
#pragma unroll
        for (int r = 0; r < RR; ++r)
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[n * RR + r] = fmaf(a[j], b[r][j], acc[n * RR + r]);
      }
    }
    lane_sums<NR * RR>(acc, lane);
    constexpr int PER = NR * RR >= 32 ? NR * RR / 32 : 1;      // values of a lane
    constexpr int SHARE = NR * RR >= 32 ? 1 : 32 / (NR * RR);  // lanes that hold the same value
    if (lane % SHARE != 0) continue;
    float* o = out + blockIdx.y * part_stride;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = lane / SHARE * PER + i, n = at / RR;
      const int64_t r = r0 + at % RR;
      if (n < rows && r < brows) o[n * ldo + r] = acc[i] + (bias != nullptr ? bias[r] : 0.f);
    }
  }
}

// out[n, c] = sum over the parts in their order (+ bias).
__global__ void __launch_bounds__(256) few_join_kernel(const float* __restrict__ parts, int count, int64_t part_stride,
                                                       const float* __restrict__ bias, float* __restrict__ out,
                                                       int64_t ldo, int rows, int64_t cols) {
  pdl_wait();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * cols) return;
  const int64_t n = i / cols, c = i - n * cols;
  float s = 0.f;
  for (int p = 0; p < count; p += 8) {
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = p + u < count ? parts[(p + u) * part_stride + i] : 0.f;
#pragma unroll
    for (int u = 0; u < 8; ++u) s += v[u];
  }
  out[n * ldo + c] = s + (bias != nullptr ? bias[c] : 0.f);
}

// out[a, c] (+)= sum_n P[n, a] Q[n, c].  A thread holds VEC columns of Q for
// NR rows and goes through a part of a.
template <int NR, int VEC>
__global__ void __launch_bounds__(THREADS) few_outer_kernel(const float* __restrict__ P, int64_t ldp,
                                                            const float* __restrict__ Q, int64_t ldq,
                                                            float* __restrict__ out, int64_t ldo, int rows, int64_t A,
                                                            int64_t cols, int64_t per, int accumulate) {
  pdl_wait();
  constexpr int AC = 128;
  __shared__ float Ps[AC][NR];
  const int64_t c = ((int64_t)blockIdx.x * THREADS + threadIdx.x) * VEC;
  const int64_t lo = blockIdx.y * per, hi = min(A, lo + per);
  float q[NR][VEC];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    if (n < rows) {
      load_cols<VEC>(Q + n * ldq, c, cols, q[n]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) q[n][j] = 0.f;
    }
  }
  for (int64_t a0 = lo; a0 < hi; a0 += AC) {
    __syncthreads();
    for (int i = threadIdx.x; i < AC * NR; i += THREADS) {
      const int n = i / AC, j = i % AC;
      Ps[j][n] = (n < rows && a0 + j < hi) ? P[n * ldp + a0 + j] : 0.f;
    }
    __syncthreads();
    if (c >= cols) continue;
    const int n_a = (int)min((int64_t)AC, hi - a0);
    for (int j = 0; j < n_a; ++j) {
      float* o = out + (a0 + j) * ldo + c;
      float v[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[k] = 0.f;
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        const float p = Ps[j][n];
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = fmaf(p, q[n][k], v[k]);
      }
      if constexpr (VEC == 4) {
        float4 u = make_float4(v[0], v[1], v[2], v[3]);
        if (accumulate) {
          const float4 w = *reinterpret_cast<const float4*>(o);
          u = make_float4(w.x + u.x, w.y + u.y, w.z + u.z, w.w + u.w);
        }
        *reinterpret_cast<float4*>(o) = u;
      } else {
        *o = accumulate ? *o + v[0] : v[0];
      }
    }
  }
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// How a product is cut: blocks of columns, parts of k, `per` of k to a part.
// Four blocks to an SM where k is long enough; parts are whole stages (KC), or
// (turned) what a block stages once (KT) or less, in multiples of 128, so that
// 16-byte reads of B's rows stay aligned.
struct Cut {
  int64_t blocks, per;
  int parts;
};
Cut cut_of(int64_t K, int64_t cols, bool turned, bool vec) {
  Cut c;
  if (turned) {
    const int64_t groups = (cols + WARPS * RR - 1) / (WARPS * RR);
    const int64_t least = (K + KT - 1) / KT, most = (K + 255) / 256;
    const int64_t want = std::max(least, std::min<int64_t>(most, (4 * 148 + groups - 1) / groups));
    c.per = ((K + want - 1) / want + 127) / 128 * 128;
    c.parts = (int)((K + c.per - 1) / c.per);
    c.blocks = std::min<int64_t>(groups, std::max<int64_t>(1, (4 * 148 + c.parts - 1) / c.parts));
    return c;
  }
  c.blocks = vec ? (cols + 127) / 128 : (cols + 31) / 32;
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>((4 * 148 + c.blocks - 1) / c.blocks, (K + KC - 1) / KC));
  c.per = ((K + want - 1) / want + KC - 1) / KC * KC;
  c.parts = (int)((K + c.per - 1) / c.per);
  return c;
}

// Calls f with the number of rows that a launch keeps, for at most 16 rows.
template <typename F>
void with_rows(int rows, F&& f) {
  if (rows == 1) f(std::integral_constant<int, 1>{});
  else if (rows <= 4) f(std::integral_constant<int, 4>{});
  else if (rows <= 8) f(std::integral_constant<int, 8>{});
  else f(std::integral_constant<int, 16>{});
}

}  // namespace

int64_t few_rows_scratch_floats(int64_t rows, int64_t K, int64_t cols, bool turned) {
  // whichever way its operands' alignment has it cut
  const int parts = std::max(cut_of(K, cols, turned, true).parts, cut_of(K, cols, turned, false).parts);
  return parts > 1 ? parts * rows * cols : 0;
}

void few_rows_product(const float* A, int64_t lda, const float* B, int64_t ldb, bool turned, const float* bias,
                      float* out, int64_t ldo, int64_t rows, int64_t K, int64_t cols, float* scratch, cudaStream_t s) {
  static_assert(KT == 1024, "FEW_ROWS_K");
  DLVK_CHECK(rows >= 1 && rows <= FEW_ROWS && K <= FEW_ROWS_K, "few_rows_product: size");
  DLVK_CHECK(scratch != nullptr || few_rows_scratch_floats(rows, K, cols, turned) == 0, "few_rows_product: scratch");
  const bool vec = al16(B) && ldb % 4 == 0 && (turned ? K : cols) % 4 == 0;
  const int n = (int)rows;
  const Cut cut = cut_of(K, cols, turned, vec);
  const int used = cut.parts;
  const int64_t per = cut.per;
  float* dst = used > 1 ? scratch : out;
  const int64_t ld = used > 1 ? cols : ldo, stride = (int64_t)n * cols;
  const float* b = used > 1 ? nullptr : bias;
  const dim3 grid((unsigned)cut.blocks, (unsigned)used);
  with_rows(n, [&](auto nr) {
    constexpr int NR = decltype(nr)::value;
    const auto go = [&](auto kernel, size_t smem) {
      launch_pdl(kernel, grid, dim3(THREADS), smem, s, A, lda, B, ldb, b, dst, ld, n, K, cols, per, stride);
    };
    if (turned) {
      static bool attr_set[kMaxDevices] = {false};  // of this NR
      const int dev = current_device_slot();
      if (!attr_set[dev]) {
        const int most = NR * KT * (int)sizeof(float);
        const auto attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
        DLVK_CUDA_CHECK(cudaFuncSetAttribute(few_nt_kernel<NR, 4>, attr, most));
        DLVK_CUDA_CHECK(cudaFuncSetAttribute(few_nt_kernel<NR, 1>, attr, most));
        attr_set[dev] = true;
      }
      // a part's columns, rounded up to whole steps of a warp
      const size_t smem = (size_t)NR * ((std::min(per, K) + 127) / 128 * 128) * sizeof(float);
      if (vec) go(few_nt_kernel<NR, 4>, smem);
      else go(few_nt_kernel<NR, 1>, smem);
    } else if (vec) {
      go(few_nn_kernel<NR, 4>, 0);
    } else {
      go(few_nn_kernel<NR, 1>, 0);
    }
  });
  DLVK_POST_LAUNCH();
  if (used > 1) {
    launch_pdl(few_join_kernel, dim3((unsigned)((n * cols + 255) / 256)), dim3(256), 0, s, scratch, used, stride, bias,
               out, ldo, n, cols);
    DLVK_POST_LAUNCH();
  }
}

void few_rows_outer(const float* P, int64_t ldp, const float* Q, int64_t ldq, float* out, int64_t ldo, int64_t rows,
                    int64_t A, int64_t cols, bool accumulate, cudaStream_t s) {
  DLVK_CHECK(rows >= 1 && rows <= FEW_ROWS, "few_rows_outer: rows");
  const bool vec = al16(Q) && al16(out) && ldq % 4 == 0 && ldo % 4 == 0 && cols % 4 == 0;
  const int64_t blocks = (cols + THREADS * (vec ? 4 : 1) - 1) / (THREADS * (vec ? 4 : 1));
  const int64_t want = std::min<int64_t>((8 * 148 + blocks - 1) / blocks, (A + 15) / 16);
  const int64_t per = (A + want - 1) / want;
  const dim3 grid((unsigned)blocks, (unsigned)((A + per - 1) / per));
  with_rows((int)rows, [&](auto nr) {
    constexpr int NR = decltype(nr)::value;
    const auto go = [&](auto kernel) {
      launch_pdl(kernel, grid, dim3(THREADS), 0, s, P, ldp, Q, ldq, out, ldo, (int)rows, A, cols, per,
                 accumulate ? 1 : 0);
    };
    if (vec) go(few_outer_kernel<NR, 4>);
    else go(few_outer_kernel<NR, 1>);
  });
  DLVK_POST_LAUNCH();
}

}  // namespace dlvk
