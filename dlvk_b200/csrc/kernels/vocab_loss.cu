// Softmax cross entropy of a vocabulary projection: the passes around the
// tensor-core ones of gemm_tc.cu (EPI 3 and 4), and the same steps on logits
// in memory for the operands those do not take (fp32, a handful of classes).
//
//   z = x W + b        loss_i = log sum_v exp(z_iv) - z_i,label
//   dz_iv = (exp(z_iv) / sum - [v = label]) * g      dx = dz W^T   dW = x^T dz   db = sum_i dz
//
// The reference computes the loss from stored probabilities
// (src/loss/loss_functions.cpp:127-160).  Here the logits of the whole
// vocabulary never reach memory: a first product keeps a maximum and a sum
// per row and 128 (64) classes, ce_finish joins them, and a second product
// makes the logits again, a piece of the vocabulary at a time, and leaves only
// their gradient, which the two gradient products then read.  That is four
// products for the three that the gradient cannot do without; what it saves
// is two [rows, classes] arrays and a pass over each.
#include <algorithm>

#include "dlvk/common.h"
#include "dlvk/kernels.h"

namespace dlvk {
namespace {

constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ int row_label(const CeRows& r, int64_t i) {
  const int64_t lab = r.labels64 ? reinterpret_cast<const int64_t*>(r.labels)[i]
                                 : (int64_t) reinterpret_cast<const int32_t*>(r.labels)[i];
  return (lab >= 0 && lab < r.classes && lab != r.ignore) ? (int)lab : -1;
}

// (m, s) joined with (m2, s2), s = sum of exp(z - m); a maximum of -inf stands
// for "every logit masked" (its s is 0, or NaN when a NaN was among them).
// The scaling to powers of 2 comes after the difference, which a mask of
// fp32's lowest value survives.
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float mn = fmaxf(m, m2);
  const float c = mn == -INFINITY ? 0.f : mn;
  s = s * exp2f((m - c) * LOG2E) + s2 * exp2f((m2 - c) * LOG2E);
  m = mn;
}

constexpr int FIN_ROWS = 32;

// A block joins 32 rows (lane = row, warps share the columns), copies their x
// rows when asked, and adds up their losses; the block that comes last adds
// the blocks' sums in their order.
template <typename T>
__global__ void __launch_bounds__(256) finish_kernel(CeRows r, const float2* __restrict__ stats, int cols,
                                                     const float* __restrict__ zlabel, float* __restrict__ rows_loss,
                                                     float2* __restrict__ norm, int mean,
                                                     const float* __restrict__ grad_scale, float* __restrict__ loss,
                                                     float* __restrict__ gscale,
                                                     unsigned long long* __restrict__ correct,
                                                     double* __restrict__ partial, unsigned* __restrict__ done,
                                                     const T* __restrict__ x, int64_t ldx, int64_t width,
                                                     T* __restrict__ x_clean, int64_t ldc, int vec) {
  __shared__ float sm_m[8][FIN_ROWS], sm_s[8][FIN_ROWS];
  __shared__ int counted[FIN_ROWS];
  __shared__ int last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row0 = (int64_t)blockIdx.x * FIN_ROWS, row = row0 + lane;
  float m = -INFINITY, s = 0.f;
  if (row < r.rows) {
    int c = warp;
    for (; c + 24 < cols; c += 32) {
      float2 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = stats[(int64_t)(c + 8 * k) * r.rows + row];
#pragma unroll
      for (int k = 0; k < 4; ++k) join(m, s, v[k].x, v[k].y);
    }
    for (; c < cols; c += 8) {
      const float2 v = stats[(int64_t)c * r.rows + row];
      join(m, s, v.x, v.y);
    }
  }
  sm_m[warp][lane] = m;
  sm_s[warp][lane] = s;
  __syncthreads();
  if (warp == 0) {
    for (int w = 1; w < 8; ++w) join(m, s, sm_m[w][lane], sm_s[w][lane]);
    int lab = -1, hit = 0;
    float l = 0.f;
    if (row < r.rows) {
      lab = row_label(r, row);
      norm[row] = make_float2(m, 1.f / s);
      if (lab >= 0) {
        const float z = zlabel[row];
        l = (m - z) + logf(s);
        hit = z >= m;
      }
      rows_loss[row] = l;
    }
    counted[lane] = lab >= 0;
    double d = l;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    const int n = __popc(__ballot_sync(0xffffffffu, lab >= 0));
    const int h = __popc(__ballot_sync(0xffffffffu, hit));
    if (lane == 0) {
      partial[3 * blockIdx.x] = d;
      partial[3 * blockIdx.x + 1] = n;
      partial[3 * blockIdx.x + 2] = h;
      __threadfence();
      last = atomicAdd(done, 1u) == gridDim.x - 1;
    }
  }
  __syncthreads();
  if (x_clean != nullptr) {
    for (int k = warp; k < FIN_ROWS && row0 + k < r.rows; k += 8) {
      const T* src = x + (row0 + k) * ldx;
      T* dst = x_clean + (row0 + k) * ldc;
      if (vec) {  // rows of whole 16-byte steps
        constexpr int V = 16 / (int)sizeof(T);
        for (int64_t c = lane * V; c < width; c += 32 * V)
          *reinterpret_cast<uint4*>(dst + c) =
              counted[k] ? *reinterpret_cast<const uint4*>(src + c) : make_uint4(0u, 0u, 0u, 0u);
      } else {
        for (int64_t c = lane; c < width; c += 32) dst[c] = counted[k] ? src[c] : from_f32<T>(0.f);
      }
    }
  }
  if (!last) return;
  // every block's sums are visible: their writers fenced before they counted
  __threadfence();
  double d = 0.0, n = 0.0, h = 0.0;
  for (unsigned b = threadIdx.x; b < gridDim.x; b += 256) {
    d += __ldcg(partial + 3 * b);
    n += __ldcg(partial + 3 * b + 1);
    h += __ldcg(partial + 3 * b + 2);
  }
  __shared__ double sm_d[3][8];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    d += __shfl_xor_sync(0xffffffffu, d, o);
    n += __shfl_xor_sync(0xffffffffu, n, o);
    h += __shfl_xor_sync(0xffffffffu, h, o);
  }
  if (lane == 0) {
    sm_d[0][warp] = d;
    sm_d[1][warp] = n;
    sm_d[2][warp] = h;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    d = n = h = 0.0;
    for (int w = 0; w < 8; ++w) {
      d += sm_d[0][w];
      n += sm_d[1][w];
      h += sm_d[2][w];
    }
    // no row counts: the loss and every gradient are 0
    const double share = mean ? (n > 0.0 ? 1.0 / n : 0.0) : 1.0;
    *loss = (float)(d * share);
    *gscale = (float)(share * (grad_scale ? (double)*grad_scale : 1.0));
    if (correct) *correct += (unsigned long long)h;
  }
}

// One row of logits per block.
__global__ void __launch_bounds__(256) piece_stats_kernel(CeRows r, const float* __restrict__ z, int64_t ldz,
                                                          int64_t col0, int64_t n, float2* __restrict__ stats,
                                                          float* __restrict__ zlabel, unsigned* __restrict__ done) {
  __shared__ float sm_m[8], sm_s[8];
  if (blockIdx.x == 0 && threadIdx.x == 0) *done = 0u;
  const int64_t row = blockIdx.x;
  const float* p = z + row * ldz;
  const int64_t at = row_label(r, row) - col0;
  float m = -INFINITY, s = 0.f;
  for (int64_t c = threadIdx.x; c < n; c += 4 * 256) {
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = c + k * 256 < n ? p[c + k * 256] : -INFINITY;
    const float mn = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), m);
    const float b = mn == -INFINITY ? 0.f : mn;
    s *= exp2f((m - b) * LOG2E);
#pragma unroll
    for (int k = 0; k < 4; ++k) s += exp2f((v[k] - b) * LOG2E);
    m = mn;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    join(m, s, m2, s2);
  }
  if ((threadIdx.x & 31) == 0) {
    sm_m[threadIdx.x >> 5] = m;
    sm_s[threadIdx.x >> 5] = s;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) join(m, s, sm_m[w], sm_s[w]);
    stats[row] = make_float2(m, s);
    if (at >= 0 && at < n && row_label(r, row) >= 0) zlabel[row] = p[at];
  }
}

__global__ void __launch_bounds__(256) piece_grad_kernel(CeRows r, float* __restrict__ z, int64_t ldz, int64_t col0,
                                                         int64_t n, const float2* __restrict__ norm,
                                                         const float* __restrict__ gscale,
                                                         __nv_bfloat16* __restrict__ dl) {
  const int64_t row = blockIdx.x;
  float* p = z + row * ldz;
  const int lab = row_label(r, row);
  const int64_t at = lab - col0;
  const float g = *gscale;
  const float2 nr = norm[row];
  const float f = nr.y * g;
  for (int64_t c = threadIdx.x; c < n; c += 256) {
    float v = 0.f;
    if (lab >= 0) {
      v = exp2f((p[c] - nr.x) * LOG2E) * f;
      if (c == at) v -= g;
    }
    p[c] = v;
    if (dl) dl[row * ldz + c] = __float2bfloat16_rn(v);
  }
}

template <typename TD, typename TS>
__global__ void __launch_bounds__(256) copy_matrix_kernel(const TS* __restrict__ src, int64_t rs, int64_t cs,
                                                          TD* __restrict__ dst, int64_t ldd, int64_t rows, int64_t cols,
                                                          int64_t pad_to, int accumulate) {
  for (int64_t i = blockIdx.y; i < rows; i += gridDim.y) {
    for (int64_t c = blockIdx.x * 1024 + threadIdx.x; c < pad_to; c += (int64_t)gridDim.x * 1024) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t j = c + k * 256;
        if (j >= pad_to) break;
        float v = j < cols ? to_f32(src[i * rs + j * cs]) : 0.f;
        if (accumulate) v += to_f32(dst[i * ldd + j]);
        dst[i * ldd + j] = from_f32<TD>(v);
      }
    }
  }
}

template <typename TD, typename TS>
void copy_matrix_t(const void* src, int64_t rs, int64_t cs, void* dst, int64_t ldd, int64_t rows, int64_t cols,
                   int64_t pad_to, bool accumulate, cudaStream_t s) {
  const dim3 grid((unsigned)std::min<int64_t>((pad_to + 1023) / 1024, 64), (unsigned)std::min<int64_t>(rows, 65535));
  copy_matrix_kernel<TD, TS><<<grid, 256, 0, s>>>(reinterpret_cast<const TS*>(src), rs, cs, reinterpret_cast<TD*>(dst),
                                                  ldd, rows, cols, pad_to, accumulate ? 1 : 0);
  DLVK_POST_LAUNCH();
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T>
void finish_t(const CeRows& r, const float2* stats, int stat_cols, const float* zlabel, float* rows_loss, float2* norm,
              bool mean, const float* grad_scale, float* loss, float* gscale, unsigned long long* correct,
              double* partial, unsigned* done, const void* x, int64_t ldx, int64_t width, void* x_clean, int64_t ldc,
              cudaStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  const int vec = al16(x) && al16(x_clean) && ldx % V == 0 && ldc % V == 0 && width % V == 0;
  finish_kernel<T><<<(unsigned)((r.rows + FIN_ROWS - 1) / FIN_ROWS), 256, 0, s>>>(
      r, stats, stat_cols, zlabel, rows_loss, norm, mean ? 1 : 0, grad_scale, loss, gscale, correct, partial, done,
      reinterpret_cast<const T*>(x), ldx, width, reinterpret_cast<T*>(x_clean), ldc, vec);
  DLVK_POST_LAUNCH();
}

}  // namespace

void ce_finish(const CeRows& r, const float2* stats, int stat_cols, const float* zlabel, float* rows_loss, float2* norm,
               bool mean, const float* grad_scale, float* loss, float* gscale, unsigned long long* correct,
               double* partial, unsigned* done, DType dt, const void* x, int64_t ldx, int64_t width, void* x_clean,
               int64_t ldc, cudaStream_t s) {
  if (dt == DType::F32)
    finish_t<float>(r, stats, stat_cols, zlabel, rows_loss, norm, mean, grad_scale, loss, gscale, correct, partial,
                    done, x, ldx, width, x_clean, ldc, s);
  else
    finish_t<__nv_bfloat16>(r, stats, stat_cols, zlabel, rows_loss, norm, mean, grad_scale, loss, gscale, correct,
                            partial, done, x, ldx, width, x_clean, ldc, s);
}

void ce_piece_stats(const CeRows& r, const float* z, int64_t ldz, int64_t col0, int64_t n, float2* stats,
                    float* zlabel, unsigned* done, cudaStream_t s) {
  piece_stats_kernel<<<(unsigned)r.rows, 256, 0, s>>>(r, z, ldz, col0, n, stats, zlabel, done);
  DLVK_POST_LAUNCH();
}

void ce_piece_grad(const CeRows& r, float* z, int64_t ldz, int64_t col0, int64_t n, const float2* norm,
                   const float* gscale, __nv_bfloat16* dl, cudaStream_t s) {
  piece_grad_kernel<<<(unsigned)r.rows, 256, 0, s>>>(r, z, ldz, col0, n, norm, gscale, dl);
  DLVK_POST_LAUNCH();
}

void copy_matrix(DType dst_dt, DType src_dt, const void* src, int64_t rs, int64_t cs, void* dst, int64_t ldd,
                 int64_t rows, int64_t cols, int64_t pad_to, bool accumulate, cudaStream_t s) {
  if (rows == 0 || pad_to == 0) return;
  if (dst_dt == DType::F32 && src_dt == DType::F32)
    copy_matrix_t<float, float>(src, rs, cs, dst, ldd, rows, cols, pad_to, accumulate, s);
  else if (dst_dt == DType::F32)
    copy_matrix_t<float, __nv_bfloat16>(src, rs, cs, dst, ldd, rows, cols, pad_to, accumulate, s);
  else if (src_dt == DType::F32)
    copy_matrix_t<__nv_bfloat16, float>(src, rs, cs, dst, ldd, rows, cols, pad_to, accumulate, s);
  else
    copy_matrix_t<__nv_bfloat16, __nv_bfloat16>(src, rs, cs, dst, ldd, rows, cols, pad_to, accumulate, s);
}

}  // namespace dlvk
