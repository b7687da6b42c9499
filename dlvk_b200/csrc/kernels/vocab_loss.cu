// Softmax cross entropy of a vocabulary projection: the passes around the
// tensor-core ones of gemm_tc.cu (EPI 3 and 4), and the same steps on logits
// in memory for the operands those do not take (fp32, a handful of classes).
//
//   z = x W + b        loss_i = log sum_v exp(z_iv) - z_i,label
//   dz_iv = (exp(z_iv) / sum - [v = label]) * g      dx = dz W^T   dW = x^T dz   db = sum_i dz
//
// The reference computes the loss from stored probabilities
// (src/loss/loss_functions.cpp:127-160).  Here the logits of the vocabulary
// are taken a tile of 256 words at a time: the first product's epilogue keeps
// a maximum and a sum per row and 128 words, ce_finish joins them.  For the
// gradients a block of rows at a time leaves exp(z - local maximum) behind
// (16 bits: 256 MB, or 4 KB a word where 2048 rows of a vocabulary above 65536
// take more), ce_rescale turns those into dz, and the two gradient products
// read dz: three products, one pass over the block.  Making the logits a second
// time instead costs a fourth product (8192 x 1024 x 32000: 1633 us of kernels
// against 1388); it is what a bias gradient takes, whose fp32 sums 16-bit
// exponentials are too coarse for.
#include <algorithm>

#include <cuda_fp16.h>

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

// x = q0 + q1 + q2 to 2^-24 of x, bf16 each (the split of Henry, Tang and
// Heinecke, 2019): what rounding leaves is exact in fp32 and goes to the next part.  An infinity or NaN is in q0 alone, and a
// finite x above bf16's range is held at its end.
__device__ __forceinline__ void three_parts(float x, __nv_bfloat16* q) {
  q[0] = __float2bfloat16_rn(x);
  q[1] = q[2] = __float2bfloat16_rn(0.f);
  if (!isfinite(x)) return;
  if (fabsf(x) > 3.38953139e38f) q[0] = __float2bfloat16_rn(copysignf(3.38953139e38f, x));
  const float a = x - __bfloat162float(q[0]);
  q[1] = __float2bfloat16_rn(a);
  q[2] = __float2bfloat16_rn(a - __bfloat162float(q[1]));
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

// 1 / counted rows (mean) or 1; no row counts: the loss and every gradient are 0.
__device__ __forceinline__ double share_of(int mean, double counted) {
  return mean ? (counted > 0.0 ? 1.0 / counted : 0.0) : 1.0;
}

__global__ void __launch_bounds__(1024) count_kernel(CeRows r, int mean, const float* __restrict__ grad_scale,
                                                     float* __restrict__ gscale, unsigned* __restrict__ done) {
  pdl_wait();
  __shared__ int sm[32];
  int n = 0;
  for (int64_t i = threadIdx.x; i < r.rows; i += 1024) n += row_label(r, i) >= 0;
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = n;
  __syncthreads();
  if (threadIdx.x < 32) {
    n = __reduce_add_sync(0xffffffffu, sm[threadIdx.x]);
    if (threadIdx.x == 0) {
      *gscale = (float)(share_of(mean, n) * (grad_scale ? (double)*grad_scale : 1.0));
      *done = 0u;
    }
  }
}

constexpr int GROUP = 32;  // rows of one group of the final sums

// The joined statistics of the rows row0 + lane, in every warp's lanes after
// a block's barrier: the warps share the columns.
template <int WARPS>
__device__ __forceinline__ void join_rows(const CeRows& r, const CeFinish& f, int64_t row, float (*sm_m)[GROUP],
                                          float (*sm_s)[GROUP], float& m, float& s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  m = -INFINITY;
  s = 0.f;
  if (row < r.rows) {
    for (int c = warp; c < f.stat_cols; c += 8 * WARPS) {
      float2 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        v[k] = c + k * WARPS < f.stat_cols ? f.stats[(int64_t)(c + k * WARPS) * r.rows + row]
                                           : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int k = 0; k < 8; ++k) join(m, s, v[k].x, v[k].y);
    }
  }
  sm_m[warp][lane] = m;
  sm_s[warp][lane] = s;
  __syncthreads();
  // WARPS neighbouring threads join one row's parts
  const int part = threadIdx.x % WARPS, of = threadIdx.x / WARPS;
  m = sm_m[part][of];
  s = sm_s[part][of];
#pragma unroll
  for (int o = WARPS / 2; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    join(m, s, m2, s2);
  }
  __syncthreads();
  if (part == 0) {
    sm_m[0][of] = m;
    sm_s[0][of] = s;
  }
  __syncthreads();
  m = sm_m[0][lane];
  s = sm_s[0][lane];
}

// Warp 0 of a group's block: the rows' losses and norms, and the group's sums.
// True in lane 0 of the block that comes last of all.
__device__ __forceinline__ bool group_sums(const CeRows& r, const CeFinish& f, int64_t group, int64_t row, bool counted,
                                           float m, float s) {
  const int lane = threadIdx.x & 31;
  int hit = 0;
  float l = 0.f;
  if (row < r.rows) {
    f.norm[row] = make_float2(m, 1.f / s);
    if (counted) {
      const float z = f.zlabel[row];
      l = (m - z) + logf(s);
      hit = z >= m;
    }
    f.rows_loss[row] = l;
  }
  double d = l;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
  const int n = __popc(__ballot_sync(0xffffffffu, counted));
  const int h = __popc(__ballot_sync(0xffffffffu, hit));
  if (lane != 0) return false;
  double* p = f.partial + 3 * ((int64_t)f.first_group + group);
  p[0] = d;
  p[1] = n;
  p[2] = h;
  __threadfence();
  return atomicAdd(f.done, 1u) == (unsigned)f.total_groups - 1u;
}

// A group's x rows, zeros in those that do not count.
template <typename T, int WARPS>
__device__ __forceinline__ void copy_rows(const CeRows& r, const CeFinish& f, int64_t row0, const int* counted,
                                          int vec) {
  const int lane = threadIdx.x & 31;
  const T* x = reinterpret_cast<const T*>(f.x);
  T* y = reinterpret_cast<T*>(f.x_clean);
  for (int k = threadIdx.x >> 5; k < GROUP && row0 + k < r.rows; k += WARPS) {
    const T* src = x + (row0 + k) * f.ldx;
    T* dst = y + (row0 + k) * f.ldc;
    if (vec) {  // rows of whole 16-byte steps
      constexpr int V = 16 / (int)sizeof(T);
      const bool keep = counted[k] != 0;
      for (int64_t c = lane * V; c < f.width; c += 4 * 32 * V) {
        uint4 u[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          u[q] = keep && c + q * 32 * V < f.width ? *reinterpret_cast<const uint4*>(src + c + q * 32 * V)
                                                  : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (c + q * 32 * V < f.width) *reinterpret_cast<uint4*>(dst + c + q * 32 * V) = u[q];
      }
    } else {
      for (int64_t c = lane; c < f.width; c += 32) dst[c] = counted[k] ? src[c] : from_f32<T>(0.f);
    }
  }
}

// The last block: adds the groups' sums in their order.
template <int WARPS>
__device__ __forceinline__ void total_sums(const CeFinish& f) {
  __shared__ double sm_d[3][WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // every group's sums are visible: their writers fenced before they counted
  __threadfence();
  double v[3] = {0.0, 0.0, 0.0};
  for (int b = threadIdx.x; b < f.total_groups; b += WARPS * 32)
#pragma unroll
    for (int k = 0; k < 3; ++k) v[k] += __ldcg(f.partial + 3 * (int64_t)b + k);
#pragma unroll
  for (int k = 0; k < 3; ++k) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    if (lane == 0) sm_d[k][warp] = v[k];
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int k = 0; k < 3; ++k) {
    v[k] = 0.0;
    for (int w = 0; w < WARPS; ++w) v[k] += sm_d[k][w];
  }
  const double share = share_of(f.mean, v[1]);
  *f.loss = (float)(v[0] * share);
  if (f.set_gscale) *f.gscale = (float)(share * (f.grad_scale ? (double)*f.grad_scale : 1.0));
  if (f.loss_sum) *f.loss_sum += (float)v[0];
  if (f.counted) *f.counted += (unsigned long long)v[1];
  if (f.correct) *f.correct += (unsigned long long)v[2];
}

// A block finishes one group of rows; another copies the group's x beside it.
constexpr int FIN_WARPS = 16;
template <typename T>
__global__ void __launch_bounds__(FIN_WARPS * 32) finish_kernel(CeRows r, CeFinish f, int vec) {
  pdl_wait();
  __shared__ float sm_m[FIN_WARPS][GROUP], sm_s[FIN_WARPS][GROUP];
  __shared__ int counted[GROUP];
  __shared__ int last;
  const int lane = threadIdx.x & 31;
  const int64_t row0 = (int64_t)blockIdx.x * GROUP, row = row0 + lane;
  if (threadIdx.x < GROUP) counted[lane] = row < r.rows && row_label(r, row) >= 0;
  if (blockIdx.y != 0) {
    __syncthreads();
    copy_rows<T, FIN_WARPS>(r, f, row0, counted, vec);
    return;
  }
  float m, s;
  join_rows<FIN_WARPS>(r, f, row, sm_m, sm_s, m, s);
  if (threadIdx.x < 32) {
    const bool end = group_sums(r, f, blockIdx.x, row, counted[lane] != 0, m, s);
    if (lane == 0) last = end;
  }
  __syncthreads();
  if (last) total_sums<FIN_WARPS>(f);
}

// e -> dz in place.  A block has a group of 32 rows and 2048 of their classes,
// a thread 8 classes of each; what a row's 2^-15 e is multiplied by, exp(local
// maximum - maximum) / sum, is made once per row and statistics column.  Bound
// by HBM: 2 bytes in, 2 out per logit.  With JOIN the blocks also join the
// statistics, each for itself, and one more block per group does the rest of
// finish_kernel's work beside them: a launch less where the statistics are few.
constexpr int RS_COLS = 2048, RS_WARPS = 8;
template <bool JOIN>
__global__ void __launch_bounds__(RS_WARPS * 32) rescale_kernel(CeRows r, CeFinish f, int vec, int width_shift,
                                                                uint16_t* __restrict__ e, int64_t lde) {
  pdl_wait();
  __shared__ float factor[RS_COLS / 64][GROUP];
  __shared__ int label[GROUP], counted[GROUP];
  __shared__ float2 norm[GROUP];
  // backwards: the exponentials that were written last are still in L2
  const int64_t group = gridDim.y - 1 - blockIdx.y, row0 = group * GROUP;
  const bool sums = JOIN && blockIdx.x == 0;
  const int64_t col0 = (int64_t)(gridDim.x - 1 - blockIdx.x) * RS_COLS;
  const int rows = (int)min((int64_t)GROUP, r.rows - row0);
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < GROUP) {
    label[lane] = lane < rows ? row_label(r, row0 + lane) : -1;
    counted[lane] = label[lane] >= 0;
    if (!JOIN && lane < rows) norm[lane] = f.norm[row0 + lane];
  }
  if constexpr (JOIN) {
    __shared__ float sm_m[RS_WARPS][GROUP], sm_s[RS_WARPS][GROUP];
    __shared__ int last;
    float m, s;
    join_rows<RS_WARPS>(r, f, row0 + lane, sm_m, sm_s, m, s);
    if (threadIdx.x < 32) norm[lane] = make_float2(m, 1.f / s);
    if (sums) {
      if (threadIdx.x < 32) {
        const bool end = group_sums(r, f, group, row0 + lane, counted[lane] != 0, m, s);
        if (lane == 0) last = end;
      }
      copy_rows<__nv_bfloat16, RS_WARPS>(r, f, row0, counted, vec);
      __syncthreads();
      if (last) total_sums<RS_WARPS>(f);
      return;
    }
  }
  __syncthreads();
  const int64_t stat0 = col0 >> width_shift, stats_all = (r.classes + (1 << width_shift) - 1) >> width_shift;
  for (int i = threadIdx.x; i < (RS_COLS >> width_shift) * GROUP; i += RS_WARPS * 32) {
    const int k = i % GROUP, t = i / GROUP;
    float v = 0.f;
    if (k < rows && stat0 + t < stats_all)
      v = exp2f((f.stats[(stat0 + t) * r.rows + row0 + k].x - norm[k].x) * LOG2E) * norm[k].y * (1.f / 32768.f);
    factor[t][k] = v;
  }
  __syncthreads();
  const int64_t col = col0 + threadIdx.x * 8;
  if (col >= r.classes) return;
  const float* mine = factor[(threadIdx.x * 8) >> width_shift];
  uint16_t* p = e + row0 * lde + col;
  for (int k0 = 0; k0 < rows; k0 += 8) {
    uint4 u[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k0 + k < rows) u[k] = *reinterpret_cast<const uint4*>(p + (k0 + k) * lde);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (k0 + k >= rows) break;
      const int lab = label[k0 + k];
      const float fac = mine[k0 + k];
      const __half2* h = reinterpret_cast<const __half2*>(&u[k]);
      float v[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 t = __half22float2(h[j]);
        v[2 * j] = t.x * fac;
        v[2 * j + 1] = t.y * fac;
      }
      const int64_t at = lab - col;
      if (lab < 0) {  // 0 whatever the row's logits were
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.f;
      } else if (at >= 0 && at < 8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] -= j == at ? 1.f : 0.f;
      }
      uint4 o;
      __nv_bfloat162* w = reinterpret_cast<__nv_bfloat162*>(&o);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
      *reinterpret_cast<uint4*>(p + (k0 + k) * lde) = o;
    }
  }
}

// A row of logits and a part of its classes per block: enough parts to fill
// the GPU when rows are few, each a statistics column of its own.
__global__ void __launch_bounds__(256) memory_stats_kernel(CeRows r, const float* __restrict__ z, int64_t ldz,
                                                           int64_t per, float2* __restrict__ stats,
                                                           float* __restrict__ zlabel, unsigned* __restrict__ done) {
  pdl_wait();
  __shared__ float sm_m[8], sm_s[8];
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0 && done != nullptr) *done = 0u;
  const int64_t row = blockIdx.x, lo = blockIdx.y * per, hi = min(r.classes, lo + per);
  const float* p = z + row * ldz;
  float m = -INFINITY, s = 0.f;
  for (int64_t c = lo + threadIdx.x; c < hi; c += 4 * 256) {
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = c + k * 256 < hi ? p[c + k * 256] : -INFINITY;
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
    stats[blockIdx.y * r.rows + row] = make_float2(m, s);
    const int lab = row_label(r, row);
    if (lab >= lo && lab < hi) zlabel[row] = p[lab];
  }
}

// A row and a part of its classes per block, four columns a thread (rows of z
// and of the parts are whole 128-byte lines).
__global__ void __launch_bounds__(256) memory_grad_kernel(CeRows r, float* __restrict__ z, int64_t ldz,
                                                          const float2* __restrict__ norm,
                                                          const float* __restrict__ gscale,
                                                          __nv_bfloat16* __restrict__ dl, int64_t pitch, int keep_z) {
  pdl_wait();
  const int64_t row = blockIdx.x;
  float* p = z + row * ldz;
  const int lab = row_label(r, row);
  const float g = *gscale;
  const float2 n = norm[row];
  const int64_t end = pitch != 0 ? pitch : (r.classes + 3) / 4 * 4;  // the padding becomes 0
  for (int64_t c = 4 * ((int64_t)blockIdx.y * 256 + threadIdx.x); c < end; c += 4 * 256 * (int64_t)gridDim.y) {
    float4 u = make_float4(0.f, 0.f, 0.f, 0.f);
    if (lab >= 0 && c < r.classes) u = *reinterpret_cast<const float4*>(p + c);
    float v[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (lab < 0 || c + k >= r.classes) {
        v[k] = 0.f;
      } else {
        v[k] = exp2f((v[k] - n.x) * LOG2E) * n.y;
        if (c + k == lab) v[k] -= 1.f;
      }
    }
    if (keep_z && c < ldz) *reinterpret_cast<float4*>(p + c) = make_float4(v[0] * g, v[1] * g, v[2] * g, v[3] * g);
    if (dl == nullptr) continue;
    if (pitch == 0) {
#pragma unroll
      for (int k = 0; k < 4; ++k) dl[row * ldz + c + k] = __float2bfloat16_rn(v[k] * g);
    } else {
      __nv_bfloat16 q[4][3];
#pragma unroll
      for (int k = 0; k < 4; ++k) three_parts(v[k], q[k]);
#pragma unroll
      for (int t = 0; t < 3; ++t) {
        __nv_bfloat162 a, b;
        a.x = q[0][t]; a.y = q[1][t]; b.x = q[2][t]; b.y = q[3][t];
        *reinterpret_cast<uint2*>(dl + (row * 3 + t) * pitch + c) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
      }
    }
  }
}

// A block splits rows blockIdx.y, ...; a thread four columns.
__global__ void __launch_bounds__(256) split_parts_kernel(const float* __restrict__ src, int64_t ld, int64_t rows,
                                                          int64_t cols, __nv_bfloat16* __restrict__ dst, int64_t pitch,
                                                          CeRows mask, int masked, int vec) {
  pdl_wait();
  const int64_t c = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x);
  if (c >= pitch) return;
  for (int64_t i = blockIdx.y; i < rows; i += gridDim.y) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (!masked || row_label(mask, i) >= 0) {
      const float* p = src + i * ld + c;
      if (vec && c + 4 <= cols) {
        const float4 u = *reinterpret_cast<const float4*>(p);
        v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (c + k < cols) v[k] = p[k];
      }
    }
    __nv_bfloat16 q[4][3];
#pragma unroll
    for (int k = 0; k < 4; ++k) three_parts(v[k], q[k]);
#pragma unroll
    for (int t = 0; t < 3; ++t) {
      __nv_bfloat162 a, b;
      a.x = q[0][t]; a.y = q[1][t]; b.x = q[2][t]; b.y = q[3][t];
      *reinterpret_cast<uint2*>(dst + i * 3 * pitch + t * pitch + c) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
  }
}

template <typename TD, typename TS>
__global__ void __launch_bounds__(256) copy_matrix_kernel(const TS* __restrict__ src, int64_t rs, int64_t cs,
                                                          TD* __restrict__ dst, int64_t ldd, int64_t rows, int64_t cols,
                                                          int64_t pad_to, int accumulate) {
  pdl_wait();
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

// bf16 rows from and to any alignment (an odd number of classes): zeros behind
// `cols` up to `pad_to`.  A thread stores eight elements as 16 aligned bytes; they
// are read as 4-byte words, five where the row's elements lie across them, which
// takes in one element before and one behind, so at the row's ends one by one.
// TX threads go along a row (552 x 54665: 28 us; an element a thread 72).
__global__ void __launch_bounds__(256) realign_kernel(const uint16_t* __restrict__ src, int64_t rs,
                                                      uint16_t* __restrict__ dst, int64_t ldd, int64_t rows,
                                                      int64_t cols, int64_t pad_to, int TX) {
  pdl_wait();
  const int tx = threadIdx.x % TX, per = 256 / TX;
  for (int64_t i = (int64_t)blockIdx.y * per + threadIdx.x / TX; i < rows; i += (int64_t)gridDim.y * per) {
    const uint16_t* s = src + i * rs;
    uint16_t* d = dst + i * ldd;
    const int64_t head = min(pad_to, (int64_t)((16 - reinterpret_cast<uintptr_t>(d) % 16) % 16 / 2));
    if (blockIdx.x == 0 && tx < head) d[tx] = tx < cols ? s[tx] : (uint16_t)0;
    for (int64_t e = head + 8 * ((int64_t)blockIdx.x * TX + tx); e < pad_to; e += 8 * (int64_t)gridDim.x * TX) {
      const bool across = (reinterpret_cast<uintptr_t>(s + e) & 2u) != 0;
      uint32_t w[4];
      if (e + 8 + across <= cols && e >= across) {
        const uint32_t* p = reinterpret_cast<const uint32_t*>(s + e - across);
        uint32_t x[5];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = p[k];
        x[4] = across ? p[4] : 0u;
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = across ? __funnelshift_r(x[k], x[k + 1], 16) : x[k];
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t lo = e + 2 * k < cols ? s[e + 2 * k] : 0u, hi = e + 2 * k + 1 < cols ? s[e + 2 * k + 1] : 0u;
          w[k] = lo | hi << 16;
        }
      }
      if (e + 8 <= pad_to) {
        *reinterpret_cast<uint4*>(d + e) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (e + k < pad_to) d[e + k] = (uint16_t)(w[k / 2] >> (k % 2 * 16));
      }
    }
  }
}

// fp32 -> bf16 of rows of whole 16-byte steps, eight elements a thread.
__global__ void __launch_bounds__(256) round_matrix_kernel(const float* __restrict__ src, int64_t rs,
                                                           __nv_bfloat16* __restrict__ dst, int64_t ldd, int64_t rows,
                                                           int64_t cols) {
  pdl_wait();
  const int64_t c = 8 * ((int64_t)blockIdx.x * 256 + threadIdx.x);
  if (c >= cols) return;
  for (int64_t i = blockIdx.y; i < rows; i += 2 * (int64_t)gridDim.y) {
    float4 u[2][2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (i + k * (int64_t)gridDim.y >= rows) break;
      const float4* p = reinterpret_cast<const float4*>(src + (i + k * (int64_t)gridDim.y) * rs + c);
      u[k][0] = p[0];
      u[k][1] = p[1];
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (i + k * (int64_t)gridDim.y >= rows) break;
      uint4 o;
      __nv_bfloat162* w = reinterpret_cast<__nv_bfloat162*>(&o);
      w[0] = __floats2bfloat162_rn(u[k][0].x, u[k][0].y);
      w[1] = __floats2bfloat162_rn(u[k][0].z, u[k][0].w);
      w[2] = __floats2bfloat162_rn(u[k][1].x, u[k][1].y);
      w[3] = __floats2bfloat162_rn(u[k][1].z, u[k][1].w);
      *reinterpret_cast<uint4*>(dst + (i + k * (int64_t)gridDim.y) * ldd + c) = o;
    }
  }
}

template <typename TD, typename TS>
void copy_matrix_t(const void* src, int64_t rs, int64_t cs, void* dst, int64_t ldd, int64_t rows, int64_t cols,
                   int64_t pad_to, bool accumulate, cudaStream_t s) {
  const dim3 grid((unsigned)std::min<int64_t>((pad_to + 1023) / 1024, 64), (unsigned)std::min<int64_t>(rows, 65535));
  launch_pdl(copy_matrix_kernel<TD, TS>, grid, dim3(256), 0, s, reinterpret_cast<const TS*>(src), rs, cs,
             reinterpret_cast<TD*>(dst), ldd, rows, cols, pad_to, accumulate ? 1 : 0);
  DLVK_POST_LAUNCH();
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Whether the x rows and their copies are whole 16-byte steps.
int whole_rows(const CeFinish& f, int step) {
  return al16(f.x) && al16(f.x_clean) && f.ldx % step == 0 && f.ldc % step == 0 && f.width % step == 0;
}

}  // namespace

void ce_count(const CeRows& r, bool mean, const float* grad_scale, float* gscale, unsigned* done, cudaStream_t s) {
  launch_pdl(count_kernel, dim3(1), dim3(1024), 0, s, r, mean ? 1 : 0, grad_scale, gscale, done);
  DLVK_POST_LAUNCH();
}

void ce_finish(const CeRows& r, const CeFinish& f, DType dt, cudaStream_t s) {
  const dim3 grid((unsigned)((r.rows + GROUP - 1) / GROUP), f.x_clean != nullptr ? 2 : 1);
  if (dt == DType::F32) launch_pdl(finish_kernel<float>, grid, dim3(FIN_WARPS * 32), 0, s, r, f, whole_rows(f, 4));
  else launch_pdl(finish_kernel<__nv_bfloat16>, grid, dim3(FIN_WARPS * 32), 0, s, r, f, whole_rows(f, 8));
  DLVK_POST_LAUNCH();
}

bool ce_rescale_joins(int64_t rows, int64_t classes, int stat_cols) {
  return stat_cols <= 512 && (classes + RS_COLS - 1) / RS_COLS * rows * stat_cols * 8 <= (8 << 20);
}

void ce_rescale(const CeRows& r, const CeFinish& f, int stat_width, bool join, void* e, int64_t lde, cudaStream_t s) {
  DLVK_CHECK((stat_width == 64 || stat_width == 128) && lde % 8 == 0 && al16(e), "ce_rescale: layout");
  const dim3 grid((unsigned)((r.classes + RS_COLS - 1) / RS_COLS + (join ? 1 : 0)),
                  (unsigned)((r.rows + GROUP - 1) / GROUP));
  DLVK_CHECK(grid.y <= 65535u, "ce_rescale: more than 2^21 rows in one block of rows");
  const int shift = stat_width == 64 ? 6 : 7, vec = whole_rows(f, 8);
  uint16_t* p = reinterpret_cast<uint16_t*>(e);
  if (join) launch_pdl(rescale_kernel<true>, grid, dim3(RS_WARPS * 32), 0, s, r, f, vec, shift, p, lde);
  else launch_pdl(rescale_kernel<false>, grid, dim3(RS_WARPS * 32), 0, s, r, f, vec, shift, p, lde);
  DLVK_POST_LAUNCH();
}

int ce_memory_stat_cols(int64_t rows, int64_t classes) {
  // about eight blocks to an SM, of at least 2048 classes
  return (int)std::max<int64_t>(1, std::min<int64_t>((8 * 148 + rows - 1) / rows, classes / 2048));
}

void ce_memory_stats(const CeRows& r, const float* z, int64_t ldz, float2* stats, float* zlabel, unsigned* done,
                     cudaStream_t s) {
  const int cols = ce_memory_stat_cols(r.rows, r.classes);
  const int64_t per = (r.classes + cols - 1) / cols;
  launch_pdl(memory_stats_kernel, dim3((unsigned)r.rows, (unsigned)cols), dim3(256), 0, s, r, z, ldz, per, stats,
             zlabel, done);
  DLVK_POST_LAUNCH();
}

void ce_memory_grad(const CeRows& r, float* z, int64_t ldz, const float2* norm, const float* gscale, __nv_bfloat16* dl,
                    int64_t pitch, bool keep_z, cudaStream_t s) {
  DLVK_CHECK(ldz % 4 == 0 && al16(z) && pitch % 4 == 0 && al16(dl), "ce_memory_grad: layout");
  const unsigned parts = (unsigned)ce_memory_stat_cols(r.rows, r.classes);
  launch_pdl(memory_grad_kernel, dim3((unsigned)r.rows, parts), dim3(256), 0, s, r, z, ldz, norm, gscale, dl, pitch,
             keep_z ? 1 : 0);
  DLVK_POST_LAUNCH();
}

void split_parts(const float* src, int64_t ld, int64_t rows, int64_t cols, __nv_bfloat16* dst, int64_t pitch,
                 const CeRows* mask, cudaStream_t s) {
  DLVK_CHECK(pitch % 64 == 0 && pitch >= cols && al16(dst), "split_parts: layout");
  if (rows == 0) return;
  const dim3 grid((unsigned)((pitch + 1023) / 1024), (unsigned)std::min<int64_t>(rows, 16384));
  launch_pdl(split_parts_kernel, grid, dim3(256), 0, s, src, ld, rows, cols, dst, pitch, mask ? *mask : CeRows{},
             mask != nullptr ? 1 : 0, al16(src) && ld % 4 == 0 ? 1 : 0);
  DLVK_POST_LAUNCH();
}

void copy_matrix(DType dst_dt, DType src_dt, const void* src, int64_t rs, int64_t cs, void* dst, int64_t ldd,
                 int64_t rows, int64_t cols, int64_t pad_to, bool accumulate, cudaStream_t s) {
  if (rows == 0 || pad_to == 0) return;
  if (dst_dt == DType::BF16 && src_dt == DType::F32 && cs == 1 && !accumulate && cols == pad_to && cols % 8 == 0 &&
      rs % 4 == 0 && ldd % 8 == 0 && al16(src) && al16(dst)) {
    const dim3 grid((unsigned)((cols / 8 + 255) / 256), (unsigned)std::min<int64_t>((rows + 1) / 2, 4096));
    launch_pdl(round_matrix_kernel, grid, dim3(256), 0, s, reinterpret_cast<const float*>(src), rs,
               reinterpret_cast<__nv_bfloat16*>(dst), ldd, rows, cols);
    DLVK_POST_LAUNCH();
    return;
  }
  if (dst_dt == DType::BF16 && src_dt == DType::BF16 && cs == 1 && !accumulate) {
    int tx = 8;
    while (tx < 256 && tx * 8 < pad_to) tx *= 2;
    const int64_t across = (pad_to + 8 * tx - 1) / (8 * tx) + 1, groups = (rows + 256 / tx - 1) / (256 / tx);
    const dim3 grid((unsigned)std::min<int64_t>(across, 64), (unsigned)std::min<int64_t>(groups, 65535));
    launch_pdl(realign_kernel, grid, dim3(256), 0, s, reinterpret_cast<const uint16_t*>(src), rs,
               reinterpret_cast<uint16_t*>(dst), ldd, rows, cols, pad_to, tx);
    DLVK_POST_LAUNCH();
    return;
  }
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
