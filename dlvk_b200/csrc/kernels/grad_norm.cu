// Global gradient norm over a list of tensors, and clipping by it.
//
//   norm = sqrt(sum over all tensors of x^2)
//   out  = x * min(1, max_norm / (norm + 1e-6))
//
// The reference clips each tensor list on the host (src/optimizers/
// optimizers.cpp:9-55: one norm per tensor, read back, then one scaling per
// tensor).  Here the whole list is one launch for the partial sums and one
// for the result: the tensors' addresses and sizes travel in the launch's
// parameters (up to 1024 tensors a launch), so nothing is copied to the
// device, nothing is kept from call to call and a call can be captured.
//
// What bounds it: HBM.  The norm reads every element once; clipping has to
// know the norm before it writes, so it reads them a second time, backwards,
// because the tensors' last 100 MB or so are still in L2 then.
//
// The sum: the squares of four elements are added in fp32, those sums in 64
// bits.  Four squares that leave fp32's range (an element beyond 1e19, or
// all of them tiny) are taken in 64 bits instead, so the norm is right over
// the whole range of fp32.  Each block's total goes to its own place and the
// totals are added in a fixed order: the result does not vary.
//
// 216 M fp32 gradients (0.86 GB): norm 128 us (6.7 TB/s), clipping into another
// buffer 407 us (two reads and a write are 395 at the measured copy rate).
#include <algorithm>
#include <cmath>

#include "dlvk/common.h"
#include "dlvk/kernels.h"

namespace dlvk {
namespace {

constexpr int THREADS = 256;
constexpr int CHUNK = 8192;      // elements of one tensor that a block takes at a time
constexpr int MAX_BLOCKS = 148 * 8;         // of the sums: a partial each
constexpr int MAX_SCALE_BLOCKS = 148 * 64;  // short blocks keep reads and writes mixed (216 M fp32: 279 -> 256 us)

template <int CAP>
struct ListTable {
  const void* in[CAP];
  void* out[CAP];
  int64_t n[CAP];
  int first[CAP];       // first chunk of each tensor
  uint8_t kind[CAP];    // bit 0: bf16 input, bit 1: bf16 output
  int count, chunks;
};
static_assert(sizeof(ListTable<NORM_LIST_MAX>) + 64 <= 32764, "the table has to fit a launch's parameters");

// The tensor that chunk c belongs to (the last one whose first chunk is <= c).
template <int CAP>
__device__ __forceinline__ int find_tensor(const ListTable<CAP>& t, int c) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ void load4(const float* p, float* v) {
  const float4 u = *reinterpret_cast<const float4*>(p);
  v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
}
__device__ __forceinline__ void load4(const __nv_bfloat16* p, float* v) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  v[0] = __uint_as_float(u.x << 16);
  v[1] = __uint_as_float(u.x & 0xffff0000u);
  v[2] = __uint_as_float(u.y << 16);
  v[3] = __uint_as_float(u.y & 0xffff0000u);
}
__device__ __forceinline__ void store4(float* p, const float* v) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float* v) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
  uint2 u;
  u.x = *reinterpret_cast<const uint32_t*>(&a);
  u.y = *reinterpret_cast<const uint32_t*>(&b);
  *reinterpret_cast<uint2*>(p) = u;
}

// Sum of four squares; see the note on range at the top.  Below 1e-30 a
// square may have lost digits to fp32's smallest numbers.
__device__ __forceinline__ double squares4(const float* v) {
  const float s = fmaf(v[0], v[0], v[1] * v[1]) + fmaf(v[2], v[2], v[3] * v[3]);
  if (s >= 1e-30f && s < INFINITY) return (double)s;
  const uint32_t any = (__float_as_uint(v[0]) | __float_as_uint(v[1]) | __float_as_uint(v[2]) | __float_as_uint(v[3])) &
                       0x7fffffffu;
  if (any == 0u) return 0.0;
  double d = 0.0;
#pragma unroll
  for (int k = 0; k < 4; ++k) d += (double)v[k] * (double)v[k];
  return d;
}
__device__ __forceinline__ double square1(float v) { return (double)v * (double)v; }

template <typename T>
__device__ __forceinline__ double chunk_squares(const T* p, int n) {
  double acc = 0.0;
  // elements before the first address that a 4-element load may have
  const int head = min(n, (int)(((4 * sizeof(T) - reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T))) / sizeof(T)) & 3));
  if ((int)threadIdx.x < head) acc += square1(to_f32(p[threadIdx.x]));
  const T* q = p + head;
  const int quads = (n - head) >> 2;
  int i = threadIdx.x;
  for (; i + 3 * THREADS < quads; i += 4 * THREADS) {
    float v[4][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) load4(q + 4 * (i + k * THREADS), v[k]);
#pragma unroll
    for (int k = 0; k < 4; ++k) acc += squares4(v[k]);
  }
  for (; i < quads; i += THREADS) {
    float v[4];
    load4(q + 4 * i, v);
    acc += squares4(v);
  }
  const int done = head + 4 * quads;
  if (done + (int)threadIdx.x < n) acc += square1(to_f32(p[done + threadIdx.x]));
  return acc;
}

__device__ __forceinline__ double block_sum_f64(double v) {
  __shared__ double sm[THREADS / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  double r = 0.0;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) r += sm[i];
  return r;
}

template <int CAP>
__global__ void __launch_bounds__(THREADS) list_squares_kernel(const __grid_constant__ ListTable<CAP> t,
                                                               double* __restrict__ partial) {
  pdl_wait();
  double acc = 0.0;
  for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    const int i = find_tensor(t, c);
    const int64_t off = (int64_t)(c - t.first[i]) * CHUNK;
    const int n = (int)min((int64_t)CHUNK, t.n[i] - off);
    if (t.kind[i] & 1) acc += chunk_squares(reinterpret_cast<const __nv_bfloat16*>(t.in[i]) + off, n);
    else acc += chunk_squares(reinterpret_cast<const float*>(t.in[i]) + off, n);
  }
  const double total = block_sum_f64(acc);
  if (threadIdx.x == 0) partial[blockIdx.x] = total;
}

// Offset of element `e` (row-major over the collapsed sizes) of a strided tensor.
__device__ __forceinline__ int64_t strided_offset(const StridedItem& s, const int64_t* stride, int64_t e) {
  int64_t o = 0;
#pragma unroll
  for (int d = 3; d >= 0; --d) {
    const int64_t q = e / s.size[d];
    o += (e - q * s.size[d]) * stride[d];
    e = q;
  }
  return o;
}
__device__ __forceinline__ float load1(const void* p, int64_t i, bool bf) {
  return bf ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store1(void* p, int64_t i, bool bf, float v) {
  if (bf) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else reinterpret_cast<float*>(p)[i] = v;
}

__global__ void __launch_bounds__(THREADS) strided_squares_kernel(const __grid_constant__ StridedItem s,
                                                                  double* __restrict__ partial) {
  pdl_wait();
  double acc = 0.0;
  const bool bf = s.kind & 1;
  for (int64_t e = blockIdx.x * (int64_t)THREADS + threadIdx.x; e < s.n; e += (int64_t)gridDim.x * THREADS)
    acc += square1(load1(s.in, strided_offset(s, s.in_stride, e), bf));
  const double total = block_sum_f64(acc);
  if (threadIdx.x == 0) partial[blockIdx.x] = total;
}

// The norm from the blocks' totals, in every thread of the block.
__device__ __forceinline__ double list_norm(const double* partial, int parts) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < parts; i += THREADS) acc += partial[i];
  return sqrt(block_sum_f64(acc));
}
// A norm that is not finite as the caller gets it, in fp32, scales nothing.
__device__ __forceinline__ float clip_coefficient(double norm, float max_norm) {
  const double c = (double)max_norm / (norm + 1e-6);
  return ((float)norm < INFINITY && c < 1.0) ? (float)c : 1.f;
}

__global__ void __launch_bounds__(THREADS) list_norm_kernel(const double* __restrict__ partial, int parts,
                                                            float* __restrict__ norm) {
  pdl_wait();
  const double r = list_norm(partial, parts);
  if (threadIdx.x == 0) *norm = (float)r;
}

template <typename TI, typename TO>
__device__ __forceinline__ void chunk_scale(const TI* p, TO* o, int n, float c) {
  constexpr int STEP = 4 * (int)sizeof(TI);
  const int head = min(n, (int)((STEP - reinterpret_cast<uintptr_t>(p) % STEP) / sizeof(TI)) & 3);
  if (reinterpret_cast<uintptr_t>(o + head) % (4 * sizeof(TO)) != 0) {
    // input and output are never aligned together: element by element
    int i = threadIdx.x;
    for (; i + 7 * THREADS < n; i += 8 * THREADS) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = to_f32(p[i + k * THREADS]);
#pragma unroll
      for (int k = 0; k < 8; ++k) o[i + k * THREADS] = from_f32<TO>(v[k] * c);
    }
    for (; i < n; i += THREADS) o[i] = from_f32<TO>(to_f32(p[i]) * c);
    return;
  }
  if ((int)threadIdx.x < head) o[threadIdx.x] = from_f32<TO>(to_f32(p[threadIdx.x]) * c);
  const TI* q = p + head;
  TO* w = o + head;
  const int quads = (n - head) >> 2;
  int i = threadIdx.x;
  for (; i + 3 * THREADS < quads; i += 4 * THREADS) {
    float v[4][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) load4(q + 4 * (i + k * THREADS), v[k]);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[k][j] *= c;
      store4(w + 4 * (i + k * THREADS), v[k]);
    }
  }
  for (; i < quads; i += THREADS) {
    float v[4];
    load4(q + 4 * i, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] *= c;
    store4(w + 4 * i, v);
  }
  const int done = head + 4 * quads;
  if (done + (int)threadIdx.x < n) o[done + threadIdx.x] = from_f32<TO>(to_f32(p[done + threadIdx.x]) * c);
}

// in == out is the usual call: no __restrict__ on the tensors, and plain loads.
template <int CAP>
__global__ void __launch_bounds__(THREADS) list_scale_kernel(const __grid_constant__ ListTable<CAP> t,
                                                             const double* __restrict__ partial, int parts,
                                                             float max_norm, float* __restrict__ norm, int in_place) {
  pdl_wait();
  const double r = list_norm(partial, parts);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)r;
  const float coef = clip_coefficient(r, max_norm);
  if (coef == 1.f && in_place) return;
  for (int c = t.chunks - 1 - blockIdx.x; c >= 0; c -= gridDim.x) {
    const int i = find_tensor(t, c);
    const int64_t off = (int64_t)(c - t.first[i]) * CHUNK;
    const int n = (int)min((int64_t)CHUNK, t.n[i] - off);
    const float* fi = reinterpret_cast<const float*>(t.in[i]) + off;
    const __nv_bfloat16* bi = reinterpret_cast<const __nv_bfloat16*>(t.in[i]) + off;
    float* fo = reinterpret_cast<float*>(t.out[i]) + off;
    __nv_bfloat16* bo = reinterpret_cast<__nv_bfloat16*>(t.out[i]) + off;
    switch (t.kind[i]) {
      case 0: chunk_scale(fi, fo, n, coef); break;
      case 1: chunk_scale(bi, fo, n, coef); break;
      case 2: chunk_scale(fi, bo, n, coef); break;
      default: chunk_scale(bi, bo, n, coef); break;
    }
  }
}

__global__ void __launch_bounds__(THREADS) strided_scale_kernel(const __grid_constant__ StridedItem s,
                                                                const double* __restrict__ partial, int parts,
                                                                float max_norm, float* __restrict__ norm) {
  pdl_wait();
  const double r = list_norm(partial, parts);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)r;
  const float coef = clip_coefficient(r, max_norm);
  if (coef == 1.f && s.in == s.out) return;
  const bool bi = s.kind & 1, bo = s.kind & 2;
  for (int64_t e = blockIdx.x * (int64_t)THREADS + threadIdx.x; e < s.n; e += (int64_t)gridDim.x * THREADS) {
    const float v = load1(s.in, strided_offset(s, s.in_stride, e), bi);
    store1(s.out, strided_offset(s, s.out_stride, e), bo, v * coef);
  }
}

template <int CAP>
int fill_table(ListTable<CAP>& t, const DenseItem* items, int count) {
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) {
    t.in[i] = items[i].in;
    t.out[i] = items[i].out;
    t.n[i] = items[i].n;
    t.kind[i] = items[i].kind;
    t.first[i] = (int)chunks;
    chunks += (items[i].n + CHUNK - 1) / CHUNK;
    DLVK_CHECK(chunks < (1LL << 31), "gradient list: more than 2^44 elements in one list");
  }
  t.count = count;
  t.chunks = (int)chunks;
  return (int)std::min<int64_t>(chunks, MAX_BLOCKS);
}

int strided_blocks(int64_t n) { return (int)std::min<int64_t>((n + 4 * THREADS - 1) / (4 * THREADS), MAX_BLOCKS); }

// Launches of the dense items, NORM_LIST_MAX tensors each.  Short lists
// travel in a smaller table: the launch copies fewer parameter bytes (150
// tensors: 37 -> 35.5 us of a call that the host bounds).
template <typename F>
void for_each_table(const DenseItem* dense, int n_dense, F&& launch) {
  for (int at = 0; at < n_dense; at += NORM_LIST_MAX) {
    const int count = std::min(NORM_LIST_MAX, n_dense - at);
    if (count <= 64) {
      ListTable<64> t;
      launch(t, fill_table(t, dense + at, count));
    } else if (count <= 256) {
      ListTable<256> t;
      launch(t, fill_table(t, dense + at, count));
    } else {
      ListTable<NORM_LIST_MAX> t;
      launch(t, fill_table(t, dense + at, count));
    }
  }
}

template <int CAP>
void squares_launch(const ListTable<CAP>& t, int blocks, double* partial, cudaStream_t s) {
  launch_pdl(list_squares_kernel<CAP>, dim3(blocks), dim3(THREADS), 0, s, t, partial);
}
template <int CAP>
void scale_launch(const ListTable<CAP>& t, const double* partial, int parts, float max_norm, float* norm,
                  int in_place, cudaStream_t s) {
  launch_pdl(list_scale_kernel<CAP>, dim3(std::min(t.chunks, MAX_SCALE_BLOCKS)), dim3(THREADS), 0, s, t, partial, parts,
             max_norm, norm, in_place);
}

}  // namespace

int grad_norm_parts(const DenseItem* dense, int n_dense, const StridedItem* strided, int n_strided) {
  int parts = 0;
  for (int at = 0; at < n_dense; at += NORM_LIST_MAX) {
    int64_t chunks = 0;
    for (int i = at; i < std::min(at + NORM_LIST_MAX, n_dense); ++i) chunks += (dense[i].n + CHUNK - 1) / CHUNK;
    parts += (int)std::min<int64_t>(chunks, MAX_BLOCKS);
  }
  for (int i = 0; i < n_strided; ++i) parts += strided_blocks(strided[i].n);
  return parts;
}

void grad_norm(const DenseItem* dense, int n_dense, const StridedItem* strided, int n_strided, bool scale,
               float max_norm, float* norm, double* partial, cudaStream_t s) {
  int parts = 0;
  for_each_table(dense, n_dense, [&](const auto& t, int blocks) {
    squares_launch(t, blocks, partial + parts, s);
    DLVK_POST_LAUNCH();
    parts += blocks;
  });
  for (int i = 0; i < n_strided; ++i) {
    const int blocks = strided_blocks(strided[i].n);
    launch_pdl(strided_squares_kernel, dim3(blocks), dim3(THREADS), 0, s, strided[i], partial + parts);
    DLVK_POST_LAUNCH();
    parts += blocks;
  }
  if (!scale || n_dense + n_strided == 0) {
    launch_pdl(list_norm_kernel, dim3(1), dim3(THREADS), 0, s, partial, parts, norm);
    DLVK_POST_LAUNCH();
    return;
  }
  bool in_place = true;
  for (int i = 0; i < n_dense; ++i) in_place = in_place && dense[i].in == dense[i].out;
  for_each_table(dense, n_dense, [&](const auto& t, int) {
    scale_launch(t, partial, parts, max_norm, norm, in_place ? 1 : 0, s);
    DLVK_POST_LAUNCH();
  });
  for (int i = 0; i < n_strided; ++i) {
    launch_pdl(strided_scale_kernel, dim3(strided_blocks(strided[i].n)), dim3(THREADS), 0, s, strided[i], partial,
               parts, max_norm, norm);
    DLVK_POST_LAUNCH();
  }
}

}  // namespace dlvk
