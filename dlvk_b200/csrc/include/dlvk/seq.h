// Device code that the kernels over sequences share: addresses of SeqRef
// elements, copies to shared memory ahead of use, gates.
#pragma once
#include "dlvk/common.h"
#include "dlvk/kernels.h"

#ifdef __CUDACC__
namespace dlvk {

template <typename T>
__device__ __forceinline__ T* at(const SeqRef& r, int64_t b, int64_t t, int64_t c) {
  return static_cast<T*>(r.p) + b * r.batch + t * r.token + c;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

// BYTES (4, 8 or 16, both addresses multiples of it) from global to shared memory
// without a register, zeros instead where not `there`.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src, bool there) {
  const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst);
  const int n = there ? BYTES : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(src), "n"(BYTES), "r"(n) : "memory");
}
// Ends a group of copies.
__device__ __forceinline__ void copies_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All copies of this thread but those of the last LEFT groups have come.
template <int LEFT>
__device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

}  // namespace dlvk
#endif  // __CUDACC__
