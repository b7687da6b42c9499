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
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float sigmoid(float x) { return rcp(1.f + ex2(x * -LOG2E)); }

// Two fp32 numbers in one register pair and one instruction.  The pipe takes as
// long as for two instructions, the issue slots are half.
using f2 = unsigned long long;
__device__ __forceinline__ f2 pack(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack(f2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 ex2_2(f2 x) {
  const float2 v = unpack(x);
  return pack(ex2(v.x), ex2(v.y));
}
__device__ __forceinline__ f2 rcp_2(f2 x) {
  const float2 v = unpack(x);
  return pack(rcp(v.x), rcp(v.y));
}
__device__ __forceinline__ f2 sigmoid_2(f2 x) {
  return rcp_2(add2(ex2_2(mul2(x, pack(-LOG2E, -LOG2E))), pack(1.f, 1.f)));
}

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
