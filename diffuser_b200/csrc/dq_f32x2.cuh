// dq_f32x2.cuh -- float32 arithmetic on register pairs (one instruction for two
// IEEE operations on sm_100) and the bf16 pairs they come from.
#pragma once

#include <cuda_bf16.h>
#include <cstdint>

namespace dq {

struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ F2 f2(float both) { return f2(both, both); }
__device__ __forceinline__ float2 unpair(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ float sum_pair(F2 a) {
  const float2 u = unpair(a);
  return u.x + u.y;
}
// bf16 pair -> float32 pair (exact), and back (RNE)
__device__ __forceinline__ F2 widen(uint32_t w) { return f2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
__device__ __forceinline__ uint32_t narrow(F2 a) {
  const float2 u = unpair(a);
  const __nv_bfloat162 b = __floats2bfloat162_rn(u.x, u.y);
  return *reinterpret_cast<const uint32_t*>(&b);
}
__device__ __forceinline__ F2 f2_neg(F2 a) {
  const float2 u = unpair(a);
  return f2(-u.x, -u.y);
}

}  // namespace dq
