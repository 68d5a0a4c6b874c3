// Two float32 operations in one instruction (sm_100's packed arithmetic), each rounded as the single one is.  The assembler
// contracts a packed product with a packed sum behind it, .rn or not (seen: a quarter of the sums differed in the last
// bit); where that matters the sum is two single ones, which it leaves alone.
#pragma once

namespace fsgs {

struct Two {
  unsigned long long v;
};
__device__ __forceinline__ Two two(float a, float b) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ Two both(float a) { return two(a, a); }
__device__ __forceinline__ void split(Two t, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(t.v)); }
__device__ __forceinline__ Two mul2(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
// a + b, not contracted with the products that a and b may be
__device__ __forceinline__ void plain_sum(Two a, Two b, float &x, float &y) {
  float a0, a1, b0, b1;
  split(a, a0, a1), split(b, b0, b1);
  x = __fadd_rn(a0, b0), y = __fadd_rn(a1, b1);
}

}  // namespace fsgs
