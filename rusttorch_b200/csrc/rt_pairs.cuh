// rt_pairs.cuh — two f32 at a time: sm_100a adds, multiplies and fuses a pair
// in one instruction.
#pragma once
#include <cstdint>

namespace rt {

// Two f32 in a 64-bit register: one instruction rounds both results.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2_of(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_to(F2 x, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v));
}
__device__ __forceinline__ F2 f2_mul(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
// The assembler joins a product of pairs and a sum to one rounding, .rn or not
// (measured: every one of 256,000 of them).  So a sum that may follow a product
// is a * one + b, which rounds the same; `one` is 1 in both halves, and must come
// from memory or an argument, or the product with it is dropped again.
__device__ __forceinline__ F2 f2_add(F2 a, F2 b, F2 one) { return f2_fma(a, one, b); }
// a + b where a and b are not products.
__device__ __forceinline__ F2 f2_sum(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

}  // namespace rt
