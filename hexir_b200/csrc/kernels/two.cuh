// two.cuh -- pairs of f32 (or f64) computed side by side.
#pragma once

#include <stdint.h>

namespace hexir {

// Two values that are computed side by side: sm_100 adds and multiplies two
// f32 with one instruction.
template <typename R>
struct Two {
  R x, y;
};
__device__ __forceinline__ uint64_t both(const Two<float> &a) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
  return r;
}
__device__ __forceinline__ Two<float> apart(uint64_t r) {
  Two<float> a;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a.x), "=f"(a.y) : "l"(r));
  return a;
}
__device__ __forceinline__ Two<float> add(const Two<float> &a, const Two<float> &b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(both(a)), "l"(both(b)));
  return apart(r);
}
__device__ __forceinline__ Two<float> mul(const Two<float> &a, const Two<float> &b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(both(a)), "l"(both(b)));
  return apart(r);
}
__device__ __forceinline__ Two<float> fma(const Two<float> &a, const Two<float> &b,
                                          const Two<float> &c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(r)
      : "l"(both(a)), "l"(both(b)), "l"(both(c)));
  return apart(r);
}
__device__ __forceinline__ Two<double> add(const Two<double> &a,
                                           const Two<double> &b) {
  return {a.x + b.x, a.y + b.y};
}
__device__ __forceinline__ Two<double> mul(const Two<double> &a,
                                           const Two<double> &b) {
  return {a.x * b.x, a.y * b.y};
}
__device__ __forceinline__ Two<double> fma(const Two<double> &a,
                                           const Two<double> &b,
                                           const Two<double> &c) {
  return {::fma(a.x, b.x, c.x), ::fma(a.y, b.y, c.y)};
}
template <typename R>
__device__ __forceinline__ R half_of(const Two<R> &a, int j) {
  return j % 2 ? a.y : a.x;
}
template <typename R>
__device__ __forceinline__ Two<R> twice(R v) {
  return {v, v};
}

}  // namespace hexir
