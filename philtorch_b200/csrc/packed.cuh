// Pairs of scalars: float32 pairs in one instruction (fma.rn.f32x2 and its kin; the same roundings as two
// scalar ones, half the arithmetic instructions), float64 pairs as two.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace ptb {

template <class S> struct Pair;

template <> struct Pair<float> {
  uint64_t v;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ explicit Pair(uint64_t bits) : v(bits) {}
  __device__ __forceinline__ Pair(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ float2 get() const {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
  }
};
__device__ __forceinline__ Pair<float> operator*(Pair<float> a, Pair<float> b) {
  Pair<float> r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair<float> operator+(Pair<float> a, Pair<float> b) {
  Pair<float> r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair<float> operator-(Pair<float> a, Pair<float> b) {
  Pair<float> r;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair<float> fma2(Pair<float> a, Pair<float> b, Pair<float> c) {
  Pair<float> r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

template <> struct Pair<double> {
  double2 v;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ Pair(double a, double b) : v(make_double2(a, b)) {}
  __device__ __forceinline__ double2 get() const { return v; }
};
__device__ __forceinline__ Pair<double> operator*(Pair<double> a, Pair<double> b) { return {a.v.x * b.v.x, a.v.y * b.v.y}; }
__device__ __forceinline__ Pair<double> operator+(Pair<double> a, Pair<double> b) { return {a.v.x + b.v.x, a.v.y + b.v.y}; }
__device__ __forceinline__ Pair<double> operator-(Pair<double> a, Pair<double> b) { return {a.v.x - b.v.x, a.v.y - b.v.y}; }
__device__ __forceinline__ Pair<double> fma2(Pair<double> a, Pair<double> b, Pair<double> c) {
  return {fma(a.v.x, b.v.x, c.v.x), fma(a.v.y, b.v.y, c.v.y)};
}

}  // namespace ptb
