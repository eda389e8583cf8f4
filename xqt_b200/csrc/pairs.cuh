// Packed fp32 arithmetic (two lanes of a register pair per instruction) with ordinary operators.
#pragma once

#include "common.cuh"
#include "sm100.cuh"

namespace xqt_b200 {
namespace sm100 {

// a pair of floats as the packed instructions take it
struct Two {
  unsigned long long v;
  __device__ __forceinline__ Two() {}
  __device__ __forceinline__ Two(float a, float b) : v(f32x2_pack(a, b)) {}
  __device__ __forceinline__ explicit Two(float a) : v(f32x2_pack(a, a)) {}
  __device__ __forceinline__ float2 both() const {
    float2 f;
    f32x2_unpack(v, f.x, f.y);
    return f;
  }
};
__device__ __forceinline__ Two operator*(Two a, Two b) { Two r; r.v = f32x2_mul(a.v, b.v); return r; }
__device__ __forceinline__ Two operator+(Two a, Two b) { Two r; r.v = f32x2_add(a.v, b.v); return r; }
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) { Two r; r.v = f32x2_fma(a.v, b.v, c.v); return r; }

}  // namespace sm100
}  // namespace xqt_b200
