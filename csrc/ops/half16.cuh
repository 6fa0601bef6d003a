// The two 16-bit floating types behind one name: conversions to and from fp32 of pairs and of eight values of a 16-byte access.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace mccl {
namespace ops {

struct Bf16 {
  using T = __nv_bfloat16;
  using T2 = __nv_bfloat162;
  static __device__ __forceinline__ float2 up(T2 v) { return __bfloat1622float2(v); }
  static __device__ __forceinline__ float up(T v) { return __bfloat162float(v); }
  static __device__ __forceinline__ T2 down(float a, float b) { return __floats2bfloat162_rn(a, b); }
  static __device__ __forceinline__ T down(float a) { return __float2bfloat16_rn(a); }
};
struct Fp16 {
  using T = __half;
  using T2 = __half2;
  static __device__ __forceinline__ float2 up(T2 v) { return __half22float2(v); }
  static __device__ __forceinline__ float up(T v) { return __half2float(v); }
  static __device__ __forceinline__ T2 down(float a, float b) { return __floats2half2_rn(a, b); }
  static __device__ __forceinline__ T down(float a) { return __float2half_rn(a); }
};

template <typename H>
__device__ __forceinline__ void unpack8_as(const uint4& raw, float (&f)[8]) {
  const typename H::T2* h = reinterpret_cast<const typename H::T2*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = H::up(h[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
template <typename H>
__device__ __forceinline__ uint4 pack8_as(const float (&f)[8]) {
  uint4 raw;
  typename H::T2* h = reinterpret_cast<typename H::T2*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = H::down(f[2 * i], f[2 * i + 1]);
  return raw;
}

}  // namespace ops
}  // namespace mccl
