// Shared by the block operators (group norm, axis rotation, attention): element types
// and vector loads of 1 to 16 bytes, the activations and their slopes.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "ptx.cuh"

namespace scb {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) {
  return __half2float(v);
}
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// V consecutive elements, loaded and stored as one access (V * sizeof(T) <= 16).
template <typename T, int V>
struct alignas(V * sizeof(T)) Pack {
  T v[V];
  __device__ __forceinline__ void load(const T* p) { *this = *reinterpret_cast<const Pack*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Pack*>(p) = *this; }
};

// Launch order of two kernels (programmatic dependent launch): the first lets the second
// start early, the second waits for the first's results before it reads or writes anything
// of theirs.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Activations; 0 to 2 number them as the GEMM epilogues do.
enum : int { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_SILU = 3, ACT_ANY = -1 };

// 1 / (1 + e^-z). e^-z overflows to inf below z = -88, where the quotient is 0 as it
// should be; relative error a few 2^-23 (__expf) wherever the result matters.
__device__ __forceinline__ float sigmoid(float z) { return __fdividef(1.f, 1.f + __expf(fminf(-z, 88.f))); }

template <int ACT>
__device__ __forceinline__ float act_fwd(float z) {
  if (ACT == ACT_RELU) return z < 0.f ? 0.f : z;  // NaN passes
  if (ACT == ACT_SILU) return z * sigmoid(z);
  if (ACT == ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  return z;
}

// d act / dz; ReLU's slope at 0 is 0.
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if (ACT == ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if (ACT == ACT_SILU) {
    const float s = sigmoid(z);
    return s * (1.f + z * (1.f - s));
  }
  if (ACT == ACT_GELU)
    return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * __expf(-0.5f * z * z) * 0.39894228040143268f;
  return 1.f;
}

// The largest power of two that divides every given byte count, at most `most`.
inline int common_alignment(int most, std::initializer_list<uint64_t> bytes) {
  uint64_t all = 0;
  for (uint64_t b : bytes) all |= b;
  int a = 1;
  while (a < most && !(all & (uint64_t)a)) a *= 2;
  return a;
}

}  // namespace scb
