// elem.cuh -- the element types of the long-context operators (ORK_B200_F32 / _F16 / _BF16) as template
// parameters: loads widen to fp32, stores round to nearest even once.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace orkb {
namespace {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class E>
__device__ __forceinline__ E from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Runs f<E>() for the element type `type` names.
template <class F>
cudaError_t with_elem(int type, F f) {
  switch (type) {
    case 0: return f((float *)nullptr);
    case 1: return f((__half *)nullptr);
    case 2: return f((__nv_bfloat16 *)nullptr);
  }
  return cudaErrorInvalidValue;
}
inline size_t elem_bytes(int type) { return type == 0 ? 4 : 2; }

}  // namespace
}  // namespace orkb
