// Shared device helpers of the decoder operators: floating types and 4-bit formats.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace b200q {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// Scale and zero point of a cache parameter word.
__device__ __forceinline__ float param_scale(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float param_zero(uint32_t p) { return static_cast<float>((p >> 16) & 0xffu); }

// A C entry's dispatch over b200q_ftype: runs `...` with T bound to the element type.
#define B200Q_DISPATCH_FTYPE(ftype, ...)   \
  switch (ftype) {                         \
    case B200Q_F32: {                      \
      using T = float;                     \
      __VA_ARGS__;                         \
    } break;                               \
    case B200Q_F16: {                      \
      using T = __half;                    \
      __VA_ARGS__;                         \
    } break;                               \
    default: {                             \
      using T = __nv_bfloat16;             \
      __VA_ARGS__;                         \
    } break;                               \
  }

}  // namespace b200q
