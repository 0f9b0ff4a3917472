// Values of the 8-bit latent cache: conversions between 8 bits, fp16 and fp32.
#pragma once
#include <cuda_fp8.h>

#include "mla_args.cuh"

namespace hk {

// largest value of a type: a block's scale is its largest magnitude over this
template <int FMT>
__device__ __forceinline__ constexpr float latent8_top() { return FMT == CACHE_I8 ? 127.f : 448.f; }

template <int FMT>
__device__ __forceinline__ float latent8_value(uint8_t b) {
  if (FMT == CACHE_I8) return (float)(int8_t)b;
  __nv_fp8_e4m3 v;
  v.__x = b;
  return (float)v;
}

// nearest 8-bit value (ties to even), saturating; NaN becomes 0, the block's scale says that it was one
template <int FMT>
__device__ __forceinline__ uint8_t latent8_round(float x) {
  if (x != x) return 0;
  if (FMT == CACHE_I8) return (uint8_t)(int8_t)__float2int_rn(fminf(fmaxf(x, -127.f), 127.f));
  return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}

}  // namespace hk
