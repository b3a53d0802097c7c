// The two element types of the policy's operators and conversions to float.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace duckb200 {

using bf16 = __nv_bfloat16;

__device__ __forceinline__ float toFloat(float x) { return x; }
__device__ __forceinline__ float toFloat(bf16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T fromFloat(float x);
template <> __device__ __forceinline__ float fromFloat<float>(float x) { return x; }
template <> __device__ __forceinline__ bf16 fromFloat<bf16>(float x) { return __float2bfloat16_rn(x); }

// The register type that VEC elements are moved as: 16 bytes, or one element.
template <class T, int VEC> struct PieceOf {
  using type = uint4;
};
template <class T> struct PieceOf<T, 1> {
  using type = T;
};

// Sum over the lanes of a warp, the same bits in every lane.
__device__ __forceinline__ float warpSum(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

}  // namespace duckb200
