// ELU whose output is kept in 8 bits for the backward pass.
//
//   y = x > 0 ? x : exp(x) - 1, rounded to the input's type
//   per group of 128 values of a row:  scale = max |y| / 127,
//   code = round(y / scale) (ties to even), the kept value is code scale
//   backward: dx = dy (kept > 0 ? 1 : 1 + kept), and the kept y itself for the
//   weight gradient of the layer that consumed it.
//
// The codes are those of the rounded y, the values that the next layer saw.
// The division by 127 and by the scale are products with their float32
// reciprocals.  A group whose scale would be zero or denormal keeps zeros; one
// that holds an infinity or NaN keeps NaN throughout (its scale is not finite),
// so a diverged activation is not hidden by its checkpoint.
#pragma once
#include "numeric_types.cuh"

namespace duckb200 {

constexpr int kGroup = 128;
constexpr int kCheckpointThreads = 256;

struct CheckpointArgs {
  const void *in;       // forward: x; backward: dy   [rows, n]
  void *y, *dx;         // [rows, n]; y may be null on the way back
  int8_t *codes;        // [rows, n]
  float *scales;        // [rows, groups]
  int64_t rows;
  int n, groups;
};

// Largest magnitude of two; NaN if either is.
__device__ __forceinline__ float maxOrNan(float a, float b) { return (a >= b || a != a) ? a : b; }

struct GroupScale {
  float scale, inverse;
};
__device__ __forceinline__ GroupScale groupScale(float largest) {
  const float scale = largest * (1.f / 127.f);
  // Denormal scales have no finite reciprocal in general.
  if (scale < 1.17549435e-38f) return {0.f, 0.f};
  return {scale, __frcp_rn(scale)};
}
// NaN converts to code 0, and 0 times a scale that is not finite is NaN.
__device__ __forceinline__ int encode(float y, float inverse) { return __float2int_rn(y * inverse); }

__device__ __forceinline__ float elu(float x) { return x > 0.f ? x : expm1f(x); }

// One warp per group, any width.
template <class T> __global__ void __launch_bounds__(kCheckpointThreads) eluCheckpointAny(CheckpointArgs p) {
  const int lane = threadIdx.x & 31;
  const int64_t total = p.rows * p.groups, warps = int64_t(gridDim.x) * (kCheckpointThreads / 32);
  for (int64_t g = int64_t(blockIdx.x) * (kCheckpointThreads / 32) + threadIdx.x / 32; g < total; g += warps) {
    const int64_t row = g / p.groups;
    const int first = int(g - row * p.groups) * kGroup;
    const int64_t at = row * p.n + first;
    float y[kGroup / 32], largest = 0.f;
#pragma unroll
    for (int i = 0; i < kGroup / 32; ++i) {
      const int c = lane + 32 * i;
      y[i] = 0.f;
      if (first + c < p.n) {
        const T rounded = fromFloat<T>(elu(toFloat(static_cast<const T *>(p.in)[at + c])));
        static_cast<T *>(p.y)[at + c] = rounded;
        y[i] = toFloat(rounded);
      }
      largest = maxOrNan(fabsf(y[i]), largest);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) largest = maxOrNan(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    const GroupScale s = groupScale(largest);
#pragma unroll
    for (int i = 0; i < kGroup / 32; ++i)
      if (first + lane + 32 * i < p.n) p.codes[at + lane + 32 * i] = int8_t(encode(y[i], s.inverse));
    if (lane == 0) p.scales[g] = s.scale;
  }
}

template <class T> __global__ void __launch_bounds__(kCheckpointThreads) eluRestoreAny(CheckpointArgs p) {
  const int lane = threadIdx.x & 31;
  const int64_t total = p.rows * p.groups, warps = int64_t(gridDim.x) * (kCheckpointThreads / 32);
  for (int64_t g = int64_t(blockIdx.x) * (kCheckpointThreads / 32) + threadIdx.x / 32; g < total; g += warps) {
    const int64_t row = g / p.groups;
    const int first = int(g - row * p.groups) * kGroup;
    const int64_t at = row * p.n + first;
    const float scale = p.scales[g];
#pragma unroll
    for (int i = 0; i < kGroup / 32; ++i) {
      const int c = lane + 32 * i;
      if (first + c >= p.n) continue;
      const float y = float(p.codes[at + c]) * scale;
      const float dy = toFloat(static_cast<const T *>(p.in)[at + c]);
      if (p.y) static_cast<T *>(p.y)[at + c] = fromFloat<T>(y);
      static_cast<T *>(p.dx)[at + c] = fromFloat<T>(dy * (y > 0.f ? 1.f : y + 1.f));
    }
  }
}

}  // namespace duckb200
