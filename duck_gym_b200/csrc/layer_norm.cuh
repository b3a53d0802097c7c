// Layer norm of the rows of a matrix, and its gradient.
//
//   unit = (x - mean) rstd,  rstd = 1 / sqrt(var + eps),  y = unit w + b
//   g    = dy w
//   dx   = rstd (g - mean(g) - unit mean(g unit))
//   dw   = sum over rows of dy unit,   db = sum over rows of dy
//
// The variance is that of the centred values (a second pass over the row), so
// a large common level costs no digits.  All sums are float32 in a fixed
// order; nothing is added with atomics, so results repeat bit for bit.  g is
// rounded before it is used (no fused product), so that it is the same number in
// its mean and in the difference from it: the gradient of a row of one value,
// or of a g that is the same throughout, is zero and not a rounding times rstd.
#pragma once
#include "numeric_types.cuh"

namespace duckb200 {

struct NormArgs {
  const void *x, *dy;
  const float *weight, *bias;   // [n] or null (1 and 0)
  void *y, *dx;
  float *stats;                 // [rows, 2]: mean, rstd (forward: may be null)
  float *partials;              // [splits, 2, n]
  float *dweight, *dbias;       // [n] or null
  int64_t rows, xStride, dyStride;
  int n;
  float eps;
};

constexpr int kNormThreads = 128;

// One warp per row, any width.
template <class T> __global__ void __launch_bounds__(kNormThreads) normForwardAny(NormArgs p) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = int64_t(gridDim.x) * (kNormThreads / 32);
  for (int64_t row = int64_t(blockIdx.x) * (kNormThreads / 32) + threadIdx.x / 32; row < p.rows; row += warps) {
    const T *x = static_cast<const T *>(p.x) + row * p.xStride;
    T *y = static_cast<T *>(p.y) + row * p.n;
    float sum = 0.f;
    for (int c = lane; c < p.n; c += 32) sum += toFloat(x[c]);
    const float mean = warpSum(sum) / float(p.n);
    float square = 0.f;
    for (int c = lane; c < p.n; c += 32) {
      const float d = toFloat(x[c]) - mean;
      square += d * d;
    }
    const float rstd = rsqrtf(warpSum(square) / float(p.n) + p.eps);
    for (int c = lane; c < p.n; c += 32) {
      const float unit = (toFloat(x[c]) - mean) * rstd;
      y[c] = fromFloat<T>(unit * (p.weight ? p.weight[c] : 1.f) + (p.bias ? p.bias[c] : 0.f));
    }
    if (p.stats && lane == 0) {
      p.stats[2 * row] = mean;
      p.stats[2 * row + 1] = rstd;
    }
  }
}

template <class T> __global__ void __launch_bounds__(kNormThreads) normBackwardAny(NormArgs p) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = int64_t(gridDim.x) * (kNormThreads / 32);
  for (int64_t row = int64_t(blockIdx.x) * (kNormThreads / 32) + threadIdx.x / 32; row < p.rows; row += warps) {
    const T *x = static_cast<const T *>(p.x) + row * p.xStride;
    const T *dy = static_cast<const T *>(p.dy) + row * p.dyStride;
    T *dx = static_cast<T *>(p.dx) + row * p.n;
    const float mean = p.stats[2 * row], rstd = p.stats[2 * row + 1];
    float s1 = 0.f, s2 = 0.f;
    for (int c = lane; c < p.n; c += 32) {
      const float g = __fmul_rn(toFloat(dy[c]), p.weight ? p.weight[c] : 1.f);
      s1 += g;
      s2 += g * ((toFloat(x[c]) - mean) * rstd);
    }
    s1 = warpSum(s1) / float(p.n);
    s2 = warpSum(s2) / float(p.n);
    for (int c = lane; c < p.n; c += 32) {
      const float g = __fmul_rn(toFloat(dy[c]), p.weight ? p.weight[c] : 1.f);
      dx[c] = fromFloat<T>(rstd * (g - s1 - (toFloat(x[c]) - mean) * rstd * s2));
    }
  }
}

// Partial sums of the weight's and bias' gradients: 32 columns by 8 rows of
// threads, every gridDim.y-th group of 8 rows.
template <class T> __global__ void __launch_bounds__(256) normColumnsAny(NormArgs p) {
  __shared__ float red[2][8][32];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float dw = 0.f, db = 0.f;
  if (c < p.n)
    for (int64_t row = int64_t(blockIdx.y) * 8 + part; row < p.rows; row += int64_t(gridDim.y) * 8) {
      const float dy = toFloat(static_cast<const T *>(p.dy)[row * p.dyStride + c]);
      const float x = toFloat(static_cast<const T *>(p.x)[row * p.xStride + c]);
      dw += dy * ((x - p.stats[2 * row]) * p.stats[2 * row + 1]);
      db += dy;
    }
  red[0][part][lane] = dw;
  red[1][part][lane] = db;
  __syncthreads();
  if (part < 2 && c < p.n) {
    float s = 0.f;
    for (int k = 0; k < 8; ++k) s += red[part][k][lane];
    p.partials[(int64_t(blockIdx.y) * 2 + part) * p.n + c] = s;
  }
}

__global__ void __launch_bounds__(256) normColumnsFinish(NormArgs p, int splits) {
  __shared__ float red[8][32];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;   // of the 2 n sums
  float s = 0.f;
  if (c < 2 * p.n)
    for (int k = part; k < splits; k += 8) s += p.partials[int64_t(k) * 2 * p.n + c];
  red[part][lane] = s;
  __syncthreads();
  if (part == 0 && c < 2 * p.n) {
    float total = 0.f;
    for (int k = 0; k < 8; ++k) total += red[k][lane];
    float *out = c < p.n ? p.dweight : p.dbias;
    if (out) out[c < p.n ? c : c - p.n] = total;
  }
}

}  // namespace duckb200
