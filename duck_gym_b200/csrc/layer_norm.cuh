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
//
// Bound by memory: forward 2 values moved per element, backward 3.  A row is held
// in the registers of a team of 8, 16 or 32 lanes, or of a block of 128 to 512
// threads (up to 16 values a lane, so rows of up to 8192), and read once; the next row's
// loads are issued before the current one is reduced.  In the backward pass a lane
// keeps the same columns for all of its rows, so the sums for the weight and the
// bias stay in its registers and leave the block as one partial row.  Wider rows
// take the kernels that read a row several times (norm...Any).  Measured cold on a
// B200, bfloat16, 393216 x 512: forward 156 us (5.2 TB/s), backward 216 us
// (5.6 TB/s) and 4 us for the partial rows; 24576 x 256: 11, 11.5 and 4.5 us, of
// which some 7 are a launch's own and the first loads'.
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

// Rows in registers: LANES lanes of a team, VEC consecutive values a load, P values a lane.
template <class T, int LANES, int VEC, int P> struct NormRow {
  static constexpr int loads = P / VEC;
  using Raw = typename PieceOf<T, VEC>::type;
  Raw raw[loads];

  __device__ __forceinline__ void load(const T *row, int lane, int n) {
#pragma unroll
    for (int i = 0; i < loads; ++i) {
      const int c = (lane + LANES * i) * VEC;
      raw[i] = c < n ? *reinterpret_cast<const Raw *>(row + c) : Raw();
    }
  }
  __device__ __forceinline__ void values(float (&x)[P]) const {
#pragma unroll
    for (int i = 0; i < loads; ++i) {
      T v[VEC];
      *reinterpret_cast<Raw *>(v) = raw[i];
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[i * VEC + j] = toFloat(v[j]);
    }
  }
  static __device__ __forceinline__ void store(T *row, const float (&x)[P], int lane, int n) {
#pragma unroll
    for (int i = 0; i < loads; ++i) {
      const int c = (lane + LANES * i) * VEC;
      Raw out;
      T *v = reinterpret_cast<T *>(&out);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = fromFloat<T>(x[i * VEC + j]);
      if (c < n) *reinterpret_cast<Raw *>(row + c) = out;
    }
  }
};

// Values of the weight or the bias for a lane's columns.
template <int LANES, int VEC, int P>
__device__ __forceinline__ void normColumns(float (&w)[P], const float *from, float otherwise, int lane, int n) {
#pragma unroll
  for (int i = 0; i < P / VEC; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int c = (lane + LANES * i) * VEC + j;
      w[i * VEC + j] = from && c < n ? from[c] : otherwise;
    }
}

// Sums of a team, the same bits in each of its lanes.  A team of more than a warp
// is the block, and `red` has two rows of its warps, used in turn.
template <int LANES> __device__ __forceinline__ float2 teamSum(float2 x, float2 *red) {
#pragma unroll
  for (int o = (LANES < 32 ? LANES : 32) / 2; o > 0; o >>= 1) {
    x.x += __shfl_xor_sync(0xffffffffu, x.x, o);
    x.y += __shfl_xor_sync(0xffffffffu, x.y, o);
  }
  if (LANES > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
    __syncthreads();
    x = red[0];
#pragma unroll
    for (int k = 1; k < LANES / 32; ++k) {
      x.x += red[k].x;
      x.y += red[k].y;
    }
  }
  return x;
}

__host__ __device__ constexpr int normBlock(int lanes) { return lanes > 32 ? lanes : 128; }
// Blocks that are to fit on a multiprocessor at once, and that are launched for
// it: a second, smaller round of blocks would cost as much as a full one
// (backward, 393216 x 512: 313 us with 3 of 4 launched blocks resident).
__host__ __device__ constexpr int normResident(int lanes, int values, bool backward) {
  const int warps = backward ? (values <= 8 ? 20 : 16) : (values <= 8 ? 28 : 16);
  return lanes > 128 ? (warps * 32 / lanes > 0 ? warps * 32 / lanes : 1) : warps / 4;
}
// Rows a team has in flight: some 32 KB a multiprocessor keep the memory busy, and
// these are the fewest that give it at that many warps.
__host__ __device__ constexpr int normAhead(int words, bool backward) {
  return words <= 4 ? (backward ? 2 : 4) : words <= 8 && !backward ? 2 : 1;
}

template <class T, int LANES, int VEC, int P>
__global__ void __launch_bounds__(normBlock(LANES), normResident(LANES, P, false)) normForwardRows(NormArgs p) {
  constexpr int THREADS = normBlock(LANES), TEAMS = THREADS / LANES;
  constexpr int AHEAD = normAhead(VEC == 1 ? P : P * int(sizeof(T)) / 4, false);
  __shared__ float2 red[2][16];
  const int lane = threadIdx.x % LANES;
  const int64_t step = int64_t(gridDim.x) * TEAMS;
  int64_t row = int64_t(blockIdx.x) * TEAMS + threadIdx.x / LANES;
  const T *x = static_cast<const T *>(p.x);
  T *y = static_cast<T *>(p.y);
  NormRow<T, LANES, VEC, P> next[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k)
    if (row + k * step < p.rows) next[k].load(x + (row + k * step) * p.xStride, lane, p.n);
  float w[P], b[P];
  normColumns<LANES, VEC, P>(w, p.weight, 1.f, lane, p.n);
  normColumns<LANES, VEC, P>(b, p.bias, 0.f, lane, p.n);
  // All teams of a warp go round as often as its first: the sums are over whole warps.
  int64_t lead = LANES < 32 ? row - (threadIdx.x & 31) / LANES : row;
  for (; lead < p.rows; lead += AHEAD * step) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k, row += step) {
      if (k > 0 && lead + k * step >= p.rows) break;
      const bool live = row < p.rows;
      float v[P];
      next[k].values(v);
      if (row + AHEAD * step < p.rows) next[k].load(x + (row + AHEAD * step) * p.xStride, lane, p.n);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < P; ++i) sum += v[i];
      const float mean = teamSum<LANES>(make_float2(sum, 0.f), red[0]).x / float(p.n);
      float square = 0.f;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int c = (lane + LANES * (i / VEC)) * VEC + i % VEC;
        v[i] -= mean;
        if (c < p.n) square = fmaf(v[i], v[i], square);
      }
      const float rstd = rsqrtf(teamSum<LANES>(make_float2(square, 0.f), red[1]).x / float(p.n) + p.eps);
#pragma unroll
      for (int i = 0; i < P; ++i) v[i] = fmaf(v[i] * rstd, w[i], b[i]);
      if (live) {
        NormRow<T, LANES, VEC, P>::store(y + row * p.n, v, lane, p.n);
        if (p.stats && lane == 0) *reinterpret_cast<float2 *>(p.stats + 2 * row) = make_float2(mean, rstd);
      }
    }
  }
}

// COLUMNS: the sums for the weight's and the bias' gradients too; DX: that of x.
template <class T, int LANES, int VEC, int P, bool DX, bool COLUMNS>
__global__ void __launch_bounds__(normBlock(LANES), normResident(LANES, P, true)) normBackwardRows(NormArgs p) {
  constexpr int THREADS = normBlock(LANES), TEAMS = THREADS / LANES;
  constexpr int AHEAD = normAhead(VEC == 1 ? P : P * int(sizeof(T)) / 4, true);
  extern __shared__ float sums[];   // [warps, 2, n] where a team is a warp or less
  __shared__ float2 red[2][16];
  const int lane = threadIdx.x % LANES;
  const int64_t step = int64_t(gridDim.x) * TEAMS;
  int64_t row = int64_t(blockIdx.x) * TEAMS + threadIdx.x / LANES;
  const T *x = static_cast<const T *>(p.x), *dy = static_cast<const T *>(p.dy);
  T *dx = static_cast<T *>(p.dx);
  const float2 *stats = reinterpret_cast<const float2 *>(p.stats);
  NormRow<T, LANES, VEC, P> nextX[AHEAD], nextY[AHEAD];
  float2 nextStats[AHEAD];
  auto load = [&](int k, int64_t r) {
    nextX[k].load(x + r * p.xStride, lane, p.n);
    nextY[k].load(dy + r * p.dyStride, lane, p.n);
    nextStats[k] = stats[r];
  };
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    nextStats[k] = make_float2(0.f, 0.f);
    if (row + k * step < p.rows) load(k, row + k * step);
  }
  float w[P], dw[P], db[P];
  if (DX) normColumns<LANES, VEC, P>(w, p.weight, 1.f, lane, p.n);
#pragma unroll
  for (int i = 0; i < P; ++i) dw[i] = db[i] = 0.f;
  const float count = float(p.n);
  int64_t lead = LANES < 32 ? row - (threadIdx.x & 31) / LANES : row;
  int turn = 0;
  auto one = [&](int k) {
    const float mean = nextStats[k].x, rstd = nextStats[k].y;
    const bool live = row < p.rows;
    float u[P], d[P];
    nextX[k].values(u);
    nextY[k].values(d);
    if (row + AHEAD * step < p.rows) load(k, row + AHEAD * step);
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = (lane + LANES * (i / VEC)) * VEC + i % VEC;
      u[i] = (u[i] - mean) * rstd;
      if (COLUMNS && live && c < p.n) {
        dw[i] = fmaf(d[i], u[i], dw[i]);
        db[i] += d[i];
      }
      if (DX) {
        d[i] = c < p.n ? __fmul_rn(d[i], w[i]) : 0.f;
        s.x += d[i];
        if (c < p.n) s.y = fmaf(d[i], u[i], s.y);
      }
    }
    if (DX) {
      s = teamSum<LANES>(s, red[turn]);
      turn ^= 1;
      s.x /= count;
      s.y /= count;
#pragma unroll
      for (int i = 0; i < P; ++i) d[i] = rstd * (d[i] - s.x - u[i] * s.y);
      if (live) NormRow<T, LANES, VEC, P>::store(dx + row * p.n, d, lane, p.n);
    }
  };
  for (; lead < p.rows; lead += AHEAD * step) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k, row += step) {
      if (k > 0 && lead + k * step >= p.rows) break;
      one(k);
    }
  }
  if (!COLUMNS) return;
  // A single block's sums are the gradients themselves.
  float *outW = p.partials + int64_t(blockIdx.x) * 2 * p.n, *outB = outW + p.n;
  if (gridDim.x == 1) outW = p.dweight, outB = p.dbias;
  if (LANES > 32) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = (lane + LANES * (i / VEC)) * VEC + i % VEC;
      if (c < p.n) {
        if (outW) outW[c] = dw[i];
        if (outB) outB[c] = db[i];
      }
    }
    return;
  }
  float *mine = sums + (threadIdx.x >> 5) * 2 * p.n;
#pragma unroll
  for (int i = 0; i < P; ++i) {
#pragma unroll
    for (int o = 16; o >= LANES; o >>= 1) {
      dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
      db[i] += __shfl_xor_sync(0xffffffffu, db[i], o);
    }
    const int c = (lane + LANES * (i / VEC)) * VEC + i % VEC;
    if (c < p.n && (threadIdx.x & 31) < LANES) {
      mine[c] = dw[i];
      mine[p.n + c] = db[i];
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * p.n; c += THREADS) {
    float total = 0.f;
#pragma unroll
    for (int k = 0; k < THREADS / 32; ++k) total += sums[k * 2 * p.n + c];
    float *out = c < p.n ? outW : outB;
    if (out) out[c < p.n ? c : c - p.n] = total;
  }
}

// The gradients from the blocks' partial rows: 32 of the 2 n sums a block, its
// warps every 32nd partial each, in a fixed order.
__global__ void __launch_bounds__(1024) normPartials(NormArgs p, int splits) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < 2 * p.n) {
#pragma unroll 4
    for (int k = part; k < splits; k += 32) s += p.partials[int64_t(k) * 2 * p.n + c];
  }
  red[part][lane] = s;
  __syncthreads();
  const float total = warpSum(red[lane][part]);
  const int column = blockIdx.x * 32 + part;
  if (lane == 0 && column < 2 * p.n) {
    float *out = column < p.n ? p.dweight : p.dbias;
    if (out) out[column < p.n ? column : column - p.n] = total;
  }
}

}  // namespace duckb200
