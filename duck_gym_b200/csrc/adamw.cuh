// AdamW over many tensors in one launch, with moments in 32 bits or in 8, and
// the norm of all gradients that they are clipped by.
//
//   g' = g min(1, max_norm / (|g| + 1e-6))      (where there is a max_norm)
//   m  = beta1 m + (1 - beta1) g',   v = beta2 v + (1 - beta2) g'^2
//   p  = p (1 - lr wd) - lr / (1 - beta1^t) m / (sqrt(v / (1 - beta2^t)) + eps)
//
// Moments in 8 bits.  128 neighbouring values share one byte, the largest
// exponent field e among their float32 forms.  A code is the float's leading
// bits, exponent and three bits of mantissa, counted from
// low = max(0, 8 e + 8 - most): most = 255 codes, 31 octaves, for v, and 127, 15
// octaves, for m, whose codes carry its sign (int8).  So both reach as far down:
// sqrt(v) over 15 octaves too.  Code 0 is the value 0; an m below the lowest code becomes 0, a
// v above 0 keeps code 1 at least, since a v rounded to zero beside an m that is
// not would make the step m / eps.
//
// The 20 bits that a code drops are rounded up or down at random.  beta2 = 0.999
// moves v by a thousandth a step where codes are an eighth of an octave apart: to
// the nearest code, v would never move.  The random bits are a hash of the step,
// the tensor's place in the list and the value's place in the tensor, so that a
// step repeats bit for bit.  bfloat16 parameters are rounded the same way: most
// steps are smaller than half a place of theirs.
//
// The moments' arithmetic is written with roundings of its own for each product
// and sum: a code depends on the last bit, and has to be the same wherever this
// formula is computed.
//
// Bound by memory: 28 bytes a value with 32-bit moments, 16 with 8-bit ones
// (float32 parameters), and 4 for the norm.  A warp has the 128 values of a
// group, two groups at once.
#pragma once
#include "numeric_types.cuh"

namespace duckb200 {

constexpr int kMomentGroup = 128;
constexpr int kAdamThreads = 256, kAdamAtOnce = 2;
constexpr int kAdamChunk = kAdamThreads / 32 * kAdamAtOnce * kMomentGroup;   // values of a block's round
constexpr int kNormChunk = 4 * kAdamChunk;
constexpr int kNormBlocks = 148 * 4;   // and sums, at most

struct AdamTensor {
  void *param;
  const void *grad;
  void *m, *v;                // float32, or codes
  uint8_t *me, *ve;           // the groups' exponents
  int64_t n;
  int32_t first;              // the tensor's first chunk
  uint32_t place : 31;        // in the caller's list
  uint32_t pieces : 1;        // four values lie on their own boundary in every array
};
// The tensors of a launch travel in its arguments (at most 32,764 bytes).
constexpr int kTensorsFew = 48, kTensorsMany = 448;
template <int MOST> struct AdamTable {
  AdamTensor t[MOST];
};
struct AdamArgs {
  int64_t *step;              // steps done, in the low 32 bits; the high ones count blocks while a step runs
  const float *rate;          // learning rate on the device, or null: rateHost
  const double *sums;         // of squares, sumCount of them
  double rateHost, beta1, beta2, weightDecay, maxNorm;
  float eps;
  int sumCount, count, chunks, finish;
};

__device__ __forceinline__ uint32_t mixBits(uint32_t x) {   // the finaliser of MurmurHash3
  x = (x ^ (x >> 16)) * 0x85ebca6bu;
  x = (x ^ (x >> 13)) * 0xc2b2ae35u;
  return x ^ (x >> 16);
}

template <int MOST> __device__ __forceinline__ int lowestCode(uint32_t exponent) {
  return max(0, int(8 * exponent) + 8 - MOST);
}
__device__ __forceinline__ float momentValue(int magnitude, int low, uint32_t exponent) {
  const uint32_t bits = magnitude ? uint32_t(magnitude + low) << 20 : 0u;
  return exponent == 255 ? __uint_as_float(0x7fffffffu) : __uint_as_float(bits);
}
// `bits` of a value's magnitude, finite or not; what a group with an infinity or a NaN gets is not read.
__device__ __forceinline__ int momentCode(uint32_t bits, uint32_t noise, int low) {
  return int(min((min(bits, 0x7f800000u) + noise) >> 20, 2039u)) - low;
}

// The chunk's tensor: the last one whose first chunk is not beyond it.
template <int MOST> __device__ __forceinline__ int tensorOf(const AdamTable<MOST> &table, int count, int chunk) {
  int low = 0, high = count;
  while (high - low > 1) {
    const int middle = (low + high) / 2;
    if (table.t[middle].first <= chunk) low = middle;
    else high = middle;
  }
  return low;
}

template <class T> struct Four;
template <> struct Four<float> {
  using Piece = float4;
};
template <> struct Four<bf16> {
  using Piece = uint2;
};
template <class T> __device__ __forceinline__ void loadFour(float (&x)[4], const T *p) {
  const typename Four<T>::Piece piece = *reinterpret_cast<const typename Four<T>::Piece *>(p);
  const T *e = reinterpret_cast<const T *>(&piece);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = toFloat(e[i]);
}
template <class T> __device__ __forceinline__ void storeFour(T *p, const T (&x)[4]) {
  typename Four<T>::Piece piece;
  T *e = reinterpret_cast<T *>(&piece);
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = x[i];
  *reinterpret_cast<typename Four<T>::Piece *>(p) = piece;
}

// Sum over a block of kAdamThreads, in every thread, in a fixed order.
__device__ __forceinline__ double blockSum(double x) {
  __shared__ double parts[kAdamThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  if (threadIdx.x % 32 == 0) parts[threadIdx.x / 32] = x;
  __syncthreads();
  double sum = 0.0;
#pragma unroll
  for (int w = 0; w < kAdamThreads / 32; ++w) sum += parts[w];
  return sum;
}

// Sums of squares, in double: block b adds its own to sums[b], which holds one
// already if b < `before`.
template <class T, int MOST>
__global__ void __launch_bounds__(kAdamThreads) gradientSquares(const __grid_constant__ AdamTable<MOST> table, int count,
                                                                int chunks, int before, double *sums) {
  double sum = 0.0;
  for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const AdamTensor &t = table.t[tensorOf(table, count, chunk)];
    const T *g = static_cast<const T *>(t.grad);
    const int64_t begin = int64_t(chunk - t.first) * kNormChunk, end = min(t.n, begin + kNormChunk);
    constexpr int R = kNormChunk / (4 * kAdamThreads);
    float x[R][4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t at = begin + 4 * (r * kAdamThreads + int(threadIdx.x));
      if (t.pieces && at + 4 <= end) {
        loadFour(x[r], g + at);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[r][i] = at + i < end ? toFloat(g[at + i]) : 0.f;
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += double(x[r][i]) * double(x[r][i]);
  }
  sum = blockSum(sum);
  if (threadIdx.x == 0) sums[blockIdx.x] = (int(blockIdx.x) < before ? sums[blockIdx.x] : 0.0) + sum;
}

struct AdamScalars {
  float clip, ahead, widen, shrink;
  uint32_t count;   // this step's number
};
__device__ __forceinline__ AdamScalars adamScalars(const AdamArgs &p) {
  __shared__ AdamScalars shared;
  double total = 0.0;
  if (p.sumCount) {
    for (int i = threadIdx.x; i < p.sumCount; i += kAdamThreads) total += p.sums[i];
    total = blockSum(total);
  }
  if (threadIdx.x == 0) {
    AdamScalars s;
    s.count = uint32_t(*reinterpret_cast<volatile int64_t *>(p.step)) + 1;
    const double rate = p.rate ? double(*p.rate) : p.rateHost;
    double clip = 1.0;
    if (p.sumCount) {
      clip = p.maxNorm / (sqrt(total) + 1e-6);
      if (clip > 1.0) clip = 1.0;   // a NaN stays one
    }
    s.clip = float(clip);
    s.ahead = float(rate / (1.0 - pow(p.beta1, double(s.count))));
    s.widen = float(rsqrt(1.0 - pow(p.beta2, double(s.count))));
    s.shrink = float(1.0 - rate * p.weightDecay);
    shared = s;
  }
  __syncthreads();
  return shared;
}

// Blocks that are done are counted in the step's high half; the last one counts the step.
__device__ __forceinline__ void finishStep(const AdamArgs &p, uint32_t count) {
  if (!p.finish) return;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    unsigned long long *step = reinterpret_cast<unsigned long long *>(p.step);
    const unsigned long long before = atomicAdd(step, 1ull << 32);
    if (uint32_t(before >> 32) == gridDim.x - 1) *reinterpret_cast<volatile int64_t *>(p.step) = int64_t(count);
  }
}

// The approximations leave 2^-21 of the step's size, which is a small part of the parameter's.
__device__ __forceinline__ float adamParameter(float p, float m, float v, const AdamScalars &s, float eps) {
  float root;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(root) : "f"(v));
  return p * s.shrink - s.ahead * __fdividef(m, root * s.widen + eps);
}
template <class T> __device__ __forceinline__ T adamRounded(float p, uint32_t noise);
template <> __device__ __forceinline__ float adamRounded<float>(float p, uint32_t) { return p; }
template <> __device__ __forceinline__ bf16 adamRounded<bf16>(float p, uint32_t noise) {
  const uint32_t bits = __float_as_uint(p);
  const bool finite = (bits & 0x7f800000u) != 0x7f800000u;
  return finite ? __ushort_as_bfloat16(uint16_t((bits + (noise & 0xffffu)) >> 16)) : __float2bfloat16_rn(p);
}

template <class T, bool EIGHT, int MOST>
__global__ void __launch_bounds__(kAdamThreads) adamStep(const __grid_constant__ AdamTable<MOST> table, AdamArgs p) {
  constexpr int U = kAdamAtOnce;
  const AdamScalars s = adamScalars(p);
  const int lane = threadIdx.x % 32;
  const float beta1 = float(p.beta1), rest1 = float(1.0 - p.beta1), beta2 = float(p.beta2), rest2 = float(1.0 - p.beta2);
  for (int chunk = blockIdx.x; chunk < p.chunks; chunk += gridDim.x) {
    const AdamTensor &t = table.t[tensorOf(table, p.count, chunk)];
    const int64_t firstGroup = int64_t(chunk - t.first) * (kAdamChunk / kMomentGroup) + threadIdx.x / 32 * U;
    const uint32_t key = mixBits(s.count + 0x9e3779b9u * (uint32_t(t.place) + 1));
    T *param = static_cast<T *>(t.param);
    const T *grad = static_cast<const T *>(t.grad);
    float x[U][4], g[U][4], m[U][4], v[U][4];
    // A lane's values: four neighbours where the group is whole and aligned, else every 32nd.
    bool whole[U];
    int left[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = (firstGroup + u) * kMomentGroup;
      left[u] = int(max(int64_t(0), min(int64_t(kMomentGroup), t.n - at)));
      whole[u] = t.pieces && left[u] == kMomentGroup;
      uint32_t me = 0, ve = 0;
      int lowM = 0, lowV = 0;
      if (EIGHT && left[u] > 0) {
        me = t.me[firstGroup + u], ve = t.ve[firstGroup + u];
        lowM = lowestCode<127>(me), lowV = lowestCode<255>(ve);
      }
      auto decode = [&](int i, int8_t cm, uint8_t cv) {
        const float magnitude = momentValue(abs(int(cm)), lowM, me);
        m[u][i] = cm < 0 ? -magnitude : magnitude;
        v[u][i] = momentValue(cv, lowV, ve);
      };
      if (whole[u]) {
        const int64_t here = at + 4 * lane;
        loadFour(x[u], param + here);
        loadFour(g[u], grad + here);
        if constexpr (EIGHT) {
          const char4 cm = *reinterpret_cast<const char4 *>(static_cast<const int8_t *>(t.m) + here);
          const uchar4 cv = *reinterpret_cast<const uchar4 *>(static_cast<const uint8_t *>(t.v) + here);
          decode(0, cm.x, cv.x);
          decode(1, cm.y, cv.y);
          decode(2, cm.z, cv.z);
          decode(3, cm.w, cv.w);
        } else {
          loadFour(m[u], static_cast<const float *>(t.m) + here);
          loadFour(v[u], static_cast<const float *>(t.v) + here);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = lane + 32 * i < left[u];
          const int64_t here = at + lane + 32 * i;
          x[u][i] = in ? toFloat(param[here]) : 0.f;
          g[u][i] = in ? toFloat(grad[here]) : 0.f;
          if constexpr (EIGHT) {
            decode(i, in ? static_cast<const int8_t *>(t.m)[here] : int8_t(0),
                   in ? static_cast<const uint8_t *>(t.v)[here] : uint8_t(0));
            if (!in) m[u][i] = v[u][i] = 0.f;   // (in a group of NaN)
          } else {
            m[u][i] = in ? static_cast<const float *>(t.m)[here] : 0.f;
            v[u][i] = in ? static_cast<const float *>(t.v)[here] : 0.f;
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = (firstGroup + u) * kMomentGroup;
      uint32_t largestM = 0, largestV = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float gi = p.sumCount ? __fmul_rn(g[u][i], s.clip) : g[u][i];
        m[u][i] = __fadd_rn(__fmul_rn(m[u][i], beta1), __fmul_rn(gi, rest1));
        v[u][i] = __fadd_rn(__fmul_rn(v[u][i], beta2), __fmul_rn(__fmul_rn(gi, gi), rest2));
        const bool in = whole[u] || lane + 32 * i < left[u];
        if (EIGHT && in) {
          largestM = max(largestM, __float_as_uint(m[u][i]) & 0x7fffffffu);
          largestV = max(largestV, __float_as_uint(v[u][i]) & 0x7fffffffu);
        }
      }
      uint32_t me = 0, ve = 0;
      int lowM = 0, lowV = 0;
      if constexpr (EIGHT) {
        me = __reduce_max_sync(0xffffffffu, largestM) >> 23;
        ve = __reduce_max_sync(0xffffffffu, largestV) >> 23;
        lowM = lowestCode<127>(me), lowV = lowestCode<255>(ve);
      }
      T out[4];
      int8_t cm[4];
      uint8_t cv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t noise = 0;
        if (EIGHT || sizeof(T) == 2)
          noise = mixBits(key ^ uint32_t(at + (whole[u] ? 4 * lane + i : lane + 32 * i)));
        out[i] = adamRounded<T>(adamParameter(x[u][i], m[u][i], v[u][i], s, p.eps), noise);
        if constexpr (EIGHT) {
          const uint32_t bits = __float_as_uint(m[u][i]), vbits = __float_as_uint(v[u][i]);
          const int magnitude = max(0, min(127, momentCode(bits & 0x7fffffffu, (noise >> 20 << 8) + 128, lowM)));
          cm[i] = int8_t(bits >> 31 ? -magnitude : magnitude);
          cv[i] = vbits == 0 ? uint8_t(0) : uint8_t(max(1, min(255, momentCode(vbits & 0x7fffffffu, noise & 0xfffffu, lowV))));
        }
      }
      if (whole[u]) {
        const int64_t here = at + 4 * lane;
        storeFour(param + here, out);
        if constexpr (EIGHT) {
          *reinterpret_cast<char4 *>(static_cast<int8_t *>(t.m) + here) = make_char4(cm[0], cm[1], cm[2], cm[3]);
          *reinterpret_cast<uchar4 *>(static_cast<uint8_t *>(t.v) + here) = make_uchar4(cv[0], cv[1], cv[2], cv[3]);
        } else {
          storeFour(static_cast<float *>(t.m) + here, m[u]);
          storeFour(static_cast<float *>(t.v) + here, v[u]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (lane + 32 * i >= left[u]) continue;
          const int64_t here = at + lane + 32 * i;
          param[here] = out[i];
          if constexpr (EIGHT) {
            static_cast<int8_t *>(t.m)[here] = cm[i];
            static_cast<uint8_t *>(t.v)[here] = cv[i];
          } else {
            static_cast<float *>(t.m)[here] = m[u][i];
            static_cast<float *>(t.v)[here] = v[u][i];
          }
        }
      }
      if (EIGHT && lane == 0 && left[u] > 0) {
        t.me[firstGroup + u] = uint8_t(me);
        t.ve[firstGroup + u] = uint8_t(ve);
      }
    }
  }
  finishStep(p, s.count);
}

// What codes stand for, in float32: param receives the values of m (signed codes)
// or, where m is null, of v.
template <int MOST>
__global__ void __launch_bounds__(kAdamThreads) momentValues(const __grid_constant__ AdamTable<MOST> table, int count, int chunks) {
  constexpr int U = kAdamAtOnce;
  const int lane = threadIdx.x % 32;
  for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const AdamTensor &t = table.t[tensorOf(table, count, chunk)];
    const int64_t firstGroup = int64_t(chunk - t.first) * (kAdamChunk / kMomentGroup) + threadIdx.x / 32 * U;
    float *out = static_cast<float *>(t.param);
    const bool sign = t.m != nullptr;
    const uint8_t *codes = static_cast<const uint8_t *>(sign ? t.m : t.v), *exponents = sign ? t.me : t.ve;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = (firstGroup + u) * kMomentGroup;
      const int left = int(max(int64_t(0), min(int64_t(kMomentGroup), t.n - at)));
      if (left == 0) continue;
      const uint32_t e = exponents[firstGroup + u];
      const int low = sign ? lowestCode<127>(e) : lowestCode<255>(e);
      auto value = [&](uint8_t code) {
        const int c = sign ? int(int8_t(code)) : int(code);
        const float magnitude = momentValue(abs(c), low, e);
        return c < 0 ? -magnitude : magnitude;
      };
      if (t.pieces && left == kMomentGroup) {
        const int64_t here = at + 4 * lane;
        const uchar4 c = *reinterpret_cast<const uchar4 *>(codes + here);
        *reinterpret_cast<float4 *>(out + here) = make_float4(value(c.x), value(c.y), value(c.z), value(c.w));
      } else {
        for (int i = lane; i < left; i += 32) out[at + i] = value(codes[at + i]);
      }
    }
  }
}

}  // namespace duckb200
