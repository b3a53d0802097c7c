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
// (float32 parameters), and 4 for the norm.  A warp has the 128 values of a group,
// and the next three groups' operands on their way through shared memory.  Measured on
// a B200, cold: 64M values, float32, moments in 8 bits 214 us (5.0 TB/s, issue slots 77 %
// busy; with the loads in registers, two groups at once, 360); a policy's 0.4M values,
// moments in 32 bits, 7 us and 3 for the norm.
#pragma once
#include "numeric_types.cuh"

namespace duckb200 {

constexpr int kMomentGroup = 128;
constexpr int kAdamThreads = 256, kAdamRound = kAdamThreads / 32 * kMomentGroup;   // one group for each warp
constexpr int kAdamRoundsMost = 16;
constexpr int kNormChunk = 8 * kAdamRound;
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
  int sumCount, count, chunks, rounds, finish;   // rounds of a chunk
};

__device__ __forceinline__ uint32_t mixBits(uint32_t x) {   // the finaliser of MurmurHash3
  x = (x ^ (x >> 16)) * 0x85ebca6bu;
  x = (x ^ (x >> 13)) * 0xc2b2ae35u;
  return x ^ (x >> 16);
}

template <int MOST> __device__ __forceinline__ int lowestCode(uint32_t exponent) {
  return max(0, int(8 * exponent) + 8 - MOST);
}
__device__ __forceinline__ float momentValue(int magnitude, int low) {
  return __uint_as_float(magnitude ? uint32_t(magnitude + low) << 20 : 0u);
}
// `bits` of a value's magnitude; LEAST for a value that is not zero.  No code stands
// for an infinity (top); what a group with one, or with a NaN, gets is not read.
template <int MOST, int LEAST> __device__ __forceinline__ int momentCode(uint32_t bits, uint32_t noise, int low) {
  const int top = min(MOST, 2039 - low);
  return max(LEAST, min(top, (int(bits) + int(noise) - (low << 20)) >> 20));
}

// The chunk's tensor, the last one whose first chunk is not beyond it; `from` that of an earlier chunk.
template <int MOST> __device__ __forceinline__ int tensorOf(const AdamTable<MOST> &table, int count, int chunk, int from) {
  if (from + 1 == count || table.t[from + 1].first > chunk) return from;
  int low = from + 1, high = count;
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
  for (int chunk = blockIdx.x, index = 0; chunk < chunks; chunk += gridDim.x) {
    index = tensorOf(table, count, chunk, index);
    const AdamTensor &t = table.t[index];
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

// The approximations leave 2^-21 of the step's size, which is a small part of the
// parameter's.  (The root of the smallest float is a normal one, and so is eps.)
__device__ __forceinline__ float adamParameter(float p, float m, float v, const AdamScalars &s, float eps) {
  float root, inverse;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(root) : "f"(v));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(fmaf(root, s.widen, eps)));
  return fmaf(p, s.shrink, -s.ahead * (m * inverse));
}
template <class T> __device__ __forceinline__ T adamRounded(float p, uint32_t noise);
template <> __device__ __forceinline__ float adamRounded<float>(float p, uint32_t) { return p; }
template <> __device__ __forceinline__ bf16 adamRounded<bf16>(float p, uint32_t noise) {
  const uint32_t bits = __float_as_uint(p);
  const bool finite = (bits & 0x7f800000u) != 0x7f800000u;
  return finite ? __ushort_as_bfloat16(uint16_t((bits + (noise & 0xffffu)) >> 16)) : __float2bfloat16_rn(p);
}

// A lane's operands on their way: slots in shared memory, of four values of each
// array, which only this thread writes and reads.
template <class T, bool EIGHT> struct AdamRing {
  static constexpr int slots = 4, value = 4 * int(sizeof(T)), moment = EIGHT ? 4 : 16;
  static constexpr int bytes = slots * 2 * (value + moment) * kAdamThreads;
  uint8_t *at;   // of slot 0: x, g, m and v of all threads, one after the other
  __device__ __forceinline__ explicit AdamRing(void *shared) : at(static_cast<uint8_t *>(shared)) {}
  template <int BYTES> __device__ __forceinline__ void copy(int offset, const void *from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(uint32_t(__cvta_generic_to_shared(at + offset))), "l"(from),
                 "n"(BYTES)
                 : "memory");
  }
  __device__ __forceinline__ int place(int slot) const { return slot * 2 * (value + moment) * kAdamThreads; }
  __device__ __forceinline__ void ask(int slot, const AdamTensor &t, int64_t here) {
    const int o = place(slot), tid = threadIdx.x;
    copy<value>(o + value * tid, static_cast<const T *>(t.param) + here);
    copy<value>(o + value * (kAdamThreads + tid), static_cast<const T *>(t.grad) + here);
    const int64_t byte = here * (EIGHT ? 1 : 4);
    copy<moment>(o + 2 * value * kAdamThreads + moment * tid, static_cast<const uint8_t *>(t.m) + byte);
    copy<moment>(o + 2 * value * kAdamThreads + moment * (kAdamThreads + tid), static_cast<const uint8_t *>(t.v) + byte);
  }
};

// One lane's four values of a group.  WHOLE: neighbours in memory, `at` the first
// lane's; else every 32nd, `left` of the group.
template <class T, bool EIGHT> struct AdamLane {
  float x[4], g[4], m[4], v[4];
  uint32_t cm[4], cv[4];   // codes; of a whole group all four in the first, until step()
  uint32_t me, ve;
  __device__ __forceinline__ void load(const AdamRing<T, EIGHT> &ring, int slot) {
    using R = AdamRing<T, EIGHT>;
    const int o = ring.place(slot), tid = threadIdx.x;
    loadFour(x, reinterpret_cast<const T *>(ring.at + o + R::value * tid));
    loadFour(g, reinterpret_cast<const T *>(ring.at + o + R::value * (kAdamThreads + tid)));
    const uint8_t *moments = ring.at + o + 2 * R::value * kAdamThreads;
    if constexpr (EIGHT) {
      cm[0] = reinterpret_cast<const uint32_t *>(moments)[tid];
      cv[0] = reinterpret_cast<const uint32_t *>(moments)[kAdamThreads + tid];
    } else {
      loadFour(m, reinterpret_cast<const float *>(moments) + 4 * tid);
      loadFour(v, reinterpret_cast<const float *>(moments) + 4 * (kAdamThreads + tid));
    }
  }
  __device__ __forceinline__ void load(const AdamTensor &t, int64_t at, int left, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t here = at + lane + 32 * i;
      const bool in = lane + 32 * i < left;
      x[i] = in ? toFloat(static_cast<const T *>(t.param)[here]) : 0.f;
      g[i] = in ? toFloat(static_cast<const T *>(t.grad)[here]) : 0.f;
      if constexpr (EIGHT) {
        cm[i] = in ? uint32_t(int(static_cast<const int8_t *>(t.m)[here])) : 0u;
        cv[i] = in ? uint32_t(static_cast<const uint8_t *>(t.v)[here]) : 0u;
      } else {
        m[i] = in ? static_cast<const float *>(t.m)[here] : 0.f;
        v[i] = in ? static_cast<const float *>(t.v)[here] : 0.f;
      }
    }
  }
  template <bool WHOLE> __device__ __forceinline__ void step(const AdamTensor &t, const AdamArgs &p, const AdamScalars &s,
                                                             uint32_t key, int64_t at, int left, int lane) {
    const float beta1 = float(p.beta1), rest1 = float(1.0 - p.beta1), beta2 = float(p.beta2), rest2 = float(1.0 - p.beta2);
    if constexpr (EIGHT) {   // values of the codes
      const int lowM = lowestCode<127>(me), lowV = lowestCode<255>(ve);
      const uint32_t packedM = cm[0], packedV = cv[0];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = WHOLE ? int(int8_t(packedM >> 8 * i)) : int(cm[i]);
        m[i] = __uint_as_float(__float_as_uint(momentValue(abs(c), lowM)) | (uint32_t(c) & 0x80000000u));
        v[i] = momentValue(WHOLE ? int(packedV >> 8 * i & 0xff) : int(cv[i]), lowV);
      }
      if (me == 255 || ve == 255) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = WHOLE || lane + 32 * i < left;
          if (me == 255 && in) m[i] = __int_as_float(0x7fffffff);
          if (ve == 255 && in) v[i] = __int_as_float(0x7fffffff);
        }
      }
    }
    uint32_t largestM = 0, largestV = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float gi = p.sumCount ? __fmul_rn(g[i], s.clip) : g[i];
      m[i] = __fadd_rn(__fmul_rn(m[i], beta1), __fmul_rn(gi, rest1));
      v[i] = __fadd_rn(__fmul_rn(v[i], beta2), __fmul_rn(__fmul_rn(gi, gi), rest2));
      if (EIGHT && (WHOLE || lane + 32 * i < left)) {
        largestM = max(largestM, __float_as_uint(m[i]) & 0x7fffffffu);
        largestV = max(largestV, __float_as_uint(v[i]) & 0x7fffffffu);
      }
    }
    int lowM = 0, lowV = 0;
    if constexpr (EIGHT) {
      me = __reduce_max_sync(0xffffffffu, largestM) >> 23;
      ve = __reduce_max_sync(0xffffffffu, largestV) >> 23;
      lowM = lowestCode<127>(me), lowV = lowestCode<255>(ve);
    }
    T out[4];
    const uint32_t mixed = key ^ uint32_t(at + (WHOLE ? 4 * lane : 0));   // (at is a multiple of 128)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t noise = 0;
      if (EIGHT || sizeof(T) == 2) noise = mixBits(WHOLE ? mixed ^ uint32_t(i) : mixed ^ uint32_t(lane + 32 * i));
      out[i] = adamRounded<T>(adamParameter(x[i], m[i], v[i], s, p.eps), noise);
      if constexpr (EIGHT) {
        const uint32_t bits = __float_as_uint(m[i]), square = __float_as_uint(v[i]) & 0x7fffffffu;
        const int magnitude = momentCode<127, 0>(bits & 0x7fffffffu, (noise >> 20 << 8) + 128, lowM), sign = int(bits) >> 31;
        cm[i] = uint32_t((magnitude ^ sign) - sign);
        cv[i] = square == 0 ? 0u : uint32_t(momentCode<255, 1>(square, noise & 0xfffffu, lowV));
      }
    }
    if constexpr (WHOLE) {
      const int64_t here = at + 4 * lane;
      storeFour(static_cast<T *>(t.param) + here, out);
      if constexpr (EIGHT) {
        auto packed = [](const uint32_t (&c)[4]) {
          return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
        };
        *reinterpret_cast<uint32_t *>(static_cast<int8_t *>(t.m) + here) = packed(cm);
        *reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(t.v) + here) = packed(cv);
      } else {
        storeFour(static_cast<float *>(t.m) + here, m);
        storeFour(static_cast<float *>(t.v) + here, v);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (lane + 32 * i >= left) continue;
        const int64_t here = at + lane + 32 * i;
        static_cast<T *>(t.param)[here] = out[i];
        if constexpr (EIGHT) {
          static_cast<int8_t *>(t.m)[here] = int8_t(cm[i]);
          static_cast<uint8_t *>(t.v)[here] = uint8_t(cv[i]);
        } else {
          static_cast<float *>(t.m)[here] = m[i];
          static_cast<float *>(t.v)[here] = v[i];
        }
      }
    }
  }
};

// A block's chunk is p.rounds groups for each of its warps, its groups in turn.
template <class T, bool EIGHT, int MOST>
__global__ void __launch_bounds__(kAdamThreads, 4) adamStep(const __grid_constant__ AdamTable<MOST> table, AdamArgs p) {
  extern __shared__ __align__(16) uint8_t shared[];
  using Ring = AdamRing<T, EIGHT>;
  Ring ring(shared);
  const AdamScalars s = adamScalars(p);
  constexpr int kWarps = kAdamThreads / 32;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  for (int chunk = blockIdx.x, index = 0; chunk < p.chunks; chunk += gridDim.x) {
    index = tensorOf(table, p.count, chunk, index);
    const AdamTensor &t = table.t[index];
    const uint32_t key = mixBits(s.count + 0x9e3779b9u * (uint32_t(t.place) + 1));
    const int64_t begin = int64_t(chunk - t.first) * p.rounds * kWarps * kMomentGroup;
    const int groups = int(min(int64_t(p.rounds) * kWarps, (t.n - begin + kMomentGroup - 1) / kMomentGroup));
    const int whole = t.pieces ? int(min(int64_t(groups), (t.n - begin) / kMomentGroup)) : 0;
    AdamLane<T, EIGHT> values;
    if (warp < whole) {
      const int count = (whole - warp + kWarps - 1) / kWarps;   // at most 32
      const int64_t first = begin + warp * kMomentGroup, mine = first / kMomentGroup + lane * kWarps;
      // The exponents of the warp's groups: lane i has the i-th one's.
      uint32_t me = 0, ve = 0;
      if (EIGHT && lane < count) me = t.me[mine], ve = t.ve[mine];
      auto ask = [&](int i) {
        if (i < count) ring.ask(i % Ring::slots, t, first + int64_t(i) * kWarps * kMomentGroup + 4 * lane);
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
#pragma unroll
      for (int i = 0; i < Ring::slots - 1; ++i) ask(i);
      for (int i = 0; i < count; ++i) {
        ask(i + Ring::slots - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(Ring::slots - 1) : "memory");
        values.load(ring, i % Ring::slots);
        if constexpr (EIGHT) values.me = __shfl_sync(0xffffffffu, me, i), values.ve = __shfl_sync(0xffffffffu, ve, i);
        values.template step<true>(t, p, s, key, first + int64_t(i) * kWarps * kMomentGroup, kMomentGroup, lane);
        if (EIGHT && lane == i) me = values.me, ve = values.ve;
      }
      if (EIGHT && lane < count) t.me[mine] = uint8_t(me), t.ve[mine] = uint8_t(ve);
    }
    for (int group = whole + warp; group < groups; group += kWarps) {
      const int64_t at = begin + int64_t(group) * kMomentGroup;
      const int left = int(min(int64_t(kMomentGroup), t.n - at));
      if constexpr (EIGHT) values.me = t.me[at / kMomentGroup], values.ve = t.ve[at / kMomentGroup];
      values.load(t, at, left, lane);
      __syncwarp();   // every lane has read the exponents
      values.template step<false>(t, p, s, key, at, left, lane);
      if (EIGHT && lane == 0) t.me[at / kMomentGroup] = uint8_t(values.me), t.ve[at / kMomentGroup] = uint8_t(values.ve);
    }
  }
  finishStep(p, s.count);
}

// What codes stand for, in float32: param receives the values of m (signed codes)
// or, where m is null, of v.  A warp has U groups at once, as many bytes of codes as
// keep the memory busy (64M values: 57 us with eight, 77 with two), or two of them
// where the values are few and blocks many.
template <int MOST, int U>
__global__ void __launch_bounds__(kAdamThreads) momentValues(const __grid_constant__ AdamTable<MOST> table, int count, int chunks) {
  const int lane = threadIdx.x % 32;
  for (int chunk = blockIdx.x, index = 0; chunk < chunks; chunk += gridDim.x) {
    index = tensorOf(table, count, chunk, index);
    const AdamTensor &t = table.t[index];
    const int64_t first = int64_t(chunk - t.first) * U * kAdamRound + threadIdx.x / 32 * U * kMomentGroup;
    float *out = static_cast<float *>(t.param);
    const bool sign = t.m != nullptr;
    const uint8_t *codes = static_cast<const uint8_t *>(sign ? t.m : t.v), *exponents = sign ? t.me : t.ve;
    auto value = [&](uint32_t code, uint32_t e, int low) {
      const int c = sign ? int(int8_t(code)) : int(code & 0xff);
      const float magnitude = e == 255 ? __int_as_float(0x7fffffff) : momentValue(abs(c), low);
      return c < 0 ? -magnitude : magnitude;
    };
    if (t.pieces && first + U * kMomentGroup <= t.n) {   // whole groups, all asked for at once
      uint32_t code[U], e[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        code[u] = *reinterpret_cast<const uint32_t *>(codes + first + u * kMomentGroup + 4 * lane);
        e[u] = exponents[first / kMomentGroup + u];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int low = sign ? lowestCode<127>(e[u]) : lowestCode<255>(e[u]);
        *reinterpret_cast<float4 *>(out + first + u * kMomentGroup + 4 * lane) =
            make_float4(value(code[u], e[u], low), value(code[u] >> 8, e[u], low), value(code[u] >> 16, e[u], low),
                        value(code[u] >> 24, e[u], low));
      }
    } else {
      for (int64_t at = first; at < min(t.n, first + U * kMomentGroup); at += kMomentGroup) {
        const uint32_t e = exponents[at / kMomentGroup];
        const int low = sign ? lowestCode<127>(e) : lowestCode<255>(e);
        for (int64_t i = at + lane; i < min(t.n, at + kMomentGroup); i += 32) out[i] = value(codes[i], e, low);
      }
    }
  }
}

}  // namespace duckb200
