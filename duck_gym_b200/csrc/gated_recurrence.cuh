// Gated linear recurrence over rollouts with episode ends, channel by channel:
//
//   f_t = sigmoid(gate_t),  h_t = f_t h_{t-1} + (1 - f_t) c_t,
//
// h_{t-1} being zero where an episode begins at t (reset_t).  With the gradient
// dh_t = dout_t + f_{t+1} dh_{t+1} (without the second term where one begins at
// t + 1)
//
//   dgate_t = dh_t (h_{t-1} - c_t) f_t (1 - f_t),   dc_t = dh_t (1 - f_t),
//   dh_initial = f_0 dh_0, or 0.
//
// A reset replaces the state instead of multiplying it by zero: what an earlier
// episode left there, infinities and NaN included, does not reach the next one.
// f and 1 - f both come from t = exp(-|gate|), 1 / (1 + t) and t / (1 + t), so
// that neither loses digits where the other is near 1.
//
// A thread has V neighbouring channels of one environment and goes along the
// steps with h in float32 registers; outputs are rounded once.  The backward
// pass needs h_{t-1} in float32: the forward pass keeps h at every kKeep-th step
// only, and the backward pass, which reads gates and values anyway, runs kKeep
// steps forwards from there in registers before it goes back through them.  So
// it moves five values an element and 8 / kKeep bytes, and out is not read.
//
// Where channels are few, the steps are split into segments.  A segment maps the
// state that it begins with to h -> P h + B; a first pass finds P and B of each
// segment, and the second one begins each segment with those before it applied
// to the initial state.  P < 0 (never a product of gates) says that an episode
// begins inside, B alone being what is left.
//
// Bound by memory, as elementwise passes are.
#pragma once
#include "numeric_types.cuh"

namespace duckb200 {

constexpr int kKeep = 16;             // steps between kept states; segments are whole multiples
constexpr int kRecurrenceThreads = 128;

struct RecurrenceRows {
  int64_t t, e;
};

struct RecurrenceArgs {
  const void *gates, *values, *dout;
  void *out, *dgates, *dvalues;        // [T, E, N] dense
  RecurrenceRows gs, vs, os;
  const float *stateIn, *dstateOut;    // [E, N] or null: zero
  float *stateOut, *dstateIn;          // or null
  const uint8_t *resets;               // [T, E] dense, or null
  float *kept;                         // [ceil(T / kKeep) - 1, E, N]: h before step kKeep, 2 kKeep, ...; or null
  float *segments;                     // [segments, 2, E, N]: P and B
  int T, E, N, segmentLength, segmentCount;
};

// V values that are moved at once.
template <class T, int V> struct Lot {
  T x[V];
};
template <> struct __align__(4) Lot<bf16, 2> { bf16 x[2]; };
template <> struct __align__(8) Lot<bf16, 4> { bf16 x[4]; };
template <> struct __align__(8) Lot<float, 2> { float x[2]; };
template <> struct __align__(16) Lot<float, 4> { float x[4]; };

template <class T, int V> __device__ __forceinline__ Lot<T, V> loadLot(const T *p) {
  return *reinterpret_cast<const Lot<T, V> *>(p);
}
template <class T, int V> __device__ __forceinline__ void storeLot(T *p, const float (&v)[V]) {
  Lot<T, V> lot;
#pragma unroll
  for (int i = 0; i < V; ++i) lot.x[i] = fromFloat<T>(v[i]);
  *reinterpret_cast<Lot<T, V> *>(p) = lot;
}

struct Gate {
  float f, rest;   // sigmoid(gate) and 1 - sigmoid(gate)
};
// For bfloat16, whose gates are known to 2^-9, the exponential and the quotient
// that the hardware approximates (2^-21); for float32 those that are rounded.
template <class T> __device__ __forceinline__ Gate gateOf(T gate) {
  const float g = toFloat(gate);
  float t, r;
  if constexpr (sizeof(T) == 2) {
    t = __expf(-fabsf(g));
    r = __fdividef(1.f, 1.f + t);
  } else {
    t = expf(-fabsf(g));
    r = 1.f / (1.f + t);
  }
  const float s = t * r;
  return g >= 0.f ? Gate{r, s} : Gate{s, r};
}

// What begins a segment: the maps of the segments before it (`forwards`) or
// after it, applied to the state of the rollout's own end.
template <int V> __device__ __forceinline__ void applySegments(const RecurrenceArgs &p, float (&h)[V], int64_t channel,
                                                               int64_t channels, int from, int count, int step) {
#pragma unroll 4
  for (int i = 0; i < count; ++i) {
    const float *at = p.segments + int64_t(from + i * step) * 2 * channels + channel;
    const Lot<float, V> P = loadLot<float, V>(at), B = loadLot<float, V>(at + channels);
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = P.x[v] < 0.f ? B.x[v] : P.x[v] * h[v] + B.x[v];
  }
}

// OUT = false: P and B of the segment instead of its outputs.
template <class T, int V, bool OUT> __global__ void __launch_bounds__(kRecurrenceThreads) recurrenceForward(RecurrenceArgs p) {
  constexpr int C = 8;   // steps whose operands are on their way while as many are computed
  const int64_t channels = int64_t(p.E) * p.N;
  const int64_t channel = (int64_t(blockIdx.x) * kRecurrenceThreads + threadIdx.x) * V;
  if (channel >= channels) return;
  const int e = int(channel / p.N), n = int(channel - int64_t(e) * p.N), segment = blockIdx.y;
  const T *gates = static_cast<const T *>(p.gates) + e * p.gs.e + n;
  const T *values = static_cast<const T *>(p.values) + e * p.vs.e + n;
  const int begin = segment * p.segmentLength, end = min(p.T, begin + p.segmentLength);
  float h[V], P[V];
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = 0.f, P[v] = 1.f;
  if (OUT) {
    if (p.stateIn) {
      const Lot<float, V> s = loadLot<float, V>(p.stateIn + channel);
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = s.x[v];
    }
    applySegments<V>(p, h, channel, channels, 0, segment, 1);
  }
  Lot<T, V> g[2][C], c[2][C];
  bool cut[2][C];
  auto load = [&](int set, int t0) {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int t = t0 + i;
      if (t < end) {
        g[set][i] = loadLot<T, V>(gates + t * p.gs.t);
        c[set][i] = loadLot<T, V>(values + t * p.vs.t);
        cut[set][i] = p.resets && p.resets[int64_t(t) * p.E + e];
      }
    }
  };
  auto advance = [&](int set, int t0) {
    if (OUT && p.kept && t0 > 0 && t0 % kKeep == 0) storeLot<float, V>(p.kept + int64_t(t0 / kKeep - 1) * channels + channel, h);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      if (t0 + i >= end) break;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Gate f = gateOf(g[set][i].x[v]);
        const float add = f.rest * toFloat(c[set][i].x[v]);
        h[v] = cut[set][i] ? add : f.f * h[v] + add;
        if (!OUT) P[v] = cut[set][i] || P[v] < 0.f ? -1.f : P[v] * f.f;
      }
      if (OUT) storeLot<T, V>(static_cast<T *>(p.out) + int64_t(t0 + i) * channels + channel, h);
    }
  };
  load(0, begin);
  for (int t0 = begin; t0 < end; t0 += 2 * C) {
    load(1, t0 + C);
    advance(0, t0);
    load(0, t0 + 2 * C);
    if (t0 + C < end) advance(1, t0 + C);
  }
  if (!OUT) {
    float *at = p.segments + int64_t(segment) * 2 * channels + channel;
    storeLot<float, V>(at, P);
    storeLot<float, V>(at + channels, h);
  } else if (p.stateOut && segment == p.segmentCount - 1) {
    storeLot<float, V>(p.stateOut + channel, h);
  }
}

// P and B of the segments of the backward pass, for the gradient that leaves a
// segment at its beginning; segment 0's is not needed.
template <class T, int V> __global__ void __launch_bounds__(kRecurrenceThreads) recurrenceBackwardSegments(RecurrenceArgs p) {
  constexpr int C = 8;
  const int64_t channels = int64_t(p.E) * p.N;
  const int64_t channel = (int64_t(blockIdx.x) * kRecurrenceThreads + threadIdx.x) * V;
  if (channel >= channels) return;
  const int e = int(channel / p.N), n = int(channel - int64_t(e) * p.N), segment = blockIdx.y + 1;
  const T *gates = static_cast<const T *>(p.gates) + e * p.gs.e + n;
  const T *dout = static_cast<const T *>(p.dout) + e * p.os.e + n;
  const int begin = segment * p.segmentLength, end = min(p.T, begin + p.segmentLength);
  float x[V], P[V];
#pragma unroll
  for (int v = 0; v < V; ++v) x[v] = 0.f, P[v] = 1.f;
  Lot<T, V> g[2][C], d[2][C];
  bool cut[2][C];
  // Backwards: step `last` - i is the i-th.
  auto load = [&](int set, int last) {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int t = last - i;
      if (t >= begin) {
        g[set][i] = loadLot<T, V>(gates + t * p.gs.t);
        d[set][i] = loadLot<T, V>(dout + t * p.os.t);
        cut[set][i] = p.resets && p.resets[int64_t(t) * p.E + e];
      }
    }
  };
  auto advance = [&](int set, int last) {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      if (last - i < begin) break;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float f = gateOf(g[set][i].x[v]).f;
        x[v] = cut[set][i] ? 0.f : f * (x[v] + toFloat(d[set][i].x[v]));
        P[v] = cut[set][i] || P[v] < 0.f ? -1.f : P[v] * f;
      }
    }
  };
  load(0, end - 1);
  for (int last = end - 1; last >= begin; last -= 2 * C) {
    load(1, last - C);
    advance(0, last);
    load(0, last - 2 * C);
    advance(1, last - C);
  }
  float *at = p.segments + int64_t(segment) * 2 * channels + channel;
  storeLot<float, V>(at, P);
  storeLot<float, V>(at + channels, x);
}

template <class T, int V> __global__ void __launch_bounds__(kRecurrenceThreads) recurrenceBackward(RecurrenceArgs p) {
  const int64_t channels = int64_t(p.E) * p.N;
  const int64_t channel = (int64_t(blockIdx.x) * kRecurrenceThreads + threadIdx.x) * V;
  if (channel >= channels) return;
  const int e = int(channel / p.N), n = int(channel - int64_t(e) * p.N), segment = blockIdx.y;
  const T *gates = static_cast<const T *>(p.gates) + e * p.gs.e + n;
  const T *values = static_cast<const T *>(p.values) + e * p.vs.e + n;
  const T *dout = static_cast<const T *>(p.dout) + e * p.os.e + n;
  const int begin = segment * p.segmentLength, end = min(p.T, begin + p.segmentLength);
  float x[V];   // the gradient that comes from later steps
#pragma unroll
  for (int v = 0; v < V; ++v) x[v] = 0.f;
  if (p.dstateOut) {
    const Lot<float, V> s = loadLot<float, V>(p.dstateOut + channel);
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = s.x[v];
  }
  applySegments<V>(p, x, channel, channels, p.segmentCount - 1, p.segmentCount - 1 - segment, -1);
  for (int t0 = begin + (end - 1 - begin) / kKeep * kKeep; t0 >= begin; t0 -= kKeep) {
    Lot<T, V> g[kKeep], c[kKeep], d[kKeep];
    float h[kKeep][V];   // before each step
    uint32_t cuts = 0;
    const float *from = t0 == 0 ? p.stateIn : p.kept + int64_t(t0 / kKeep - 1) * channels;
    Lot<float, V> first{};
    if (from) first = loadLot<float, V>(from + channel);
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
      const int t = t0 + i;
      if (t < end) {
        g[i] = loadLot<T, V>(gates + t * p.gs.t);
        c[i] = loadLot<T, V>(values + t * p.vs.t);
        d[i] = loadLot<T, V>(dout + t * p.os.t);
        if (p.resets) cuts |= uint32_t(p.resets[int64_t(t) * p.E + e] != 0) << i;
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float now = first.x[v];
#pragma unroll
      for (int i = 0; i < kKeep; ++i) {
        if (t0 + i >= end) break;
        if (cuts >> i & 1) now = 0.f;
        h[i][v] = now;
        const Gate f = gateOf(g[i].x[v]);
        now = f.f * now + f.rest * toFloat(c[i].x[v]);
      }
    }
#pragma unroll
    for (int i = kKeep - 1; i >= 0; --i) {
      if (t0 + i >= end) continue;
      float dg[V], dc[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Gate f = gateOf(g[i].x[v]);
        const float dh = x[v] + toFloat(d[i].x[v]);
        dc[v] = dh * f.rest;
        dg[v] = dc[v] * f.f * (h[i][v] - toFloat(c[i].x[v]));
        x[v] = cuts >> i & 1 ? 0.f : dh * f.f;
      }
      const int64_t at = int64_t(t0 + i) * channels + channel;
      storeLot<T, V>(static_cast<T *>(p.dgates) + at, dg);
      storeLot<T, V>(static_cast<T *>(p.dvalues) + at, dc);
    }
  }
  if (p.dstateIn && segment == 0) storeLot<float, V>(p.dstateIn + channel, x);
}

// One step of every environment, the state updated in place.
struct RecurrenceStep {
  const void *gates, *values;
  void *out;
  float *state;
  const uint8_t *resets;   // [E] or null
  int64_t gatesE, valuesE;
  int64_t channels;
  int N;
};
template <class T, int V> __global__ void __launch_bounds__(kRecurrenceThreads) recurrenceStep(RecurrenceStep p) {
  const int64_t channel = (int64_t(blockIdx.x) * kRecurrenceThreads + threadIdx.x) * V;
  if (channel >= p.channels) return;
  const int64_t e = channel / p.N;
  const int n = int(channel - e * p.N);
  const Lot<T, V> g = loadLot<T, V>(static_cast<const T *>(p.gates) + e * p.gatesE + n);
  const Lot<T, V> c = loadLot<T, V>(static_cast<const T *>(p.values) + e * p.valuesE + n);
  const Lot<float, V> s = loadLot<float, V>(p.state + channel);
  const bool cut = p.resets && p.resets[e];
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const Gate f = gateOf(g.x[v]);
    const float add = f.rest * toFloat(c.x[v]);
    h[v] = cut ? add : f.f * s.x[v] + add;
  }
  storeLot<float, V>(p.state + channel, h);
  storeLot<T, V>(static_cast<T *>(p.out) + channel, h);
}

}  // namespace duckb200
