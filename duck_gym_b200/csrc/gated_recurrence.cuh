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
// f and 1 - f both come from one exponential t, as 1 / (1 + t) and t / (1 + t), so
// that neither loses digits where the other is near 1.
//
// A thread has V neighbouring channels of one environment and goes along the
// steps with h in float32 registers; outputs are rounded once.  The backward
// pass needs h_{t-1} in float32: the forward pass keeps h at every kKeep-th step
// only, and the backward pass, which reads gates and values anyway, runs kKeep
// steps forwards from there in registers before it goes back through them.  So
// it moves five values an element and 4 / kKeep bytes each way, and out is not read.
//
// Where channels are few, the steps are split into segments.  A segment maps the
// state that it begins with to h -> P h + B; a first pass finds P and B of each
// segment, and the second one begins each segment with those before it applied
// to the initial state.  P's sign bit (products of gates have none) says that an
// episode begins inside, B alone being what is left.
//
// Bound by memory in principle; 24 instructions a value in the forward pass (issue
// slots 56 % busy) and warps that wait for their copies keep it at 60 % of the copy's
// rate.  Measured on a B200, cold,
// bfloat16: 24 steps of 1024 x 256 channels, forward 12 us, backward 15.5 (38 and
// 65 MB); 1000 steps of 256 x 256, 108 and 153 us (3.6 and 4.3 TB/s, both of them with
// the kept states); 16384 steps of 1024 channels in 74 segments, 24 us for P and B and
// 32 for the outputs.  One step of 4096 x 256 channels 4.6 us.
#pragma once
#include "numeric_types.cuh"

namespace duckb200 {

constexpr int kKeep = 8;             // steps between kept states; segments are whole multiples
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

// V values that are moved at once, as one word, pair or quad of words.
template <int BYTES> struct Word;
template <> struct Word<2> { using type = unsigned short; };
template <> struct Word<4> { using type = unsigned; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<16> { using type = uint4; };
template <class T, int V> struct Lot {
  typename Word<V * int(sizeof(T))>::type w;
  __device__ __forceinline__ float at(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(reinterpret_cast<const unsigned *>(&w)[i]);
    else if constexpr (V == 1) return __uint_as_float(unsigned(w) << 16);
    else {
      const unsigned two = reinterpret_cast<const unsigned *>(&w)[i / 2];
      return __uint_as_float(i % 2 ? two & 0xffff0000u : two << 16);
    }
  }
};
template <class T, int V> __device__ __forceinline__ Lot<T, V> loadLot(const T *p) {
  return {*reinterpret_cast<const typename Word<V * int(sizeof(T))>::type *>(p)};
}
template <class T, int V> __device__ __forceinline__ void storeLot(T *p, const float (&v)[V]) {
  typename Word<V * int(sizeof(T))>::type w;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) reinterpret_cast<unsigned *>(&w)[i] = __float_as_uint(v[i]);
  } else if constexpr (V == 1) {
    w = __bfloat16_as_ushort(__float2bfloat16_rn(v[0]));
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const __nv_bfloat162 two = __floats2bfloat162_rn(v[i], v[i + 1]);
      reinterpret_cast<unsigned *>(&w)[i / 2] = *reinterpret_cast<const unsigned *>(&two);
    }
  }
  *reinterpret_cast<typename Word<V * int(sizeof(T))>::type *>(p) = w;
}

struct Gate {
  float f, rest;   // sigmoid(gate) and 1 - sigmoid(gate)
};
// For bfloat16, whose gates are known to 2^-9, the exponential and the quotient
// that the hardware approximates (2^-21), exp(-gate) held at 2^126 (a NaN stays one),
// whose reciprocal is the smallest normal number, and taken off: a gate from -87.3 down
// leaves nothing of a state, however large; for float32 the rounded exponential, of -|gate|, and the hardware's
// reciprocal of a number between 1 and 2 after one of Newton's iterations, so that
// neither f nor 1 - f loses digits where the other is near 1.
template <class T> __device__ __forceinline__ Gate gateOf(float g) {
  if constexpr (sizeof(T) == 2) {
    float t, r;
    asm("min.NaN.f32 %0, %1, 0f42FC0000;" : "=f"(t) : "f"(g * -1.4426950408889634f));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(t));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + t));
    return {r - 1.17549435e-38f, t * r};
  } else {
    const float t = expf(-fabsf(g)), d = 1.f + t;
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    r = fmaf(r, fmaf(-d, r, 1.f), r);
    const float s = t * r;
    return g >= 0.f ? Gate{r, s} : Gate{s, r};
  }
}

// What begins a segment: the maps of the segments before it (`forwards`) or
// after it, applied to the state of the rollout's own end.
template <int V> __device__ __forceinline__ void applySegments(const RecurrenceArgs &p, float (&h)[V], int64_t channel,
                                                               int64_t channels, int from, int count, int step) {
#pragma unroll 8
  for (int i = 0; i < count; ++i) {
    const float *at = p.segments + int64_t(from + i * step) * 2 * channels + channel;
    const Lot<float, V> P = loadLot<float, V>(at), B = loadLot<float, V>(at + channels);
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = __float_as_int(P.at(v)) < 0 ? B.at(v) : P.at(v) * h[v] + B.at(v);
  }
}

// A thread's operands on their way: slots of kKeep steps in shared memory, of A
// arrays, which only this thread writes and reads.  So few registers wait for
// memory, and where threads are few more slots keep as many bytes under way.
template <class T, int V, int A, int SLOTS> struct Ring {
  using W = typename Word<V * int(sizeof(T))>::type;
  static constexpr int words = A * kKeep * kRecurrenceThreads;   // of a slot
  static constexpr int bytes = SLOTS * words * int(sizeof(W));
  W *at;
  __device__ __forceinline__ explicit Ring(void *shared) : at(static_cast<W *>(shared) + threadIdx.x) {}
  __device__ __forceinline__ void copy(int slot, int array, int step, const T *from) {
    W *to = at + slot * words + (array * kKeep + step) * kRecurrenceThreads;
    if constexpr (sizeof(W) >= 4)
      asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(uint32_t(__cvta_generic_to_shared(to))), "l"(from),
                   "n"(int(sizeof(W)))
                   : "memory");
    else
      *to = *reinterpret_cast<const W *>(from);
  }
  __device__ __forceinline__ Lot<T, V> get(int slot, int array, int step) const {
    return {at[slot * words + (array * kKeep + step) * kRecurrenceThreads]};
  }
};
__device__ __forceinline__ void copiesIssued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LATER> __device__ __forceinline__ void copiesWait() { asm volatile("cp.async.wait_group %0;" ::"n"(LATER) : "memory"); }

// What a thread works on.
template <int V> struct Place {
  int64_t channels, channel;
  int e, n;
  int group;   // of the warp's environments, if all its threads have channels of at most four; else -1
  __device__ __forceinline__ explicit Place(const RecurrenceArgs &p)
      : channels(int64_t(p.E) * p.N), channel((int64_t(blockIdx.x) * kRecurrenceThreads + threadIdx.x) * V),
        e(int(channel / p.N)), n(int(channel - int64_t(e) * p.N)) {
    const int first = __shfl_sync(0xffffffffu, e, 0);   // (by all lanes: not in a condition)
    const bool few = channel < channels && e - first < 4;
    group = __all_sync(0xffffffffu, few) ? e - first : -1;
  }
};

// The resets of kAsked chunks, asked for as many chunks ahead and left as they are
// in memory meanwhile (a comparison, or a copy, would wait for them): a lane has
// one of a chunk's eight steps of one of four environments.  In a warp of more
// environments, or at the last channels, each thread reads its own when it needs
// them.
constexpr int kAsked = 4;
struct Resets {
  const uint8_t *at;
  int64_t E;
  int group, step, by;        // the lane's step of a chunk, and from chunk to chunk
  uint8_t asked[kAsked];
  uint32_t masks;             // a byte for each chunk
  static_assert(kKeep == 8, "lanes of a chunk");
  template <class P> __device__ __forceinline__ Resets(const RecurrenceArgs &p, const P &place, int by)
      : at(nullptr), E(p.E), group(place.group), step(threadIdx.x % 8), by(by), masks(0) {
    const int other = place.e - place.group + threadIdx.x % 32 / 8;   // environment whose steps this lane asks for
    if (p.resets) at = p.resets + (group >= 0 ? min(other, p.E - 1) : place.e);
  }
  __device__ __forceinline__ void ask(int t0, int begin, int end) {
    if (at == nullptr || group < 0) return;
#pragma unroll
    for (int k = 0; k < kAsked; ++k) {
      const int t = t0 + k * by + step;
      asked[k] = 0;
      if (t >= begin && t < end) asked[k] = at[t * E];
    }
  }
  __device__ __forceinline__ void take() {
    if (at == nullptr || group < 0) return;
    masks = 0;
#pragma unroll
    for (int k = 0; k < kAsked; ++k) masks |= (__ballot_sync(0xffffffffu, asked[k] != 0) >> 8 * group & 0xffu) << 8 * k;
  }
  // Of the k-th of the chunks, which begins at t0.
  __device__ __forceinline__ uint32_t chunk(int k, int t0, int end) const {
    if (at == nullptr) return 0;
    if (group >= 0) return masks >> 8 * k & 0xffu;
    uint32_t mask = 0;
#pragma unroll
    for (int i = 0; i < kKeep; ++i) mask |= uint32_t(t0 + i < end && at[int64_t(t0 + i) * E] != 0) << i;
    return mask;
  }
};

// OUT = false: P and B of the segment instead of its outputs.
template <class T, int V, int SLOTS, bool OUT>
__global__ void __launch_bounds__(kRecurrenceThreads) recurrenceForward(RecurrenceArgs p) {
  extern __shared__ __align__(16) uint8_t shared[];
  const Place<V> at(p);
  if (at.channel >= at.channels) return;
  const int segment = blockIdx.y;
  const int begin = segment * p.segmentLength, end = min(p.T, begin + p.segmentLength);
  const T *gates = static_cast<const T *>(p.gates) + at.e * p.gs.e + at.n + begin * p.gs.t;
  const T *values = static_cast<const T *>(p.values) + at.e * p.vs.e + at.n + begin * p.vs.t;
  Ring<T, V, 2, SLOTS> ring(shared);
  Resets resets(p, at, kKeep);
  int asked = begin, slot = 0;   // the next step to be copied, and where to
  auto ask = [&] {
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
      if (asked + i < end) {
        ring.copy(slot, 0, i, gates);
        ring.copy(slot, 1, i, values);
      }
      gates += p.gs.t, values += p.vs.t;
    }
    copiesIssued();
    asked += kKeep;
    slot = slot + 1 == SLOTS ? 0 : slot + 1;
  };
  resets.ask(begin, begin, end);
#pragma unroll
  for (int k = 0; k < SLOTS - 1; ++k) ask();
  float h[V], P[V];
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = 0.f, P[v] = 1.f;
  if (OUT) {
    if (p.stateIn) {
      const Lot<float, V> s = loadLot<float, V>(p.stateIn + at.channel);
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = s.at(v);
    }
    applySegments<V>(p, h, at.channel, at.channels, 0, segment, 1);
  }
  T *out = static_cast<T *>(p.out) + int64_t(begin) * at.channels + at.channel;
  for (int t0 = begin, from = 0, k = 0; t0 < end; t0 += kKeep, k = (k + 1) % kAsked) {
    if (k == 0) {
      resets.take();
      resets.ask(t0 + kAsked * kKeep, begin, end);
    }
    const uint32_t cuts = resets.chunk(k, t0, end);
    ask();
    copiesWait<SLOTS - 1>();
    if (OUT && p.kept && t0 > 0) storeLot<float, V>(p.kept + int64_t(t0 / kKeep - 1) * at.channels + at.channel, h);
    // The gates of a chunk do not wait on one another; the states do, by one product a step.
    float f[kKeep][V], add[kKeep][V];
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
      const Lot<T, V> g = ring.get(from, 0, i), c = ring.get(from, 1, i);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Gate gate = gateOf<T>(g.at(v));
        f[i][v] = gate.f;
        add[i][v] = gate.rest * c.at(v);
      }
    }
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
      const bool in = t0 + i < end, cut = cuts >> i & 1;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float next = cut ? add[i][v] : f[i][v] * h[v] + add[i][v];
        h[v] = in ? next : h[v];
        if (!OUT) {
          const float product = cut ? -1.f : P[v] * f[i][v];
          P[v] = in ? product : P[v];
        }
      }
      if (OUT && in) storeLot<T, V>(out, h);
      out += at.channels;
    }
    from = from + 1 == SLOTS ? 0 : from + 1;
  }
  if (!OUT) {
    float *to = p.segments + int64_t(segment) * 2 * at.channels + at.channel;
    storeLot<float, V>(to, P);
    storeLot<float, V>(to + at.channels, h);
  } else if (p.stateOut && segment == p.segmentCount - 1) {
    storeLot<float, V>(p.stateOut + at.channel, h);
  }
}

// P and B of the segments of the backward pass, for the gradient that leaves a
// segment at its beginning; segment 0's is not needed.  Chunks as below.
template <class T, int V, int SLOTS>
__global__ void __launch_bounds__(kRecurrenceThreads) recurrenceBackwardSegments(RecurrenceArgs p) {
  extern __shared__ __align__(16) uint8_t shared[];
  const Place<V> at(p);
  if (at.channel >= at.channels) return;
  const int segment = blockIdx.y + 1;
  const int begin = segment * p.segmentLength, end = min(p.T, begin + p.segmentLength);
  int t0 = begin + (end - 1 - begin) / kKeep * kKeep, asked = t0, slot = 0;
  const T *gates = static_cast<const T *>(p.gates) + at.e * p.gs.e + at.n + t0 * p.gs.t;
  const T *dout = static_cast<const T *>(p.dout) + at.e * p.os.e + at.n + t0 * p.os.t;
  Ring<T, V, 2, SLOTS> ring(shared);
  Resets resets(p, at, -kKeep);
  auto ask = [&] {
    const T *gt = gates, *ot = dout;
#pragma unroll
    for (int i = 0; i < kKeep; ++i, gt += p.gs.t, ot += p.os.t)
      if (asked >= begin && asked + i < end) {
        ring.copy(slot, 0, i, gt);
        ring.copy(slot, 1, i, ot);
      }
    copiesIssued();
    asked -= kKeep, gates -= kKeep * p.gs.t, dout -= kKeep * p.os.t;
    slot = slot + 1 == SLOTS ? 0 : slot + 1;
  };
  resets.ask(t0, begin, end);
#pragma unroll
  for (int k = 0; k < SLOTS - 1; ++k) ask();
  float x[V], P[V];
#pragma unroll
  for (int v = 0; v < V; ++v) x[v] = 0.f, P[v] = 1.f;
  for (int from = 0, k = 0; t0 >= begin; t0 -= kKeep, k = (k + 1) % kAsked) {
    if (k == 0) {
      resets.take();
      resets.ask(t0 - kAsked * kKeep, begin, end);
    }
    const uint32_t cuts = resets.chunk(k, t0, end);
    ask();
    copiesWait<SLOTS - 1>();
    float f[kKeep][V], d[kKeep][V];
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
      const Lot<T, V> g = ring.get(from, 0, i), o = ring.get(from, 1, i);
#pragma unroll
      for (int v = 0; v < V; ++v) f[i][v] = gateOf<T>(g.at(v)).f, d[i][v] = o.at(v);
    }
#pragma unroll
    for (int i = kKeep - 1; i >= 0; --i) {
      const bool in = t0 + i < end, cut = cuts >> i & 1;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float next = cut ? 0.f : f[i][v] * (x[v] + d[i][v]);
        const float product = cut ? -1.f : P[v] * f[i][v];
        x[v] = in ? next : x[v];
        P[v] = in ? product : P[v];
      }
    }
    from = from + 1 == SLOTS ? 0 : from + 1;
  }
  float *to = p.segments + int64_t(segment) * 2 * at.channels + at.channel;
  storeLot<float, V>(to, P);
  storeLot<float, V>(to + at.channels, x);
}

template <class T, int V, int SLOTS> __global__ void __launch_bounds__(kRecurrenceThreads) recurrenceBackward(RecurrenceArgs p) {
  extern __shared__ __align__(16) uint8_t shared[];
  const Place<V> at(p);
  if (at.channel >= at.channels) return;
  const int segment = blockIdx.y;
  const int begin = segment * p.segmentLength, end = min(p.T, begin + p.segmentLength);
  int t0 = begin + (end - 1 - begin) / kKeep * kKeep, asked = t0, slot = 0;
  const T *gates = static_cast<const T *>(p.gates) + at.e * p.gs.e + at.n + t0 * p.gs.t;
  const T *values = static_cast<const T *>(p.values) + at.e * p.vs.e + at.n + t0 * p.vs.t;
  const T *dout = static_cast<const T *>(p.dout) + at.e * p.os.e + at.n + t0 * p.os.t;
  Ring<T, V, 3, SLOTS> ring(shared);
  Resets resets(p, at, -kKeep);
  auto ask = [&] {
    const T *gt = gates, *vt = values, *ot = dout;
#pragma unroll
    for (int i = 0; i < kKeep; ++i, gt += p.gs.t, vt += p.vs.t, ot += p.os.t)
      if (asked >= begin && asked + i < end) {
        ring.copy(slot, 0, i, gt);
        ring.copy(slot, 1, i, vt);
        ring.copy(slot, 2, i, ot);
      }
    copiesIssued();
    asked -= kKeep, gates -= kKeep * p.gs.t, values -= kKeep * p.vs.t, dout -= kKeep * p.os.t;
    slot = slot + 1 == SLOTS ? 0 : slot + 1;
  };
  auto before = [&](int t) {   // the state before step t, the first one of a chunk
    Lot<float, V> s{};
    if (t < begin) return s;
    if (t > 0) return loadLot<float, V>(p.kept + int64_t(t / kKeep - 1) * at.channels + at.channel);
    return p.stateIn ? loadLot<float, V>(p.stateIn + at.channel) : s;
  };
  resets.ask(t0, begin, end);
#pragma unroll
  for (int k = 0; k < SLOTS - 1; ++k) ask();
  Lot<float, V> state = before(t0);
  float x[V];   // the gradient that comes from later steps
#pragma unroll
  for (int v = 0; v < V; ++v) x[v] = 0.f;
  if (p.dstateOut) {
    const Lot<float, V> s = loadLot<float, V>(p.dstateOut + at.channel);
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = s.at(v);
  }
  applySegments<V>(p, x, at.channel, at.channels, p.segmentCount - 1, p.segmentCount - 1 - segment, -1);
  T *dg = static_cast<T *>(p.dgates) + int64_t(t0) * at.channels + at.channel;
  T *dc = static_cast<T *>(p.dvalues) + int64_t(t0) * at.channels + at.channel;
  for (int from = 0, k = 0; t0 >= begin; t0 -= kKeep, k = (k + 1) % kAsked) {
    if (k == 0) {
      resets.take();
      resets.ask(t0 - kAsked * kKeep, begin, end);
    }
    const uint32_t cuts = resets.chunk(k, t0, end);
    ask();
    const Lot<float, V> first = state;
    state = before(t0 - kKeep);
    copiesWait<SLOTS - 1>();
    // Forwards through the states, of which dgate = dh slope needs the one before each step.
    float f[kKeep][V], rest[kKeep][V], slope[kKeep][V], now[V];
#pragma unroll
    for (int v = 0; v < V; ++v) now[v] = first.at(v);
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
      const Lot<T, V> g = ring.get(from, 0, i), c = ring.get(from, 1, i);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Gate gate = gateOf<T>(g.at(v));
        const float value = c.at(v);
        f[i][v] = gate.f, rest[i][v] = gate.rest;
        if (cuts >> i & 1) now[v] = 0.f;
        slope[i][v] = gate.f * gate.rest * (now[v] - value);
        now[v] = gate.f * now[v] + gate.rest * value;
      }
    }
#pragma unroll
    for (int i = kKeep - 1; i >= 0; --i) {
      const bool in = t0 + i < end, cut = cuts >> i & 1;
      const Lot<T, V> d = ring.get(from, 2, i);
      float a[V], b[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float dh = x[v] + d.at(v);
        a[v] = dh * slope[i][v];
        b[v] = dh * rest[i][v];
        const float next = cut ? 0.f : dh * f[i][v];
        x[v] = in ? next : x[v];
      }
      if (in) {
        storeLot<T, V>(dg + i * at.channels, a);
        storeLot<T, V>(dc + i * at.channels, b);
      }
    }
    dg -= kKeep * at.channels, dc -= kKeep * at.channels;
    from = from + 1 == SLOTS ? 0 : from + 1;
  }
  if (p.dstateIn && segment == 0) storeLot<float, V>(p.dstateIn + at.channel, x);
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
    const Gate f = gateOf<T>(g.at(v));
    const float add = f.rest * c.at(v);
    h[v] = cut ? add : f.f * s.at(v) + add;
  }
  storeLot<float, V>(p.state + channel, h);
  storeLot<T, V>(static_cast<T *>(p.out) + channel, h);
}

}  // namespace duckb200
