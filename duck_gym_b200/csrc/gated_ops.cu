// C entries of the gated recurrence (declared in include/duck_b200.h): argument
// checks, the choice of a kernel, launches.
#include "capi.hpp"
#include "gated_recurrence.cuh"

#include <algorithm>
#include <initializer_list>

using namespace duckb200;

namespace {

int64_t ceilDiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
void requireType(int type) { require(type == DUCK_FLOAT32 || type == DUCK_BFLOAT16, "Invalid element type"); }

constexpr int kStepsMax = INT32_MAX - (1 << 24);   // steps are counted in 32 bits, a few chunks past the last one

bool recurrenceChecked(const duck_recurrence *a) {
  require(a != nullptr, "Invalid arguments");
  requireType(a->type);
  require(a->T >= 0 && a->E >= 0 && a->N >= 0, "Invalid recurrence sizes");
  require(int64_t(a->E) * a->N < (int64_t(1) << 31), "Too many environments and channels");
  require(a->T <= kStepsMax, "Too many steps");
  return a->E > 0 && a->N > 0;
}
void requireAligned(std::initializer_list<const void *> pointers) {
  for (const void *p : pointers)
    require(reinterpret_cast<uintptr_t>(p) % 16 == 0, "States, outputs and workspaces have to be 16-byte aligned");
}

// How the steps are split where two channels a thread leave fewer than eight warps on a multiprocessor.
struct RecurrencePlan {
  int segmentLength, segments;
  int64_t scratchBytes, keptBytes;
};
RecurrencePlan planRecurrence(const duck_recurrence &a) {
  RecurrencePlan p{};
  const int64_t channels = int64_t(a.E) * a.N, threads = ceilDiv(channels, 2);
  const int64_t want = threads >= 148 * 256 ? 1 : std::max<int64_t>(1, std::min<int64_t>(a.T / 64, 148 * 512 / threads));
  p.segmentLength = int(ceilDiv(ceilDiv(std::max(1, a.T), want), kKeep) * kKeep);
  p.segments = std::max(1, int(ceilDiv(a.T, p.segmentLength)));
  if (p.segments > 1) p.scratchBytes = int64_t(p.segments) * 2 * channels * 4;
  p.keptBytes = a.T > 0 ? (ceilDiv(a.T, kKeep) - 1) * channels * 4 : 0;
  return p;
}

// Whether V channels can be moved at once: a lot of them belongs to one environment and lies on its own boundary.
bool lotsOf(int V, int N, int type, std::initializer_list<const void *> pointers, std::initializer_list<int64_t> strides) {
  const int size = V * (type == DUCK_FLOAT32 ? 4 : 2);
  bool ok = N % V == 0;
  for (const void *p : pointers) ok = ok && reinterpret_cast<uintptr_t>(p) % size == 0;
  for (int64_t s : strides) ok = ok && s % V == 0;
  return ok;
}

RecurrenceArgs argsOf(const duck_recurrence &a, const RecurrencePlan &plan) {
  RecurrenceArgs r{};
  r.gates = a.gates, r.values = a.values, r.dout = a.dout;
  r.out = a.out, r.dgates = a.dgates, r.dvalues = a.dvalues;
  r.gs = {a.gates_stride[0], a.gates_stride[1]};
  r.vs = {a.values_stride[0], a.values_stride[1]};
  r.os = {a.dout_stride[0], a.dout_stride[1]};
  r.stateIn = a.state_in, r.dstateOut = a.dstate_out;
  r.stateOut = a.state_out, r.dstateIn = a.dstate_in;
  r.resets = a.resets;
  r.kept = a.saved, r.segments = a.scratch;
  r.T = a.T, r.E = a.E, r.N = a.N;
  r.segmentLength = plan.segmentLength, r.segmentCount = plan.segments;
  return r;
}

// No steps: the state before them is the one after them.
void copyState(const duck_recurrence &a, const float *from, float *to, cudaStream_t stream) {
  if (!to) return;
  const size_t bytes = size_t(a.E) * a.N * sizeof(float);
  check(from ? cudaMemcpyAsync(to, from, bytes, cudaMemcpyDeviceToDevice, stream) : cudaMemsetAsync(to, 0, bytes, stream),
        "gated recurrence state");
}

dim3 recurrenceGrid(int64_t channels, int V, int segments) {
  return dim3(unsigned(ceilDiv(channels, int64_t(kRecurrenceThreads) * V)), unsigned(segments));
}

template <class T, int V> void launchForward(const RecurrenceArgs &r, cudaStream_t stream) {
  const int64_t channels = int64_t(r.E) * r.N;
  if (r.segmentCount > 1)
    recurrenceForward<T, V, false><<<recurrenceGrid(channels, V, r.segmentCount - 1), kRecurrenceThreads, 0, stream>>>(r);
  recurrenceForward<T, V, true><<<recurrenceGrid(channels, V, r.segmentCount), kRecurrenceThreads, 0, stream>>>(r);
}
template <class T, int V> void launchBackward(const RecurrenceArgs &r, cudaStream_t stream) {
  const int64_t channels = int64_t(r.E) * r.N;
  if (r.segmentCount > 1)
    recurrenceBackwardSegments<T, V><<<recurrenceGrid(channels, V, r.segmentCount - 1), kRecurrenceThreads, 0, stream>>>(r);
  recurrenceBackward<T, V><<<recurrenceGrid(channels, V, r.segmentCount), kRecurrenceThreads, 0, stream>>>(r);
}

}  // namespace

extern "C" {

int duck_gated_recurrence_sizes(const duck_recurrence *args, int64_t *out) {
  return guarded([&] {
    require(out != nullptr, "Invalid arguments");
    out[0] = out[1] = 0;
    if (!recurrenceChecked(args)) return;
    const RecurrencePlan plan = planRecurrence(*args);
    out[0] = plan.scratchBytes;
    out[1] = plan.keptBytes;
  });
}

int duck_gated_recurrence_forward(const duck_recurrence *args, duck_stream stream) {
  return guarded([&] {
    if (!recurrenceChecked(args)) return;
    const duck_recurrence &a = *args;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    requireAligned({a.out, a.state_in, a.state_out, a.saved, a.scratch});
    if (a.T == 0) return copyState(a, a.state_in, a.state_out, s);
    require(a.gates && a.values && a.out, "Invalid arguments");
    const RecurrencePlan plan = planRecurrence(a);
    require(plan.segments == 1 || a.scratch, "Invalid arguments");
    const RecurrenceArgs r = argsOf(a, plan);
    auto lots = [&](int V) {
      return lotsOf(V, a.N, a.type, {a.gates, a.values, a.out},
                    {a.gates_stride[0], a.gates_stride[1], a.values_stride[0], a.values_stride[1]});
    };
    const bool four = int64_t(a.E) * a.N >= int64_t(148) * 2048 && lots(4), two = lots(2);
    if (a.type == DUCK_FLOAT32)
      four ? launchForward<float, 4>(r, s) : two ? launchForward<float, 2>(r, s) : launchForward<float, 1>(r, s);
    else
      four ? launchForward<bf16, 4>(r, s) : two ? launchForward<bf16, 2>(r, s) : launchForward<bf16, 1>(r, s);
    check(cudaGetLastError(), "gated recurrence launch");
  });
}

int duck_gated_recurrence_backward(const duck_recurrence *args, duck_stream stream) {
  return guarded([&] {
    if (!recurrenceChecked(args)) return;
    const duck_recurrence &a = *args;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    requireAligned({a.state_in, a.dstate_out, a.dgates, a.dvalues, a.dstate_in, a.saved, a.scratch});
    if (a.T == 0) return copyState(a, a.dstate_out, a.dstate_in, s);
    require(a.gates && a.values && a.dout && a.dgates && a.dvalues, "Invalid arguments");
    const RecurrencePlan plan = planRecurrence(a);
    require((plan.segments == 1 || a.scratch) && (plan.keptBytes == 0 || a.saved), "Invalid arguments");
    const RecurrenceArgs r = argsOf(a, plan);
    const bool two = lotsOf(2, a.N, a.type, {a.gates, a.values, a.dout, a.dgates, a.dvalues},
                            {a.gates_stride[0], a.gates_stride[1], a.values_stride[0], a.values_stride[1],
                             a.dout_stride[0], a.dout_stride[1]});
    if (a.type == DUCK_FLOAT32) two ? launchBackward<float, 2>(r, s) : launchBackward<float, 1>(r, s);
    else two ? launchBackward<bf16, 2>(r, s) : launchBackward<bf16, 1>(r, s);
    check(cudaGetLastError(), "gated recurrence backward launch");
  });
}

int duck_gated_recurrence_step(const duck_recurrence *args, duck_stream stream) {
  return guarded([&] {
    if (!recurrenceChecked(args)) return;
    const duck_recurrence &a = *args;
    require(a.gates && a.values && a.out && a.state_out, "Invalid arguments");
    require(reinterpret_cast<uintptr_t>(a.state_out) % 4 == 0, "Invalid arguments");
    const int64_t channels = int64_t(a.E) * a.N;
    RecurrenceStep r{a.gates, a.values, a.out, a.state_out, a.resets, a.gates_stride[1], a.values_stride[1], channels, a.N};
    const bool four = reinterpret_cast<uintptr_t>(a.state_out) % 16 == 0 &&
                      lotsOf(4, a.N, a.type, {a.gates, a.values, a.out}, {a.gates_stride[1], a.values_stride[1]});
    const unsigned blocks = unsigned(ceilDiv(channels, int64_t(kRecurrenceThreads) * (four ? 4 : 1)));
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (a.type == DUCK_FLOAT32)
      four ? recurrenceStep<float, 4><<<blocks, kRecurrenceThreads, 0, s>>>(r)
           : recurrenceStep<float, 1><<<blocks, kRecurrenceThreads, 0, s>>>(r);
    else
      four ? recurrenceStep<bf16, 4><<<blocks, kRecurrenceThreads, 0, s>>>(r)
           : recurrenceStep<bf16, 1><<<blocks, kRecurrenceThreads, 0, s>>>(r);
    check(cudaGetLastError(), "gated recurrence step launch");
  });
}

}  // extern "C"
