// C entries of the gated recurrence and of the gated linear layer (declared in
// include/duck_b200.h): argument checks, the choice of a kernel, launches.
#include "capi.hpp"
#include "gated_linear.cuh"
#include "gated_recurrence.cuh"

#include <algorithm>
#include <atomic>
#include <initializer_list>
#include <new>

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

// How the steps are split where two channels a thread leave fewer than four warps on a multiprocessor: into segments of 64
// steps at least that give it eight.  They are read twice, so that where threads are enough one pass is faster (1000 steps,
// 256 x 256 channels: 261 us forward and backward, 396 in two segments); a replay of 16384 steps of 1024 channels takes 56 us.
struct RecurrencePlan {
  int segmentLength, segments;
  int64_t scratchBytes, keptBytes;
};
RecurrencePlan planRecurrence(const duck_recurrence &a) {
  RecurrencePlan p{};
  const int64_t channels = int64_t(a.E) * a.N, threads = ceilDiv(channels, 2);
  const int64_t want = threads >= 148 * 128 ? 1 : std::max<int64_t>(1, std::min<int64_t>(a.T / 64, 148 * 256 / threads));
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

// Dynamic shared memory above 48 KB has to be asked for, once per kernel and device
// (by whichever thread comes first: autograd calls from its own).
template <auto kernel> void allowShared(int bytes) {
  static std::atomic<bool> done[64] = {};
  int device = 0;
  check(cudaGetDevice(&device), "cudaGetDevice");
  if (device < 64 && done[device]) return;
  check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "cudaFuncSetAttribute");
  if (device < 64) done[device] = true;
}

dim3 recurrenceGrid(int64_t channels, int V, int segments) {
  return dim3(unsigned(ceilDiv(channels, int64_t(kRecurrenceThreads) * V)), unsigned(segments));
}

template <class T, int V, int SLOTS> void launchForward(const RecurrenceArgs &r, cudaStream_t stream) {
  const int64_t channels = int64_t(r.E) * r.N;
  constexpr int bytes = Ring<T, V, 2, SLOTS>::bytes;
  constexpr auto find = recurrenceForward<T, V, SLOTS, false>, run = recurrenceForward<T, V, SLOTS, true>;
  if constexpr (bytes > 48 * 1024) allowShared<find>(bytes), allowShared<run>(bytes);
  if (r.segmentCount > 1) find<<<recurrenceGrid(channels, V, r.segmentCount - 1), kRecurrenceThreads, bytes, stream>>>(r);
  run<<<recurrenceGrid(channels, V, r.segmentCount), kRecurrenceThreads, bytes, stream>>>(r);
}
template <class T, int V, int SLOTS> void launchBackward(const RecurrenceArgs &r, cudaStream_t stream) {
  const int64_t channels = int64_t(r.E) * r.N;
  constexpr int findBytes = Ring<T, V, 2, SLOTS>::bytes, bytes = Ring<T, V, 3, SLOTS>::bytes;
  constexpr auto find = recurrenceBackwardSegments<T, V, SLOTS>;
  constexpr auto run = recurrenceBackward<T, V, SLOTS>;
  if constexpr (findBytes > 48 * 1024) allowShared<find>(findBytes);
  if constexpr (bytes > 48 * 1024) allowShared<run>(bytes);
  if (r.segmentCount > 1) find<<<recurrenceGrid(channels, V, r.segmentCount - 1), kRecurrenceThreads, findBytes, stream>>>(r);
  run<<<recurrenceGrid(channels, V, r.segmentCount), kRecurrenceThreads, bytes, stream>>>(r);
}
// Two channels a thread where they can be moved at once (four take twice the registers: a second, partly filled round of
// blocks).  Four slots where there are fewer than 512 threads a multiprocessor (1000 steps, 256 x 256 channels: forward 108 us,
// backward 153; eight slots the same, blocks of 32 or 64 threads too), two where there are more and their copies fill the
// memory's queue.
constexpr int kFewThreads = 148 * 512, kFewSlots = 4;
template <class T, class F> void withSlots(const RecurrenceArgs &r, bool two, F &&f) {
  const bool few = ceilDiv(int64_t(r.E) * r.N, two ? 2 : 1) * r.segmentCount < kFewThreads;
  auto slots = [&](auto v) {
    if (few) f(v, std::integral_constant<int, kFewSlots>());
    else f(v, std::integral_constant<int, 2>());
  };
  if (two) slots(std::integral_constant<int, 2>());
  else slots(std::integral_constant<int, 1>());
}
template <class F> void withLots(const duck_recurrence &a, const RecurrenceArgs &r, bool two, F &&f) {
  if (a.type == DUCK_FLOAT32) withSlots<float>(r, two, [&](auto v, auto slots) { f(0.f, v, slots); });
  else withSlots<bf16>(r, two, [&](auto v, auto slots) { f(bf16(), v, slots); });
}

// ---------------------------------------------------------------- gated linear
// Products that a tensor core adds up in one accumulator.  It cuts its sums off where float32 rounds them, so that sums of one
// sign come out too small: 65536 products by 6e-4, a third of a rounding to bfloat16 in the mean square, a million by 6e-3.
// Longer sums are made of parts, added in float32; those of the projections, whose accumulators go nowhere but into the
// activation, are refused.
constexpr int kTensorSum = 1 << 16;

bool gatedChecked(const duck_gated *a) {
  require(a != nullptr, "Invalid arguments");
  requireType(a->type);
  require(a->rows >= 0 && a->D > 0 && a->F > 0, "Invalid layer sizes");
  require(a->rows < (int64_t(1) << 31) - 4096 && a->D <= (1 << 20) && a->F <= (1 << 20), "Too many rows or columns");
  require(a->type == DUCK_FLOAT32 || a->D <= kTensorSum, "bfloat16 layers have 65536 columns at most");
  require(a->activation >= DUCK_SILU && a->activation <= DUCK_SIGMOID, "Invalid activation");
  require(a->type == DUCK_FLOAT32 || a->D % 8 || a->rows <= 1 || a->x == nullptr || a->x_stride >= a->D,
          "bfloat16 rows must not overlap");
  return a->rows > 0;
}

int64_t wholeColumns(int64_t D) { return ceilDiv(D, 8) * 8; }
// How a backward call's workspace is laid out.
struct GatedPlan {
  int stride;                // bfloat16: of da and du
  int weightColumns;         // of a tile of the weights' gradients
  int splits;                // of the rows, for the weights' gradients
  int weightTile;            // float32: rows and columns of a tile of them
  int inputColumns, inputSplits;   // of a tile of the gradient of x (float32: rows too), and of F
  int64_t biasCount;
  int64_t bothBytes, biasBytes, partBytes, inputBytes, keptBytes;   // in this order
};
// Where tiles leave multiprocessors idle, the steps of their products are split, so that each part has `least` at least;
// and where they are more than `most`.
int splitsOf(int64_t tiles, int64_t fit, int64_t steps, int64_t least, int64_t most = INT64_MAX) {
  const int64_t splits = std::max({int64_t(1), std::min<int64_t>(fit / tiles, steps / least), (steps - 1) / most + 1});
  return int(std::max<int64_t>(1, ceilDiv(steps, ceilDiv(std::max<int64_t>(1, steps), splits))));   // none without steps
}
int64_t padded(int64_t bytes) { return ceilDiv(bytes, 256) * 256; }
// Columns of a tile, of which a row of tiles has `columns`: rounds of tiles over the multiprocessors, times a tile's time.  A
// product of 128 columns takes 0.77 of the time of one of 256: its operands' way out of shared memory bounds it (16384 x 4096
// by 1024 twice: 291 us in tiles of 128 columns, 216 in those of 256).
int tileColumns(int64_t rowTiles, int64_t columns) {
  int best = 0;
  int64_t least = 0;
  for (int n : {256, 128, 64}) {
    if (n > 64 && n / 2 >= columns) continue;
    const int64_t cost = ceilDiv(rowTiles * ceilDiv(columns, n), 148) * (n == 256 ? 100 : n == 128 ? 77 : 65);
    if (best == 0 || cost < least) best = n, least = cost;
  }
  return best;
}
// float32 products in tiles of 128 by 128, or of 64 by 64 where those are less than the multiprocessors or half empty (4999
// rows, 61 x 301: the gradient of x 85 us in 40 tiles of 128, 35 in 79 of 64, 21 with their steps split three ways).
int productTile(int64_t rows, int64_t columns) {
  return columns <= 64 || ceilDiv(rows, 128) * ceilDiv(columns, 128) < 148 ? 64 : 128;
}
GatedPlan planGated(const duck_gated &a) {
  GatedPlan p{};
  const bool weights = a.dw_gate != nullptr, biases = a.db_gate != nullptr;
  const int64_t rows = a.rows;
  if (a.type == DUCK_BFLOAT16) {
    p.stride = int(ceilDiv(a.F, 8) * 8);
    if (a.D % 8) p.keptBytes = (rows + 2 * int64_t(a.F)) * wholeColumns(a.D) * 2;
    p.bothBytes = padded(rows * 2 * p.stride * 2);
    p.biasCount = ceilDiv(rows, kTileRows) * 4;
    // Rows are split so that the tiles fill the GPU once, into parts of 512 rows at least: a part's sums are written and read
    // once more (24576 rows, 256 x 512: 17 us in 18 parts of 256 columns, 20 in 9 of 128).
    p.weightColumns = a.D > 128 ? 256 : a.D > 64 ? 128 : 64;
    constexpr int most = kTensorSum / kTileSteps;
    p.splits = splitsOf(2 * ceilDiv(a.F, kTileRows) * ceilDiv(a.D, p.weightColumns), 148, ceilDiv(rows, kTileSteps), 8, most);
    // x's gradient of few rows (66 rows, 136 x 3788: three tiles of 120 steps each otherwise).
    const int64_t rowTiles = ceilDiv(rows, kTileRows);
    p.inputColumns = tileColumns(rowTiles, a.D);
    p.inputSplits = splitsOf(rowTiles * ceilDiv(a.D, p.inputColumns), 148, 2 * ceilDiv(a.F, kTileSteps), 8, most);
  } else {
    p.bothBytes = padded(rows * 2 * a.F * 4);
    p.keptBytes = rows * 2 * a.F * 4;
    p.biasCount = ceilDiv(rows, kGradientRows);
    // Parts of 128 rows at least, or of 128 features.
    const int64_t large = 2 * ceilDiv(a.F, 128) * ceilDiv(a.D, 128) * std::max<int64_t>(1, rows / 128);
    p.weightTile = a.D <= 64 || large < 148 ? 64 : 128;
    p.splits = splitsOf(2 * ceilDiv(a.F, p.weightTile) * ceilDiv(a.D, p.weightTile), 2 * 148,
                        ceilDiv(rows, productSteps(p.weightTile)), 128 / productSteps(p.weightTile));
    p.inputColumns = productTile(rows, a.D);
    p.inputSplits = splitsOf(ceilDiv(rows, p.inputColumns) * ceilDiv(a.D, p.inputColumns), 2 * 148,
                             2 * ceilDiv(a.F, productSteps(p.inputColumns)), 128 / productSteps(p.inputColumns));
  }
  if (biases) p.biasBytes = padded(p.biasCount * 2 * a.F * 4);
  if (weights && (a.type == DUCK_FLOAT32 || p.splits > 1)) p.partBytes = padded(int64_t(p.splits) * 2 * a.F * a.D * 4);
  if (a.dx && p.inputSplits > 1) p.inputBytes = padded(p.inputSplits * rows * a.D * 4);
  return p;
}

// A map over bfloat16 rows for boxes of boxColumns values (64, 32 or 16: as wide as the swizzle) by boxRows rows.
CUtensorMap mapOf(const void *base, int64_t columns, int64_t rows, int64_t stride, int boxRows, int boxColumns = 64) {
  using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                              const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void *entry = nullptr;
    cudaDriverEntryPointQueryResult found;
    check(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &entry, 12000, cudaEnableDefault, &found),
          "cuTensorMapEncodeTiled");
    if (found != cudaDriverEntryPointSuccess || !entry) throw CudaError("cuTensorMapEncodeTiled: not in the driver");
    return reinterpret_cast<Encode>(entry);
  }();
  CUtensorMap map;
  const cuuint64_t sizes[2] = {cuuint64_t(columns), cuuint64_t(rows)}, strides[1] = {cuuint64_t(stride) * 2};
  const cuuint32_t box[2] = {cuuint32_t(boxColumns), cuuint32_t(boxRows)}, steps[2] = {1, 1};
  const CUtensorMapSwizzle swizzle = boxColumns == 64   ? CU_TENSOR_MAP_SWIZZLE_128B
                                     : boxColumns == 32 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                        : CU_TENSOR_MAP_SWIZZLE_32B;
  auto fill = [&] {
    return encode(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(base), sizes, strides, box, steps,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult status = fill();
  if (status == CUDA_ERROR_INVALID_CONTEXT || status == CUDA_ERROR_NOT_INITIALIZED) {
    // A thread's first call, before any that made its device's context current (autograd has threads of its own).
    int device = 0;
    check(cudaGetDevice(&device), "cudaGetDevice");
    check(cudaSetDevice(device), "cudaSetDevice");
    status = fill();
  }
  require(status != CUDA_ERROR_INVALID_VALUE, "Rows have to be whole 16-byte pieces on 16-byte boundaries");
  if (status != CUDA_SUCCESS) throw CudaError("cuTensorMapEncodeTiled: error " + std::to_string(int(status)));
  return map;
}

template <Pass PASS, int BN> void launchTiles(const TileMaps &maps, const TileArgs &t, cudaStream_t stream) {
  constexpr auto kernel = gatedTiles<PASS, BN>;
  constexpr int bytes = TileShared<PASS, BN>::bytes;
  allowShared<kernel>(bytes);
  kernel<<<std::min(t.tiles, 148), kTileThreads, bytes, stream>>>(maps, t);
  check(cudaGetLastError(), "gated linear launch");
}

template <class F> void withColumns(int columns, F &&f) {
  if (columns == 256) f(std::integral_constant<int, 256>());
  else if (columns == 128) f(std::integral_constant<int, 128>());
  else f(std::integral_constant<int, 64>());
}

// Both projections, side by side.
template <Pass PASS> void launchProjections(const duck_gated &a, TileArgs t, cudaStream_t stream) {   // a: operandsOf()
  const int64_t rowTiles = ceilDiv(a.rows, kTileRows);
  auto run = [&](auto columns) {
    constexpr int BN = columns.value;
    constexpr int part = TileShared<PASS, BN>::part;
    TileMaps maps{};   // (those that a pass does not use are not read)
    if (PASS == Pass::gradients) {
      if (t.wholeDh) maps.dh = mapOf(t.dh, a.F, a.rows, a.rows > 1 ? t.dhStride : t.stride, 32, part);
      maps.out0 = mapOf(t.both, a.F, a.rows, 2 * int64_t(t.stride), 32, part);
      maps.out1 = mapOf(t.both + t.stride, a.F, a.rows, 2 * int64_t(t.stride), 32, part);
    } else if (t.wholeH) {
      maps.out0 = mapOf(t.h, a.F, a.rows, a.F, 32, part);
    }
    maps.a0 = mapOf(a.x, a.D, a.rows, a.rows > 1 ? a.x_stride : a.D, kTileRows);
    maps.b0 = mapOf(a.w_gate, a.D, a.F, a.D, BN / 2);
    maps.b1 = mapOf(a.w_up, a.D, a.F, a.D, BN / 2);
    t.steps = int(ceilDiv(a.D, kTileSteps));
    t.columnTiles = int(ceilDiv(a.F, BN / 2));
    const int64_t tiles = rowTiles * t.columnTiles;
    require(tiles < (int64_t(1) << 31), "Too many rows and columns");
    t.tiles = int(tiles);
    launchTiles<PASS, BN>(maps, t, stream);
  };
  withColumns(tileColumns(rowTiles, 2 * int64_t(a.F)), run);
}
std::atomic<int64_t> waitLimit{int64_t(kWaitLimit)};
// A word of host memory that the kernels of every device reach, and set where a wait ran out.
std::atomic<int> &ranOut() {
  static std::atomic<int> *const word = [] {
    // The first call may be a captured one, and this is no work of its stream.
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    check(cudaThreadExchangeStreamCaptureMode(&mode), "cudaThreadExchangeStreamCaptureMode");
    void *memory = nullptr;
    const cudaError_t status = cudaHostAlloc(&memory, sizeof(std::atomic<int>), cudaHostAllocPortable | cudaHostAllocMapped);
    check(cudaThreadExchangeStreamCaptureMode(&mode), "cudaThreadExchangeStreamCaptureMode");
    check(status, "cudaHostAlloc");
    return new (memory) std::atomic<int>(0);
  }();
  return *word;
}
void waitsChecked() {
  if (ranOut().load(std::memory_order_relaxed) && ranOut().exchange(0))
    throw CudaError("gated linear: a wait of an earlier call's kernel ran out, and results of it are NaN");
}
TileArgs tileArgs(const duck_gated &a) {
  TileArgs t{};
  t.waitLimit = uint64_t(waitLimit.load());
  t.ranOut = reinterpret_cast<volatile int *>(&ranOut());
  t.bGate = static_cast<const bf16 *>(a.b_gate);
  t.bUp = static_cast<const bf16 *>(a.b_up);
  t.rows = a.rows, t.D = a.D, t.F = a.F, t.activation = a.activation;
  t.wholeD = a.D % 8 == 0;
  t.wholeBias = reinterpret_cast<uintptr_t>(a.b_gate) % 16 == 0 && reinterpret_cast<uintptr_t>(a.b_up) % 16 == 0;
  t.splits = 1;
  return t;
}
// The operands that the tiles read, with D for their rows: the call's own, or the copies that a forward call has padded.
duck_gated operandsOf(const duck_gated &a) {
  duck_gated o = a;
  if (a.D % 8 == 0) return o;
  const int64_t stride = wholeColumns(a.D);
  const bf16 *kept = static_cast<const bf16 *>(a.kept);
  o.x = kept, o.x_stride = stride, o.D = int(stride);
  o.w_gate = kept + a.rows * stride, o.w_up = kept + (a.rows + a.F) * stride;
  return o;
}
ProductArgs productArgs(const duck_gated &a) {
  ProductArgs g{};
  g.x = static_cast<const float *>(a.x);
  g.wGate = static_cast<const float *>(a.w_gate);
  g.wUp = static_cast<const float *>(a.w_up);
  g.bGate = static_cast<const float *>(a.b_gate);
  g.bUp = static_cast<const float *>(a.b_up);
  g.rows = a.rows, g.xStride = a.x_stride, g.D = a.D, g.F = a.F, g.activation = a.activation, g.splits = 1;
  g.wholeX = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.x_stride % 4 == 0;
  g.wholeD = a.D % 4 == 0 && reinterpret_cast<uintptr_t>(a.w_gate) % 16 == 0 && reinterpret_cast<uintptr_t>(a.w_up) % 16 == 0;
  g.wholeF = a.F % 4 == 0;
  return g;
}
template <Pass PASS> void launchProducts(const ProductArgs &g, int tile, int64_t rows, int64_t columns, int splits, cudaStream_t stream) {
  const int64_t rowTiles = (PASS == Pass::weights ? 2 : 1) * ceilDiv(rows, tile);
  const dim3 grid(unsigned(rowTiles), unsigned(ceilDiv(columns, tile)), unsigned(splits));
  auto run = [&](auto t, auto runs) {
    constexpr int T = t.value;
    constexpr int bytes = PASS == Pass::forward && runs.value ? T * T * int(sizeof(float)) : 0;
    constexpr auto kernel = gatedProducts<PASS, T, runs.value>;
    if constexpr (bytes > 0) allowShared<kernel>(bytes);
    kernel<<<grid, kProductThreads, bytes, stream>>>(g);
  };
  auto withRuns = [&](auto t) {   // (the code of runs costs a forward pass without them 1.5 %, 16384 rows, 1024 x 1024)
    if constexpr (PASS == Pass::forward)
      if (g.D <= kRunSteps) return run(t, std::false_type());
    run(t, std::true_type());
  };
  if (tile == 128) withRuns(std::integral_constant<int, 128>());
  else withRuns(std::integral_constant<int, 64>());
  check(cudaGetLastError(), "gated linear launch");
}
// Sums of parts to one or two arrays, and of the biases' parts.
template <class T>
void launchSums(const duck_gated &a, const float *parts, int splits, void *first, int64_t cut, void *second, int64_t count,
                const float *biasParts, int64_t biasCount, cudaStream_t stream) {
  SumArgs<T> s{parts, biasParts, static_cast<T *>(first), static_cast<T *>(second), static_cast<T *>(a.db_gate),
               static_cast<T *>(a.db_up), cut, count, a.F, splits, int(biasCount), 0};
  const int64_t some = parts ? ceilDiv(count, kSumThreads * 4) : 0, all = some + (biasParts ? ceilDiv(2 * int64_t(a.F), kSumColumns) : 0);
  if (all == 0) return;
  require(all < (int64_t(1) << 31), "Too many rows and columns");
  s.blocks = int(some);
  sumParts<T><<<unsigned(all), kSumThreads, 0, stream>>>(s);
  check(cudaGetLastError(), "gated linear sums launch");
}
template <class T>
void launchSums(const duck_gated &a, const GatedPlan &plan, const float *parts, const float *biasParts, const float *inputParts,
                cudaStream_t stream) {
  const int64_t weights = int64_t(a.F) * a.D, input = a.rows * a.D;
  launchSums<T>(a, parts, plan.splits, a.dw_gate, weights, a.dw_up, 2 * weights, biasParts, plan.biasCount, stream);
  if (inputParts) launchSums<T>(a, inputParts, plan.inputSplits, a.dx, input, nullptr, input, nullptr, 0, stream);
}

void gatedBackward16(const duck_gated &a, const GatedPlan &plan, cudaStream_t stream) {
  TileArgs t = tileArgs(a);
  unsigned char *scratch = static_cast<unsigned char *>(a.scratch);
  t.both = reinterpret_cast<bf16 *>(scratch);
  t.stride = plan.stride;
  float *biasParts = a.db_gate ? reinterpret_cast<float *>(scratch + plan.bothBytes) : nullptr;
  float *parts = plan.partBytes ? reinterpret_cast<float *>(scratch + plan.bothBytes + plan.biasBytes) : nullptr;
  float *inputParts = plan.inputBytes ? reinterpret_cast<float *>(scratch + plan.bothBytes + plan.biasBytes + plan.partBytes) : nullptr;
  t.dh = static_cast<const bf16 *>(a.dh);
  t.dhStride = a.dh_stride;
  t.wholeDh = reinterpret_cast<uintptr_t>(a.dh) % 16 == 0 && a.dh_stride % 8 == 0 && a.dh_stride >= a.F;
  t.biasParts = biasParts;
  const duck_gated o = operandsOf(a);
  launchProjections<Pass::gradients>(o, t, stream);
  const int64_t rowTiles = ceilDiv(a.rows, kTileRows);
  if (a.dx) {
    t.dx = static_cast<bf16 *>(a.dx);
    t.steps = int(ceilDiv(a.F, kTileSteps));
    t.rowTiles = int(rowTiles);
    t.splits = plan.inputSplits;
    t.parts = inputParts;
    withColumns(plan.inputColumns, [&](auto n) {
      TileMaps maps{};
      maps.a0 = mapOf(t.both, a.F, a.rows, 2 * int64_t(plan.stride), kTileRows);
      maps.a1 = mapOf(t.both + plan.stride, a.F, a.rows, 2 * int64_t(plan.stride), kTileRows);
      maps.b0 = mapOf(o.w_gate, o.D, a.F, o.D, 64);
      maps.b1 = mapOf(o.w_up, o.D, a.F, o.D, 64);
      t.columnTiles = int(ceilDiv(a.D, n.value));
      const int64_t tiles = rowTiles * t.columnTiles * t.splits;
      require(tiles < (int64_t(1) << 31), "Too many rows and columns");
      t.tiles = int(tiles);
      launchTiles<Pass::input, n.value>(maps, t, stream);
    });
  }
  if (a.dw_gate) {
    t.dwGate = static_cast<bf16 *>(a.dw_gate);
    t.dwUp = static_cast<bf16 *>(a.dw_up);
    t.parts = parts;
    t.splits = plan.splits;
    t.steps = int(ceilDiv(a.rows, kTileSteps));
    t.rowTiles = int(ceilDiv(a.F, kTileRows));
    withColumns(plan.weightColumns, [&](auto n) {
      TileMaps maps{};
      maps.a0 = mapOf(t.both, a.F, a.rows, 2 * int64_t(plan.stride), 64);
      maps.a1 = mapOf(t.both + plan.stride, a.F, a.rows, 2 * int64_t(plan.stride), 64);
      maps.b0 = mapOf(o.x, o.D, a.rows, a.rows > 1 ? o.x_stride : o.D, 64);
      t.columnTiles = int(ceilDiv(a.D, n.value));
      const int64_t tiles = int64_t(t.columnTiles) * 2 * t.rowTiles * t.splits;
      require(tiles < (int64_t(1) << 31), "Too many rows and columns");
      t.tiles = int(tiles);
      launchTiles<Pass::weights, n.value>(maps, t, stream);
    });
  }
  launchSums<bf16>(a, plan, parts, biasParts, inputParts, stream);
}

void gatedBackward32(const duck_gated &a, const GatedPlan &plan, cudaStream_t stream) {
  ProductArgs g = productArgs(a);
  unsigned char *scratch = static_cast<unsigned char *>(a.scratch);
  float *both = reinterpret_cast<float *>(scratch);
  float *biasParts = a.db_gate ? reinterpret_cast<float *>(scratch + plan.bothBytes) : nullptr;
  float *parts = a.dw_gate ? reinterpret_cast<float *>(scratch + plan.bothBytes + plan.biasBytes) : nullptr;
  float *inputParts = plan.inputBytes ? reinterpret_cast<float *>(scratch + plan.bothBytes + plan.biasBytes + plan.partBytes) : nullptr;
  const int64_t rowBlocks = ceilDiv(a.rows, kGradientRows);
  const GradientArgs e{static_cast<const float *>(a.kept), static_cast<const float *>(a.dh), both, biasParts, a.rows, a.dh_stride,
                       a.F, a.activation};
  gatedGradients<<<dim3(unsigned(rowBlocks), unsigned(ceilDiv(a.F, 32))), 256, 0, stream>>>(e);
  check(cudaGetLastError(), "gated linear launch");
  g.both = both;
  if (a.dx) {
    g.dx = static_cast<float *>(a.dx);
    g.parts = inputParts;
    g.splits = plan.inputSplits;
    launchProducts<Pass::input>(g, plan.inputColumns, a.rows, a.D, plan.inputSplits, stream);
  }
  if (a.dw_gate) {
    g.parts = parts;
    g.splits = plan.splits;
    launchProducts<Pass::weights>(g, plan.weightTile, a.F, a.D, plan.splits, stream);
  }
  launchSums<float>(a, plan, parts, biasParts, inputParts, stream);
}

}  // namespace

extern "C" {

int duck_gated_linear_sizes(const duck_gated *args, int64_t *out) {
  return guarded([&] {
    require(out != nullptr, "Invalid arguments");
    out[0] = out[1] = 0;
    if (!gatedChecked(args)) return;
    const GatedPlan plan = planGated(*args);
    out[0] = plan.bothBytes + plan.biasBytes + plan.partBytes + plan.inputBytes;
    out[1] = plan.keptBytes;
  });
}

int duck_wait_limit(int64_t nanoseconds) {
  return guarded([&] {
    require(nanoseconds >= 0, "A wait's limit is 0 or more");
    waitLimit = nanoseconds;
  });
}

int duck_wait_status(void) {
  return guarded([&] { waitsChecked(); });
}

int duck_gated_linear_forward(const duck_gated *args, duck_stream stream) {
  return guarded([&] {
    if (!gatedChecked(args)) return;
    if (args->type == DUCK_BFLOAT16) waitsChecked();
    const duck_gated &a = *args;
    require(a.x && a.w_gate && a.w_up && a.h && !a.b_gate == !a.b_up, "Invalid arguments");
    requireAligned({a.h, a.kept});
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (a.type == DUCK_BFLOAT16) {
      TileArgs t = tileArgs(a);
      t.h = static_cast<bf16 *>(a.h);
      t.wholeH = a.F % 8 == 0;
      const duck_gated o = operandsOf(a);
      if (a.D % 8) {
        require(a.kept, "Invalid arguments");
        const PadArgs p{static_cast<const bf16 *>(a.x), static_cast<const bf16 *>(a.w_gate), static_cast<const bf16 *>(a.w_up),
                        static_cast<bf16 *>(a.kept), a.rows, a.x_stride, a.D, a.F, o.D};
        const int64_t blocks = ceilDiv((a.rows + 2 * int64_t(a.F)) * (o.D / 8), kPadThreads);
        padRows<<<unsigned(std::min<int64_t>(blocks, 148 * 8)), kPadThreads, 0, s>>>(p);
        check(cudaGetLastError(), "gated linear launch");
      }
      return launchProjections<Pass::forward>(o, t, s);
    }
    ProductArgs g = productArgs(a);
    g.h = static_cast<float *>(a.h);
    g.kept = static_cast<float *>(a.kept);
    launchProducts<Pass::forward>(g, productTile(a.rows, 2 * int64_t(a.F)), a.rows, 2 * int64_t(a.F), 1, s);
  });
}

int duck_gated_linear_backward(const duck_gated *args, duck_stream stream) {
  return guarded([&] {
    const bool some = gatedChecked(args);
    const duck_gated &a = *args;
    if (a.type == DUCK_BFLOAT16) waitsChecked();
    require(!a.dw_gate == !a.dw_up && !a.db_gate == !a.db_up && !a.b_gate == !a.b_up, "Invalid arguments");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (!some) {   // no rows: no sums
      const size_t size = a.type == DUCK_FLOAT32 ? 4 : 2;
      for (void *p : {a.dw_gate, a.dw_up})
        if (p) check(cudaMemsetAsync(p, 0, size_t(a.F) * a.D * size, s), "gated linear gradients");
      for (void *p : {a.db_gate, a.db_up})
        if (p) check(cudaMemsetAsync(p, 0, size_t(a.F) * size, s), "gated linear gradients");
      return;
    }
    if (!a.dx && !a.dw_gate && !a.db_gate) return;
    require(a.x && a.w_gate && a.w_up && a.dh && a.scratch && (a.kept || (a.type == DUCK_BFLOAT16 && a.D % 8 == 0)), "Invalid arguments");
    requireAligned({a.dx, a.dw_gate, a.dw_up, a.kept, a.scratch});
    const GatedPlan plan = planGated(a);
    if (a.type == DUCK_BFLOAT16) gatedBackward16(a, plan, s);
    else gatedBackward32(a, plan, s);
  });
}

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
    const bool two = lotsOf(2, a.N, a.type, {a.gates, a.values, a.out},
                            {a.gates_stride[0], a.gates_stride[1], a.values_stride[0], a.values_stride[1]});
    withLots(a, r, two, [&](auto zero, auto v, auto slots) { launchForward<decltype(zero), v.value, slots.value>(r, s); });
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
    withLots(a, r, two, [&](auto zero, auto v, auto slots) { launchBackward<decltype(zero), v.value, slots.value>(r, s); });
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
