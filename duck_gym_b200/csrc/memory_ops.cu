// C entries of the operators of a policy with memory (declared in
// include/duck_b200.h): argument checks, the choice of a kernel, launches.
#include "attention_chunks.cuh"
#include "capi.hpp"
#include "checkpoint8.cuh"
#include "layer_norm.cuh"
#include "linear_attention.cuh"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <initializer_list>
#include <type_traits>

using namespace duckb200;

namespace {

// Calls f with a value of the element type.
template <class F> void withType(int type, F &&f) {
  if (type == DUCK_FLOAT32) f(0.f);
  else f(bf16());
}
void requireType(int type) { require(type == DUCK_FLOAT32 || type == DUCK_BFLOAT16, "Invalid element type"); }

int64_t ceilDiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Whether rows at these addresses and distances (in elements) are made of whole
// 16-byte pieces; a null pointer is.
bool pieces16(std::initializer_list<const void *> pointers, std::initializer_list<int64_t> strides, int type) {
  const int64_t piece = type == DUCK_FLOAT32 ? 4 : 8;
  for (const void *p : pointers)
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  for (int64_t s : strides)
    if (s % piece) return false;
  return true;
}

// Mean and rstd are moved together.
void requireStats(const float *stats) {
  require(reinterpret_cast<uintptr_t>(stats) % 8 == 0, "Statistics have to be 8-byte aligned");
}

// Layer norm kernels that hold a row in registers: 16-byte pieces where rows are
// made of them, else single values; up to 8192 values.  Calls f with a kernel's
// lanes, values a load and values a lane.
constexpr int kNormWidest = 8192;
template <int N> using Constant = std::integral_constant<int, N>;
template <class T, class F> void withNormRows(int n, bool pieces, F &&f) {
  constexpr int V = 16 / sizeof(T);
  auto wide = [&](auto vec) {
    if (n <= 256) f(Constant<32>(), vec, Constant<8>());
    else if (n <= 512) f(Constant<32>(), vec, Constant<16>());
    else if (n <= 1024) f(Constant<128>(), vec, Constant<8>());
    else if (n <= 2048) f(Constant<256>(), vec, Constant<8>());
    else if (n <= 4096) f(Constant<256>(), vec, Constant<16>());
    else f(Constant<512>(), vec, Constant<16>());
  };
  if (pieces && n <= 64) f(Constant<8>(), Constant<V>(), Constant<8>());
  else if (pieces && n <= 128) f(Constant<16>(), Constant<V>(), Constant<8>());
  else if (pieces) wide(Constant<V>());
  else if (n <= 64) f(Constant<32>(), Constant<1>(), Constant<2>());
  else wide(Constant<1>());
}
// Blocks of a pass over the rows.
int64_t normBlocks(int64_t rows, int n, bool pieces, bool backward) {
  int64_t blocks = 1;
  withNormRows<float>(n, pieces, [&](auto lanes, auto, auto values) {
    constexpr int L = lanes.value;
    // Up to 16 rows a team, one block: its sums need no second kernel, which costs as much as the rows do.
    if (backward && rows <= 16 * (normBlock(L) / L)) return;
    blocks = std::min<int64_t>(ceilDiv(rows, normBlock(L) / L),
                               148 * (backward ? normResident(L, values.value, true) : normResident(L, values.value, false)));
  });
  return std::max<int64_t>(1, blocks);
}

// Partial rows that the sums of the weight's and bias' gradients come in.
int64_t normSplits(int64_t rows, int n) {
  if (n <= kNormWidest) return std::max(normBlocks(rows, n, true, true), normBlocks(rows, n, false, true));
  const int64_t columns = ceilDiv(n, 32);
  return std::max<int64_t>(1, std::min<int64_t>(ceilDiv(rows, 64), ceilDiv(148 * 8, columns)));
}

// Codes are moved 8 or 4 at a time beside pieces of 16 bytes of values; their array
// has to be aligned for that.
enum class Groups { keep, restore, restoreBounded };
void launchGroups(const CheckpointArgs &a, int type, bool pieces, duck_stream stream, Groups what) {
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  pieces = pieces && reinterpret_cast<uintptr_t>(a.codes) % 8 == 0;
  withType(type, [&](auto zero) {
    using T = decltype(zero);
    const int groups = pieces ? kCheckpointThreads / Piece<T>::lanes : kCheckpointThreads / 32 * kGroupsAtOnce;
    const unsigned blocks = unsigned(std::min<int64_t>(ceilDiv(a.rows * a.groups, groups), 148 * 8));
    auto kernel = what == Groups::keep      ? (pieces ? eluCheckpointPieces<T> : eluCheckpointAny<T>)
                  : what == Groups::restore ? (pieces ? eluRestorePieces<T, false> : eluRestoreAny<T, false>)
                                            : (pieces ? eluRestorePieces<T, true> : eluRestoreAny<T, true>);
    kernel<<<blocks, kCheckpointThreads, 0, s>>>(a);
  });
}

int restoreElu(const void *dy, const int8_t *codes, const float *scales, void *y, void *dx, int64_t rows, int n, int type,
               Groups what, duck_stream stream) {
  return guarded([&] {
    requireType(type);
    require(rows >= 0 && n > 0, "Invalid checkpoint sizes");
    if (rows == 0) return;
    require(dy && codes && scales && dx, "Invalid arguments");
    CheckpointArgs a{dy, y, dx, const_cast<int8_t *>(codes), const_cast<float *>(scales), rows, n,
                     int(ceilDiv(n, kGroup))};
    launchGroups(a, type, pieces16({dy, y, dx}, {int64_t(n)}, type), stream, what);
    check(cudaGetLastError(), "checkpoint launch");
  });
}

constexpr int kStepsMax = INT32_MAX - (1 << 24);
bool attentionChecked(const duck_attention *a) {
  require(a != nullptr, "Invalid arguments");
  requireType(a->type);
  require(a->T >= 0 && a->E >= 0 && a->H >= 0, "Invalid attention sizes");
  require(a->Dk > 0 && a->Dk <= kHeadMax && a->Dv > 0 && a->Dv <= kHeadMax, "Head sizes have to be 1 to 128");
  require(int64_t(a->E) * a->H < (int64_t(1) << 31), "Too many environments and heads");
  // Steps are counted in 32 bits, up to a chunk for each of some hundred segments past the last one.
  require(a->T <= kStepsMax, "Too many steps");
  return a->E > 0 && a->H > 0;
}
Rows rowsOf(const int64_t *s) { return {s[0], s[1], s[2]}; }
void requireAligned(std::initializer_list<const void *> pointers) {
  for (const void *p : pointers)
    require(reinterpret_cast<uintptr_t>(p) % 16 == 0, "States, outputs and workspaces have to be 16-byte aligned");
}

// The most rows and columns of some sweeps' states.
int mostRows(const Sweeps &p, int count) {
  int n = 0;
  for (int i = 0; i < count; ++i) n = std::max(n, p.s[i].Di);
  return n;
}
int mostColumns(const Sweeps &p, int count) {
  int n = 0;
  for (int i = 0; i < count; ++i) n = std::max(n, p.s[i].Dj);
  return n;
}
template <int DI, bool OUT> void launchScan(const Sweeps &p, int count, int segments, cudaStream_t stream) {
  const int tiles = int(ceilDiv(mostColumns(p, count), kScanColumns));
  const dim3 grid{unsigned(int64_t(p.s[0].E) * p.s[0].H), unsigned(tiles * segments), unsigned(count)};
  bool padded = false;
  for (int i = 0; i < count; ++i) padded |= p.s[i].Di < DI;
  if (OUT && padded) attentionScan<float, DI, OUT, OUT><<<grid, scanThreads(DI), 0, stream>>>(p, tiles);
  else attentionScan<float, DI, OUT, false><<<grid, scanThreads(DI), 0, stream>>>(p, tiles);
  check(cudaGetLastError(), "linear attention launch");
}
template <bool OUT> void launchScan(const Sweeps &p, int count, int segments, cudaStream_t stream) {
  const int rows = mostRows(p, count);
  if (rows <= 16) launchScan<16, OUT>(p, count, segments, stream);
  else if (rows <= 32) launchScan<32, OUT>(p, count, segments, stream);
  else if (rows <= 64) launchScan<64, OUT>(p, count, segments, stream);
  else launchScan<128, OUT>(p, count, segments, stream);
}

// How a call's steps are split where it has fewer blocks than four a multiprocessor: segments of 64 steps at least.
struct ScanPlan {
  int segmentLength, segments;
  int64_t stateBytes, cutBytes;   // of one sweep
};
ScanPlan planScan(const duck_attention &a) {
  const int64_t blocks = int64_t(a.E) * a.H * ceilDiv(std::max(a.Dk, a.Dv), kScanColumns);
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(a.T / 64, 4 * 148 / blocks));
  ScanPlan p{};
  p.segmentLength = int(ceilDiv(ceilDiv(std::max(1, a.T), want), kScanSteps) * kScanSteps);
  p.segments = std::max(1, int(ceilDiv(a.T, p.segmentLength)));
  if (p.segments > 1) {
    p.cutBytes = ceilDiv(int64_t(a.E) * a.H * p.segments, 16) * 16;
    p.stateBytes = ceilDiv(int64_t(a.E) * a.H * p.segments * a.Dk * a.Dv, 4) * 16;
  }
  return p;
}
// float32 operands.  `own`: which sweeps find their segments' starts; the others share another's.
void runScan(const duck_attention &a, Sweeps p, int count, std::initializer_list<int> own, cudaStream_t stream) {
  const ScanPlan plan = planScan(a);
  for (int i = 0; i < count; ++i) {
    p.s[i].segmentLength = plan.segmentLength;
    p.s[i].segments = plan.segments;
  }
  if (plan.segments > 1) {
    require(a.scratch, "Invalid arguments");
    Sweeps first{};
    int n = 0;
    for (int i : own) {
      unsigned char *at = reinterpret_cast<unsigned char *>(a.scratch) + n * (plan.stateBytes + plan.cutBytes);
      p.s[i].starts = reinterpret_cast<float *>(at);
      p.s[i].cuts = at + plan.stateBytes;
      first.s[n++] = p.s[i];
    }
    for (int i = 0; i < count; ++i)   // (the gradient of k goes along that of v, its state turned)
      if (!p.s[i].starts) p.s[i].starts = first.s[n - 1].starts, p.s[i].cuts = first.s[n - 1].cuts;
    launchScan<false>(first, n, plan.segments - 1, stream);
    const dim3 grid{unsigned(int64_t(a.E) * a.H), unsigned(ceilDiv(int64_t(a.Dk) * a.Dv, 256)), unsigned(n)};
    joinSweeps<<<grid, 256, 0, stream>>>(first);
    check(cudaGetLastError(), "linear attention launch");
  }
  launchScan<true>(p, count, plan.segments, stream);
}
// One round of blocks: there is usually nothing to do but to look at the flags.
void launchRedo(const Sweeps &p, int count, const uint8_t *flags, int flagCount, cudaStream_t stream) {
  const int64_t tiles = ceilDiv(mostColumns(p, count), kScanColumns);
  const int64_t blocks = std::min<int64_t>(int64_t(p.s[0].E) * p.s[0].H, 148 / (tiles * count));
  const dim3 grid{unsigned(blocks), unsigned(tiles), unsigned(count)};
  if (mostRows(p, count) <= 32) redoAttention<32><<<grid, scanThreads(32), 0, stream>>>(p, flags, flagCount);
  else redoAttention<128><<<grid, scanThreads(128), 0, stream>>>(p, flags, flagCount);
  check(cudaGetLastError(), "linear attention launch");
}

// No steps: the state before them is the one after them.
void copyState(const duck_attention &a, const float *from, float *to, cudaStream_t stream) {
  if (!to) return;
  const size_t bytes = size_t(a.E) * a.H * a.Dk * a.Dv * sizeof(float);
  check(from ? cudaMemcpyAsync(to, from, bytes, cudaMemcpyDeviceToDevice, stream) : cudaMemsetAsync(to, 0, bytes, stream),
        "linear attention state");
}

Sweep forwardSweep(const duck_attention &a) {
  return {a.k, a.v, a.q, a.out, rowsOf(a.k_stride), rowsOf(a.v_stride), rowsOf(a.q_stride), a.state_in, a.state_out,
          a.decay, a.resets, a.T, a.E, a.H, a.Dk, a.Dv, a.Dv, 1, 0, 1.f, a.scale, a.T, 1, nullptr, nullptr};
}
Sweep gradientOfQ(const duck_attention &a) {
  return {a.v, a.k, a.dout, a.dq, rowsOf(a.v_stride), rowsOf(a.k_stride), rowsOf(a.dout_stride), a.state_in, nullptr,
          a.decay, a.resets, a.T, a.E, a.H, a.Dv, a.Dk, 1, a.Dv, 0, 1.f, a.scale, a.T, 1, nullptr, nullptr};
}
Sweep gradientOfK(const duck_attention &a) {
  return {a.dout, a.q, a.v, a.dk, rowsOf(a.dout_stride), rowsOf(a.q_stride), rowsOf(a.v_stride), a.dstate_out, nullptr,
          a.decay, a.resets, a.T, a.E, a.H, a.Dv, a.Dk, 1, a.Dv, 1, a.scale, 1.f, a.T, 1, nullptr, nullptr};
}
Sweep gradientOfV(const duck_attention &a) {   // and of the state
  return {a.q, a.dout, a.k, a.dv, rowsOf(a.q_stride), rowsOf(a.dout_stride), rowsOf(a.k_stride), a.dstate_out,
          a.dstate_in, a.decay, a.resets, a.T, a.E, a.H, a.Dk, a.Dv, a.Dv, 1, 1, a.scale, 1.f, a.T, 1, nullptr, nullptr};
}

// How a forward or backward call in bfloat16 is laid out.
struct ChunkPlan {
  int C, columnTiles, segmentLength, segmentCount, chunks;
  int64_t stateSize, segmentBytes, cutBytes, flagBytes;   // of the scratch, in this order
};
// With fewer blocks than half of what fits on the GPU at once, T is split so that
// the segments' blocks fill it once: a second, partly filled round costs as much as a
// full one (a replay of 16384 steps, 8 heads of 128: 187 us in 26 segments).  Of the
// backward pass at head sizes up to 64 a fourth block would fit.
ChunkPlan planChunks(const duck_attention &a, bool backward) {
  ChunkPlan p{};
  p.C = a.T <= 32 ? 32 : 64;
  p.columnTiles = backward ? 1 : int(ceilDiv(a.Dv, 64));
  p.chunks = int(ceilDiv(a.T, p.C));
  p.stateSize = int64_t(a.Dk) * a.Dv;
  const int64_t blocks = int64_t(a.E) * a.H * p.columnTiles;
  const int64_t fit = std::max(a.Dk, a.Dv) <= 64 ? 3 * 148 : backward ? 148 : 2 * 148;
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(p.chunks / 4, fit / blocks));
  p.segmentLength = int(ceilDiv(std::max(1, p.chunks), want)) * p.C;
  p.segmentCount = std::max(1, int(ceilDiv(a.T, p.segmentLength)));
  const int64_t states = int64_t(a.E) * a.H * p.segmentCount;
  if (p.segmentCount > 1) {
    p.segmentBytes = states * p.stateSize * 4;
    p.cutBytes = states;
  }
  p.flagBytes = states * p.columnTiles;
  return p;
}

bool dense16(const void *base, const int64_t *strides, int width) {
  return reinterpret_cast<uintptr_t>(base) % 16 == 0 && strides[0] % 8 == 0 && strides[1] % 8 == 0 &&
         strides[2] % 8 == 0 && width % 8 == 0;
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

template <int C, int DK, int DV, bool OUT, bool STATE>
void launchChunks(const ChunkArgs &a, int segments, int buffers, cudaStream_t stream) {
  const dim3 grid(unsigned(int64_t(a.E) * a.H), unsigned(segments * a.columnTiles));
  constexpr auto kernel = attentionChunks<C, DK, DV, OUT, STATE>;
  constexpr int most = chunkSharedBytes<C, DK, DV, OUT>(STATE ? 2 : 1);
  if constexpr (most > 48 * 1024) allowShared<kernel>(most);
  kernel<<<grid, C * 2, chunkSharedBytes<C, DK, DV, OUT>(buffers), stream>>>(a, buffers);
  check(cudaGetLastError(), "linear attention launch");
}
template <int C, bool OUT, bool STATE>
void launchChunks(const ChunkArgs &a, int segments, int buffers, cudaStream_t stream) {
  const bool narrow = a.Dv <= 32;
  if (a.Dk <= 32) narrow ? launchChunks<C, 32, 32, OUT, STATE>(a, segments, buffers, stream)
                         : launchChunks<C, 32, 64, OUT, STATE>(a, segments, buffers, stream);
  else if (a.Dk <= 64) narrow ? launchChunks<C, 64, 32, OUT, STATE>(a, segments, buffers, stream)
                              : launchChunks<C, 64, 64, OUT, STATE>(a, segments, buffers, stream);
  else narrow ? launchChunks<C, 128, 32, OUT, STATE>(a, segments, buffers, stream)
              : launchChunks<C, 128, 64, OUT, STATE>(a, segments, buffers, stream);
}

void forwardChunks(const duck_attention &a, cudaStream_t stream) {
  const ChunkPlan plan = planChunks(a, false);
  const bool split = plan.segmentCount > 1;
  require(a.scratch, "Invalid arguments");
  ChunkArgs c{};
  c.q = static_cast<const bf16 *>(a.q);
  c.k = static_cast<const bf16 *>(a.k);
  c.v = static_cast<const bf16 *>(a.v);
  c.out = static_cast<bf16 *>(a.out);
  c.qs = rowsOf(a.q_stride);
  c.ks = rowsOf(a.k_stride);
  c.vs = rowsOf(a.v_stride);
  c.decay = a.decay;
  c.resets = a.resets;
  c.stateIn = a.state_in;
  c.stateOut = a.state_out;
  c.saved = static_cast<bf16 *>(a.saved);
  c.T = a.T, c.E = a.E, c.H = a.H, c.Dk = a.Dk, c.Dv = a.Dv;
  c.segmentLength = plan.segmentLength;
  c.segmentCount = plan.segmentCount;
  c.columnTiles = plan.columnTiles;
  c.vecQ = dense16(a.q, a.q_stride, a.Dk);
  c.vecK = dense16(a.k, a.k_stride, a.Dk);
  c.vecV = dense16(a.v, a.v_stride, a.Dv);
  c.scale = a.scale;
  c.precise = a.state_out != nullptr;
  c.flags = reinterpret_cast<uint8_t *>(a.scratch) + plan.segmentBytes + plan.cutBytes;
  // Two sets of tiles, except where they are so large (128 rows of state) that two blocks on a multiprocessor hide
  // a chunk's loads better than one block's own next set: 107 -> 90 us for the replay of 16384 steps.
  const bool more = std::min(plan.chunks, plan.segmentLength / plan.C) > 1;
  const int buffers = more && a.Dk <= 64 ? 2 : 1;
  if (split) {
    c.segments = a.scratch;
    c.segmentCut = reinterpret_cast<uint8_t *>(a.scratch) + plan.segmentBytes;
    launchChunks<64, false, true>(c, plan.segmentCount - 1, more ? 2 : 1, stream);
    const dim3 grid(unsigned(int64_t(a.E) * a.H), unsigned(ceilDiv(plan.stateSize, 256)));
    joinSegments<<<grid, 256, 0, stream>>>(c.segments, c.segmentCut, a.state_in, a.decay, a.H, a.T, plan.segmentCount,
                                           plan.segmentLength, plan.stateSize, 0);
    check(cudaGetLastError(), "linear attention launch");
  }
  const bool advance = plan.chunks > 1 || a.state_out;
  if (plan.C == 32) advance ? launchChunks<32, true, true>(c, 1, 1, stream) : launchChunks<32, true, false>(c, 1, 1, stream);
  else advance ? launchChunks<64, true, true>(c, plan.segmentCount, buffers, stream)
               : launchChunks<64, true, false>(c, 1, 1, stream);
  launchRedo({{forwardSweep(a)}}, 1, c.flags, plan.segmentCount * plan.columnTiles, stream);
}

template <int C, int D, bool OUT, bool STATE>
void launchBackward(const BackwardArgs &a, int segments, cudaStream_t stream) {
  const dim3 grid(unsigned(int64_t(a.E) * a.H), unsigned(segments));
  constexpr auto kernel = attentionChunksBackward<C, D, OUT, STATE>;
  constexpr int most = backwardSharedBytes<C, D, OUT>(true);
  if constexpr (most > 48 * 1024) allowShared<kernel>(most);
  const bool later = STATE || a.dstateOut;
  kernel<<<grid, backwardWarps<C, D, OUT>() * 32, backwardSharedBytes<C, D, OUT>(later), stream>>>(a);
  check(cudaGetLastError(), "linear attention backward launch");
}
template <int C, bool OUT, bool STATE>
void launchBackward(const BackwardArgs &a, int segments, cudaStream_t stream) {
  const int d = std::max(a.Dk, a.Dv);
  if (d <= 32) launchBackward<C, 32, OUT, STATE>(a, segments, stream);
  else if (d <= 64) launchBackward<C, 64, OUT, STATE>(a, segments, stream);
  else launchBackward<C, 128, OUT, STATE>(a, segments, stream);
}

void backwardChunks(const duck_attention &a, cudaStream_t stream) {
  const ChunkPlan plan = planChunks(a, true);
  const bool split = plan.segmentCount > 1;
  require(a.scratch && (plan.chunks <= 1 || a.saved), "Invalid arguments");
  BackwardArgs c{};
  c.q = static_cast<const bf16 *>(a.q);
  c.k = static_cast<const bf16 *>(a.k);
  c.v = static_cast<const bf16 *>(a.v);
  c.dout = static_cast<const bf16 *>(a.dout);
  c.dq = static_cast<bf16 *>(a.dq);
  c.dk = static_cast<bf16 *>(a.dk);
  c.dv = static_cast<bf16 *>(a.dv);
  c.qs = rowsOf(a.q_stride);
  c.ks = rowsOf(a.k_stride);
  c.vs = rowsOf(a.v_stride);
  c.os = rowsOf(a.dout_stride);
  c.decay = a.decay;
  c.resets = a.resets;
  c.stateIn = a.state_in;
  c.dstateOut = a.dstate_out;
  c.dstateIn = a.dstate_in;
  c.saved = static_cast<const bf16 *>(a.saved);
  c.T = a.T, c.E = a.E, c.H = a.H, c.Dk = a.Dk, c.Dv = a.Dv;
  c.segmentLength = plan.segmentLength;
  c.segmentCount = plan.segmentCount;
  c.vecQ = dense16(a.q, a.q_stride, a.Dk);
  c.vecK = dense16(a.k, a.k_stride, a.Dk);
  c.vecV = dense16(a.v, a.v_stride, a.Dv);
  c.vecO = dense16(a.dout, a.dout_stride, a.Dv);
  c.scale = a.scale;
  c.precise = a.dstate_in != nullptr;
  c.flags = reinterpret_cast<uint8_t *>(a.scratch) + plan.segmentBytes + plan.cutBytes;
  if (split) {
    c.segments = a.scratch;
    c.segmentCut = reinterpret_cast<uint8_t *>(a.scratch) + plan.segmentBytes;
    launchBackward<64, false, true>(c, plan.segmentCount - 1, stream);
    const dim3 grid(unsigned(int64_t(a.E) * a.H), unsigned(ceilDiv(plan.stateSize, 256)));
    joinSegments<<<grid, 256, 0, stream>>>(c.segments, c.segmentCut, a.dstate_out, a.decay, a.H, a.T,
                                           plan.segmentCount, plan.segmentLength, plan.stateSize, 1);
    check(cudaGetLastError(), "linear attention backward launch");
  }
  const bool advance = plan.chunks > 1 || a.dstate_in;
  if (plan.C == 32) advance ? launchBackward<32, true, true>(c, 1, stream) : launchBackward<32, true, false>(c, 1, stream);
  else advance ? launchBackward<64, true, true>(c, plan.segmentCount, stream)
               : launchBackward<64, true, false>(c, 1, stream);
  launchRedo({{gradientOfQ(a), gradientOfK(a), gradientOfV(a)}}, 3, c.flags, plan.segmentCount, stream);
}

}  // namespace

extern "C" {

int duck_layer_norm_forward(const void *x, const float *weight, const float *bias, void *y, float *stats,
                            int64_t rows, int n, int64_t x_stride, double eps, int type, duck_stream stream) {
  return guarded([&] {
    requireType(type);
    require(rows >= 0 && n > 0 && x_stride >= 0, "Invalid layer norm sizes");
    require(eps >= 0 && std::isfinite(eps), "Invalid layer norm eps");
    if (rows == 0) return;
    require(x && y, "Invalid arguments");
    requireStats(stats);
    NormArgs a{};
    a.x = x; a.weight = weight; a.bias = bias; a.y = y; a.stats = stats;
    a.rows = rows; a.n = n; a.xStride = x_stride; a.eps = float(eps);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const bool pieces = pieces16({x, y}, {x_stride, int64_t(n)}, type);
    withType(type, [&](auto zero) {
      using T = decltype(zero);
      if (n > kNormWidest) {
        const int64_t blocks = std::min<int64_t>(ceilDiv(rows, kNormThreads / 32), int64_t(148) * 16);
        normForwardAny<T><<<unsigned(blocks), kNormThreads, 0, s>>>(a);
        return;
      }
      withNormRows<T>(n, pieces, [&](auto lanes, auto vec, auto values) {
        constexpr int L = lanes.value;
        normForwardRows<T, L, vec.value, values.value>
            <<<unsigned(normBlocks(rows, n, pieces, false)), normBlock(L), 0, s>>>(a);
      });
    });
    check(cudaGetLastError(), "layer norm launch");
  });
}

int64_t duck_layer_norm_scratch(int64_t rows, int n) {
  if (rows < 0 || n <= 0) return -1;
  return normSplits(rows, n) * 2 * n;
}

int duck_layer_norm_backward(const void *x, const void *dy, const float *weight, const float *stats, void *dx,
                             float *dweight, float *dbias, float *scratch, int64_t rows, int n, int64_t x_stride,
                             int64_t dy_stride, int type, duck_stream stream) {
  return guarded([&] {
    requireType(type);
    require(rows >= 0 && n > 0 && x_stride >= 0 && dy_stride >= 0, "Invalid layer norm sizes");
    const bool columns = dweight || dbias;
    if (!columns && !dx) return;
    require(!columns || scratch, "Invalid arguments");
    require(rows == 0 || (x && dy && stats), "Invalid arguments");
    requireStats(stats);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    NormArgs a{};
    a.x = x; a.dy = dy; a.weight = weight; a.dx = dx; a.stats = const_cast<float *>(stats); a.partials = scratch;
    a.dweight = dweight; a.dbias = dbias; a.rows = rows; a.n = n; a.xStride = x_stride; a.dyStride = dy_stride;
    const bool pieces = pieces16({x, dy, dx}, {x_stride, dy_stride, int64_t(n)}, type);
    int splits = 0;
    withType(type, [&](auto zero) {
      using T = decltype(zero);
      if (n > kNormWidest) {
        if (dx && rows > 0) {
          const int64_t blocks = std::min<int64_t>(ceilDiv(rows, kNormThreads / 32), int64_t(148) * 16);
          normBackwardAny<T><<<unsigned(blocks), kNormThreads, 0, s>>>(a);
        }
        splits = int(normSplits(rows, n));
        if (columns) normColumnsAny<T><<<dim3(unsigned(ceilDiv(n, 32)), unsigned(splits)), 256, 0, s>>>(a);
        return;
      }
      withNormRows<T>(n, pieces, [&](auto lanes, auto vec, auto values) {
        constexpr int L = lanes.value, V = vec.value, P = values.value;
        const int64_t blocks = normBlocks(rows, n, pieces, true);
        const int shared = L > 32 ? 0 : normBlock(L) / 32 * 2 * n * int(sizeof(float));
        splits = int(blocks);
        if (dx && columns) normBackwardRows<T, L, V, P, true, true><<<unsigned(blocks), normBlock(L), shared, s>>>(a);
        else if (dx) normBackwardRows<T, L, V, P, true, false><<<unsigned(blocks), normBlock(L), 0, s>>>(a);
        else normBackwardRows<T, L, V, P, false, true><<<unsigned(blocks), normBlock(L), shared, s>>>(a);
      });
    });
    if (columns && (splits > 1 || n > kNormWidest)) normPartials<<<unsigned(ceilDiv(int64_t(2) * n, 32)), 1024, 0, s>>>(a, splits);
    check(cudaGetLastError(), "layer norm backward launch");
  });
}

int duck_elu_checkpoint(const void *x, void *y, int8_t *codes, float *scales, int64_t rows, int n, int type,
                        duck_stream stream) {
  return guarded([&] {
    requireType(type);
    require(rows >= 0 && n > 0, "Invalid checkpoint sizes");
    if (rows == 0) return;
    require(x && y && codes && scales, "Invalid arguments");
    CheckpointArgs a{x, y, nullptr, codes, scales, rows, n, int(ceilDiv(n, kGroup))};
    launchGroups(a, type, pieces16({x, y}, {int64_t(n)}, type), stream, Groups::keep);
    check(cudaGetLastError(), "checkpoint launch");
  });
}

int duck_elu_restore(const void *dy, const int8_t *codes, const float *scales, void *y, void *dx, int64_t rows, int n,
                     int type, duck_stream stream) {
  return restoreElu(dy, codes, scales, y, dx, rows, n, type, Groups::restore, stream);
}

int duck_elu_restore_bounded(const void *dy, const int8_t *codes, const float *scales, void *y, void *dx, int64_t rows,
                             int n, int type, duck_stream stream) {
  return restoreElu(dy, codes, scales, y, dx, rows, n, type, Groups::restoreBounded, stream);
}

int duck_linear_attention_sizes(const duck_attention *args, int64_t *out) {
  return guarded([&] {
    require(out != nullptr, "Invalid arguments");
    out[0] = out[1] = out[2] = 0;
    if (!attentionChecked(args) || args->T == 0) return;
    if (args->type != DUCK_BFLOAT16) {
      const ScanPlan plan = planScan(*args);
      out[0] = plan.stateBytes + plan.cutBytes;
      out[1] = 2 * out[0];
      return;
    }
    const ChunkPlan plan = planChunks(*args, false), back = planChunks(*args, true);
    out[0] = plan.segmentBytes + plan.cutBytes + plan.flagBytes;
    out[1] = back.segmentBytes + back.cutBytes + back.flagBytes;
    out[2] = plan.chunks > 1 ? int64_t(args->E) * args->H * plan.chunks * plan.stateSize * 2 : 0;
  });
}

int duck_linear_attention_forward(const duck_attention *args, duck_stream stream) {
  return guarded([&] {
    if (!attentionChecked(args)) return;
    const duck_attention &a = *args;
    require(a.decay && (a.T == 0 || (a.q && a.k && a.v && a.out)), "Invalid arguments");
    requireAligned({a.out, a.state_in, a.state_out, a.saved, a.scratch});
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (a.T == 0) copyState(a, a.state_in, a.state_out, s);
    else if (a.type == DUCK_BFLOAT16) forwardChunks(a, s);
    else runScan(a, {{forwardSweep(a)}}, 1, {0}, s);
  });
}

int duck_linear_attention_backward(const duck_attention *args, duck_stream stream) {
  return guarded([&] {
    if (!attentionChecked(args)) return;
    const duck_attention &a = *args;
    require(a.decay && (a.T == 0 || (a.q && a.k && a.v && a.dout && a.dq && a.dk && a.dv)), "Invalid arguments");
    requireAligned({a.state_in, a.dstate_out, a.dq, a.dk, a.dv, a.dstate_in, a.saved, a.scratch});
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (a.T == 0) copyState(a, a.dstate_out, a.dstate_in, s);
    else if (a.type == DUCK_BFLOAT16) backwardChunks(a, s);
    else runScan(a, {{gradientOfQ(a), gradientOfK(a), gradientOfV(a)}}, 3, {0, 2}, s);
  });
}

int duck_linear_attention_step(const duck_attention *args, duck_stream stream) {
  return guarded([&] {
    if (!attentionChecked(args)) return;
    const duck_attention &a = *args;
    require(a.q && a.k && a.v && a.out && a.decay && a.state_out, "Invalid arguments");
    StepOf s{a.q, a.k, a.v, a.out, a.state_out, a.decay, a.resets, a.q_stride[1], a.q_stride[2], a.k_stride[1],
             a.k_stride[2], a.v_stride[1], a.v_stride[2], a.E, a.H, a.Dk, a.Dv, a.scale};
    // Four columns a thread where rows of the state are whole 16-byte pieces.
    const bool quads = a.Dv % 4 == 0 && reinterpret_cast<uintptr_t>(a.state_out) % 16 == 0;
    withType(a.type, [&](auto zero) {
      using T = decltype(zero);
      const unsigned blocks = unsigned(int64_t(a.E) * a.H);
      cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
      if (quads) attentionStepQuads<T><<<blocks, 128, 0, st>>>(s);
      else attentionStepAny<T><<<blocks, 128, 0, st>>>(s);
    });
    check(cudaGetLastError(), "linear attention step launch");
  });
}

}  // extern "C"
