// C entries of the operators of a policy with memory (declared in
// include/duck_b200.h): argument checks, the choice of a kernel, launches.
#include "capi.hpp"
#include "checkpoint8.cuh"
#include "layer_norm.cuh"
#include "linear_attention.cuh"

#include <algorithm>
#include <cmath>

using namespace duckb200;

namespace {

int multiprocessors() {
  int device = 0, n = 0;
  check(cudaGetDevice(&device), "cudaGetDevice");
  check(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device), "cudaDeviceGetAttribute");
  return n;
}

// Calls f with a value of the element type.
template <class F> void withType(int type, F &&f) {
  if (type == DUCK_FLOAT32) f(0.f);
  else f(bf16());
}
void requireType(int type) { require(type == DUCK_FLOAT32 || type == DUCK_BFLOAT16, "Invalid element type"); }

int64_t ceilDiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Row groups that the sums of the weight's gradient are split into.
int normSplits(int64_t rows, int n) {
  const int64_t columns = ceilDiv(n, 32);
  return int(std::max<int64_t>(1, std::min<int64_t>(ceilDiv(rows, 64), ceilDiv(148 * 8, columns))));
}

bool attentionChecked(const duck_attention *a) {
  require(a != nullptr, "Invalid arguments");
  requireType(a->type);
  require(a->T >= 0 && a->E >= 0 && a->H >= 0, "Invalid attention sizes");
  require(a->Dk > 0 && a->Dk <= kHeadMax && a->Dv > 0 && a->Dv <= kHeadMax, "Head sizes have to be 1 to 128");
  require(int64_t(a->E) * a->H < (int64_t(1) << 31), "Too many environments and heads");
  return a->E > 0 && a->H > 0;
}
Rows rowsOf(const int64_t *s) { return {s[0], s[1], s[2]}; }

template <class T> void launchScan(const Sweep &s, cudaStream_t stream) {
  const int threads = std::min(128, int(ceilDiv(s.Dj, 32)) * 32);
  const dim3 grid(unsigned(int64_t(s.E) * s.H), unsigned(ceilDiv(s.Dj, threads)));
  if (s.Di <= 16) attentionScan<T, 16><<<grid, threads, 0, stream>>>(s);
  else if (s.Di <= 32) attentionScan<T, 32><<<grid, threads, 0, stream>>>(s);
  else if (s.Di <= 64) attentionScan<T, 64><<<grid, threads, 0, stream>>>(s);
  else attentionScan<T, 128><<<grid, threads, 0, stream>>>(s);
  check(cudaGetLastError(), "linear attention launch");
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
    NormArgs a{};
    a.x = x; a.weight = weight; a.bias = bias; a.y = y; a.stats = stats;
    a.rows = rows; a.n = n; a.xStride = x_stride; a.eps = float(eps);
    const int64_t blocks = std::min<int64_t>(ceilDiv(rows, kNormThreads / 32), int64_t(multiprocessors()) * 16);
    withType(type, [&](auto zero) {
      normForwardAny<decltype(zero)><<<unsigned(blocks), kNormThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a);
    });
    check(cudaGetLastError(), "layer norm launch");
  });
}

int64_t duck_layer_norm_scratch(int64_t rows, int n) {
  if (rows < 0 || n <= 0) return -1;
  return int64_t(normSplits(rows, n)) * 2 * n;
}

int duck_layer_norm_backward(const void *x, const void *dy, const float *weight, const float *stats, void *dx,
                             float *dweight, float *dbias, float *scratch, int64_t rows, int n, int64_t x_stride,
                             int64_t dy_stride, int type, duck_stream stream) {
  return guarded([&] {
    requireType(type);
    require(rows >= 0 && n > 0 && x_stride >= 0 && dy_stride >= 0, "Invalid layer norm sizes");
    const bool columns = dweight || dbias;
    require(!columns || scratch, "Invalid arguments");
    require(rows == 0 || (x && dy && stats), "Invalid arguments");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    NormArgs a{};
    a.x = x; a.dy = dy; a.weight = weight; a.dx = dx; a.stats = const_cast<float *>(stats); a.partials = scratch;
    a.dweight = dweight; a.dbias = dbias; a.rows = rows; a.n = n; a.xStride = x_stride; a.dyStride = dy_stride;
    const int splits = normSplits(rows, n);
    withType(type, [&](auto zero) {
      using T = decltype(zero);
      if (dx && rows > 0) {
        const int64_t blocks = std::min<int64_t>(ceilDiv(rows, kNormThreads / 32), int64_t(multiprocessors()) * 16);
        normBackwardAny<T><<<unsigned(blocks), kNormThreads, 0, s>>>(a);
      }
      if (columns) normColumnsAny<T><<<dim3(unsigned(ceilDiv(n, 32)), unsigned(splits)), 256, 0, s>>>(a);
    });
    if (columns) normColumnsFinish<<<unsigned(ceilDiv(int64_t(2) * n, 32)), 256, 0, s>>>(a, splits);
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
    const int64_t blocks = std::min<int64_t>(ceilDiv(rows * a.groups, kCheckpointThreads / 32),
                                             int64_t(multiprocessors()) * 32);
    withType(type, [&](auto zero) {
      eluCheckpointAny<decltype(zero)>
          <<<unsigned(blocks), kCheckpointThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a);
    });
    check(cudaGetLastError(), "checkpoint launch");
  });
}

int duck_elu_restore(const void *dy, const int8_t *codes, const float *scales, void *y, void *dx, int64_t rows, int n,
                     int type, duck_stream stream) {
  return guarded([&] {
    requireType(type);
    require(rows >= 0 && n > 0, "Invalid checkpoint sizes");
    if (rows == 0) return;
    require(dy && codes && scales && dx, "Invalid arguments");
    CheckpointArgs a{dy, y, dx, const_cast<int8_t *>(codes), const_cast<float *>(scales), rows, n,
                     int(ceilDiv(n, kGroup))};
    const int64_t blocks = std::min<int64_t>(ceilDiv(rows * a.groups, kCheckpointThreads / 32),
                                             int64_t(multiprocessors()) * 32);
    withType(type, [&](auto zero) {
      eluRestoreAny<decltype(zero)>
          <<<unsigned(blocks), kCheckpointThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a);
    });
    check(cudaGetLastError(), "checkpoint launch");
  });
}

int duck_linear_attention_sizes(const duck_attention *args, int64_t *out) {
  return guarded([&] {
    require(out != nullptr, "Invalid arguments");
    attentionChecked(args);
    out[0] = out[1] = out[2] = 0;
  });
}

int duck_linear_attention_forward(const duck_attention *args, duck_stream stream) {
  return guarded([&] {
    if (!attentionChecked(args)) return;
    const duck_attention &a = *args;
    require(a.decay && (a.T == 0 || (a.q && a.k && a.v && a.out)), "Invalid arguments");
    Sweep s{a.k, a.v, a.q, a.out, rowsOf(a.k_stride), rowsOf(a.v_stride), rowsOf(a.q_stride), a.state_in, a.state_out,
            a.decay, a.resets, a.T, a.E, a.H, a.Dk, a.Dv, a.Dv, 1, 0, 1.f, a.scale};
    withType(a.type, [&](auto zero) { launchScan<decltype(zero)>(s, reinterpret_cast<cudaStream_t>(stream)); });
  });
}

int duck_linear_attention_backward(const duck_attention *args, duck_stream stream) {
  return guarded([&] {
    if (!attentionChecked(args)) return;
    const duck_attention &a = *args;
    require(a.decay && (a.T == 0 || (a.q && a.k && a.v && a.dout && a.dq && a.dk && a.dv)), "Invalid arguments");
    const Rows q = rowsOf(a.q_stride), k = rowsOf(a.k_stride), v = rowsOf(a.v_stride), o = rowsOf(a.dout_stride);
    const Sweep dq{a.v, a.k, a.dout, a.dq, v, k, o, a.state_in, nullptr, a.decay, a.resets,
                   a.T, a.E, a.H, a.Dv, a.Dk, 1, a.Dv, 0, 1.f, a.scale};
    const Sweep dk{a.dout, a.q, a.v, a.dk, o, q, v, a.dstate_out, nullptr, a.decay, a.resets,
                   a.T, a.E, a.H, a.Dv, a.Dk, 1, a.Dv, 1, a.scale, 1.f};
    const Sweep dv{a.q, a.dout, a.k, a.dv, q, o, k, a.dstate_out, a.dstate_in, a.decay, a.resets,
                   a.T, a.E, a.H, a.Dk, a.Dv, a.Dv, 1, 1, a.scale, 1.f};
    withType(a.type, [&](auto zero) {
      using T = decltype(zero);
      launchScan<T>(dq, reinterpret_cast<cudaStream_t>(stream));
      launchScan<T>(dk, reinterpret_cast<cudaStream_t>(stream));
      launchScan<T>(dv, reinterpret_cast<cudaStream_t>(stream));
    });
  });
}

int duck_linear_attention_step(const duck_attention *args, duck_stream stream) {
  return guarded([&] {
    if (!attentionChecked(args)) return;
    const duck_attention &a = *args;
    require(a.q && a.k && a.v && a.out && a.decay && a.state_out, "Invalid arguments");
    StepOf s{a.q, a.k, a.v, a.out, a.state_out, a.decay, a.resets, a.q_stride[1], a.q_stride[2], a.k_stride[1],
             a.k_stride[2], a.v_stride[1], a.v_stride[2], a.E, a.H, a.Dk, a.Dv, a.scale};
    withType(a.type, [&](auto zero) {
      attentionStepAny<decltype(zero)>
          <<<unsigned(int64_t(a.E) * a.H), 128, 0, reinterpret_cast<cudaStream_t>(stream)>>>(s);
    });
    check(cudaGetLastError(), "linear attention step launch");
  });
}

}  // extern "C"
