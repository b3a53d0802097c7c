// C entries of the optimizer (declared in include/duck_b200.h): argument checks,
// the tables of tensors that launches carry, launches.
#include "adamw.cuh"
#include "capi.hpp"

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <vector>

using namespace duckb200;

namespace {

static_assert(DUCK_GRADIENT_SUMS == kNormBlocks, "the header says how many sums there are");
static_assert(sizeof(AdamTable<kTensorsMany>) + sizeof(AdamArgs) <= 32764, "arguments of a launch");

int64_t ceilDiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool on(const void *p, int boundary) { return reinterpret_cast<uintptr_t>(p) % boundary == 0; }

// The launches of a call: tensors of one element type, as many as fit in a launch's arguments.
struct Launch {
  int type;
  std::vector<AdamTensor> tensors;
  int chunks = 0;
};
std::vector<Launch> launchesOf(const duck_adamw_tensor *tensors, int count, int chunkValues, bool eight) {
  std::vector<Launch> launches;
  for (int type : {DUCK_FLOAT32, DUCK_BFLOAT16}) {
    int64_t chunks = 0;
    for (int i = 0; i < count; ++i) {
      const duck_adamw_tensor &a = tensors[i];
      if (a.type != type || a.n == 0) continue;
      if (launches.empty() || launches.back().type != type || int(launches.back().tensors.size()) == kTensorsMany) {
        launches.push_back({type, {}, 0});
        chunks = 0;
      }
      const int four = type == DUCK_FLOAT32 ? 16 : 8, moment = eight ? 4 : 16;
      AdamTensor t{a.param, a.grad, a.exp_avg, a.exp_avg_sq, a.exp_avg_exponents, a.exp_avg_sq_exponents, a.n,
                   int32_t(chunks), uint32_t(a.place) & 0x7fffffffu,
                   on(a.param, four) && on(a.grad, four) && on(a.exp_avg, moment) && on(a.exp_avg_sq, moment)};
      launches.back().tensors.push_back(t);
      chunks += ceilDiv(a.n, chunkValues);
      require(chunks < (int64_t(1) << 31), "Too many values");
      launches.back().chunks = int(chunks);
    }
  }
  return launches;
}
int64_t valuesOf(const duck_adamw_tensor *tensors, int count) {
  int64_t values = 0;
  for (int i = 0; i < count; ++i) values += tensors[i].n;
  return values;
}
template <class F> void withTable(const Launch &l, F &&f) {
  auto fill = [&](auto table) {
    std::copy(l.tensors.begin(), l.tensors.end(), table.t);
    f(table);
  };
  if (l.tensors.size() <= kTensorsFew) fill(AdamTable<kTensorsFew>{});
  else fill(AdamTable<kTensorsMany>{});
}

void tensorsChecked(const duck_adamw_tensor *tensors, int count) {
  require(count >= 0 && (count == 0 || tensors), "Invalid arguments");
  for (int i = 0; i < count; ++i) {
    require(tensors[i].n >= 0 && tensors[i].place >= 0, "Invalid tensor sizes");
    require(tensors[i].type == DUCK_FLOAT32 || tensors[i].type == DUCK_BFLOAT16, "Invalid element type");
  }
}

// Dynamic shared memory above 48 KB has to be asked for, once per kernel and device
// (by whichever thread comes first).
template <auto kernel> void allowShared(int bytes) {
  static std::atomic<bool> done[64] = {};
  int device = 0;
  check(cudaGetDevice(&device), "cudaGetDevice");
  if (device < 64 && done[device]) return;
  check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "cudaFuncSetAttribute");
  if (device < 64) done[device] = true;
}

template <class T, bool EIGHT, int MOST>
void launchStep(const AdamTable<MOST> &table, const AdamArgs &args, cudaStream_t stream) {
  const int blocks = std::max(1, std::min(args.chunks, 148 * 4));
  constexpr auto kernel = adamStep<T, EIGHT, MOST>;
  constexpr int bytes = AdamRing<T, EIGHT>::bytes;
  if constexpr (bytes + 1024 > 48 * 1024) allowShared<kernel>(bytes);   // (there is some beside it)
  kernel<<<blocks, kAdamThreads, bytes, stream>>>(table, args);
}

}  // namespace

extern "C" {

int duck_gradient_squares(const duck_adamw_tensor *tensors, int count, int before, double *sums, int *sum_count,
                          duck_stream stream) {
  return guarded([&] {
    tensorsChecked(tensors, count);
    require(before >= 0 && before <= kNormBlocks && sums && sum_count, "Invalid arguments");
    for (int i = 0; i < count; ++i) require(tensors[i].n == 0 || tensors[i].grad, "Invalid arguments");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    *sum_count = before;
    for (const Launch &l : launchesOf(tensors, count, kNormChunk, false)) {
      const int blocks = std::min(l.chunks, kNormBlocks);
      withTable(l, [&](const auto &table) {
        constexpr int M = sizeof(table.t) / sizeof(AdamTensor);
        if (l.type == DUCK_FLOAT32)
          gradientSquares<float, M><<<blocks, kAdamThreads, 0, s>>>(table, int(l.tensors.size()), l.chunks, *sum_count, sums);
        else
          gradientSquares<bf16, M><<<blocks, kAdamThreads, 0, s>>>(table, int(l.tensors.size()), l.chunks, *sum_count, sums);
      });
      check(cudaGetLastError(), "gradient norm launch");
      *sum_count = std::max(*sum_count, blocks);
    }
  });
}

int duck_adamw_step(const duck_adamw_tensor *tensors, int count, const duck_adamw *options, duck_stream stream) {
  return guarded([&] {
    tensorsChecked(tensors, count);
    require(options != nullptr, "Invalid arguments");
    const duck_adamw &o = *options;
    require(o.step && on(o.step, 8), "The step count is an int64 on an 8-byte boundary");
    require(o.bits == 8 || o.bits == 32, "Moments have 8 or 32 bits");
    require(o.beta1 >= 0 && o.beta1 < 1 && o.beta2 >= 0 && o.beta2 < 1, "Invalid betas");
    require((o.eps == 0 || o.eps >= FLT_MIN) && std::isfinite(float(o.eps)) && o.weight_decay >= 0 && std::isfinite(o.weight_decay),
            "Invalid eps or weight decay");
    require(o.rate || std::isfinite(o.rate_value), "Invalid learning rate");
    require(o.sum_count >= 0 && o.sum_count <= kNormBlocks && (o.sum_count == 0 || (o.sums && o.max_norm >= 0)),
            "Invalid norm");
    for (int i = 0; i < count; ++i) {
      const duck_adamw_tensor &t = tensors[i];
      require(t.n == 0 || (t.param && t.grad && t.exp_avg && t.exp_avg_sq), "Invalid arguments");
      require(t.n == 0 || o.bits == 32 || (t.exp_avg_exponents && t.exp_avg_sq_exponents), "Invalid arguments");
    }
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    // As many rounds a chunk as leave every block one: a chunk finds its tensor and fills its ring anew.
    const int rounds = int(std::max<int64_t>(
        1, std::min<int64_t>(kAdamRoundsMost, valuesOf(tensors, count) / (int64_t(148) * 4 * kAdamRound))));
    std::vector<Launch> launches = launchesOf(tensors, count, rounds * kAdamRound, o.bits == 8);
    if (launches.empty()) launches.push_back({DUCK_FLOAT32, {}, 0});   // the step is counted all the same
    for (size_t i = 0; i < launches.size(); ++i) {
      const Launch &l = launches[i];
      const AdamArgs args{o.step, o.rate, o.sums, o.rate_value, o.beta1, o.beta2, o.weight_decay, o.max_norm, float(o.eps),
                          o.sum_count, int(l.tensors.size()), l.chunks, rounds, i + 1 == launches.size()};
      withTable(l, [&](const auto &table) {
        if (l.type == DUCK_FLOAT32) o.bits == 8 ? launchStep<float, true>(table, args, s) : launchStep<float, false>(table, args, s);
        else o.bits == 8 ? launchStep<bf16, true>(table, args, s) : launchStep<bf16, false>(table, args, s);
      });
      check(cudaGetLastError(), "optimizer step launch");
    }
  });
}

int duck_moment_values(const duck_adamw_tensor *tensors, int count, duck_stream stream) {
  return guarded([&] {
    tensorsChecked(tensors, count);
    for (int i = 0; i < count; ++i) {
      const duck_adamw_tensor &t = tensors[i];
      require(t.type == DUCK_FLOAT32, "Values of moments are float32");
      require(t.n == 0 || (t.param && (t.exp_avg ? !t.exp_avg_sq && t.exp_avg_exponents : t.exp_avg_sq && t.exp_avg_sq_exponents)),
              "Invalid arguments");
    }
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int groups = valuesOf(tensors, count) >= int64_t(148) * 8 * 8 * kAdamRound ? 8 : 2;
    for (const Launch &l : launchesOf(tensors, count, groups * kAdamRound, true)) {
      withTable(l, [&](const auto &table) {
        constexpr int M = sizeof(table.t) / sizeof(AdamTensor);
        const int blocks = std::min(l.chunks, 148 * 8);
        if (groups == 8) momentValues<M, 8><<<blocks, kAdamThreads, 0, s>>>(table, int(l.tensors.size()), l.chunks);
        else momentValues<M, 2><<<blocks, kAdamThreads, 0, s>>>(table, int(l.tensors.size()), l.chunks);
      });
      check(cudaGetLastError(), "moment values launch");
    }
  });
}

}  // extern "C"
