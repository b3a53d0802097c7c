// Gated linear layer: two projections of the same rows, one of them through an
// activation, multiplied.
//
//   a = x Wg^T + bg,  u = x Wu^T + bu,  h = act(a) u
//   da = dh u act'(a),  du = dh act(a)
//   dx = da Wg + du Wu,  dWg = da^T x,  dWu = du^T x,  dbg = sum of da,  dbu = sum of du
//
// bfloat16 (gatedTiles): products on the tensor cores, operands by the TMA into a
// ring of shared memory tiles, accumulators in tensor memory.  Both projections of
// a tile are one product, the rows of Wg and of Wu side by side as its columns, and
// leave tensor memory together, so that a and u are never in memory.  The backward
// pass computes them again (a third more products than from stored ones), in
// float32, and rounds da and du once: a and u as bfloat16 would add two roundings to
// each, and their two arrays cost as much memory as the layer's output twice.  So
// forward passes keep x only; and, where the TMA does not take rows as they are, the
// padded copies of x and the weights that it read.
//
// One block a multiprocessor goes through tiles of 128 rows: one thread issues the
// copies, one the products, sixteen warps take finished accumulators out, while the
// products of the next tile go to the other half of tensor memory.  Measured on a
// B200, cold: 16384 rows, 1024 x 4096, forward 182 us (1.51 PFLOP/s, tensor pipe 79 %),
// da and du 251, dx 207, weights 205 (80 %, of which four rounds for 3.5 of tiles); 24576
// rows, 256 x 512: 21, 41, 19, 18 and 5 us for the sums, where the accumulators' way out
// bounds the first two (forward: 10 us of it alone, 10 of products and copies alone, 13
// together, and 7 for the start and the end; da and du: 18 of 41 for shuffles of the bias
// sums, dh and stores).
//
// float32 (gatedProducts): FMA in pairs; a and u are kept, since they are exact and
// their products are what the time goes to: 34 to 41 TFLOP/s in large ones (18115 rows,
// 933 x 198, forward 393 us; 4091 rows, 112 x 3920, 173), 27, 21 and 19 us for the
// products of 4999 rows, 61 x 301.
#pragma once
#include "numeric_types.cuh"
#include "umma.cuh"

#include <type_traits>

namespace duckb200 {

enum Activation { kSilu = 0, kGelu = 1, kSigmoid = 2 };

struct Activated {
  float y, slope;
};
// act(a) and its derivative.  FAST: the exponential and the quotient of the
// hardware (2^-21), for results that are rounded to bfloat16.
template <int ACT, bool FAST> __device__ __forceinline__ Activated activate(float a) {
  if constexpr (ACT == kGelu) {
    const float below = 0.5f * (1.f + erff(a * 0.70710678f));
    const float density = 0.39894228f * (FAST ? __expf(-0.5f * a * a) : expf(-0.5f * a * a));
    return {a * below, below + a * density};
  } else {
    float s, rest;
    // FAST: exp(-a) is held at 2^127, whose reciprocal is flushed to zero, so that s is 0 from a = -87.3 down and no
    // infinity meets a zero (rest is 0 there, too, where it is 1, but has s as a factor).  A NaN stays one.
    if constexpr (FAST) {
      float t;
      asm("min.NaN.f32 %0, %1, 0f42FE0000;" : "=f"(t) : "f"(a * -1.4426950408889634f));
      asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(t));
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + t));
      rest = t * s;
    } else {
      s = 1.f / (1.f + expf(-a)), rest = 1.f / (1.f + expf(a));
    }
    if constexpr (ACT == kSilu) return {a * s, s + a * s * rest};
    else return {s, s * rest};
  }
}
template <class F> __device__ __forceinline__ void withActivation(int kind, F &&f) {
  if (kind == kSilu) f(std::integral_constant<int, kSilu>());
  else if (kind == kGelu) f(std::integral_constant<int, kGelu>());
  else f(std::integral_constant<int, kSigmoid>());
}

// ------------------------------------------------------------------- bfloat16
// What a pass of gatedTiles computes.
enum class Pass {
  forward,     // h
  gradients,   // da and du, from x, the weights and dh
  input,       // dx
  weights      // dWg and dWu, or parts of them
};

struct TileArgs {
  const bf16 *bGate, *bUp;   // or null
  bf16 *h;                   // forward
  const bf16 *dh;            // gradients
  bf16 *both;                // [rows, 2, stride]: da and du
  float *biasParts;          // [128-row tiles x 4, 2, F]: sums over 32 rows, or null
  bf16 *dx;                  // input
  bf16 *dwGate, *dwUp;       // weights, where they are not split
  float *parts;              // weights: [splits, 2, F, D], input: [splits, rows, D]
  int64_t rows, dhStride;
  int D, F, stride, activation;
  int tiles, columnTiles, rowTiles, splits, steps;   // steps of 64 of a tile's product
  bool wholeH, wholeDh, wholeBias, wholeD;   // rows of 16-byte pieces: h and dh move by the TMA
  uint64_t waitLimit;
  volatile int *ranOut;      // host memory: set where a wait ran out
};
struct TileMaps {
  CUtensorMap a0, a1, b0, b1;   // operands
  CUtensorMap dh, out0, out1;   // gradients: dh, da and du; forward: out0 is h
};

constexpr int kTileWarps = 16, kTileThreads = 128 + 32 * kTileWarps, kTileRows = 128, kTileSteps = 64, kTileChunk = 16;
template <Pass PASS, int BN> struct TileShared {
  static constexpr bool dual = PASS == Pass::forward || PASS == Pass::gradients;
  static constexpr int columns = dual ? BN / 2 : BN;                                      // of the output that a tile has
  static constexpr int part = columns / 4 < kTileChunk ? kTileChunk : columns / 4;        // and that a warp has
  static constexpr int stages = PASS == Pass::gradients ? (BN == 256 ? 3 : BN == 128 ? 5 : 6) : (BN == 256 ? 4 : BN == 128 ? 6 : 8);
  static constexpr int a = kTileRows * kTileSteps * 2, b = BN * kTileSteps * 2;
  static constexpr int staging = dual ? 32 * part * 2 : 32 * 32;                          // of a warp: its rows, or 32 bytes of them
  static constexpr int incoming = PASS == Pass::gradients ? staging : 0;                  // its rows of dh
  static constexpr int bytes = 1024 + stages * (a + b) + kTileWarps * (staging + incoming) + 512;
};

// A warp's 32 rows of 32 bytes: two pieces of 16 bytes, so placed that neither rows
// of pieces nor columns of them meet in a bank.
__device__ __forceinline__ uint4 *stagedPiece(uint4 *staging, int row, int piece) {
  return staging + row * 2 + (piece ^ (row >> 2 & 1));
}

// Column sums over the 32 lanes: lane i is left with column i % 16's.
__device__ __forceinline__ float columnSum(float (&x)[kTileChunk], int lane) {
#pragma unroll
  for (int half = kTileChunk / 2; half > 0; half /= 2) {
    const bool upper = lane & half;
#pragma unroll
    for (int i = 0; i < half; ++i) {
      const float send = upper ? x[i] : x[i + half], keep = upper ? x[i + half] : x[i];
      x[i] = keep + __shfl_xor_sync(0xffffffffu, send, half);
    }
  }
  return x[0] + __shfl_xor_sync(0xffffffffu, x[0], 16);
}

// A warp's rows of 32 bytes, one row a lane as two pieces, to memory, a row's pieces
// by neighbouring lanes: `values` of E a row exist; whole pieces where rows are made
// of them.
template <class E> __device__ __forceinline__ void storeRows(uint4 *staging, uint4 first, uint4 second, E *to, int64_t rowStride,
                                                             int64_t rowsLeft, int values, bool pieces, int lane) {
  constexpr int V = 16 / sizeof(E);
  *stagedPiece(staging, lane, 0) = first;
  *stagedPiece(staging, lane, 1) = second;
  __syncwarp();
  const int piece = lane % 2;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = lane / 2 + 16 * i;
    if (row >= rowsLeft || piece * V >= values) continue;
    const uint4 v = *stagedPiece(staging, row, piece);
    E *at = to + row * rowStride + piece * V;
    if (pieces && piece * V + V <= values) {
      *reinterpret_cast<uint4 *>(at) = v;
    } else {
      const E *e = reinterpret_cast<const E *>(&v);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (piece * V + j < values) at[j] = e[j];
    }
  }
  __syncwarp();
}
// Eight floats, rounded.
__device__ __forceinline__ uint4 eightOf(const float *x) {
  uint4 v;
  uint32_t *w = reinterpret_cast<uint32_t *>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 two = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t *>(&two);
  }
  return v;
}
__device__ __forceinline__ uint4 fourOf(const float *x) {
  return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
}

template <Pass PASS, int BN> __global__ void __launch_bounds__(kTileThreads, 1)
gatedTiles(const __grid_constant__ TileMaps maps, TileArgs p) {
  using S = TileShared<PASS, BN>;
  constexpr bool kDual = PASS == Pass::forward || PASS == Pass::gradients;
  constexpr bool kAlongA = PASS != Pass::weights, kAlongB = kDual;
  constexpr int kColumns = S::columns, kPart = S::part, kChunk = kTileChunk;
  extern __shared__ uint8_t raw[];
  uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint8_t *tileA = base, *tileB = base + S::stages * S::a;
  uint8_t *staging = tileB + S::stages * S::b;
  uint8_t *incoming = staging + kTileWarps * S::staging;
  uint64_t *full = reinterpret_cast<uint64_t *>(incoming + kTileWarps * S::incoming);
  uint64_t *empty = full + S::stages, *done = empty + S::stages, *taken = done + 2, *came = taken + 2;
  uint64_t *ended = came + kTileWarps;
  uint32_t *tensor = reinterpret_cast<uint32_t *>(ended + 1);
  volatile int *broken = reinterpret_cast<volatile int *>(tensor + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    *broken = p.waitLimit == 0;   // (given up from the start)
    for (int i = 0; i < S::stages; ++i) barrierInit(full + i, 1), barrierInit(empty + i, 1);
    for (int i = 0; i < 2; ++i) barrierInit(done + i, 1), barrierInit(taken + i, kTileWarps);
    for (int i = 0; i < kTileWarps; ++i) barrierInit(came + i, 1);
    barrierInit(ended, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 2) tensorAllocate(tensor, 2 * BN);
  tensorFenceBefore();
  __syncthreads();
  tensorFenceAfter();
  const uint32_t accumulators = *tensor;

  // Where a tile lies.
  struct Tile {
    int row, column, split, half;   // first output row (of Wg or Wu: half 1) and column
  };
  auto tileAt = [&](int t) {
    Tile at{};
    const int column = t % p.columnTiles, rest = t / p.columnTiles;
    at.column = column * kColumns;
    if constexpr (PASS == Pass::weights) {
      const int row = rest % (2 * p.rowTiles);
      at.split = rest / (2 * p.rowTiles);
      at.half = row >= p.rowTiles;
      at.row = (row - at.half * p.rowTiles) * kTileRows;
    } else if constexpr (PASS == Pass::input) {
      at.split = rest / p.rowTiles;
      at.row = (rest - at.split * p.rowTiles) * kTileRows;
    } else {
      at.row = rest * kTileRows;
    }
    return at;
  };
  auto stepsOf = [&](const Tile &at, int &first) {
    if constexpr (PASS == Pass::weights || PASS == Pass::input) {
      const int all = PASS == Pass::input ? 2 * p.steps : p.steps, each = (all + p.splits - 1) / p.splits;
      first = at.split * each;
      return max(0, min(all, first + each) - first);
    } else {
      first = 0;
      return p.steps;
    }
  };

  if (warp == 0) {
    if (lane == 0) {
      prefetchMap(&maps.a0);
      prefetchMap(&maps.b0);
      int stage = 0, issued = 0;
      uint32_t parity = 0;
      bool fine = true;
      for (int t = blockIdx.x; t < p.tiles && fine; t += gridDim.x) {
        const Tile at = tileAt(t);
        int first;
        const int steps = stepsOf(at, first);
        for (int k = 0; k < steps; ++k) {
          fine = barrierWait(empty + stage, parity ^ 1, broken, p.waitLimit);
          if (!fine) break;
          uint64_t *bar = full + stage;
          uint8_t *a = tileA + stage * S::a, *b = tileB + stage * S::b;
          barrierExpect(bar, S::a + S::b);
          if constexpr (kDual) {
            const int x = k * kTileSteps;
            copyBox(a, &maps.a0, x, at.row, bar);
            copyBox(b, &maps.b0, x, at.column, bar);
            copyBox(b + S::b / 2, &maps.b1, x, at.column, bar);
          } else if constexpr (PASS == Pass::input) {
            const bool up = first + k >= p.steps;   // du and Wu after da and Wg
            const int x = (first + k - (up ? p.steps : 0)) * kTileSteps;
            copyBox(a, up ? &maps.a1 : &maps.a0, x, at.row, bar);
#pragma unroll
            for (int j = 0; j < BN / 64; ++j) copyBox(b + j * 8192, up ? &maps.b1 : &maps.b0, at.column + 64 * j, x, bar);
          } else {
            const int y = (first + k) * kTileSteps;
#pragma unroll
            for (int j = 0; j < 2; ++j) copyBox(a + j * 8192, at.half ? &maps.a1 : &maps.a0, at.row + 64 * j, y, bar);
#pragma unroll
            for (int j = 0; j < BN / 64; ++j) copyBox(b + j * 8192, &maps.b0, at.column + 64 * j, y, bar);
          }
          issued = min(issued + 1, S::stages);
          if (++stage == S::stages) stage = 0, parity ^= 1;
        }
      }
      // The copies come to their end before the block does, whoever gave up.
      for (int i = 0; i < issued; ++i) {
        if (--stage < 0) stage = S::stages - 1, parity ^= 1;
        barrierSettle(full + stage, parity);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0, n = 0;
      uint32_t parity = 0;
      bool fine = true;
      constexpr uint32_t shape = productShape(BN, kAlongA, kAlongB);
      for (int t = blockIdx.x; t < p.tiles && fine; t += gridDim.x, ++n) {
        const Tile at = tileAt(t);
        int first;
        const int steps = stepsOf(at, first), buffer = n & 1;
        fine = barrierWait(taken + buffer, (n >> 1 & 1) ^ 1, broken, p.waitLimit);
        tensorFenceAfter();
        for (int k = 0; k < steps && fine; ++k) {
          fine = barrierWait(full + stage, parity, broken, p.waitLimit);
          if (!fine) break;
          tensorFenceAfter();
          const uint64_t a = operandDescriptor<kAlongA>(sharedAddress(tileA + stage * S::a));
          const uint64_t b = operandDescriptor<kAlongB>(sharedAddress(tileB + stage * S::b));
#pragma unroll
          for (int i = 0; i < kTileSteps / 16; ++i)
            tensorProduct(accumulators + buffer * BN, a + i * kDescriptorStep<kAlongA>, b + i * kDescriptorStep<kAlongB>, shape,
                          k > 0 || i > 0);
          tensorCommit(empty + stage);
          if (++stage == S::stages) stage = 0, parity ^= 1;
        }
        if (fine) tensorCommit(done + buffer);
      }
      // So do the products, before their tensor memory is freed.
      tensorCommit(ended);
      barrierSettle(ended, 0);
    }
  } else if (warp >= 4) {
    // A warp has a quarter of the tile's rows (that of tensor memory which it reaches) and of its columns.
    constexpr int kChunks = kPart / kChunk;
    const int quarter = warp % 4, part = (warp - 4) / 4;
    uint4 *stage = reinterpret_cast<uint4 *>(staging + (warp - 4) * S::staging);
    // Accumulators of a tile: zero where it has no steps, NaN where a wait ran out.
    auto take = [&](float (&x)[kChunk], uint32_t from, bool fine, bool some) {
      if (fine && some) {
        tensorLoad16(x, from);
      } else {
#pragma unroll
        for (int i = 0; i < kChunk; ++i) x[i] = fine ? 0.f : __int_as_float(0x7fffffff);
      }
    };
    if constexpr (kDual) {
      // Rows of the warp's part as pieces of 16 bytes, where the TMA's swizzle has them: neither rows of pieces nor columns
      // of them meet in a bank.
      constexpr int kPieces = kPart / 8;
      auto pieceOf = [&](uint4 *base, int piece) { return base + lane * kPieces + (piece ^ (kPieces == 4 ? lane >> 1 & 3 : lane >> 2 & 1)); };
      uint4 *gradients = reinterpret_cast<uint4 *>(incoming + (warp - 4) * S::incoming);
      uint64_t *bar = came + (warp - 4);
      uint32_t parity = 0;
      bool asked = false, fine = p.waitLimit > 0;
      auto ours = [&](const Tile &at) {   // the tile has rows and columns for this warp
        return part * kPart < kColumns && at.row + quarter * 32 < p.rows && at.column + part * kPart < p.F;
      };
      auto askGradients = [&](int t) {
        if (t >= p.tiles) return;
        const Tile at = tileAt(t);
        if (!ours(at)) return;
        barrierExpect(bar, S::incoming);
        copyBox(gradients, &maps.dh, at.column + part * kPart, at.row + quarter * 32, bar);
        asked = true;
      };
      if (PASS == Pass::gradients && p.wholeDh && lane == 0) askGradients(blockIdx.x);
      int n = 0;
      for (int t = blockIdx.x; t < p.tiles; t += gridDim.x, ++n) {
        const Tile at = tileAt(t);
        const bool own = ours(at);
        const int buffer = n & 1, first = at.column + part * kPart;
        const int64_t row = at.row + quarter * 32, rowsLeft = p.rows - row;
        const bool mine = lane < rowsLeft;
        // (given up once, no tile waits again)
        fine = fine && __all_sync(0xffffffffu, barrierAwait(done + buffer, n >> 1 & 1, broken, p.waitLimit));
        if (PASS == Pass::gradients && p.wholeDh && own && fine) {
          fine = __all_sync(0xffffffffu, barrierAwait(bar, parity, broken, p.waitLimit));
          if (fine) asked = false, parity ^= 1;
        }
        tensorFenceAfter();
        const uint32_t tensorRow = accumulators + buffer * BN + (uint32_t(quarter * 32) << 16) + part * kPart;
        uint4 later[kChunks][2];   // du, until da has left
        if (own) {
          if (lane == 0) storesRead();   // of the tile before
#pragma unroll
          for (int k = 0; k < kChunks; ++k) {
            const int column = first + k * kChunk, columns = min(kChunk, p.F - column);
            if (columns <= 0) break;
            float a[kChunk], u[kChunk];
            __syncwarp();   // loads from tensor memory are the whole warp's
            take(a, tensorRow + k * kChunk, fine, p.steps > 0);
            take(u, tensorRow + BN / 2 + k * kChunk, fine, p.steps > 0);
            uint4 dh[2];
            if constexpr (PASS == Pass::gradients) {
              if (p.wholeDh) {
#pragma unroll
                for (int i = 0; i < 2; ++i) dh[i] = *pieceOf(gradients, 2 * k + i);
              } else {
                const bf16 *from = p.dh + (row + lane) * p.dhStride + column;
                uint32_t *w = reinterpret_cast<uint32_t *>(dh);
#pragma unroll
                for (int i = 0; i < kChunk; i += 2) {
                  const uint32_t low = mine && i < columns ? __bfloat16_as_ushort(from[i]) : 0u;
                  const uint32_t high = mine && i + 1 < columns ? __bfloat16_as_ushort(from[i + 1]) : 0u;
                  w[i / 2] = high << 16 | low;
                }
              }
            }
            uint4 bias[2][2];
            if (p.bGate) {
              if (p.wholeBias && columns == kChunk) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  bias[0][i] = reinterpret_cast<const uint4 *>(p.bGate + column)[i];
                  bias[1][i] = reinterpret_cast<const uint4 *>(p.bUp + column)[i];
                }
              } else {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                  for (int i = 0; i < kChunk; i += 2) {
                    const bf16 *from = (b ? p.bUp : p.bGate) + column;
                    const uint32_t low = i < columns ? __bfloat16_as_ushort(from[i]) : 0u;
                    const uint32_t high = i + 1 < columns ? __bfloat16_as_ushort(from[i + 1]) : 0u;
                    reinterpret_cast<uint32_t *>(bias[b])[i / 2] = high << 16 | low;
                  }
              }
            }
            tensorLoadWait();
            tensorLoaded(a);
            tensorLoaded(u);
            auto half = [](const uint4 (&v)[2], int i) {
              const uint32_t two = reinterpret_cast<const uint32_t *>(v)[i / 2];
              return __uint_as_float(i % 2 ? two & 0xffff0000u : two << 16);
            };
            if (p.bGate) {
#pragma unroll
              for (int i = 0; i < kChunk; ++i) a[i] += half(bias[0], i), u[i] += half(bias[1], i);
            }
            withActivation(p.activation, [&](auto kind) {
#pragma unroll
              for (int i = 0; i < kChunk; ++i) {
                const Activated f = activate<kind.value, true>(a[i]);
                if constexpr (PASS == Pass::forward) {
                  a[i] = f.y * u[i];
                } else {
                  const float d = half(dh, i);
                  a[i] = d * u[i] * f.slope;
                  u[i] = d * f.y;
                }
              }
            });
            if (PASS == Pass::gradients || p.wholeH) {
              *pieceOf(stage, 2 * k) = eightOf(a);
              *pieceOf(stage, 2 * k + 1) = eightOf(a + 8);
            } else {
              storeRows(stage, eightOf(a), eightOf(a + 8), p.h + row * p.F + column, p.F, rowsLeft, columns, false, lane);
            }
            if constexpr (PASS == Pass::gradients) {
              later[k][0] = eightOf(u), later[k][1] = eightOf(u + 8);
              if (p.biasParts) {
                if (rowsLeft < 32) {   // (a row that is not there may have become NaN beside an infinite bias)
#pragma unroll
                  for (int i = 0; i < kChunk; ++i) a[i] = mine ? a[i] : 0.f, u[i] = mine ? u[i] : 0.f;
                }
                const float sumA = columnSum(a, lane), sumU = columnSum(u, lane);
                float *parts = p.biasParts + (int64_t(at.row / kTileRows) * 4 + quarter) * 2 * p.F + column;
                if (lane < columns) parts[lane] = sumA, parts[p.F + lane] = sumU;
              }
            }
          }
          if (PASS == Pass::gradients || p.wholeH) {
            fenceForCopies();
            __syncwarp();
            if (lane == 0) storeBox(&maps.out0, stage, first, int(row));
          }
        } else if (PASS == Pass::gradients && p.biasParts && part * kPart < kColumns && first < p.F) {
          // No rows: their sums are zero.
          float *parts = p.biasParts + (int64_t(at.row / kTileRows) * 4 + quarter) * 2 * p.F;
          for (int column = first + lane; column < min(p.F, first + kPart); column += 32) parts[column] = parts[p.F + column] = 0.f;
        }
        tensorFenceBefore();
        __syncwarp();
        if (lane == 0 && fine) barrierArrive(taken + buffer);   // (without it the products do not go on)
        if constexpr (PASS == Pass::gradients) {
          if (p.wholeDh && fine && lane == 0) askGradients(t + gridDim.x);   // every lane has its row of this tile's
          if (own) {
            if (lane == 0) storesRead();
            __syncwarp();
#pragma unroll
            for (int k = 0; k < kChunks; ++k) {
              *pieceOf(stage, 2 * k) = later[k][0];
              *pieceOf(stage, 2 * k + 1) = later[k][1];
            }
            fenceForCopies();
            __syncwarp();
            if (lane == 0) storeBox(&maps.out1, stage, first, int(row));
          }
        }
      }
      if (lane == 0) {
        storesDone();
        if (asked) barrierSettle(bar, parity);   // given up: its own copy comes to its end
      }
      __syncwarp();
    } else {
      int n = 0;
      bool fine = p.waitLimit > 0;
      for (int t = blockIdx.x; t < p.tiles; t += gridDim.x, ++n) {
        const Tile at = tileAt(t);
        const int buffer = n & 1;
        int first;
        const int steps = stepsOf(at, first);
        const int64_t row = at.row + quarter * 32, rowsLeft = (PASS == Pass::weights ? int64_t(p.F) : p.rows) - row;
        fine = fine && __all_sync(0xffffffffu, barrierWait(done + buffer, n >> 1 & 1, broken, p.waitLimit));
        tensorFenceAfter();
        const uint32_t tensorRow = accumulators + buffer * BN + (uint32_t(quarter * 32) << 16) + part * kPart;
#pragma unroll
        for (int k = 0; k < kChunks; ++k) {
          const int column = at.column + part * kPart + k * kChunk, columns = min(kChunk, p.D - column);
          if (columns <= 0) break;
          float x[kChunk];
          __syncwarp();
          take(x, tensorRow + k * kChunk, fine, steps > 0);
          tensorLoadWait();
          tensorLoaded(x);
          if (p.splits == 1) {
            bf16 *to = PASS == Pass::input ? p.dx : at.half ? p.dwUp : p.dwGate;
            storeRows(stage, eightOf(x), eightOf(x + 8), to + row * p.D + column, p.D, rowsLeft, columns, p.wholeD, lane);
          } else {
            const int64_t before = PASS == Pass::input ? at.split * p.rows : (int64_t(at.split) * 2 + at.half) * p.F;
            float *to = p.parts + (before + row) * p.D + column;
            storeRows(stage, fourOf(x), fourOf(x + 4), to, p.D, rowsLeft, columns, p.wholeD, lane);
            if (columns > 8) storeRows(stage, fourOf(x + 8), fourOf(x + 12), to + 8, p.D, rowsLeft, columns - 8, p.wholeD, lane);
          }
        }
        tensorFenceBefore();
        __syncwarp();
        if (lane == 0 && fine) barrierArrive(taken + buffer);   // (without it the products do not go on)
      }
    }
  }
  tensorFenceBefore();
  __syncthreads();
  tensorFenceAfter();
  if (warp == 2) tensorFree(accumulators, 2 * BN);
  if (threadIdx.x == 0 && *broken) *p.ranOut = 1, __threadfence_system();
}

// Rows of x, of Wg and of Wu, one after the other, as rows of whole 16-byte pieces: the
// TMA takes no others.
struct PadArgs {
  const bf16 *x, *wGate, *wUp;
  bf16 *to;            // [rows + 2 F, stride]
  int64_t rows, xStride;
  int D, F, stride;
};
constexpr int kPadThreads = 256;
__global__ void __launch_bounds__(kPadThreads) padRows(PadArgs p) {
  const int pieces = p.stride / 8;
  const int64_t all = (p.rows + 2 * int64_t(p.F)) * pieces;
  for (int64_t i = int64_t(blockIdx.x) * kPadThreads + threadIdx.x; i < all; i += int64_t(gridDim.x) * kPadThreads) {
    const int64_t row = i / pieces, weight = row - p.rows;
    const int column = int(i - row * pieces) * 8;
    const bf16 *from = weight < 0       ? p.x + row * p.xStride
                       : weight < p.F ? p.wGate + weight * p.D
                                      : p.wUp + (weight - p.F) * p.D;
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const uint32_t low = column + j < p.D ? __bfloat16_as_ushort(from[column + j]) : 0u;
      const uint32_t high = column + j + 1 < p.D ? __bfloat16_as_ushort(from[column + j + 1]) : 0u;
      w[j / 2] = high << 16 | low;
    }
    *reinterpret_cast<uint4 *>(p.to + row * p.stride + column) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// -------------------------------------------------------------------- float32
// Tiles of 128 rows and 128 columns, 16 steps at a time, 8 by 8 values a thread as
// pairs; the operands of the next steps are on their way in registers.  Where that
// leaves multiprocessors without a tile, of 64 by 64, 4 by 4 and 32 steps (with 16 the
// next steps' way from memory takes longer than their products).  The forward pass's
// columns are half of Wg's and half the same of Wu's: a thread has both of a value.
// A sum of n values of random sign is off by 2^-25 sqrt(n / 2) of itself where each is
// added to one register; after kRunSteps it goes to memory, and is added to
// there, so that long ones are off by no more than 7e-7.  That is where the outputs
// are, but for the forward pass, whose sums are not outputs: shared memory (16384
// rows, 4096 x 1024: 5.20 ms, in one run 4.99).
struct ProductArgs {
  const float *x, *wGate, *wUp, *bGate, *bUp;
  float *h, *kept;             // forward: h, and a and u [2, rows, F] or null
  const float *both;           // [2, rows, F]: da and du
  float *dx, *parts;           // weights: [splits, 2, F, D], input: [splits, rows, D] where it is split
  int64_t rows, xStride;
  int D, F, activation, splits;
  bool wholeX, wholeD, wholeF;   // rows of x, of D and of F values are 16-byte pieces
};
constexpr int kProductThreads = 256;
__host__ __device__ constexpr int productSteps(int tile) { return tile == 64 ? 32 : 16; }
constexpr int kRunSteps = 1024;

// The first `count` of four values.
__device__ __forceinline__ float4 fetchFour(const float *p, int64_t count, bool whole) {
  if (count >= 4 && whole) return *reinterpret_cast<const float4 *>(p);
  return make_float4(count > 0 ? p[0] : 0.f, count > 1 ? p[1] : 0.f, count > 2 ? p[2] : 0.f, count > 3 ? p[3] : 0.f);
}
using Two = unsigned long long;
__device__ __forceinline__ Two twoOf(float a, float b) {
  Two p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ float2 partsOf(Two p) {
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ void addProduct(Two &d, Two a, Two b) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(d) : "l"(a), "l"(b));
}

// RUNS: sums may be longer than one run; the forward pass has T T floats of dynamic shared memory then.
template <Pass PASS, int T, bool RUNS> __global__ void __launch_bounds__(kProductThreads, 2) gatedProducts(ProductArgs p) {
  static_assert(PASS != Pass::gradients, "gatedGradients");
  constexpr int K = productSteps(T), P = T + 4, R = T / 16, H = R / 2;   // R rows and columns a thread, H in each half of the columns
  constexpr int kLoads = T * K / (4 * kProductThreads), kGroups = T / 4, kSteps = K / 4;   // a thread's, and of four values side by side
  constexpr bool kAlongA = PASS != Pass::weights, kAlongB = PASS == Pass::forward;   // steps are contiguous
  __shared__ __align__(16) float as[2][K][P], bs[2][K][P];
  extern __shared__ __align__(16) Two earlier[];   // forward: sums of the runs before, R H of each thread
  const int tid = threadIdx.x;
  const int64_t row0 = int64_t(blockIdx.x) * T;   // weights: of Wg's and then Wu's tiles
  const int rowTiles = (p.F + T - 1) / T;
  const int half = PASS == Pass::weights && int(blockIdx.x) >= rowTiles;
  const int64_t m0 = PASS == Pass::weights ? row0 - int64_t(half) * rowTiles * T : row0;
  const int n0 = blockIdx.y * (PASS == Pass::forward ? T / 2 : T);
  const int64_t plane = p.rows * p.F;
  const int halfSteps = (p.F + K - 1) / K;   // input: steps of the first product, then those of the second
  const int64_t allSteps = PASS == Pass::forward ? (p.D + K - 1) / K : PASS == Pass::input ? 2 * halfSteps : (p.rows + K - 1) / K;
  const int64_t each = (allSteps + p.splits - 1) / p.splits;
  const int64_t first = blockIdx.z * each, last = min(allSteps, first + each);

  auto fetchA = [&](int64_t step, int i) {
    const int at = tid + i * kProductThreads;
    if constexpr (PASS == Pass::forward) {
      const int64_t m = m0 + at / kSteps, k = step * K + at % kSteps * 4;
      return fetchFour(p.x + m * p.xStride + k, m < p.rows ? p.D - k : 0, p.wholeX);
    } else if constexpr (PASS == Pass::input) {
      const bool up = step >= halfSteps;
      const int64_t m = m0 + at / kSteps, k = (step - (up ? halfSteps : 0)) * K + at % kSteps * 4;
      return fetchFour(p.both + (up ? plane : 0) + m * p.F + k, m < p.rows ? p.F - k : 0, p.wholeF);
    } else {
      const int64_t k = step * K + at / kGroups, m = m0 + at % kGroups * 4;
      return fetchFour(p.both + (half ? plane : 0) + k * p.F + m, k < p.rows ? p.F - m : 0, p.wholeF);
    }
  };
  auto fetchB = [&](int64_t step, int i) {
    const int at = tid + i * kProductThreads;
    if constexpr (PASS == Pass::forward) {
      const int row = at / kSteps, f = n0 + row % (T / 2);
      const int64_t k = step * K + at % kSteps * 4;
      return fetchFour((row < T / 2 ? p.wGate : p.wUp) + int64_t(f) * p.D + k, f < p.F ? p.D - k : 0, p.wholeD);
    } else if constexpr (PASS == Pass::input) {
      const bool up = step >= halfSteps;
      const int64_t k = (step - (up ? halfSteps : 0)) * K + at / kGroups, n = n0 + at % kGroups * 4;
      return fetchFour((up ? p.wUp : p.wGate) + k * p.D + n, k < p.F ? p.D - n : 0, p.wholeD);
    } else {
      const int64_t k = step * K + at / kGroups, n = n0 + at % kGroups * 4;
      return fetchFour(p.x + k * p.xStride + n, k < p.rows ? p.D - n : 0, p.wholeX);
    }
  };
  // Operands whose steps are contiguous are turned over on their way: fours of rows are placed so that the lanes of four
  // and eight steps' fours do not meet in a bank.
  auto turned = [](int k) { return (k / 4 & 7) * 4; };
  auto put = [&](float (&tile)[K][P], bool along, int i, float4 v) {
    const int at = tid + i * kProductThreads;
    if (along) {
      const int k = at % kSteps * 4, row = (at / kSteps) ^ turned(k);
      tile[k][row] = v.x, tile[k + 1][row] = v.y, tile[k + 2][row] = v.z, tile[k + 3][row] = v.w;
    } else {
      *reinterpret_cast<float4 *>(&tile[at / kGroups][at % kGroups * 4]) = v;
    }
  };

  const int ty = tid / 16, tx = tid % 16;
  Two sum[R][H];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < H; ++j) sum[i][j] = 0;
  float4 a[kLoads], b[kLoads];
  if (first < last) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) put(as[0], kAlongA, i, fetchA(first, i)), put(bs[0], kAlongB, i, fetchB(first, i));
  }
  __syncthreads();
  // What the tile's sums go to.
  auto store = [&](bool add) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t m = m0 + (i / 4) * 64 + ty * 4 + i % 4;
      if (m >= (PASS == Pass::weights ? int64_t(p.F) : p.rows)) continue;
      float *to = PASS == Pass::weights ? p.parts + ((int64_t(blockIdx.z) * 2 + half) * p.F + m) * p.D
                  : p.splits > 1        ? p.parts + (blockIdx.z * p.rows + m) * p.D
                                        : p.dx + m * p.D;
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const int n = n0 + (j / H) * (T / 2) + tx * H + j % H;
        const float2 two = partsOf(sum[i][j / 2]);
        const float v = j % 2 ? two.y : two.x;
        if (n < p.D) to[n] = add ? to[n] + v : v;
      }
#pragma unroll
      for (int j = 0; j < H; ++j) sum[i][j] = 0;
    }
  };
  int64_t run = first;
  do {
    const int64_t end = RUNS ? min(last, run + kRunSteps / K) : last;
    for (int64_t step = run; step < end; ++step) {
      const int now = int(step - first) & 1;
      if (step + 1 < last) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) a[i] = fetchA(step + 1, i), b[i] = fetchB(step + 1, i);
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float rows[R];
#pragma unroll
        for (int i = 0; i < R; i += 4)
          *reinterpret_cast<float4 *>(rows + i) = *reinterpret_cast<const float4 *>(&as[now][k][(i * 16 + ty * 4) ^ (kAlongA ? turned(k) : 0)]);
        const int turn = kAlongB ? turned(k) : 0;
        Two columns[H];
        if constexpr (H == 4) {
          *reinterpret_cast<ulonglong2 *>(columns) = *reinterpret_cast<const ulonglong2 *>(&bs[now][k][tx * 4 ^ turn]);
          *reinterpret_cast<ulonglong2 *>(columns + 2) = *reinterpret_cast<const ulonglong2 *>(&bs[now][k][T / 2 + (tx * 4 ^ turn)]);
        } else {
          columns[0] = *reinterpret_cast<const Two *>(&bs[now][k][tx * 2 ^ turn]);
          columns[1] = *reinterpret_cast<const Two *>(&bs[now][k][T / 2 + (tx * 2 ^ turn)]);
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const Two r = twoOf(rows[i], rows[i]);
#pragma unroll
          for (int j = 0; j < H; ++j) addProduct(sum[i][j], r, columns[j]);
        }
      }
      if (step + 1 < last) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) put(as[now ^ 1], kAlongA, i, a[i]), put(bs[now ^ 1], kAlongB, i, b[i]);
      }
      __syncthreads();
    }
    if constexpr (PASS != Pass::forward) {
      store(run > first);
    } else if constexpr (RUNS) {   // (a thread's own sums: no barrier)
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < H; ++j) {
          Two &at = earlier[(i * H + j) * kProductThreads + tid];
          const float2 now = partsOf(sum[i][j]), before = run > first ? partsOf(at) : make_float2(0.f, 0.f);
          const Two both = twoOf(before.x + now.x, before.y + now.y);
          if (end < last) at = both, sum[i][j] = 0;
          else sum[i][j] = both;
        }
    }
    run = end;
  } while (run < last);
  if constexpr (PASS == Pass::forward) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t m = m0 + (i / 4) * 64 + ty * 4 + i % 4;
      if (m >= p.rows) continue;
      float v[R];
#pragma unroll
      for (int j = 0; j < H; ++j) {
        const float2 two = partsOf(sum[i][j]);
        v[2 * j] = two.x, v[2 * j + 1] = two.y;
      }
      const int f = n0 + tx * H;
#pragma unroll
      for (int j = 0; j < H; ++j) {
        if (f + j >= p.F) break;
        float gate = v[j], up = v[H + j];
        if (p.bGate) gate += p.bGate[f + j], up += p.bUp[f + j];
        const int64_t at = m * p.F + f + j;
        if (p.kept) p.kept[at] = gate, p.kept[plane + at] = up;
        withActivation(p.activation, [&](auto kind) { p.h[at] = activate<kind.value, false>(gate).y * up; });
      }
    }
  }
}

// da and du from what the forward pass kept, and sums over kGradientRows rows for
// the biases' gradients.  A warp has 32 columns of every eighth row.
struct GradientArgs {
  const float *kept, *dh;
  float *both, *biasParts;   // [row blocks, 2, F] or null
  int64_t rows, dhStride;
  int F, activation;
};
constexpr int kGradientRows = 64;
__global__ void __launch_bounds__(256) gatedGradients(GradientArgs p) {
  __shared__ float sums[8][2][32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, f = blockIdx.y * 32 + lane;
  const int64_t row0 = int64_t(blockIdx.x) * kGradientRows, plane = p.rows * p.F;
  float sumA = 0.f, sumU = 0.f;
  if (f < p.F)
    withActivation(p.activation, [&](auto kind) {
#pragma unroll 4
      for (int r = warp; r < kGradientRows; r += 8) {
        const int64_t row = row0 + r, at = row * p.F + f;
        if (row >= p.rows) break;
        const float d = p.dh[row * p.dhStride + f], u = p.kept[plane + at];
        const Activated y = activate<kind.value, false>(p.kept[at]);
        const float da = d * u * y.slope, du = d * y.y;
        p.both[at] = da, p.both[plane + at] = du;
        sumA += da, sumU += du;
      }
    });
  if (!p.biasParts) return;
  sums[warp][0][lane] = sumA, sums[warp][1][lane] = sumU;
  __syncthreads();
  if (warp >= 2 || f >= p.F) return;
  float sum = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) sum += sums[w][warp][lane];
  p.biasParts[(int64_t(blockIdx.x) * 2 + warp) * p.F + f] = sum;
}

// -------------------------------------------------------------- sums of parts
// out[i] = sum over n of parts[n, i], in float32, to the layer's type; the first
// `cut` of the `count` values to one array, the others to another.  Bias sums likewise.
template <class T> struct SumArgs {
  const float *parts, *biasParts;
  T *first, *second, *dbGate, *dbUp;
  int64_t cut, count;
  int F, splits, biasCount, blocks;   // blocks for `parts`
};
constexpr int kSumThreads = 256, kSumColumns = 8;
template <class T> __global__ void __launch_bounds__(kSumThreads) sumParts(SumArgs<T> p) {
  if (int(blockIdx.x) < p.blocks) {
    const int64_t i = (int64_t(blockIdx.x) * kSumThreads + threadIdx.x) * 4;
    if (i >= p.count) return;
    if (p.cut % 4 == 0 && p.count % 4 == 0) {
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int n = 0; n < p.splits; ++n) {
        const float4 v = *reinterpret_cast<const float4 *>(p.parts + n * p.count + i);
        sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
      }
      T *to = i < p.cut ? p.first + i : p.second + (i - p.cut);
      to[0] = fromFloat<T>(sum.x), to[1] = fromFloat<T>(sum.y), to[2] = fromFloat<T>(sum.z), to[3] = fromFloat<T>(sum.w);
    } else {
      for (int64_t j = i; j < min(i + 4, p.count); ++j) {
        float sum = 0.f;
        for (int n = 0; n < p.splits; ++n) sum += p.parts[n * p.count + j];
        (j < p.cut ? p.first[j] : p.second[j - p.cut]) = fromFloat<T>(sum);
      }
    }
    return;
  }
  // Biases: a block has eight columns, a sector of each part, and as many parts at once as that leaves threads for.
  constexpr int kAtOnce = kSumThreads / kSumColumns;
  __shared__ float sums[kAtOnce][kSumColumns];
  const int own = threadIdx.x % kSumColumns, from = threadIdx.x / kSumColumns;
  const int column = (int(blockIdx.x) - p.blocks) * kSumColumns + own;
  float sum = 0.f;
  if (column < 2 * p.F) {
#pragma unroll 8
    for (int n = from; n < p.biasCount; n += kAtOnce) sum += p.biasParts[int64_t(n) * 2 * p.F + column];
  }
  sums[from][own] = sum;
  __syncthreads();
  if (from > 0 || column >= 2 * p.F) return;
#pragma unroll
  for (int k = 1; k < kAtOnce; ++k) sum += sums[k][own];
  (column < p.F ? p.dbGate[column] : p.dbUp[column - p.F]) = fromFloat<T>(sum);
}

}  // namespace duckb200
