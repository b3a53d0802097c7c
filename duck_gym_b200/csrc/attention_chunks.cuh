// Linear attention with a decay in chunks of C steps, bfloat16 operands.
//
// Within a chunk that starts from the state S (i, j steps of the chunk, L its
// length, decay l, everything of one environment and head):
//
//   o_i  = scale [ l^(i+1) S^T q_i + sum_{j <= i} l^(i-j) (q_i . k_j) v_j ]
//   S'   = l^L S + sum_j l^(L-1-j) k_j v_j^T
//
// which are the products Q K^T, (Q K^T . decays) V, Q S and K^T V.  A warp owns
// 16 steps of the chunk and a slice of S, which stays in its registers in
// float32 from chunk to chunk; a bfloat16 copy in shared memory is the operand
// of the next chunk's Q S.
//
// Decays without an exponential per pair: a table of l^n in shared memory, read at
// i - j (the lanes of a tile read 14 neighbouring words).  The table is zero below
// n = 0, which is the causal mask.
//
// Roundings to bfloat16, each of 8 significant bits: the decayed scores, and the
// copy of S.  The state's own operand l^(L-1-j) k_j is not rounded to 8 bits: it is
// split into the sum of two bfloat16 numbers (16 bits), a product each, so that an
// output has one rounding on its way besides its own; and of three (24 bits) where
// the state is an output, in every chunk: the steps after a chunk may add nothing, so
// that what has faded is all there is.  (Measured against 64 bits: outputs and
// gradients 2.3e-3 in the 2-norm, where one rounding is 1.7e-3; states and their
// gradients 1.4e-7 to 1.04e-6, the more the longer they remember.  With three parts
// throughout, 1000 x 256 takes 224 us forward and 353 backward.)
//
// Episodes: step i sees step j only if no reset lies in (j, i]; S only if none
// lies at or before i.  Scores and states that are masked are replaced, not
// multiplied by zero.  A product still multiplies a masked zero with whatever
// the other operand holds, so an infinity or NaN of an earlier episode (or of a
// later step in the same tile) would come out as NaN.  So a block that saw
// anything in its outputs or its state that is not finite says so in a flag, and
// redoAttention() computes the environments and heads of such blocks once more
// step by step, where nothing masked is ever touched.  (What is wrong in this way is
// never finite, the saved states and those of segments included, and whoever reads
// those sees it too.)
//
// Warp-level products of 16x8x16, because a chunk of one head is small (64 x 64
// times 64, 24 steps a rollout) and half of a score matrix is masked; a warp's 16
// steps are a natural piece of both.  What bounds them on a B200 is the operands' way from
// shared memory and the latency of short chains of products, with 12 to 16 warps a
// multiprocessor: 1000 steps, 256 environments, 4 heads of 64, forward 202 us (tensor
// pipe 34 % active, shared memory's data pipe 40 %, issue slots 36 %, DRAM 36 %),
// backward 320 to 344 us by the run (42 %, 53 %, 42 %, 35 %); 24 steps, 1024
// environments: 29 and 44 us (3.9 and 3.5 TB/s); 16384 steps, one environment, 8 heads
// of 128, in 18 segments: 49 us for what each adds, 8 for the join, 88 us.
// Tried and slower: two warps for the same 16 steps (235 us), 32 steps a warp (241 us
// with a third fewer reads of shared memory), rows of V read once for scores and state
// (258 us), the backward blocks unrolled (357 us).
#pragma once
#include "linear_attention.cuh"
#include "tensor_tiles.cuh"

#include <type_traits>

namespace duckb200 {

struct ChunkArgs {
  const bf16 *q, *k, *v;
  bf16 *out;                   // [T, E, H, Dv] dense
  Rows qs, ks, vs;
  const float *decay;
  const uint8_t *resets;       // [T, E] or null
  const float *stateIn;        // [E, H, Dk, Dv] or null
  float *stateOut;             // or null
  bf16 *saved;                 // [E, H, chunks, Dk, Dv]: the state before each chunk, or null
  float *segments;             // [E, H, segmentCount, Dk, Dv] where T is split, else null
  uint8_t *segmentCut;         // [E, H, segmentCount]
  uint8_t *flags;              // [E, H, segmentCount, columnTiles]: blocks that saw what is not finite
  int T, E, H, Dk, Dv;
  int segmentLength, segmentCount, columnTiles;
  int vecQ, vecK, vecV;        // rows can be read in 16-byte pieces
  int precise;                 // the state is an output: its operand is split in three
  float scale;
};

// A power of a decay to a few units in the last place, however far it has faded (2 to
// the n times a float32 logarithm would be off by 2^-24 of the exponent: 2e-6 of what
// 500 steps at 0.9 leave).  Of a negative or NaN decay: NaN, which leaves a block to
// redoAttention().
__device__ __forceinline__ float powerOf(float decay, int n) {
  return decay >= 0.f ? powf(decay, float(n)) : __int_as_float(0x7fc00000);
}

// Where episodes begin in steps t0 .. t0 + 63 before `end`: a lane looks at two of
// them; read a chunk ahead.
struct Resets {
  uint32_t a = 0, b = 0;   // the bytes as they are: looked at only when they are needed
  __device__ __forceinline__ void read(const uint8_t *resets, int E, int e, int t0, int end) {
    if (!resets) return;
    const int t = t0 + (threadIdx.x & 31);
    const uint8_t *at = resets + int64_t(t) * E + e;
    a = b = 0;
    if (t < end) a = at[0];
    if (t + 32 < end) b = at[int64_t(32) * E];
  }
  // Bit i: at step t0 + i.
  __device__ __forceinline__ unsigned long long mask() const {
    const unsigned low = __ballot_sync(0xffffffffu, a != 0), high = __ballot_sync(0xffffffffu, b != 0);
    return (static_cast<unsigned long long>(high) << 32) | low;
  }
};
// Last step of a chunk up to i at which an episode begins, or -1: step i sees the
// steps from there on, and the state before the chunk if there is none.
__device__ __forceinline__ int episodeStart(unsigned long long mask, int i) {
  return 63 - __clzll(static_cast<long long>(mask & (~0ull >> (63 - i))));
}
// First step after j at which an episode begins: the steps before it see step j.
__device__ __forceinline__ int episodeEnd(unsigned long long mask, int j) {
  const unsigned long long after = mask & ~(~0ull >> (63 - j));
  return after ? __ffsll(static_cast<long long>(after)) - 1 : 1 << 30;
}

// Rows t0.. (count of them, the rest zero) of an operand, columns c0..c0+D-1
// (those from `width` on zero), into a tile of C rows.
template <int C, int D, int THREADS>
__device__ __forceinline__ void loadTile(bf16 *tile, const bf16 *base, int64_t stride, int t0, int count, int c0,
                                         int width, bool vec) {
  constexpr int L = D + 8;
  if (vec) {
    constexpr int pieces = D / 8, rows = THREADS / pieces;   // rows that the block's threads copy at once
    const int r0 = threadIdx.x / pieces, c = (threadIdx.x % pieces) * 8;
    const bool inside = c0 + c < width;
    const bf16 *from = base + int64_t(t0 + r0) * stride + c0 + c;
    bf16 *to = tile + r0 * L + c;
    if (count == C && width >= c0 + D) {
#pragma unroll
      for (int x = 0; x < C / rows; ++x) copyAsync16(to + x * rows * L, from + x * (rows * stride));
      return;
    }
#pragma unroll
    for (int x = 0; x < C / rows; ++x) {
      const bool valid = inside && r0 + x * rows < count;
      copyAsync16(to + x * rows * L, valid ? from + x * (rows * stride) : base, valid);
    }
  } else {
    for (int id = threadIdx.x; id < C * D; id += THREADS) {
      const int r = id / D, c = id % D;
      tile[r * L + c] = r < count && c0 + c < width ? base[int64_t(t0 + r) * stride + c0 + c] : fromFloat<bf16>(0.f);
    }
  }
}

// Rows of 16 steps by N tiles of 8 columns of a dense [T, E, H, width] output,
// as the products leave them: lane 4 g + q has columns 2 q and 2 q + 1 of row g
// (and g + 8) of each tile.  `finite` becomes NaN if one of them is not finite.
// Where rows are whole 16-byte pieces, the four lanes of a row exchange their
// pairs of four tiles (a 4 x 4 transpose, two rounds), so that each stores all of
// one tile: 64 bytes of a row at a time.
template <int N>
__device__ __forceinline__ void storeTile(bf16 *out, const float (&x)[N][4], int64_t stepStride, int first, int count,
                                          int row0, int col0, int width, uint32_t &finite) {
  const int lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
  if (N % 4 == 0 && width % 8 == 0) {
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int i = row0 + g + y * 8;
      bf16 *to = out + int64_t(first + i) * stepStride + col0 + tq * 8;
#pragma unroll
      for (int n = 0; n < N / 4 * 4; n += 4) {
        uint32_t p[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          p[m] = packPair(x[n + m][2 * y], x[n + m][2 * y + 1]);
          finite = addZeroTimes(p[m], finite);
        }
        const bool odd = tq & 1, upper = tq & 2;
        const uint32_t a = __shfl_xor_sync(0xffffffffu, odd ? p[0] : p[1], 1);
        const uint32_t b = __shfl_xor_sync(0xffffffffu, odd ? p[2] : p[3], 1);
        // Of tiles (0, 2) + odd: columns of the lower and the upper lane of the pair.
        const uint32_t l0 = odd ? a : p[0], u0 = odd ? p[1] : a, l2 = odd ? b : p[2], u2 = odd ? p[3] : b;
        const uint32_t c = __shfl_xor_sync(0xffffffffu, upper ? l0 : l2, 2);
        const uint32_t d = __shfl_xor_sync(0xffffffffu, upper ? u0 : u2, 2);
        const uint4 whole = upper ? make_uint4(c, d, l2, u2) : make_uint4(l0, u0, c, d);
        if (i < count && col0 + (n + tq) * 8 < width) *reinterpret_cast<uint4 *>(to + n * 8) = whole;
      }
    }
    return;
  }
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const uint32_t p = packPair(x[n][2 * y], x[n][2 * y + 1]);
      finite = addZeroTimes(p, finite);
      const int i = row0 + g + y * 8, j = col0 + n * 8 + 2 * tq;
      if (i >= count) continue;
      bf16 *to = out + int64_t(first + i) * stepStride + j;
      if (j + 1 < width && width % 2 == 0) *reinterpret_cast<uint32_t *>(to) = p;
      else {
        if (j < width) to[0] = fromFloat<bf16>(x[n][2 * y]);
        if (j + 1 < width) to[1] = fromFloat<bf16>(x[n][2 * y + 1]);
      }
    }
}
// The same through 16 rows of shared memory (D of them wide at least) that only
// this warp uses.
template <int D, int N>
__device__ __forceinline__ void storeTileStaged(bf16 *out, bf16 *stage, const float (&x)[N][4], int64_t stepStride,
                                                int first, int count, int row0, int col0, int width,
                                                uint32_t &finite) {
  constexpr int L = D + 8, pieces = N, rows = 32 / pieces;   // lanes of a row, rows of an instruction
  if (width % 8 != 0) {
    storeTile(out, x, stepStride, first, count, row0, col0, width, finite);
    return;
  }
#pragma unroll
  for (int n = 0; n < N; n += 2) {
    const uint32_t p[4] = {packPair(x[n][0], x[n][1]), packPair(x[n][2], x[n][3]), packPair(x[n + 1][0], x[n + 1][1]),
                           packPair(x[n + 1][2], x[n + 1][3])};
#pragma unroll
    for (int m = 0; m < 4; ++m) finite = addZeroTimes(p[m], finite);
    storeMatrices<L>(stage, 0, n * 8, p);
  }
  __syncwarp();
  const int lane = threadIdx.x & 31, r0 = lane / pieces, c = (lane % pieces) * 8;
  bf16 *to = out + int64_t(first + row0 + r0) * stepStride + col0 + c;
  const bool inside = col0 + c < width;
#pragma unroll
  for (int r = 0; r < 16 / rows; ++r)
    if (inside && row0 + r0 + r * rows < count)
      *reinterpret_cast<uint4 *>(to + r * (rows * stepStride)) =
          *reinterpret_cast<const uint4 *>(stage + (r0 + r * rows) * L + c);
}

template <int N> __device__ __forceinline__ bool notFinite(const float (&x)[N][4]) {
  float sum = 0.f;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int y = 0; y < 4; ++y) sum = fmaf(x[n][y], 0.f, sum);
  return sum != 0.f;
}

// A float32 state [rows, width] (from column c0 on, D columns) as a bfloat16 tile.
template <int DK, int D, int THREADS>
__device__ __forceinline__ void loadState(bf16 *tile, const float *from, int rows, int c0, int width) {
  constexpr int L = D + 8, quads = D / 4;
  if (width % 4 == 0) {
    constexpr int each = DK * quads / THREADS, AHEAD = each < 16 ? each : 16;   // loads in flight
    for (int n0 = 0; n0 < each; n0 += AHEAD) {
      float4 v[AHEAD];
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) {
        const int id = (n0 + n) * THREADS + threadIdx.x, i = id / quads, j = (id % quads) * 4;
        v[n] = i < rows && c0 + j < width ? *reinterpret_cast<const float4 *>(from + i * width + c0 + j)
                                          : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) {
        const int id = (n0 + n) * THREADS + threadIdx.x, i = id / quads, j = (id % quads) * 4;
        *reinterpret_cast<uint2 *>(tile + i * L + j) = make_uint2(packPair(v[n].x, v[n].y), packPair(v[n].z, v[n].w));
      }
    }
  } else {
    for (int id = threadIdx.x; id < DK * D; id += THREADS) {
      const int i = id / D, j = id % D;
      tile[i * L + j] = fromFloat<bf16>(i < rows && c0 + j < width ? from[i * width + c0 + j] : 0.f);
    }
  }
}

// The warp's slice of a float32 state: row tiles of 16 from m0 on by column tiles
// of 8 from n0 on (of those from column c0 of the state on).
template <int SM, int SN>
__device__ __forceinline__ void readSlice(float (&S)[SM][SN][4], const float *from, int m0, int n0, int c0, int rows,
                                          int width) {
  const int lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
#pragma unroll
  for (int m = 0; m < SM; ++m)
#pragma unroll
    for (int n = 0; n < SN; ++n)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int i = (m0 + m) * 16 + g + y * 8, j = c0 + (n0 + n) * 8 + 2 * tq;
        float2 v = make_float2(0.f, 0.f);
        if (from && i < rows) {
          const float *at = from + int64_t(i) * width + j;
          if (width % 2 == 0) {
            if (j < width) v = *reinterpret_cast<const float2 *>(at);
          } else {
            if (j < width) v.x = at[0];
            if (j + 1 < width) v.y = at[1];
          }
        }
        S[m][n][2 * y] = v.x;
        S[m][n][2 * y + 1] = v.y;
      }
}
template <int SM, int SN>
__device__ __forceinline__ void writeSlice(float *to, const float (&S)[SM][SN][4], int m0, int n0, int c0, int rows,
                                           int width) {
  const int lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
#pragma unroll
  for (int m = 0; m < SM; ++m)
#pragma unroll
    for (int n = 0; n < SN; ++n)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int i = (m0 + m) * 16 + g + y * 8, j = c0 + (n0 + n) * 8 + 2 * tq;
        if (i >= rows) continue;
        float *at = to + int64_t(i) * width + j;
        if (width % 2 == 0) {
          if (j < width) *reinterpret_cast<float2 *>(at) = make_float2(S[m][n][2 * y], S[m][n][2 * y + 1]);
        } else {
          if (j < width) at[0] = S[m][n][2 * y];
          if (j + 1 < width) at[1] = S[m][n][2 * y + 1];
        }
      }
}
// ... and its bfloat16 copy in a tile with rows of L.
template <int L, int SM, int SN>
__device__ __forceinline__ void copySlice(bf16 *tile, const float (&S)[SM][SN][4], int m0, int n0) {
#pragma unroll
  for (int m = 0; m < SM; ++m)
#pragma unroll
    for (int n = 0; n < SN; n += 2) {
      const uint32_t p[4] = {packPair(S[m][n][0], S[m][n][1]), packPair(S[m][n][2], S[m][n][3]),
                             packPair(S[m][n + 1][0], S[m][n + 1][1]), packPair(S[m][n + 1][2], S[m][n + 1][3])};
      storeMatrices<L>(tile, (m0 + m) * 16, (n0 + n) * 8, p);
    }
}

// Shared memory of a block: tiles in `buffers` copies.
template <int C, int DK, int DV, bool OUT> constexpr int chunkTileElements() {
  return C * (DK + 8) * (OUT ? 2 : 1) + C * (DV + 8);
}
template <int C, int DK, int DV, bool OUT> constexpr int chunkSharedBytes(int buffers) {
  return buffers * (chunkTileElements<C, DK, DV, OUT>() + (OUT ? DK * (DV + 8) : 0)) * 2 + 4 * (3 * C + 21);
}

// One block per (environment, head), segment of T and tile of DV columns; C / 16
// warps.  OUT = false computes the state at the segment's end only; STATE = false
// is for one chunk whose last state nobody wants.
template <int C, int DK, int DV, bool OUT, bool STATE>
__global__ void __launch_bounds__(C * 2, (DK == 128 ? 128 : STATE ? 192 : 256) / C)
    attentionChunks(ChunkArgs p, int buffers) {
  constexpr int N = DV / 8;                                    // column tiles of the outputs
  constexpr int W = C / 16, THREADS = W * 32, LQ = DK + 8, LV = DV + 8;
  constexpr int RT = DK / 16;                                  // row tiles of the state
  constexpr int SM = RT >= W ? RT / W : 1;                     // of which a warp has
  constexpr int SPLIT = RT >= W ? 1 : W / RT;                  // warps that share a row tile
  constexpr int SN = DV / 8 / SPLIT;                           // tiles of 8 columns of a warp's slice
  static_assert(SN % 2 == 0, "operands of the state come two column tiles at a time");
  extern __shared__ __align__(16) unsigned char shared[];
  bf16 *tiles = reinterpret_cast<bf16 *>(shared);
  bf16 *copies = tiles + buffers * chunkTileElements<C, DK, DV, OUT>();      // the state in bfloat16
  float *toEnd = reinterpret_cast<float *>(copies + (OUT ? buffers * DK * LV : 0));   // l^(L - 1 - j)
  float *powers = toEnd + C;                                                  // scale l^(x - 16), 0 for x < 16
  float *decays = powers + C + 20;                                            // l^x, x up to C

  const int64_t eh = blockIdx.x;
  const int e = int(eh / p.H), h = int(eh - int64_t(e) * p.H);
  const int seg = blockIdx.y / p.columnTiles, col0 = (blockIdx.y - seg * p.columnTiles) * DV;
  const int t0 = seg * p.segmentLength, t1 = min(p.T, t0 + p.segmentLength);
  const int chunks = (t1 - t0 + C - 1) / C;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, tq = lane & 3;
  const bf16 *q = p.q + e * p.qs.e + h * p.qs.h, *k = p.k + e * p.ks.e + h * p.ks.h, *v = p.v + e * p.vs.e + h * p.vs.h;
  const int64_t stateSize = int64_t(p.Dk) * p.Dv;
  const float *init = p.segments && OUT ? p.segments + (eh * p.segmentCount + seg) * stateSize
                      : p.stateIn && !p.segments ? p.stateIn + eh * stateSize : nullptr;
  float *last = !OUT ? p.segments + (eh * p.segmentCount + seg) * stateSize
                : p.stateOut && seg == p.segmentCount - 1 ? p.stateOut + eh * stateSize : nullptr;

  auto load = [&](int c, int buffer) {
    bf16 *tile = tiles + buffer * chunkTileElements<C, DK, DV, OUT>();
    const int first = t0 + c * C, count = min(C, t1 - first);
    loadTile<C, DK, THREADS>(tile, k, p.ks.t, first, count, 0, p.Dk, p.vecK);
    loadTile<C, DV, THREADS>(tile + C * LQ, v, p.vs.t, first, count, col0, p.Dv, p.vecV);
    if (OUT) loadTile<C, DK, THREADS>(tile + C * (LQ + LV), q, p.qs.t, first, count, 0, p.Dk, p.vecQ);
    commitCopies();
  };
  load(0, 0);
  Resets resets;
  resets.read(p.resets, p.E, e, t0, min(t1, t0 + C));

  // The warp's slice of the state, and its copy.
  const int sm0 = RT >= W ? warp * SM : warp / SPLIT, sn0 = RT >= W ? 0 : (warp % SPLIT) * SN;
  float S[SM][SN][4];
  if (STATE) {
    readSlice(S, init, sm0, sn0, col0, p.Dk, p.Dv);
    if (OUT) copySlice<LV>(copies, S, sm0, sn0);
  } else if (init) {
    loadState<DK, DV, THREADS>(copies, init, p.Dk, col0, p.Dv);
  }

  // Powers of the decay.
  const float decay = p.decay[h];
  for (int x = threadIdx.x; x < C + 20; x += THREADS) {
    const int n = x - 16;
    const float f = powerOf(decay, n < 0 ? 0 : n);
    powers[x] = n < 0 ? 0.f : p.scale * f;
    if (n >= 0 && n <= C) decays[n] = f;
    if (n >= 0 && n < C) toEnd[C - 1 - n] = f;
  }
  const int i0 = 16 * warp;   // the warp's steps
  const float fullChunk = powerOf(decay, C);

  uint32_t finite = 0;
  bool anyReset = false, later = init != nullptr;   // later: S is not zero
  for (int c = 0; c < chunks; ++c) {
    const int buffer = buffers > 1 ? c & 1 : 0, first = t0 + c * C, count = min(C, t1 - first);
    const unsigned long long mask = resets.mask();
    anyReset |= mask != 0;
    if (STATE && buffers == 1 && c > 0) {
      __syncthreads();   // the tiles and the copy of the state are free
      if (OUT) copySlice<LV>(copies, S, sm0, sn0);
      load(c, 0);
    }
    waitCopies();
    __syncthreads();
    if (c + 1 < chunks) {
      if (buffers > 1) load(c + 1, (c + 1) & 1);
      resets.read(p.resets, p.E, e, first + C, min(t1, first + 2 * C));
    }
    const bf16 *K = tiles + buffer * chunkTileElements<C, DK, DV, OUT>(), *V = K + C * LQ, *Q = V + C * LV;
    if (STATE && count < C)
      for (int x = threadIdx.x; x < C; x += THREADS) toEnd[x] = x < count ? decays[count - 1 - x] : 0.f;

    const bool advance = STATE && (c + 1 < chunks || last);
    const bf16 *copy = copies + buffer * DK * LV;
    if (OUT && STATE && p.saved) {
      const int chunk = seg * (p.segmentLength / C) + c;
      bf16 *to = p.saved + (eh * ((p.T + C - 1) / C) + chunk) * stateSize + col0;
      if (chunk == 0) {
        // the caller has it
      } else if (p.Dv % 8 == 0) {
#pragma unroll
        for (int x = threadIdx.x; x < DK * DV / 8; x += THREADS) {
          const int i = x / (DV / 8), j = x % (DV / 8) * 8;
          if (i < p.Dk && col0 + j < p.Dv)
            *reinterpret_cast<uint4 *>(to + i * p.Dv + j) = *reinterpret_cast<const uint4 *>(copy + i * LV + j);
        }
      } else {
        for (int x = threadIdx.x; x < p.Dk * DV; x += THREADS)
          if (col0 + x % DV < p.Dv) to[x / DV * p.Dv + x % DV] = copy[x / DV * LV + x % DV];
      }
    }
    const int start0 = episodeStart(mask, i0 + g), start1 = episodeStart(mask, i0 + g + 8);
    const int lowest = episodeStart(mask, i0), highest = episodeStart(mask, i0 + 15);   // of the warp's steps
    const int start = episodeStart(mask, 63);   // the state after the chunk sees the steps from there on
    uint32_t a[DK / 16][4];
    float o[N][4];
    if (OUT) {
#pragma unroll
      for (int kk = 0; kk < DK / 16; ++kk) operandA<LQ>(a[kk], Q, i0, kk * 16);
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[n][x] = 0.f;
      if (later && lowest < 0) {   // Q S
#pragma unroll
        for (int kk = 0; kk < DK / 16; ++kk)
#pragma unroll
          for (int n = 0; n < N / 2; ++n) {
            uint32_t b[4];
            operandBTransposed<LV>(b, copy, kk * 16, n * 16);
            multiplyAdd(o[2 * n], a[kk], b[0], b[1]);
            multiplyAdd(o[2 * n + 1], a[kk], b[2], b[3]);
          }
        const float f0 = powers[16 + i0 + g + 1], f1 = powers[16 + i0 + g + 9];
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[n][x] *= x < 2 ? f0 : f1;
        if (highest >= 0) {
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[n][x] = (x < 2 ? start0 : start1) < 0 ? o[n][x] : 0.f;
        }
      }
    }
    if (OUT) {
#pragma unroll
      for (int block = 0; block < C / 16; ++block) {   // of 16 steps
        if (block > warp) break;
        float s[2][4] = {};
#pragma unroll
        for (int kk = 0; kk < DK / 16; ++kk) {
          uint32_t b[4];
          operandB<LQ>(b, K, block * 16, kk * 16);
          multiplyAdd(s[0], a[kk], b[0], b[1]);
          multiplyAdd(s[1], a[kk], b[2], b[3]);
        }
        const float *f = powers + 16 + i0 - block * 16 + g - 2 * tq;   // of the distance i - j, 0 below zero
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[n][x] *= f[(x >> 1) * 8 - (x & 1) - n * 8];
        if (block * 16 < highest) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (block * 16 + 2 * tq + n * 8 + (x & 1) < (x < 2 ? start0 : start1)) s[n][x] = 0.f;
        }
        const uint32_t w[4] = {packPair(s[0][0], s[0][1]), packPair(s[0][2], s[0][3]), packPair(s[1][0], s[1][1]),
                               packPair(s[1][2], s[1][3])};
#pragma unroll
        for (int n = 0; n < N / 2; ++n) {
          uint32_t b[4];
          operandBTransposed<LV>(b, V, block * 16, n * 16);
          multiplyAdd(o[2 * n], w, b[0], b[1]);
          multiplyAdd(o[2 * n + 1], w, b[2], b[3]);
        }
      }
      // The warp has its rows of Q for itself and is done with them.
      bf16 *out = p.out + eh * p.Dv;
      const int64_t stepStride = int64_t(p.E) * p.H * p.Dv;
      if constexpr (DV <= DK)
        storeTileStaged<DK>(out, const_cast<bf16 *>(Q) + i0 * LQ, o, stepStride, first, count, i0, col0, p.Dv, finite);
      else storeTile(out, o, stepStride, first, count, i0, col0, p.Dv, finite);
    }

    // The state at the chunk's end.
    if (advance) {
      if (count < C) __syncthreads();   // toEnd
      const float f = count == C ? fullChunk : decays[count];
#pragma unroll
      for (int m = 0; m < SM; ++m)
#pragma unroll
        for (int n = 0; n < SN; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) S[m][n][x] *= f;
      if (start >= 0) {
#pragma unroll
        for (int m = 0; m < SM; ++m)
#pragma unroll
          for (int n = 0; n < SN; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) S[m][n][x] = 0.f;
      }
      auto add = [&](auto terms) {   // without a branch among the products
        constexpr int TERMS = decltype(terms)::value;
#pragma unroll
      for (int block = 0; block < C / 16; ++block) {
        const int j = block * 16 + 2 * tq;
        float2 f0 = *reinterpret_cast<const float2 *>(toEnd + j), f1 = *reinterpret_cast<const float2 *>(toEnd + j + 8);
        if (mask) {
          f0.x = j >= start ? f0.x : 0.f;
          f0.y = j + 1 >= start ? f0.y : 0.f;
          f1.x = j + 8 >= start ? f1.x : 0.f;
          f1.y = j + 9 >= start ? f1.y : 0.f;
        }
        uint32_t part[SM][TERMS][4];
#pragma unroll
        for (int m = 0; m < SM; ++m) {
          uint32_t kt[4];
          operandATransposed<LQ>(kt, K, (sm0 + m) * 16, block * 16);
#pragma unroll
          for (int x = 0; x < 4; ++x)   // registers 0, 1: steps 2 tq, + 1; registers 2, 3: 8 later
            splitPair<TERMS>(part[m], x, lowOf(kt[x]) * (x < 2 ? f0.x : f1.x), highOf(kt[x]) * (x < 2 ? f0.y : f1.y));
        }
#pragma unroll
        for (int n = 0; n < SN / 2; ++n) {
          uint32_t b[4];
          operandBTransposed<LV>(b, V, block * 16, (sn0 + 2 * n) * 8);
#pragma unroll
          for (int m = 0; m < SM; ++m)
#pragma unroll
            for (int t = 0; t < TERMS; ++t) {
              multiplyAdd(S[m][2 * n], part[m][t], b[0], b[1]);
              multiplyAdd(S[m][2 * n + 1], part[m][t], b[2], b[3]);
            }
        }
      }
      };
      if (p.precise && (!OUT || last)) add(std::integral_constant<int, 3>());   // it reaches the last state
      else add(std::integral_constant<int, 2>());
      later = true;
      if (OUT && buffers > 1 && c + 1 < chunks) copySlice<LV>(copies + ((c + 1) & 1) * DK * LV, S, sm0, sn0);
    }
  }
  bool bad = (finite & 0x7fff7fffu) != 0;   // NaN
  if (STATE && last) {
    writeSlice(last, S, sm0, sn0, col0, p.Dk, p.Dv);
#pragma unroll
    for (int m = 0; m < SM; ++m) bad |= notFinite(S[m]);
  }
  if (!OUT && col0 == 0 && threadIdx.x == 0) p.segmentCut[eh * p.segmentCount + seg] = anyReset;
  if (OUT) {
    const bool redo = __syncthreads_or(bad);
    if (threadIdx.x == 0) p.flags[eh * gridDim.y + blockIdx.y] = redo;
  }
}

using Forwards = std::integral_constant<int, 1>;
using Backwards = std::integral_constant<int, -1>;

// Operands and arrays of a backward call.
struct BackwardArgs {
  const bf16 *q, *k, *v, *dout;
  bf16 *dq, *dk, *dv;          // dense
  Rows qs, ks, vs, os;
  const float *decay;
  const uint8_t *resets;
  const float *stateIn, *dstateOut;
  float *dstateIn;
  const bf16 *saved;           // the state before each chunk but the first
  float *segments;             // [E, H, segmentCount, Dk, Dv]: gradient of the state after each segment, or null
  uint8_t *segmentCut;
  uint8_t *flags;              // [E, H, segmentCount]
  int T, E, H, Dk, Dv;
  int segmentLength, segmentCount;
  int vecQ, vecK, vecV, vecO;
  int precise;                 // the gradient of the state is an output
  float scale;
};

template <int C, int D, bool OUT> constexpr int backwardWarps() { return OUT && D == 128 ? C / 8 : C / 16; }
// Where `later` states' gradients never exist, no room for X.
template <int C, int D, bool OUT> constexpr int backwardSharedBytes(bool later) {
  return (OUT ? 4 * C + (later ? 2 : 1) * D : 2 * C) * (D + 8) * 2 + (2 * C + 24) * 4;
}

// One block per (environment, head) and segment of T, chunks from the last to the
// first.  With X the gradient of the state after the chunk and S the state before
// it, steps i and j, L the chunk's length:
//
//   dq_i = scale [ l^(i+1) S do_i + sum_{j <= i} l^(i-j) (do_i . v_j) k_j ]
//   dk_j = l^(L-1-j) X v_j   + scale sum_{i >= j} l^(i-j) (v_j . do_i) q_i
//   dv_j = l^(L-1-j) X^T k_j + scale sum_{i >= j} l^(i-j) (k_j . q_i) do_i
//   X'   = l^L X + scale sum_i l^(i+1) q_i do_i^T
//
// S comes from the forward pass in bfloat16, X stays in registers in float32 as
// S does there, with the same split of its operand.  Each of the three outputs
// takes its scores from products of its own, in the layout in which they are the
// next product's operand: six instead of five products of C x C x D, and no score
// passes through shared memory.  OUT = false: X' of a segment alone.
// STATE = false is for one chunk whose first state's gradient nobody wants.
template <int C, int D, bool OUT, bool STATE>
__global__ void __launch_bounds__(backwardWarps<C, D, OUT>() * 32, (D == 128 ? 64 : STATE && C == 32 ? 192 : 256) / C)
    attentionChunksBackward(BackwardArgs p) {
  constexpr int W = backwardWarps<C, D, OUT>(), THREADS = W * 32, LD = D + 8;
  constexpr int PARTS = W / (C / 16);                          // warps that share 16 rows of the outputs
  constexpr int N = D / 8 / PARTS;                             // tiles of 8 columns of a warp's outputs
  constexpr int RT = D / 16, SM = RT >= W ? RT / W : 1, SPLIT = RT >= W ? 1 : W / RT, SN = D / 8 / SPLIT;
  extern __shared__ __align__(16) unsigned char shared[];
  float *powers = reinterpret_cast<float *>(shared);   // scale l^(x - 16), 0 for x < 16; C + 20 of them
  float *decays = powers + C + 20;                     // l^x, x up to C; C + 4 of them, for the tiles' alignment
  bf16 *Q = reinterpret_cast<bf16 *>(decays + C + 4), *O = Q + C * LD, *K = O + C * LD, *V = K + C * LD, *S = V + C * LD,
       *X = S + D * LD;
  const int64_t eh = blockIdx.x;
  const int e = int(eh / p.H), h = int(eh - int64_t(e) * p.H), seg = OUT ? blockIdx.y : blockIdx.y + 1;
  const int t0 = seg * p.segmentLength, t1 = min(p.T, t0 + p.segmentLength);
  const int chunks = (t1 - t0 + C - 1) / C, allChunks = (p.T + C - 1) / C;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, tq = lane & 3;
  const int row = (warp / PARTS) * 16, col = (warp % PARTS) * N * 8;
  const bf16 *q = p.q + e * p.qs.e + h * p.qs.h, *o = p.dout + e * p.os.e + h * p.os.h;
  const bf16 *k = p.k + e * p.ks.e + h * p.ks.h, *v = p.v + e * p.vs.e + h * p.vs.h;
  const int64_t stateSize = int64_t(p.Dk) * p.Dv;
  const float *init = p.segments ? (OUT ? p.segments + (eh * p.segmentCount + seg) * stateSize : nullptr)
                                 : p.dstateOut ? p.dstateOut + eh * stateSize : nullptr;
  float *last = !OUT ? p.segments + (eh * p.segmentCount + seg) * stateSize
                : p.dstateIn && seg == 0 ? p.dstateIn + eh * stateSize : nullptr;

  const float decay = p.decay[h];
  for (int x = threadIdx.x; x < C + 20; x += THREADS) {
    const int n = x - 16;
    const float f = powerOf(decay, n < 0 ? 0 : n);
    powers[x] = n < 0 ? 0.f : p.scale * f;
    if (n >= 0) decays[n] = f;
  }
  const bool precise = p.precise && (!OUT || last);   // what this block adds reaches the first state's gradient
  const int sm0 = RT >= W ? warp * SM : warp / SPLIT, sn0 = RT >= W ? 0 : (warp % SPLIT) * SN;
  float dS[SM][SN][4];
  if (STATE) readSlice(dS, init, sm0, sn0, 0, p.Dk, p.Dv);

  uint32_t finite = 0;
  bool anyReset = false, later = init != nullptr;   // later: X is not zero
  for (int c = chunks - 1; c >= 0; --c) {
    const int first = t0 + c * C, count = min(C, t1 - first);
    loadTile<C, D, THREADS>(Q, q, p.qs.t, first, count, 0, p.Dk, p.vecQ);
    loadTile<C, D, THREADS>(O, o, p.os.t, first, count, 0, p.Dv, p.vecO);
    const int chunk = seg * (p.segmentLength / C) + c;
    const bool earlier = OUT && (chunk > 0 || p.stateIn);          // S is not zero
    if (OUT) {
      loadTile<C, D, THREADS>(K, k, p.ks.t, first, count, 0, p.Dk, p.vecK);
      loadTile<C, D, THREADS>(V, v, p.vs.t, first, count, 0, p.Dv, p.vecV);
      if (chunk > 0) {
        loadTile<D, D, THREADS>(S, p.saved + (eh * allChunks + chunk) * stateSize, p.Dv, 0, p.Dk, 0, p.Dv,
                                p.Dv % 8 == 0);
      } else if (p.stateIn) {
        loadState<D, D, THREADS>(S, p.stateIn + eh * stateSize, p.Dk, 0, p.Dv);
      }
      if (STATE) {
        if (later) copySlice<LD>(X, dS, sm0, sn0);
      } else if (init) {
        loadState<D, D, THREADS>(X, init, p.Dk, 0, p.Dv);
      }
    }
    commitCopies();
    Resets resets;
    resets.read(p.resets, p.E, e, first, min(t1, first + C));
    const unsigned long long mask = resets.mask();
    anyReset |= mask != 0;
    waitCopies();
    __syncthreads();
    const int endStart = episodeStart(mask, 63);   // the state after the chunk sees the steps from there on

    if (OUT) {
      const int blockRow = row / 16, blocks = (count + 15) / 16;
      uint32_t a[D / 16][4];
      float out[N][4];
      // The scores of the warp's rows with a block of 16 other steps, times their decays; `sign` 1: the rows are
      // the later steps.
      const int start0 = episodeStart(mask, row + g), start1 = episodeStart(mask, row + g + 8);
      const int end0 = episodeEnd(mask, row + g), end1 = episodeEnd(mask, row + g + 8);
      auto weights = [&](uint32_t (&w)[4], const bf16 *other, int block, auto sign_) {
        constexpr int sign = decltype(sign_)::value;
        float s[2][4] = {};
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t b[4];
          operandB<LD>(b, other, block * 16, kk * 16);
          multiplyAdd(s[0], a[kk], b[0], b[1]);
          multiplyAdd(s[1], a[kk], b[2], b[3]);
        }
        const float *f = powers + 16 + sign * (row - block * 16 + g - 2 * tq);
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[n][x] *= f[sign * ((x >> 1) * 8 - (x & 1) - n * 8)];
        if (mask) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int at = block * 16 + n * 8 + 2 * tq + (x & 1);
              if (sign > 0 ? at < (x < 2 ? start0 : start1) : at >= (x < 2 ? end0 : end1)) s[n][x] = 0.f;
            }
        }
        w[0] = packPair(s[0][0], s[0][1]);
        w[1] = packPair(s[0][2], s[0][3]);
        w[2] = packPair(s[1][0], s[1][1]);
        w[3] = packPair(s[1][2], s[1][3]);
      };
      auto accumulate = [&](const uint32_t (&w)[4], const bf16 *rows, int block) {
#pragma unroll
        for (int n = 0; n < N / 2; ++n) {
          uint32_t b[4];
          operandBTransposed<LD>(b, rows, block * 16, col + n * 16);
          multiplyAdd(out[2 * n], w, b[0], b[1]);
          multiplyAdd(out[2 * n + 1], w, b[2], b[3]);
        }
      };
      auto rowsOfA = [&](const bf16 *x) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) operandA<LD>(a[kk], x, row, kk * 16);
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) out[n][x] = 0.f;
      };
      auto scaleRows = [&](float f0, float f1) {   // a factor of zero replaces
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) out[n][x] *= x < 2 ? f0 : f1;
        if (mask || count < C) {
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) out[n][x] = (x < 2 ? f0 : f1) == 0.f ? 0.f : out[n][x];
        }
      };
      const int64_t stepK = int64_t(p.E) * p.H * p.Dk, stepV = int64_t(p.E) * p.H * p.Dv;
      if (row < count) {
        // dq
        rowsOfA(O);
        if (earlier) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int n = 0; n < N / 2; ++n) {
              uint32_t b[4];
              operandB<LD>(b, S, col + n * 16, kk * 16);
              multiplyAdd(out[2 * n], a[kk], b[0], b[1]);
              multiplyAdd(out[2 * n + 1], a[kk], b[2], b[3]);
            }
          scaleRows(start0 < 0 ? powers[16 + row + g + 1] : 0.f, start1 < 0 ? powers[16 + row + g + 9] : 0.f);
        }
        for (int block = 0; block <= blockRow; ++block) {
          uint32_t w[4];
          weights(w, V, block, Forwards());
          accumulate(w, K, block);
        }
        storeTile(p.dq + eh * p.Dk, out, stepK, first, count, row, col, p.Dk, finite);
        // dv, dk
        const int left0 = count - 1 - row - g, left1 = left0 - 8;
        const float f0 = row + g >= endStart && left0 >= 0 ? decays[left0] : 0.f;
        const float f1 = row + g + 8 >= endStart && left1 >= 0 ? decays[left1] : 0.f;
        rowsOfA(K);
        if (later) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int n = 0; n < N / 2; ++n) {
              uint32_t b[4];
              operandBTransposed<LD>(b, X, kk * 16, col + n * 16);
              multiplyAdd(out[2 * n], a[kk], b[0], b[1]);
              multiplyAdd(out[2 * n + 1], a[kk], b[2], b[3]);
            }
          scaleRows(f0, f1);
        }
        for (int block = blockRow; block < blocks; ++block) {
          uint32_t w[4];
          weights(w, Q, block, Backwards());
          accumulate(w, O, block);
        }
        storeTile(p.dv + eh * p.Dv, out, stepV, first, count, row, col, p.Dv, finite);
        rowsOfA(V);
        if (later) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int n = 0; n < N / 2; ++n) {
              uint32_t b[4];
              operandB<LD>(b, X, col + n * 16, kk * 16);
              multiplyAdd(out[2 * n], a[kk], b[0], b[1]);
              multiplyAdd(out[2 * n + 1], a[kk], b[2], b[3]);
            }
          scaleRows(f0, f1);
        }
        for (int block = blockRow; block < blocks; ++block) {
          uint32_t w[4];
          weights(w, O, block, Backwards());
          accumulate(w, Q, block);
        }
        storeTile(p.dk + eh * p.Dk, out, stepK, first, count, row, col, p.Dk, finite);
      }
    }

    if (STATE && (c > 0 || last)) {
      const int firstReset = episodeEnd(mask, 0);   // of the steps after 0
      const float f = decays[count];
#pragma unroll
      for (int m = 0; m < SM; ++m)
#pragma unroll
        for (int n = 0; n < SN; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) dS[m][n][x] *= f;
      if (endStart >= 0) {
#pragma unroll
        for (int m = 0; m < SM; ++m)
#pragma unroll
          for (int n = 0; n < SN; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) dS[m][n][x] = 0.f;
      }
      auto add = [&](auto terms) {
        constexpr int TERMS = decltype(terms)::value;
      for (int kk = 0; kk < (count + 15) / 16; ++kk) {
        float w[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int i = kk * 16 + 2 * tq + (x & 1) + (x >> 1) * 8;
          w[x] = !(mask & 1) && i < firstReset ? powers[16 + i + 1] : 0.f;
        }
        uint32_t part[SM][TERMS][4];
#pragma unroll
        for (int m = 0; m < SM; ++m) {
          uint32_t a[4];
          operandATransposed<LD>(a, Q, (sm0 + m) * 16, kk * 16);
#pragma unroll
          for (int x = 0; x < 4; ++x)
            splitPair<TERMS>(part[m], x, lowOf(a[x]) * w[(x >> 1) * 2], highOf(a[x]) * w[(x >> 1) * 2 + 1]);
        }
#pragma unroll
        for (int n = 0; n < SN / 2; ++n) {
          uint32_t b[4];
          operandBTransposed<LD>(b, O, kk * 16, (sn0 + 2 * n) * 8);
#pragma unroll
          for (int m = 0; m < SM; ++m)
#pragma unroll
            for (int t = 0; t < TERMS; ++t) {
              multiplyAdd(dS[m][2 * n], part[m][t], b[0], b[1]);
              multiplyAdd(dS[m][2 * n + 1], part[m][t], b[2], b[3]);
            }
        }
      }
      };
      if (precise) add(std::integral_constant<int, 3>());
      else add(std::integral_constant<int, 2>());
      later = true;
      __syncthreads();   // the tiles and X are free
    }
  }
  bool bad = (finite & 0x7fff7fffu) != 0;   // NaN
  if (STATE && last) {
    writeSlice(last, dS, sm0, sn0, 0, p.Dk, p.Dv);
#pragma unroll
    for (int m = 0; m < SM; ++m) bad |= notFinite(dS[m]);
  }
  if (!OUT && threadIdx.x == 0) p.segmentCut[eh * p.segmentCount + seg] = anyReset;
  if (OUT) {
    const bool redo = __syncthreads_or(bad);
    if (threadIdx.x == 0) p.flags[eh * p.segmentCount + seg] = redo;
  }
}

// States at the segments' ends that a sweep enters them by, from what each
// segment adds, in place: forwards in time from `init`, or backwards.  The
// last segment of the sweep adds nothing that is needed.
__global__ void __launch_bounds__(256) joinSegments(float *segments, const uint8_t *cut, const float *init,
                                                    const float *decay, int H, int T, int segmentCount,
                                                    int segmentLength, int64_t stateSize, int reverse) {
  const int64_t eh = blockIdx.x, x = int64_t(blockIdx.y) * blockDim.x + threadIdx.x;
  if (x >= stateSize) return;
  const float d = decay[eh % H], whole = powerOf(d, segmentLength);
  float S = init ? init[eh * stateSize + x] : 0.f;
  float *states = segments + eh * segmentCount * stateSize + x;
  constexpr int AHEAD = 8;   // loads in flight: the chain itself is a multiplication a segment
  for (int u0 = 0; u0 < segmentCount; u0 += AHEAD) {
    float added[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int u = u0 + k, s = reverse ? segmentCount - 1 - u : u;
      added[k] = u + 1 < segmentCount ? states[s * stateSize] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int u = u0 + k, s = reverse ? segmentCount - 1 - u : u;
      if (u >= segmentCount) break;
      states[s * stateSize] = S;
      if (u + 1 == segmentCount) break;
      const int length = min(segmentLength, T - s * segmentLength);
      const float f = length == segmentLength ? whole : powerOf(d, length);
      S = cut[eh * segmentCount + s] ? added[k] : fmaf(f, S, added[k]);
    }
  }
}

// Sweeps of a call step by step, for the environments and heads that have one of
// their `count` flags set; usually none has (2.4 us).  A block has a run of them and
// looks at all its flags at once first.  Where many are set this is slow, one head
// after the other: 24 steps of 4096 environments, 4 heads of 64, forward and backward,
// 149 us a call with none, 343 us with one environment, 11.2 ms with all.
template <int DI>
__global__ void __launch_bounds__(scanThreads(DI))
    redoAttention(const __grid_constant__ Sweeps p, const uint8_t *flags, int count) {
  const Sweep &s = p.s[blockIdx.z];
  const int64_t all = int64_t(s.E) * s.H, run = (all + gridDim.x - 1) / gridDim.x;
  const int64_t first = blockIdx.x * run, end = min(all, first + run);
  bool any = false;
  for (int64_t x = first * count + threadIdx.x; x < end * count; x += blockDim.x) any |= flags[x] != 0;
  if (!__syncthreads_or(any)) return;
  for (int64_t eh = first; eh < end; ++eh) {
    any = false;
    for (int x = threadIdx.x; x < count; x += blockDim.x) any |= flags[eh * count + x] != 0;
    if (__syncthreads_or(any)) scanSteps<bf16, DI, true, true>(s, eh, blockIdx.y, 0);
  }
}

}  // namespace duckb200
