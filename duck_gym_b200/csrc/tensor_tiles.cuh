// 16x8x16 bfloat16 matrix products on shared-memory tiles.  The tiles are rows
// of D + 8 elements: 16 bytes more than a multiple of 32 bytes puts the eight
// rows of an 8x8 matrix on distinct banks.
#pragma once
#include "numeric_types.cuh"

namespace duckb200 {

__device__ __forceinline__ uint32_t sharedAddress(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void loadMatrices(uint32_t (&r)[4], const bf16 *p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(sharedAddress(p))
               : "memory");
}
__device__ __forceinline__ void loadMatricesTransposed(uint32_t (&r)[4], const bf16 *p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(sharedAddress(p))
               : "memory");
}
// c += a b
__device__ __forceinline__ void multiplyAdd(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Operands of a tile X with rows `stride` apart.
// A: rows row0.., columns col0.. of X.
template <int stride> __device__ __forceinline__ void operandA(uint32_t (&a)[4], const bf16 *x, int row0, int col0) {
  const int lane = threadIdx.x & 31;
  loadMatrices(a, x + (row0 + (lane & 15)) * stride + col0 + (lane >> 4) * 8);
}
// A: the transpose of X's rows k0.. and columns m0.. (m the rows of the operand).
template <int stride>
__device__ __forceinline__ void operandATransposed(uint32_t (&a)[4], const bf16 *x, int m0, int k0) {
  const int lane = threadIdx.x & 31;
  loadMatricesTransposed(a, x + (k0 + (lane & 7) + (lane >> 4) * 8) * stride + m0 + ((lane >> 3) & 1) * 8);
}
// B for two tiles of 8 columns, X holding a row per column n of the operand: b[0..1] of n0, b[2..3] of n0 + 8.
template <int stride> __device__ __forceinline__ void operandB(uint32_t (&b)[4], const bf16 *x, int n0, int k0) {
  const int lane = threadIdx.x & 31;
  loadMatrices(b, x + (n0 + (lane & 7) + (lane >> 4) * 8) * stride + k0 + ((lane >> 3) & 1) * 8);
}
// B for two tiles of 8 columns, X holding a row per k.
template <int stride>
__device__ __forceinline__ void operandBTransposed(uint32_t (&b)[4], const bf16 *x, int k0, int n0) {
  const int lane = threadIdx.x & 31;
  loadMatricesTransposed(b, x + (k0 + (lane & 15)) * stride + n0 + (lane >> 4) * 8);
}

__device__ __forceinline__ uint32_t packPair(float low, float high) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(low, high);
  return *reinterpret_cast<const uint32_t *>(&p);
}
__device__ __forceinline__ float lowOf(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float highOf(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }

// Results of products, packed in pairs, into a tile: rows row0.. by columns col0.. (16 x 16): p[0] rows 0-7 and p[1]
// rows 8-15 of the first 8 columns, p[2] and p[3] of the second.
template <int stride>
__device__ __forceinline__ void storeMatrices(bf16 *x, int row0, int col0, const uint32_t (&p)[4]) {
  const int lane = threadIdx.x & 31;
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(
                   sharedAddress(x + (row0 + (lane & 15)) * stride + col0 + (lane >> 4) * 8)),
               "r"(p[0]), "r"(p[1]), "r"(p[2]), "r"(p[3])
               : "memory");
}
// NaN in the sum if either number of the pair is not finite.
__device__ __forceinline__ uint32_t addZeroTimes(uint32_t pair, uint32_t sum) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(pair), "r"(0u), "r"(sum));
  return d;
}

// Two numbers as the sum of N pairs of bfloat16 numbers, each the rounding of what the ones before leave.
template <int N> __device__ __forceinline__ void splitPair(uint32_t (&part)[N][4], int at, float low, float high) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    part[n][at] = packPair(low, high);
    low -= lowOf(part[n][at]);
    high -= highOf(part[n][at]);
  }
}

// 16 bytes from global to shared memory without a register; zeros where !valid
// (the address is then not read).
__device__ __forceinline__ void copyAsync16(bf16 *to, const bf16 *from, bool valid) {
  const int bytes = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(sharedAddress(to)), "l"(from), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void copyAsync16(bf16 *to, const bf16 *from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(sharedAddress(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void commitCopies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void waitCopies() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

}  // namespace duckb200
