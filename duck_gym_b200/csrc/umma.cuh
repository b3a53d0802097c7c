// The pieces of a matrix product on the fifth-generation tensor cores: copies of
// tiles by the TMA, mbarriers, tensor memory, and products of bfloat16 tiles that
// are accumulated there in float32.
//
// Every wait has a limit.  A thread whose wait runs out says so in `broken`, which
// ends the others' waits; a kernel then marks its outputs as not computed, waits for
// the copies and products that it has begun (with kWaitLimit), and ends as it would
// otherwise.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace duckb200 {

__device__ __forceinline__ uint32_t sharedAddress(const void *p) { return uint32_t(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void barrierInit(uint64_t *bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(sharedAddress(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void barrierExpect(uint64_t *bar, int bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(sharedAddress(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void barrierArrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(sharedAddress(bar)) : "memory");
}
__device__ __forceinline__ bool barrierTry(uint64_t *bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(sharedAddress(bar)), "r"(parity)
      : "memory");
  return done;
}
__device__ __forceinline__ uint64_t nanoseconds() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
constexpr uint64_t kWaitLimit = 2000000000;   // nanoseconds; callers may choose another one
constexpr uint64_t kLookAgain = 10000000;     // a thread that did not look for longer was not running
// Whether the barrier's phase came to its end; false once a wait ran out.  The time
// that the GPU was taken away from the kernel does not count.
__device__ __forceinline__ bool barrierWait(uint64_t *bar, uint32_t parity, volatile int *broken, uint64_t limit) {
  if (barrierTry(bar, parity)) return true;
  uint64_t looked = nanoseconds(), waited = 0;
  for (;;) {
    for (int i = 0; i < 64; ++i)
      if (barrierTry(bar, parity)) return true;
    if (*broken) return false;
    const uint64_t now = nanoseconds();
    waited += min(now - looked, kLookAgain);
    looked = now;
    if (waited > limit) {
      *broken = 1;
      return false;
    }
  }
}

// The same, the loop out of line: for warps whose registers are full (da and du of 24576
// rows, 256 x 512: 41 us, 43.5 with it in line).
__device__ __noinline__ bool barrierLoop(uint64_t *bar, uint32_t parity, volatile int *broken, uint64_t limit) {
  return barrierWait(bar, parity, broken, limit);
}
__device__ __forceinline__ bool barrierAwait(uint64_t *bar, uint32_t parity, volatile int *broken, uint64_t limit) {
  return barrierTry(bar, parity) || barrierLoop(bar, parity, broken, limit);
}

// A box of the map at {x, y} into shared memory.
__device__ __forceinline__ void copyBox(void *to, const CUtensorMap *map, int x, int y, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          sharedAddress(to)),
      "l"(map), "r"(x), "r"(y), "r"(sharedAddress(bar))
      : "memory");
}
// A box from shared memory to the map's array at {x, y}; what lies beyond the array is
// left out.  The box's memory was written before fenceForCopies().
__device__ __forceinline__ void storeBox(const CUtensorMap *map, const void *from, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y),
               "r"(sharedAddress(from))
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void fenceForCopies() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// For what this thread has begun, whether others have given up or not.
__device__ __forceinline__ void barrierSettle(uint64_t *bar, uint32_t parity) {
  int none = 0;
  barrierWait(bar, parity, &none, kWaitLimit);
}
// Until this thread's stored boxes have been read, or are in memory.
__device__ __forceinline__ void storesRead() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void storesDone() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void prefetchMap(const CUtensorMap *map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// Tensor memory: `columns` (a power of two from 32 on) by one whole warp.
__device__ __forceinline__ void tensorAllocate(uint32_t *address, int columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sharedAddress(address)), "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tensorFree(uint32_t address, int columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(address), "r"(columns));
}
__device__ __forceinline__ void tensorFenceBefore() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensorFenceAfter() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Arrives at the barrier once the products issued before are done.
__device__ __forceinline__ void tensorCommit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(sharedAddress(bar))
               : "memory");
}
// 32 lanes, 16 columns of the accumulator: column i of the thread's lane in x[i].
__device__ __forceinline__ void tensorLoad16(float *x, uint32_t address) {
  uint32_t *r = reinterpret_cast<uint32_t *>(x);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(address));
}
__device__ __forceinline__ void tensorLoadWait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// What was loaded is not used before the wait: no use of a register moves over this.
template <int N> __device__ __forceinline__ void tensorLoaded(float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+f"(x[i]));
}

// Descriptors of bfloat16 operands in tiles of 128-byte rows, swizzled as the TMA
// writes them (CU_TENSOR_MAP_SWIZZLE_128B), on 1024-byte boundaries.
// A row of the operand lies along the 64 values of a tile row (`ALONG` = true: its
// steps are contiguous): groups of 8 rows are 1024 bytes apart.  Or steps are the
// tile's rows: 64 operand rows side by side, the next 64 in a tile of 64 steps, 8192
// bytes on; groups of 8 steps are 1024 bytes apart.
template <bool ALONG> __device__ __forceinline__ uint64_t operandDescriptor(uint32_t address) {
  const uint64_t lead = ALONG ? 1 : 8192 >> 4;
  return uint64_t((address & 0x3ffff) >> 4) | lead << 16 | uint64_t(1024 >> 4) << 32 | uint64_t(1) << 46 | uint64_t(2) << 61;
}
// 16 steps on.
template <bool ALONG> constexpr uint64_t kDescriptorStep = ALONG ? 32 >> 4 : 2048 >> 4;

// 128 rows by n columns, 16 steps of bfloat16, float32 accumulators.
constexpr uint32_t productShape(int n, bool aAlong, bool bAlong) {
  return 1u << 4 | 1u << 7 | 1u << 10 | uint32_t(!aAlong) << 15 | uint32_t(!bAlong) << 16 | uint32_t(n >> 3) << 17 |
         uint32_t(128 >> 4) << 24;
}
__device__ __forceinline__ void tensorProduct(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a),
      "l"(b), "r"(shape), "r"(uint32_t(add))
      : "memory");
}

}  // namespace duckb200
