// sym_b200 -- shared-memory barriers with bounded waits, and the encoding of
// tensor maps: what every kernel that is fed by asynchronous copies uses.
#pragma once

#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <atomic>
#include <cstdint>

namespace sbc {

/// Launch counters and the wait limit of this library (defined in
/// relocate.cu; sbc_launch_count, sbc_wait_launch_count,
/// sbc_set_wait_limit_ns).
void count_launch();
void count_wait_launch();
uint64_t wait_limit_ns();

/// Lets a kernel use `bytes` of dynamic shared memory (the same number in every
/// call for a kernel) on the current device; the driver is asked once per
/// kernel and device.
template <auto KERNEL> cudaError_t allow_shared(int bytes) {
  static std::atomic<bool> allowed[64];
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess || (device < 64 && allowed[device].load(std::memory_order_relaxed)))
    return e;
  e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && device < 64)
    allowed[device].store(true, std::memory_order_relaxed);
  return e;
}

/// A tiled tensor map (unit element strides, what lies past the end reads as
/// 0); false where the driver lacks or refuses it. May be a thread's first CUDA
/// call.
bool encode_tiled(CUtensorMap *map, CUtensorMapDataType type, uint32_t rank, const void *base, const cuuint64_t *dims,
                  const cuuint64_t *strides, const cuuint32_t *box, CUtensorMapSwizzle swizzle);

__device__ __forceinline__ uint32_t smem_addr(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void mbar_init(uint64_t *bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}

__device__ __forceinline__ void mbar_expect_tx(uint64_t *bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes)
               : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

__device__ __forceinline__ uint64_t global_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

__device__ __forceinline__ bool mbar_try(uint32_t a, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
               " selp.u32 %0, 1, 0, p;\n}"
               : "=r"(done)
               : "r"(a), "r"(parity)
               : "memory");
  return done != 0;
}

/// Wait for `parity` for at most `limit_ns` of the global timer (read only
/// once the first poll failed); true when the phase completed.
__device__ __forceinline__ bool mbar_wait(uint64_t *bar, uint32_t parity, uint64_t limit_ns) {
  const uint32_t a = smem_addr(bar);
  if (mbar_try(a, parity))
    return true;
  const uint64_t t0 = global_ns();
  for (;;) {
    if (mbar_try(a, parity))
      return true;
    if (global_ns() - t0 > limit_ns)
      return false;
  }
}

/// The same for kernels whose latency counts: the global timer is read only
/// once in 64 failed polls, each of which sleeps for a while by itself.
__device__ __forceinline__ bool mbar_wait_often(uint64_t *bar, uint32_t parity, uint64_t limit_ns) {
  const uint32_t a = smem_addr(bar);
  uint64_t t0 = 0;
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (mbar_try(a, parity))
        return true;
    const uint64_t now = global_ns();
    if (t0 == 0)
      t0 = now;
    else if (now - t0 > limit_ns)
      return false;
  }
}

} // namespace sbc
