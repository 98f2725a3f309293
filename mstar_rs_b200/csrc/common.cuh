// What the library's translation units share: bounded waits and bulk copies
// on the device, the error text and the cached device properties on the host
// (both defined in sampler.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <mutex>
#include <string>

#include "../../include/mstar_sampler.h"

namespace mstar {

// Bound on one wait for a bulk copy: 2 ms of %globaltimer (a copy of at
// most 64 KB lands within microseconds), with an iteration cap behind it.
constexpr uint64_t kWaitNs = 2000000ull;
constexpr unsigned kWaitIters = 1u << 26;

__device__ __forceinline__ uint32_t smem_u32(const void *p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}

__device__ __forceinline__ void mbar_init(uint64_t *bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}

__device__ __forceinline__ void mbar_expect_tx(uint64_t *bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)),
               "r"(bytes)
               : "memory");
}

__device__ __forceinline__ uint64_t global_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

// Bounded wait on phase `parity` (kWaitNs); false if the limit ran out.
__device__ __forceinline__ bool mbar_wait(uint64_t *bar, uint32_t parity) {
  const uint32_t a = smem_u32(bar);
  uint64_t t0 = 0;
  for (unsigned i = 0; i < kWaitIters; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(a), "r"(parity)
        : "memory");
    if (ok) return true;
    const uint64_t t = global_ns();
    if (i == 0) t0 = t;
    else if (t - t0 > kWaitNs) return false;
  }
  return false;
}

__device__ __forceinline__ void bulk_g2s(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// ------------------------------------------------------------ host side

constexpr int kMaxDevices = 64;

int fail(int code, const std::string &msg);  // keeps `msg` for mstar_sampler_last_error, returns `code`
int current_device();
int sm_count();
int max_smem_optin();

// Lets kernel K use `bytes` of dynamic shared memory on the current device;
// the runtime is asked once per device and larger size (by one thread at a time:
// a smaller size set last would undo a larger one).
template <auto K>
inline int allow_smem(int bytes) {
  static std::atomic<int> allowed[kMaxDevices];
  static std::mutex setting;
  std::atomic<int> &have = allowed[current_device()];
  if (have.load(std::memory_order_acquire) >= bytes) return MSTAR_OK;
  const std::lock_guard<std::mutex> lock(setting);
  if (have.load(std::memory_order_relaxed) >= bytes) return MSTAR_OK;
  const cudaError_t e = cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(MSTAR_ERR_CUDA, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
  have.store(bytes, std::memory_order_release);
  return MSTAR_OK;
}

int check_w4(const mstar_w4_t *w);  // a 4-bit matrix's sizes and pointers (w4head.cu)

}  // namespace mstar
