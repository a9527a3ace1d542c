// What the kernels of the per-token operators share: waits of one-warp roles, loads whose lines leave L2 first, casts, launches.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <mutex>

#include "common_host.h"
#include "ptx.cuh"

namespace tb {

bool pdl_enabled();  // api.cu

// mbar_wait_warp with its slow part out of line: the roles' loops are one warp each, so every taken branch in them is exposed.
static __device__ __noinline__ bool wait_slow(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status,
                                              unsigned long long timeout_ns, int code) {
  return mbar_wait_warp(bar, parity, WaitCtx{abort_flag, status, timeout_ns}, code);
}
static __device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, const WaitCtx& w, int code) {
  if (__builtin_expect(__all_sync(0xffffffffu, mbar_try_wait(bar, parity)), 1)) return true;
  return wait_slow(bar, parity, w.abort_flag, w.status, w.timeout_ns, code);
}

static __device__ __forceinline__ uint64_t evict_first_policy() {
  uint64_t policy;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  return policy;
}

template <typename T>
__device__ __forceinline__ T cast16(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 cast16<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half cast16<__half>(float v) { return __float2half_rn(v); }

// One launch, counted; with programmatic dependent launch as the GEMM kernels use it, in clusters of `cluster` blocks along x (0: none).
template <typename... Params, typename... Args>
int launch_token_kernel(void (*kernel)(Params...), dim3 grid, int threads, int smem_bytes, int cluster, cudaStream_t stream, const char* what,
                        Args... args) {
  cudaLaunchConfig_t lc = {};
  lc.gridDim = grid;
  lc.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  lc.dynamicSmemBytes = static_cast<size_t>(smem_bytes);
  lc.stream = stream;
  cudaLaunchAttribute attr[2];
  lc.attrs = attr;
  lc.numAttrs = 0;
  if (cluster > 0) {
    attr[lc.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[lc.numAttrs].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[lc.numAttrs].val.clusterDim.y = 1;
    attr[lc.numAttrs].val.clusterDim.z = 1;
    ++lc.numAttrs;
  }
  if (pdl_enabled()) {
    attr[lc.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[lc.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++lc.numAttrs;
  }
  cudaError_t e = cudaLaunchKernelEx(&lc, kernel, args...);
  if (e != cudaSuccess) return cuda_fail(e, what);
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return TB_OK;
}

// The opt-in to `smem_bytes` of shared memory, once per kernel instantiation (each has a `configured` of its own) and device, and
// again if a launch needs more.
struct SmemOptIn {
  std::mutex mu;
  int bytes[64] = {};
};
template <typename K>
int opt_in_smem(K kernel, int smem_bytes, int device, SmemOptIn& configured, const char* what) {
  std::lock_guard<std::mutex> lk(configured.mu);
  int& have = configured.bytes[device & 63];
  if (smem_bytes > have) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes);
    if (e != cudaSuccess) return cuda_fail(e, what);
    have = smem_bytes;
  }
  return TB_OK;
}

}  // namespace tb
