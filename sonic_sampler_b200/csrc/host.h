// Host-side helpers shared by the translation units behind include/sonic_b200.h.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/sonic_b200.h"

namespace sonic {

// Record `message` as the calling thread's last error and return `code`. Never throws.
sonic_status fail_with(sonic_status code, const char* message) noexcept;

inline sonic_status launch_status(cudaError_t e) noexcept {
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? SONIC_OK : fail_with(SONIC_ERR_CUDA, cudaGetErrorString(e));
}

// Launch with `smem` bytes of dynamic shared memory; with `pdl` the kernel may start before the
// stream's previous kernel has ended (it waits with griddepcontrol.wait before its first access);
// `cluster` CTAs form a cluster.
template <typename Kern, typename... Args>
cudaError_t launch_kernel(Kern kern, dim3 grid, dim3 block, size_t smem, cudaStream_t stream, bool pdl, int cluster,
                          const Args&... args) noexcept {
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  cfg.numAttrs = 0;
  if (pdl) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = cluster;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

inline bool is_aligned(const void* p, uintptr_t bytes) { return (uintptr_t)p % bytes == 0; }

// Checks of the descriptors that several entry points take; `who` names the entry point's messages.
sonic_status check_cache(const SonicPagedCache& c) noexcept;
sonic_status check_sequences(const SonicSequences& s, bool lengths) noexcept;

}  // namespace sonic
