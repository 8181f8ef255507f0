// Paged attention: bf16 queries over a bf16 cache.

#include "attention_kernel.cuh"

sonic_status sonic::attention_bf16(const AttentionLaunch& p, cudaStream_t stream) {
  return launch_shape<__nv_bfloat16, false>(p, stream);
}
