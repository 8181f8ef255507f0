// Paged attention: fp16 queries over an fp16 cache.

#include "attention_kernel.cuh"

sonic_status sonic::attention_f16(const AttentionLaunch& p, cudaStream_t stream) {
  return launch_shape<__half, false>(p, stream);
}
