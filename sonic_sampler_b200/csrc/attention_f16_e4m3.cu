// Paged attention: fp16 queries over an e4m3 cache.

#include "attention_kernel.cuh"

sonic_status sonic::attention_f16_e4m3(const AttentionLaunch& p, cudaStream_t stream) {
  return launch_shape<__half, true>(p, stream);
}
