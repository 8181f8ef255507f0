// Entry points of the paged attention: argument checks, workspace and the choice of types. The
// kernel is in attention_kernel.cuh, compiled once for each pair of types.

#include <algorithm>
#include <cmath>

#include "attention.h"

using namespace sonic;

extern "C" size_t sonic_paged_attention_workspace_size(const SonicPagedAttentionArgs* a) {
  return a ? WORKSPACE_BYTES : 0;
}

extern "C" sonic_status sonic_paged_attention(const SonicPagedAttentionArgs* a, void* stream) {
  if (!a) return fail_with(SONIC_ERR_INVALID_ARGUMENT, "args must not be NULL");
  if (sonic_status s = check_cache(a->cache)) return s;
  if (sonic_status s = check_sequences(a->sequences, true)) return s;
  if (a->dtype != SONIC_DTYPE_BF16 && a->dtype != SONIC_DTYPE_F16)
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "queries must be bf16 or f16");
  if (a->cache.dtype != SONIC_DTYPE_E4M3 && a->cache.dtype != a->dtype)
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "queries must be of the cache's dtype unless it is e4m3");
  if (a->q_heads < 1 || a->q_heads % a->cache.kv_heads)
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "q_heads must be a multiple of kv_heads");
  if (a->window < 0 || a->max_tokens < 0) return fail_with(SONIC_ERR_INVALID_ARGUMENT, "window and max_tokens must not be negative");
  if (!std::isfinite(a->scale)) return fail_with(SONIC_ERR_INVALID_ARGUMENT, "scale must be finite");
  if ((int64_t)a->sequences.tokens * a->q_heads * (a->cache.head_dim / 4) > INT32_MAX)
    return fail_with(SONIC_ERR_UNSUPPORTED, "tokens x q_heads is too large for one call");
  // the kernel's division of query rows by the group is exact below 2^32 / group rows
  const int64_t group = a->q_heads / a->cache.kv_heads;
  if ((int64_t)a->sequences.tokens * group * group >= (1ll << 32))
    return fail_with(SONIC_ERR_UNSUPPORTED, "tokens x q_heads is too large for one call");
  if (a->sequences.tokens == 0) return SONIC_OK;
  if (!a->queries || !a->out) return fail_with(SONIC_ERR_INVALID_ARGUMENT, "queries and out must not be NULL");
  if (!is_aligned(a->queries, 16) || a->q_token_stride % 8 || a->q_head_stride % 8)
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "query rows must start on 16-byte boundaries");
  if (!is_aligned(a->out, 8) || a->out_token_stride % 4 || a->out_head_stride % 4)
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "output rows must start on 8-byte boundaries");
  if (!a->workspace || a->workspace_bytes < WORKSPACE_BYTES || !is_aligned(a->workspace, 16))
    return fail_with(SONIC_ERR_WORKSPACE, "workspace smaller than sonic_paged_attention_workspace_size(), or not 16-byte aligned");
  AttentionLaunch p;
  p.a = *a;
  char* w = static_cast<char*>(a->workspace);
  p.ws.error = reinterpret_cast<uint32_t*>(w);
  p.ws.tickets = reinterpret_cast<uint32_t*>(w + HEADER);
  p.ws.stats = reinterpret_cast<float2*>(w + HEADER + TICKET_BYTES);
  p.ws.parts = reinterpret_cast<float4*>(w + HEADER + TICKET_BYTES + STAT_BYTES);
  p.group = a->q_heads / a->cache.kv_heads;
  p.group_inverse = (uint32_t)((1ull << 32) / p.group + 1);
  // page_size <= 2^l: the inverse is 2^32 (2^l - page_size) / page_size + 1, the shift l - 1
  int l = 0;
  while ((1ll << l) < a->cache.page_size) ++l;
  p.page_inverse = (uint32_t)(((1ull << 32) * ((1ull << l) - a->cache.page_size)) / a->cache.page_size + 1);
  p.page_shift = l - 1;
  p.packed = a->cache.slot_stride != a->cache.head_dim || a->cache.page_size % 16 ? 0 : a->cache.page_size % 32 ? 1 : 2;
  const SonicSequences& s = a->sequences;
  p.room = (int)std::min<int64_t>((int64_t)s.table_width * a->cache.page_size, 1 << 30);
  p.window = a->window > p.room ? 0 : a->window;
  p.each = s.tokens / s.requests;
  p.most = s.cu_seqlens ? (a->max_tokens > 0 ? a->max_tokens : (s.tokens + s.requests - 1) / s.requests) : p.each;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool q8 = a->cache.dtype == SONIC_DTYPE_E4M3;
  if (a->dtype == SONIC_DTYPE_BF16) return q8 ? attention_bf16_e4m3(p, st) : attention_bf16(p, st);
  return q8 ? attention_f16_e4m3(p, st) : attention_f16(p, st);
}
