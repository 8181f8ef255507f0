// What the units of the paged attention share: the workspace's layout, and a launch by types.
#pragma once

#include "host.h"

namespace sonic {

constexpr int WARPS = 4;                   // of a CTA
constexpr int MAX_CTAS = 296;              // 148 SMs x 2
constexpr int MAX_WARPS = MAX_CTAS * WARPS;
constexpr int PART_FLOATS = 4096;          // a partial result: 8 NT query rows x head_dim at most
constexpr int PART_ROWS = 32;

// Partial results: MAX_WARPS slots for what a warp has of the first unit of its share, where others
// follow it; then 2 MAX_CTAS for what a CTA has of units that it shares, and 2 MAX_CTAS for sets of
// CTAs.
constexpr int SLOTS = MAX_WARPS + 4 * MAX_CTAS;
struct AttentionWorkspace {
  uint32_t* error;
  uint32_t* tickets;  // [2][2 * MAX_CTAS], zero between calls
  float2* stats;      // [SLOTS][PART_ROWS] (m, l)
  float4* parts;      // [SLOTS][PART_FLOATS / 4], in the order of the accumulator fragments
};

constexpr size_t HEADER = 256;             // error word
constexpr size_t TICKET_BYTES = (size_t)4 * MAX_CTAS * 4 + 128;
constexpr size_t STAT_BYTES = (size_t)SLOTS * PART_ROWS * 8;
constexpr size_t PART_BYTES = (size_t)SLOTS * PART_FLOATS * 4;
constexpr size_t WORKSPACE_BYTES = HEADER + TICKET_BYTES + STAT_BYTES + PART_BYTES;
static_assert((HEADER + TICKET_BYTES) % 128 == 0 && STAT_BYTES % 128 == 0, "partial results are 16-byte aligned");

struct AttentionLaunch {
  SonicPagedAttentionArgs a;
  AttentionWorkspace ws;
  int group;               // query heads a kv head
  uint32_t group_inverse;  // floor(2^32 / group) + 1: r / group is the high half of r times it
  // k / page_size = (h + (k - h) / 2) >> page_shift with h the high half of k times page_inverse
  // (Granlund and Montgomery, Division by invariant integers using multiplication, 1994); pages of one
  // slot have the shift -1
  uint32_t page_inverse;
  int page_shift;
  int packed;              // a page's rows follow one another, and a page holds a multiple of 16 (1) or 32 (2)
  int room;                // longest request: what a page-table row holds, at most 2^30
  int window;              // 0 where no request is longer than it
  int each;                // new tokens a request has, without cu_seqlens
  int most;                // new tokens a request has at most, as far as the host knows
  int direct;              // 0: balanced shares; else this many row tiles a (request, kv head) at once
  int unit_warps;          // warps of each then: 1, or 4 to 32 (a cluster of CTAs)
};

// The kernel for the types of a call (one translation unit each).
sonic_status attention_bf16(const AttentionLaunch& p, cudaStream_t stream);
sonic_status attention_f16(const AttentionLaunch& p, cudaStream_t stream);
sonic_status attention_bf16_e4m3(const AttentionLaunch& p, cudaStream_t stream);
sonic_status attention_f16_e4m3(const AttentionLaunch& p, cudaStream_t stream);

}  // namespace sonic
