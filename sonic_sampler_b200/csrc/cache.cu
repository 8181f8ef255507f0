// The paged key-value cache: new rows into their pages (quantised on the way), and pages read back
// into rows. Both are copies bound by memory: a row is read once and written once.
//
// A CTA takes a run of consecutive token rows. Its first threads look the tokens up (request,
// position, page), one token a thread, so the chain of dependent reads is paid once a CTA; then all
// threads move 16-byte pieces, every (token, keys or values, head) row by a group of neighbouring
// lanes.

#include <algorithm>

#include "host.h"
#include "values.cuh"

namespace sonic {
namespace {

constexpr int NT = 128;  // (256: 4 % slower read-back, 2 % slower append)
constexpr int MAX_RUN = 64;  // tokens a CTA takes at most

// Request of row `row`: the last b with bounds[b] <= row (bounds non-decreasing, bounds[0] <= row).
__device__ __forceinline__ int request_of(const int32_t* bounds, int requests, int row) {
  int lo = 0, hi = requests - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (bounds[mid] <= row)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// Element offset of (page, slot) in the pages, and of its scales; head 0.
struct Slot {
  int64_t at = -1;  // -1: nothing there
  int64_t scale = 0;
};

__device__ __forceinline__ Slot find_slot(const SonicPagedCache& c, const SonicSequences& s, int request, int64_t position,
                                          uint32_t* error) {
  Slot found;
  if (position < 0) return found;
  // (a position is below some int32 length: a 32-bit division will do)
  const uint32_t index = (uint32_t)position / (uint32_t)c.page_size;
  int page = -1;
  if (index < (uint32_t)s.table_width) page = s.page_table[request * s.table_stride + index];
  if (page < 0 || page >= c.pages) {
    if (error) atomicOr(error, (uint32_t)SONIC_DEVICE_ERR_PAGE);
    return found;
  }
  const int slot = (int)((uint32_t)position - index * (uint32_t)c.page_size);
  found.at = page * c.page_stride + slot * c.slot_stride;
  found.scale = page * c.scale_page_stride + slot;
  return found;
}

// Pieces of the run's tokens, `lanes` neighbouring threads a (token, keys or values, head) row: piece
// i of a thread, of `items` a thread.
constexpr int APPEND_ITEMS = 2;
constexpr int GATHER_ITEMS = 4;

struct Work {
  int run;             // tokens a CTA takes
  int row_shift;       // log2 of the lanes a row has
  uint32_t per_token;  // rows a token has
  uint32_t inverse;    // floor(2^32 / per_token) + 1: r / per_token is the high half of r times it
};

struct Item {
  bool live;
  int t, half, head, lane;
};

__device__ __forceinline__ Item item_of(const Work& w, int i, int count, int heads, int items) {
  Item x;
  const uint32_t r = ((blockIdx.y * items + i) * NT + threadIdx.x) >> w.row_shift;
  x.lane = threadIdx.x & ((1 << w.row_shift) - 1);
  x.live = r < count * w.per_token;
  x.t = __umulhi(r, w.inverse);
  const int rest = r - x.t * w.per_token;
  x.half = rest >= heads;
  x.head = x.half ? rest - heads : rest;
  return x;
}

// Largest magnitude of a packed pair's lanes and of `top`'s, as 16-bit patterns (NaN above infinity).
__device__ __forceinline__ uint32_t top_pair(uint32_t top, uint32_t x) { return __vmaxu2(top, x & 0x7fff7fffu); }

// Each thread moves 16 activations an item: 32 bytes in; 32 bytes (16-bit cache) or 16 codes out. A row
// is head_dim / 16 neighbouring lanes (4, 8 or 16), which reduce its largest magnitude by shuffles, on
// packed 16-bit patterns. The activations are asked for before the tokens are looked up, all items' at
// once. Bound by instructions more than by memory: 16000 tokens of 8 heads of 128 into e4m3 take
// 21 us (8 activations an item, fp32 maxima: 31 us; one item at a time: 34 us).
template <typename T, bool Q8>
__global__ void __launch_bounds__(NT) append_kernel(SonicCacheAppendArgs a, Work work) {
  __shared__ Slot slots[MAX_RUN];
  grid_dependency_trigger();
  const SonicSequences& s = a.sequences;
  const SonicPagedCache& c = a.cache;
  const int first = blockIdx.x * work.run;
  const int count = min(work.run, s.tokens - first);
  grid_dependency_wait();
  uint4 x[APPEND_ITEMS][2];
#pragma unroll
  for (int i = 0; i < APPEND_ITEMS; ++i) {
    const Item item = item_of(work, i, count, c.kv_heads, APPEND_ITEMS);
    x[i][0] = x[i][1] = make_uint4(0, 0, 0, 0);
    if (item.live) {
      const int64_t at = item.half ? (first + item.t) * a.value_token_stride + item.head * a.value_head_stride
                                   : (first + item.t) * a.key_token_stride + item.head * a.key_head_stride;
      const uint4* from = reinterpret_cast<const uint4*>(static_cast<const T*>(item.half ? a.values : a.keys) + at + item.lane * 16);
      x[i][0] = from[0];
      x[i][1] = from[1];
    }
  }
  if (threadIdx.x < count) {
    const int row = first + threadIdx.x;
    Slot found;
    if (s.cu_seqlens) {
      const int b = request_of(s.cu_seqlens, s.requests, row);
      // rows outside every request have no place in the cache
      if (row >= s.cu_seqlens[b] && row < s.cu_seqlens[b + 1])
        found = find_slot(c, s, b, (int64_t)s.lengths[b] - s.cu_seqlens[b + 1] + row, a.error);
    } else {
      const int each = s.tokens / s.requests, b = row / each;
      found = find_slot(c, s, b, (int64_t)s.lengths[b] - each + row % each, a.error);
    }
    slots[threadIdx.x] = found;
  }
  __syncthreads();
  const int lanes = 1 << work.row_shift;
#pragma unroll
  for (int i = 0; i < APPEND_ITEMS; ++i) {
    const Item item = item_of(work, i, count, c.kv_heads, APPEND_ITEMS);
    Slot slot;
    if (item.live) slot = slots[item.t];
    void* pages = item.half ? c.values : c.keys;
    const int64_t to = slot.at + item.head * c.head_stride + item.lane * 16;
    if constexpr (!Q8) {
      if (slot.at >= 0) {
        reinterpret_cast<uint4*>(static_cast<T*>(pages) + to)[0] = x[i][0];
        reinterpret_cast<uint4*>(static_cast<T*>(pages) + to)[1] = x[i][1];
      }
    } else {
      const uint32_t w[8] = {x[i][0].x, x[i][0].y, x[i][0].z, x[i][0].w, x[i][1].x, x[i][1].y, x[i][1].z, x[i][1].w};
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) top = top_pair(top, w[k]);
      // (all lanes, live or not: the shuffles are warp-wide)
      for (int d = lanes >> 1; d >= 1; d >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, d));
      top = max(top & 0xffffu, top >> 16);
      float scale, inverse;
      e4m3_scale(magnitude_bits(Pair<T>::unpack(top).x), scale, inverse);
      if (slot.at >= 0) {
        uint32_t codes[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 lo = Pair<T>::unpack(w[2 * k]), hi = Pair<T>::unpack(w[2 * k + 1]);
          codes[k] = e4m3_pack4(lo.x * inverse, lo.y * inverse, hi.x * inverse, hi.y * inverse);
        }
        *reinterpret_cast<uint4*>(static_cast<uint8_t*>(pages) + to) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
        if (item.lane == 0) (item.half ? c.value_scales : c.key_scales)[slot.scale + item.head * c.scale_head_stride] = scale;
      }
    }
  }
}

// Each thread moves 16 cached bytes an item: 8 values of a 16-bit cache, all items' loads at once, or 16
// codes into 32 bytes, one item after the other (three bytes move for each one asked for, and
// more reads in flight only disturb the writes: 215000 tokens of 8 heads of 128 take 206 us, 95 % of the
// measured copy rate, 241 to 256 us with 2 or 4 items' loads at once; 16-bit: 44 us against 48).
template <typename T, bool Q8>
__global__ void __launch_bounds__(NT) gather_kernel(SonicCacheGatherArgs a, Work work) {
  __shared__ Slot slots[MAX_RUN];
  grid_dependency_trigger();
  const SonicSequences& s = a.sequences;
  const SonicPagedCache& c = a.cache;
  const int first = blockIdx.x * work.run;
  const int count = min(work.run, s.tokens - first);
  grid_dependency_wait();
  if (threadIdx.x < count) {
    const int row = first + threadIdx.x;
    const int b = request_of(a.starts, s.requests, row);
    Slot found;
    if (row >= a.starts[b] && row < a.starts[b + 1]) found = find_slot(c, s, b, row - a.starts[b], a.error);
    slots[threadIdx.x] = found;
  }
  __syncthreads();
  constexpr int PER = Q8 ? 16 : 8;  // values an item
  constexpr int AT_ONCE = Q8 ? 1 : GATHER_ITEMS;
#pragma unroll 1
  for (int i0 = 0; i0 < GATHER_ITEMS; i0 += AT_ONCE) {
    uint4 x[AT_ONCE];
    float scale[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const Item item = item_of(work, i0 + i, count, c.kv_heads, GATHER_ITEMS);
      x[i] = make_uint4(0, 0, 0, 0);
      scale[i] = 0.0f;
      if (!item.live) continue;
      const Slot slot = slots[item.t];
      if (slot.at < 0) continue;
      const int64_t at = slot.at + item.head * c.head_stride + item.lane * PER;
      const void* pages = item.half ? c.values : c.keys;
      if constexpr (Q8) {
        x[i] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(pages) + at);
        scale[i] = (item.half ? c.value_scales : c.key_scales)[slot.scale + item.head * c.scale_head_stride];
      } else {
        x[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(pages) + at);
      }
    }
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const Item item = item_of(work, i0 + i, count, c.kv_heads, GATHER_ITEMS);
      if (!item.live) continue;
      T* out = static_cast<T*>(item.half ? a.values : a.keys) +
               ((int64_t)(first + item.t) * c.kv_heads + item.head) * c.head_dim + item.lane * PER;
      if constexpr (!Q8) {
        *reinterpret_cast<uint4*>(out) = x[i];
      } else {
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        uint32_t y[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 lo = Pair<__half>::unpack(e4m3_to_half2((uint16_t)w[k]));
          const float2 hi = Pair<__half>::unpack(e4m3_to_half2((uint16_t)(w[k] >> 16)));
          y[2 * k] = Pair<T>::pack(lo.x * scale[i], lo.y * scale[i]);
          y[2 * k + 1] = Pair<T>::pack(hi.x * scale[i], hi.y * scale[i]);
        }
        reinterpret_cast<uint4*>(out)[0] = make_uint4(y[0], y[1], y[2], y[3]);
        reinterpret_cast<uint4*>(out)[1] = make_uint4(y[4], y[5], y[6], y[7]);
      }
    }
  }
}

int log2_of(int v) {
  int l = 0;
  while ((1 << l) < v) ++l;
  return l;
}

// As many tokens a CTA as its threads take with `items` pieces each (one at least, in several rounds of
// CTAs where a token has more); a small call's are spread over more CTAs.
Work work_of(int tokens, int heads, int lanes, int items) {
  Work w;
  w.row_shift = log2_of(lanes);
  w.per_token = 2 * heads;
  w.inverse = (uint32_t)((1ull << 32) / w.per_token + 1);
  const int full = items * NT / (2 * heads * lanes), spread = std::max(1, tokens / 296);
  w.run = std::max(1, std::min(MAX_RUN, std::min(full, spread)));
  return w;
}

// blockIdx.y: rounds of a token with more pieces than one CTA takes
dim3 grid_of(const Work& w, int tokens, int lanes, int items) {
  const int pieces = w.run * w.per_token * lanes;
  return dim3((unsigned)(((int64_t)tokens + w.run - 1) / w.run), (pieces + items * NT - 1) / (items * NT));
}

bool is_16bit(int dtype) { return dtype == SONIC_DTYPE_BF16 || dtype == SONIC_DTYPE_F16; }

}  // namespace

sonic_status check_cache(const SonicPagedCache& c) noexcept {
  if (!c.keys || !c.values) return fail_with(SONIC_ERR_INVALID_ARGUMENT, "cache keys and values must not be NULL");
  if (!is_16bit(c.dtype) && c.dtype != SONIC_DTYPE_E4M3)
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "cache dtype must be bf16, f16 or e4m3");
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256)
    return fail_with(SONIC_ERR_UNSUPPORTED, "head_dim must be 64, 128 or 256");
  if (c.pages < 1 || c.page_size < 1 || c.kv_heads < 1)
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "pages, page_size and kv_heads must be positive");
  if (c.kv_heads > 1024) return fail_with(SONIC_ERR_INVALID_ARGUMENT, "kv_heads must be at most 1024");
  const int per = c.dtype == SONIC_DTYPE_E4M3 ? 16 : 8;
  if (!is_aligned(c.keys, 16) || !is_aligned(c.values, 16) || c.page_stride % per || c.head_stride % per || c.slot_stride % per)
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "cache rows must start on 16-byte boundaries");
  if (c.page_stride < 0 || c.head_stride < 0 || c.slot_stride < 0 || c.scale_page_stride < 0 || c.scale_head_stride < 0)
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "cache strides must not be negative");
  if (c.dtype == SONIC_DTYPE_E4M3 && (!c.key_scales || !c.value_scales))
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "an e4m3 cache needs key_scales and value_scales");
  return SONIC_OK;
}

sonic_status check_sequences(const SonicSequences& s, bool lengths) noexcept {
  if (s.requests < 1 || s.tokens < 0) return fail_with(SONIC_ERR_INVALID_ARGUMENT, "requests must be positive and tokens not negative");
  if (!s.page_table || s.table_width < 1 || s.table_stride < 0)
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "page_table must have at least one column");
  if (lengths && !s.lengths) return fail_with(SONIC_ERR_INVALID_ARGUMENT, "lengths must not be NULL");
  if (lengths && !s.cu_seqlens && s.tokens % s.requests)
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "without cu_seqlens, tokens must be a multiple of requests");
  return SONIC_OK;
}

}  // namespace sonic

using namespace sonic;

extern "C" sonic_status sonic_cache_append(const SonicCacheAppendArgs* a, void* stream) {
  if (!a) return fail_with(SONIC_ERR_INVALID_ARGUMENT, "args must not be NULL");
  if (sonic_status s = check_cache(a->cache)) return s;
  if (sonic_status s = check_sequences(a->sequences, true)) return s;
  if (a->sequences.tokens == 0) return SONIC_OK;
  if (!is_16bit(a->dtype) || (a->cache.dtype != SONIC_DTYPE_E4M3 && a->cache.dtype != a->dtype))
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "keys and values must be bf16 or f16, and of the cache's dtype unless it is e4m3");
  if (!a->keys || !a->values) return fail_with(SONIC_ERR_INVALID_ARGUMENT, "keys and values must not be NULL");
  if (!is_aligned(a->keys, 16) || !is_aligned(a->values, 16) || a->key_token_stride % 8 || a->key_head_stride % 8 ||
      a->value_token_stride % 8 || a->value_head_stride % 8)
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "rows of keys and values must start on 16-byte boundaries");
  const int lanes = a->cache.head_dim / 16;
  const Work work = work_of(a->sequences.tokens, a->cache.kv_heads, lanes, APPEND_ITEMS);
  const dim3 grid = grid_of(work, a->sequences.tokens, lanes, APPEND_ITEMS);
  const bool pdl = a->flags & SONIC_FLAG_PDL;
  const auto go = [&](auto kernel) {
    return launch_status(launch_kernel(kernel, grid, dim3(NT), 0, (cudaStream_t)stream, pdl, 1, *a, work));
  };
  const bool q8 = a->cache.dtype == SONIC_DTYPE_E4M3;
  if (a->dtype == SONIC_DTYPE_BF16) return q8 ? go(append_kernel<__nv_bfloat16, true>) : go(append_kernel<__nv_bfloat16, false>);
  return q8 ? go(append_kernel<__half, true>) : go(append_kernel<__half, false>);
}

extern "C" sonic_status sonic_cache_gather(const SonicCacheGatherArgs* a, void* stream) {
  if (!a) return fail_with(SONIC_ERR_INVALID_ARGUMENT, "args must not be NULL");
  if (sonic_status s = check_cache(a->cache)) return s;
  if (sonic_status s = check_sequences(a->sequences, false)) return s;
  if (a->sequences.tokens == 0) return SONIC_OK;
  if (!is_16bit(a->dtype) || (a->cache.dtype != SONIC_DTYPE_E4M3 && a->cache.dtype != a->dtype))
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "outputs must be bf16 or f16, and of the cache's dtype unless it is e4m3");
  if (!a->starts || !a->keys || !a->values) return fail_with(SONIC_ERR_INVALID_ARGUMENT, "starts, keys and values must not be NULL");
  if (!is_aligned(a->keys, 16) || !is_aligned(a->values, 16))
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "outputs must start on 16-byte boundaries");
  const bool q8 = a->cache.dtype == SONIC_DTYPE_E4M3;
  const int lanes = a->cache.head_dim / (q8 ? 16 : 8);
  const Work work = work_of(a->sequences.tokens, a->cache.kv_heads, lanes, GATHER_ITEMS);
  const dim3 grid = grid_of(work, a->sequences.tokens, lanes, GATHER_ITEMS);
  const bool pdl = a->flags & SONIC_FLAG_PDL;
  const auto go = [&](auto kernel) {
    return launch_status(launch_kernel(kernel, grid, dim3(NT), 0, (cudaStream_t)stream, pdl, 1, *a, work));
  };
  if (a->dtype == SONIC_DTYPE_BF16) return q8 ? go(gather_kernel<__nv_bfloat16, true>) : go(gather_kernel<__nv_bfloat16, false>);
  return q8 ? go(gather_kernel<__half, true>) : go(gather_kernel<__half, false>);
}
