// Attention of a call's new tokens over a paged key-value cache.
//
// With s_j = c q.k_j (c = scale * log2 e) and any reference m, out = sum_j 2^(s_j - m) v_j / l,
// l = sum_j 2^(s_j - m): the kernel streams the keys once and keeps m (the running maximum), l and
// the unnormalised out in registers, rescaling when m rises. Sums over disjoint key ranges join the
// same way, so a sequence may be cut anywhere.
//
// Bound by memory: G = q_heads / kv_heads query heads share a key, so a cached byte meets 2 G n
// multiply-adds (n new tokens), far below the tensor cores' balance. The work is laid out for a
// continuous stream of the cache:
// - A unit is (request, kv head, tile of up to 16 MT query rows). All units' steps (4 KT keys each)
//   are laid end to end and cut into equal shares, one a CTA, whatever the lengths: a CTA finds its
//   place with a scan over `lengths`. A unit that several CTAs share is joined by the last of them
//   to finish, from partial results in the workspace, in the order of the keys.
// - Inside a CTA each of 4 warps takes KT of a step's keys through its own ring of asynchronous
//   16-byte copies, with its own m, l and out: no block barrier inside a share's unit.
// - Rows of the matrix instructions (m16n8k16) are query rows, so 16 rows cost one instruction's
//   height; tcgen05 tiles are 128 rows high and would be mostly empty here.
// - An e4m3 key row is code * scale: the scale multiplies the score after the product. A value row's
//   scale vs multiplies the softmax weight, and the reference is the running maximum of
//   s_j + log2 vs_j, so that the fp16 weights keep their precision whatever the scales. Codes
//   become fp16 exactly; query rows are brought to fp16's range by a power of two.

#include <algorithm>
#include <cmath>

#include "host.h"
#include "values.cuh"

namespace sonic {
namespace {

constexpr int WARPS = 4;
constexpr int NT = 32 * WARPS;
constexpr int MAX_CTAS = 296;        // 148 SMs x 2
constexpr size_t HEADER = 256;       // error word
constexpr int PART_FLOATS = 4096;    // rows x head_dim of one partial result (16 MT x D at most)
constexpr int PART_ROWS = 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr unsigned ALL = 0xffffffffu;

__host__ __device__ constexpr int imax(int a, int b) { return a > b ? a : b; }
__host__ __device__ constexpr int imin(int a, int b) { return a < b ? a : b; }

struct Workspace {
  uint32_t* error;
  uint32_t* tickets;  // [2 * MAX_CTAS], zero between calls
  float2* stats;      // [2 * MAX_CTAS][PART_ROWS] (m, l)
  float* parts;       // [2 * MAX_CTAS][PART_FLOATS]
};

constexpr size_t TICKET_BYTES = (2 * MAX_CTAS * 4 + 255) / 256 * 256;
constexpr size_t STAT_BYTES = (size_t)2 * MAX_CTAS * PART_ROWS * 8;
constexpr size_t PART_BYTES = (size_t)2 * MAX_CTAS * PART_FLOATS * 4;
constexpr size_t WORKSPACE_BYTES = HEADER + TICKET_BYTES + STAT_BYTES + PART_BYTES;

// 2^x; 0 for -infinity
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float log2_fast(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 16 bytes global -> shared, zeros when !live
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void load_matrices_transposed(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ uint4 load_shared16(uint32_t at) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at) : "memory");
  return r;
}
__device__ __forceinline__ uint2 load_shared8(uint32_t at) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(at) : "memory");
  return r;
}

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

struct Launch {
  SonicPagedAttentionArgs a;
  Workspace ws;
  int group;       // query heads a kv head
  int page_shift;  // log2(page_size), or -1
};

// A: activations; Q8: e4m3 cache; D: head_dim; MT: tiles of 16 query rows.
template <typename A, bool Q8, int D, int MT>
struct Shape {
  using M = std::conditional_t<Q8, __half, A>;  // type of the products' operands
  static constexpr int ROW = D * (Q8 ? 1 : 2);  // bytes of a cached row
  static constexpr int CPR = ROW / 16;          // 16-byte pieces of it
  static constexpr int KT = imin(32, imax(16, 4096 / ROW));  // keys of a warp's tile
  static constexpr int STEP = WARPS * KT;
  static constexpr int TILE = KT * ROW;
  static constexpr int STAGE = 2 * TILE + (Q8 ? 2 * KT * 4 : 0);  // keys, values, their scales
  static constexpr int STAGES = imax(3, 24 * 1024 / STAGE);
  static constexpr int RING = WARPS * STAGES * STAGE;
  static constexpr int ROWS = 16 * MT;
  // row pitch of the block's reduction buffer: 4 floats of padding every 32
  static constexpr int PITCH = D + D / 8 + (D == 128 ? 0 : D == 64 ? 8 : 16);
  static constexpr int REDUCE = WARPS * ROWS * PITCH * 4;
  static constexpr bool Q_REGISTERS = MT == 1 && D <= 128;
  static constexpr int Q_BYTES = Q_REGISTERS ? 0 : MT * (D / 16) * 512;
  static constexpr int SMEM = imax(imax(RING, REDUCE), MAX_CTAS * ROWS * 4) + Q_BYTES;
  static constexpr int OCC = SMEM <= 112 * 1024 ? 2 : 1;
  // weights of fp16 products reach 2^14, so that small ones stay above fp16's smallest normal
  static constexpr float SHIFT = std::is_same<M, __half>::value ? 14.0f : 0.0f;

  // byte offset of piece c of key row r, and of value row r: the pieces are permuted so that the
  // fragment reads below are free of bank conflicts
  static __device__ __forceinline__ int key_at(int r, int c) {
    if constexpr (!Q8)
      return r * ROW + ((c ^ (r & 7)) << 4);
    else if constexpr (D == 64)
      return r * ROW + (c << 4);
    else
      return r * ROW + ((c ^ ((r & 1) << 2)) << 4);
  }
  static __device__ __forceinline__ int value_at(int r, int c) {
    if constexpr (!Q8) {
      return r * ROW + ((c ^ (r & 7)) << 4);
    } else if constexpr (D == 64) {
      const int x = ((r & 1) << 2 | c) ^ (((r >> 1) & 3) << 1);
      return (r >> 1) * 128 + (x << 4);
    } else {
      return r * ROW + ((c ^ (r & 6)) << 4);
    }
  }
};

// position of dimension d in a row of the reduction buffer
__device__ __forceinline__ int padded(int d) { return d + (d >> 5) * 4; }

struct Request {
  int new_tokens, first_row, length, begin, steps, tiles;  // begin: first key any query sees
};

template <class S>
__device__ __forceinline__ Request read_request(const Launch& p, int b) {
  const SonicSequences& s = p.a.sequences;
  Request q;
  if (s.cu_seqlens) {
    const int lo = min(max(s.cu_seqlens[b], 0), s.tokens), hi = min(max(s.cu_seqlens[b + 1], lo), s.tokens);
    q.first_row = lo;
    q.new_tokens = hi - lo;
  } else {
    q.new_tokens = s.tokens / s.requests;
    q.first_row = b * q.new_tokens;
  }
  const int64_t room = min((int64_t)s.table_width * p.a.cache.page_size, (int64_t)INT32_MAX - S::STEP);
  const int length = s.lengths[b];
  q.length = (int)min((int64_t)max(length, 0), room);
  if (length != q.length) atomicOr(p.ws.error, (uint32_t)SONIC_DEVICE_ERR_PAGE);
  q.begin = p.a.window > 0 ? (int)max((int64_t)0, (int64_t)q.length - q.new_tokens - p.a.window + 1) : 0;
  q.begin = min(q.begin, q.length);
  q.steps = q.new_tokens > 0 ? (q.length + S::STEP - 1) / S::STEP - q.begin / S::STEP : 0;
  if (q.length == q.begin) q.steps = 0;
  q.tiles = (int)(((int64_t)q.new_tokens * p.group + S::ROWS - 1) / S::ROWS);
  return q;
}

// One warp's place in its keys: where its next tile lies.
struct Keys {
  int64_t at;     // element offset of this lane's key row (head included)
  int64_t scale;  // and of its scales
  uint32_t live;  // bit r: key r of the tile exists
};

template <typename A, bool Q8, int D, int MT>
__global__ void __launch_bounds__(NT, (Shape<A, Q8, D, MT>::OCC)) attention_kernel(const __grid_constant__ Launch p) {
  using S = Shape<A, Q8, D, MT>;
  using M = typename S::M;
  constexpr int KT = S::KT;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint32_t scan[WARPS];
  __shared__ uint32_t place[2];
  __shared__ float2 warp_stats[WARPS][S::ROWS];
  __shared__ int is_last;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;  // fragment row and column pair
  const SonicSequences& seq = p.a.sequences;
  const SonicPagedCache& cache = p.a.cache;
  const int heads = cache.kv_heads;

  grid_dependency_trigger();
  grid_dependency_wait();

  // ---- this CTA's share of the steps ----
  const int per = (seq.requests + NT - 1) / NT;
  const int b_lo = min(tid * per, seq.requests), b_hi = min(b_lo + per, seq.requests);
  uint32_t mine = 0;
  for (int b = b_lo; b < b_hi; ++b) {
    const Request q = read_request<S>(p, b);
    mine += (uint32_t)q.steps * heads * q.tiles;
  }
  uint32_t upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t o = __shfl_up_sync(ALL, upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 31) scan[warp] = upto;
  if (tid == 0) place[0] = 0, place[1] = 0;
  __syncthreads();
  uint32_t before = upto - mine, total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += scan[w];
    total += scan[w];
  }
  const uint32_t share = (total + gridDim.x - 1) / gridDim.x;
  const uint32_t begin = min((uint64_t)blockIdx.x * share, (uint64_t)total), end = min((uint64_t)begin + share, (uint64_t)total);
  if (begin < end && begin >= before && begin < before + mine) {
    uint32_t base = before;
    for (int b = b_lo; b < b_hi; ++b) {
      const Request q = read_request<S>(p, b);
      const uint32_t w = (uint32_t)q.steps * heads * q.tiles;
      if (begin < base + w) {
        place[0] = b;
        place[1] = base;
        break;
      }
      base += w;
    }
  }
  __syncthreads();

  // ---- requests without a visible key: zeros ----
  for (int b = blockIdx.x; b < seq.requests; b += gridDim.x) {
    const Request q = read_request<S>(p, b);
    if (q.steps != 0) continue;
    const int pieces = q.new_tokens * p.a.q_heads * (D / 4);
    for (int i = tid; i < pieces; i += NT) {
      const int d = i % (D / 4) * 4, head = i / (D / 4) % p.a.q_heads, row = q.first_row + i / (D / 4) / p.a.q_heads;
      A* out = static_cast<A*>(p.a.out) + (int64_t)row * p.a.out_token_stride + (int64_t)head * p.a.out_head_stride + d;
      *reinterpret_cast<uint2*>(out) = make_uint2(0, 0);
      if (d == 0 && p.a.lse) p.a.lse[(int64_t)row * p.a.q_heads + head] = -INFINITY;
    }
  }

  const uint32_t ring = shared_address(smem) + warp * S::STAGES * S::STAGE;
  unsigned char* const q_smem = smem + (S::SMEM - S::Q_BYTES);
  const float score_scale = p.a.scale * kLog2e;

  int b = (int)place[0];
  uint32_t base = place[1];
  Request q = begin < end ? read_request<S>(p, b) : Request{};
  for (uint32_t pos = begin; pos < end;) {
    while (pos >= base + (uint32_t)q.steps * heads * q.tiles) {
      base += (uint32_t)q.steps * heads * q.tiles;
      q = read_request<S>(p, ++b);
    }
    const uint32_t unit = (pos - base) / q.steps;
    const int from = (int)(pos - base - unit * q.steps);           // first step of the piece
    const int steps = (int)min((uint32_t)(q.steps - from), end - pos);
    const int head = unit / q.tiles, tile = unit % q.tiles;
    const uint32_t unit_begin = base + unit * q.steps;
    pos += steps;

    // ---- query rows ----
    const int all_rows = q.new_tokens * p.group;
    const int rows = min(S::ROWS, all_rows - tile * S::ROWS);      // valid rows of the tile
    // positions of the keys that fragment rows g and g + 8 see: (limit - window, limit]
    int limit[MT][2];
    float row_scale[MT][2];
    uint32_t qf[S::Q_REGISTERS ? D / 16 : 1][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = m * 16 + g + 8 * i, row = tile * S::ROWS + r;
        limit[m][i] = r < rows ? q.length - q.new_tokens + row / p.group : -1;
        row_scale[m][i] = score_scale;
      }
    __syncthreads();  // the last piece's reduction buffer and queries are free
    // queries in fragment order; with e4m3 keys a lane's products run over 16 consecutive
    // dimensions (one 16-byte piece of codes), so the queries are permuted alike
    const auto query_fragments = [&](int m, uint32_t (&f)[D / 16][4]) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = m * 16 + g + 8 * i, row = tile * S::ROWS + r;
        const bool live = r < rows;
        const A* src = static_cast<const A*>(p.a.queries);
        if (live)
          src += (int64_t)(q.first_row + row / p.group) * p.a.q_token_stride + (int64_t)(head * p.group + row % p.group) * p.a.q_head_stride;
        if constexpr (!Q8) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            f[k][i] = live ? *reinterpret_cast<const uint32_t*>(src + 16 * k + 2 * t) : 0u;
            f[k][2 + i] = live ? *reinterpret_cast<const uint32_t*>(src + 16 * k + 8 + 2 * t) : 0u;
          }
        } else {
          float2 x[D / 16][2];
          uint32_t top = 0;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const int d = 64 * (k / 4) + 16 * t + 4 * (k % 4);
            const uint2 v = live ? *reinterpret_cast<const uint2*>(src + d) : make_uint2(0, 0);
            x[k][0] = Pair<A>::unpack(v.x);
            x[k][1] = Pair<A>::unpack(v.y);
            top = max(max(top, max(magnitude_bits(x[k][0].x), magnitude_bits(x[k][0].y))),
                      max(magnitude_bits(x[k][1].x), magnitude_bits(x[k][1].y)));
          }
          top = max(top, __shfl_xor_sync(ALL, top, 1));
          top = max(top, __shfl_xor_sync(ALL, top, 2));
          // the power of two that brings the row's largest magnitude to [2^14, 2^15); rows of zeros,
          // infinities or NaN stay as they are
          const int exponent = (int)(top >> 23);  // biased
          const int up = exponent == 0 || exponent == 255 ? 0 : min(max(127 + 14 - exponent, -126), 126);
          const float factor = __uint_as_float((uint32_t)(127 + up) << 23);
          row_scale[m][i] = score_scale * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            f[k][i] = Pair<__half>::pack(x[k][0].x * factor, x[k][0].y * factor);
            f[k][2 + i] = Pair<__half>::pack(x[k][1].x * factor, x[k][1].y * factor);
          }
        }
      }
    };
    if constexpr (S::Q_REGISTERS) {
      query_fragments(0, qf);
    } else {
      // the same for every warp: warp w keeps what it computes for the row scales, warp 0 stores
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        uint32_t f[D / 16][4];
        query_fragments(m, f);
        if (warp == 0)
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            reinterpret_cast<uint4*>(q_smem)[(m * (D / 16) + k) * 32 + lane] = make_uint4(f[k][0], f[k][1], f[k][2], f[k][3]);
      }
      __syncthreads();
    }
    // keys that every row of the tile sees: [all_from, all_to)
    const int first_limit = q.length - q.new_tokens + tile * S::ROWS / p.group;
    const int last_limit = q.length - q.new_tokens + (tile * S::ROWS + rows - 1) / p.group;
    const int all_to = first_limit + 1;
    const int all_from = p.a.window > 0 ? (int)max((int64_t)0, (int64_t)last_limit - p.a.window + 1) : 0;
    // keys that some row sees: copied, the rest of a tile is zeros
    const int some_from = p.a.window > 0 ? max(q.begin, (int)max((int64_t)0, (int64_t)first_limit - p.a.window + 1)) : 0;
    const int some_to = min(q.length, last_limit + 1);

    // ---- the stream of keys ----
    const int first_key = (q.begin / S::STEP + from) * S::STEP + warp * KT;
    const int32_t* table = seq.page_table + (int64_t)b * seq.table_stride;
    const auto find = [&](int step) {
      Keys k;
      const int key = first_key + step * S::STEP + (lane & (KT - 1));
      bool live = step < steps && key >= some_from && key < some_to;
      k.at = k.scale = 0;
      if (live) {
        const int index = p.page_shift >= 0 ? key >> p.page_shift : key / cache.page_size;
        const int slot = key - index * cache.page_size;
        const int page = __ldg(table + index);
        if (page < 0 || page >= cache.pages) {
          atomicOr(p.ws.error, (uint32_t)SONIC_DEVICE_ERR_PAGE);
          live = false;
        } else {
          k.at = page * cache.page_stride + head * cache.head_stride + slot * cache.slot_stride;
          if constexpr (Q8) k.scale = page * cache.scale_page_stride + head * cache.scale_head_stride + slot;
        }
      }
      k.live = __ballot_sync(ALL, live);
      return k;
    };
    const auto copy = [&](int step, const Keys& k) {
      if (step < steps) {
        const uint32_t stage = ring + (uint32_t)(step % S::STAGES) * S::STAGE;
#pragma unroll
        for (int i = 0; i < KT * S::CPR / 32; ++i) {
          const int r = (i * 32 + lane) / S::CPR, c = (i * 32 + lane) % S::CPR;
          const int64_t at = __shfl_sync(ALL, k.at, r);
          const bool live = (k.live >> r) & 1;
          const int64_t bytes = at * (Q8 ? 1 : 2) + c * 16;
          copy16(stage + S::key_at(r, c), static_cast<const char*>(cache.keys) + bytes, live);
          copy16(stage + S::TILE + S::value_at(r, c), static_cast<const char*>(cache.values) + bytes, live);
        }
        if constexpr (Q8) {
          if (lane < KT) {
            const bool live = (k.live >> lane) & 1;
            copy4(stage + 2 * S::TILE + lane * 4, cache.key_scales + k.scale, live);
            copy4(stage + 2 * S::TILE + KT * 4 + lane * 4, cache.value_scales + k.scale, live);
          }
        }
      }
      copies_commit();
    };

    float o[MT][D / 8][4];
    float top[MT][2], sum[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[m][j][i] = 0.0f;
      top[m][0] = top[m][1] = -INFINITY;
      sum[m][0] = sum[m][1] = 0.0f;
    }

    Keys next = find(0);
#pragma unroll
    for (int i = 0; i < S::STAGES - 1; ++i) {
      const Keys now = next;
      next = find(i + 1);
      copy(i, now);
    }

    for (int step = 0; step < steps; ++step) {
      copies_wait<S::STAGES - 2>();
      __syncwarp();
      {
        const Keys now = next;
        next = find(step + S::STAGES);
        copy(step + S::STAGES - 1, now);
      }
      const int key0 = first_key + step * S::STEP;
      if (key0 >= some_to || key0 + KT <= some_from) continue;
      const uint32_t keys = ring + (uint32_t)(step % S::STAGES) * S::STAGE, values = keys + S::TILE;

      // ---- scores ----
      float s[MT][KT / 8][4];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < KT / 8; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[m][n][i] = 0.0f;
      const auto query = [&](int m, int k, uint32_t (&f)[4]) {
        if constexpr (S::Q_REGISTERS) {
#pragma unroll
          for (int i = 0; i < 4; ++i) f[i] = qf[k][i];
        } else {
          const uint4 v = load_shared16(shared_address(q_smem) + ((m * (D / 16) + k) * 32 + lane) * 16);
          f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
        }
      };
      if constexpr (!Q8) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          uint32_t f[MT][4];
#pragma unroll
          for (int m = 0; m < MT; ++m) query(m, k, f[m]);
#pragma unroll
          for (int n = 0; n < KT / 16; ++n) {
            uint32_t kf[4];
            load_matrices(kf, keys + S::key_at(n * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              mma<M>(s[m][2 * n], f[m], kf[0], kf[1]);
              mma<M>(s[m][2 * n + 1], f[m], kf[2], kf[3]);
            }
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
          uint4 codes[KT / 8];
#pragma unroll
          for (int n = 0; n < KT / 8; ++n) codes[n] = load_shared16(keys + S::key_at(n * 8 + g, 4 * j + t));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t f[MT][4];
#pragma unroll
            for (int m = 0; m < MT; ++m) query(m, 4 * j + i, f[m]);
#pragma unroll
            for (int n = 0; n < KT / 8; ++n) {
              const uint32_t w = i == 0 ? codes[n].x : i == 1 ? codes[n].y : i == 2 ? codes[n].z : codes[n].w;
              const uint32_t lo = e4m3_to_half2((uint16_t)w), hi = e4m3_to_half2((uint16_t)(w >> 16));
#pragma unroll
              for (int m = 0; m < MT; ++m) mma<M>(s[m][n], f[m], lo, hi);
            }
          }
        }
      }

      // ---- softmax weights ----
      const bool masked = key0 < all_from || key0 + KT > all_to;
      float value_scale[KT / 8][2], log_scale[KT / 8][2];
#pragma unroll
      for (int n = 0; n < KT / 8; ++n) {
        float2 ks = make_float2(1.0f, 1.0f), vs = ks;
        if constexpr (Q8) {
          const uint2 x = load_shared8(keys + 2 * S::TILE + (n * 8 + 2 * t) * 4);
          const uint2 y = load_shared8(keys + 2 * S::TILE + KT * 4 + (n * 8 + 2 * t) * 4);
          ks = make_float2(__uint_as_float(x.x), __uint_as_float(x.y));
          vs = make_float2(__uint_as_float(y.x), __uint_as_float(y.y));
          value_scale[n][0] = vs.x, value_scale[n][1] = vs.y;
          // (a scale of zero or NaN still leaves its key in the sum)
          log_scale[n][0] = fmaxf(log2_fast(vs.x), -126.0f), log_scale[n][1] = fmaxf(log2_fast(vs.y), -126.0f);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float v = s[m][n][i] * row_scale[m][i >> 1];
            if constexpr (Q8) v *= (i & 1) ? ks.y : ks.x;
            if (masked) {
              const int key = key0 + n * 8 + 2 * t + (i & 1);
              const bool sees = key <= limit[m][i >> 1] && (p.a.window <= 0 || key > limit[m][i >> 1] - p.a.window);
              v = sees ? v : -INFINITY;
            }
            s[m][n][i] = v;
          }
      }
      bool rose = false;
      float reference[MT][2], alpha[MT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float v = top[m][i];
#pragma unroll
          for (int n = 0; n < KT / 8; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) v = fmaxf(v, Q8 ? s[m][n][2 * i + c] + log_scale[n][c] : s[m][n][2 * i + c]);
          v = fmaxf(v, __shfl_xor_sync(ALL, v, 1));
          v = fmaxf(v, __shfl_xor_sync(ALL, v, 2));
          rose = rose || v > top[m][i];
          reference[m][i] = (v == -INFINITY ? 0.0f : v) - S::SHIFT;
          alpha[m][i] = exp2_fast(top[m][i] - v);  // NaN where both are -infinity: o and sum are 0 there
          if (top[m][i] == -INFINITY) alpha[m][i] = 0.0f;
          top[m][i] = v;
        }
      if (__any_sync(ALL, rose)) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          sum[m][0] *= alpha[m][0];
          sum[m][1] *= alpha[m][1];
#pragma unroll
          for (int j = 0; j < D / 8; ++j) {
            o[m][j][0] *= alpha[m][0];
            o[m][j][1] *= alpha[m][0];
            o[m][j][2] *= alpha[m][1];
            o[m][j][3] *= alpha[m][1];
          }
        }
      }
      // the weights as the second product's left operand
      uint32_t w[MT][KT / 16][4];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < KT / 8; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float e0 = exp2_fast(s[m][n][2 * i] - reference[m][i]);
            float e1 = exp2_fast(s[m][n][2 * i + 1] - reference[m][i]);
            sum[m][i] += e0 + e1;
            if constexpr (Q8) {
              // a masked key weighs 0 whatever its scale holds
              e0 = s[m][n][2 * i] == -INFINITY ? 0.0f : e0 * value_scale[n][0];
              e1 = s[m][n][2 * i + 1] == -INFINITY ? 0.0f : e1 * value_scale[n][1];
            }
            w[m][n / 2][(n & 1) * 2 + i] = Pair<M>::pack(e0, e1);
          }

      // ---- out += weights x values ----
      // fragments of the values' keys [16 n, 16 n + 16), dimensions of column tiles j ... j + 3
      const auto products = [&](auto&& only, auto&& add) {
#pragma unroll
        for (int n = 0; n < KT / 16; ++n) {
          if constexpr (!Q8) {
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
              uint32_t vf[4];
              load_matrices_transposed(vf, values + S::value_at(n * 16 + (lane & 7) + (((lane >> 3) & 1) << 3), 2 * j + (lane >> 4)));
              only(n, vf[0], vf[1]);
              only(n, vf[2], vf[3]);
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                add(m, o[m][2 * j], w[m][n], vf[0], vf[1]);
                add(m, o[m][2 * j + 1], w[m][n], vf[2], vf[3]);
              }
            }
          } else {
            // lane (g, t) reads keys 2t, 2t + 1, 2t + 8, 2t + 9, dimensions [D/8 g, D/8 (g + 1))
            // (16 at a time): column tile j, column g stands for dimension 16 g + j (+ 128)
            constexpr int SPAN = D == 64 ? 8 : 16;
#pragma unroll
            for (int h = 0; h < imax(1, D / 128); ++h) {
              uint32_t x[4][SPAN / 4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int r = n * 16 + 2 * t + (i & 1) + (i >> 1) * 8;
                if constexpr (D == 64) {
                  const uint2 v = load_shared8(values + S::value_at(r, g >> 1) + (g & 1) * 8);
                  x[i][0] = v.x, x[i][1] = v.y;
                } else {
                  const uint4 v = load_shared16(values + S::value_at(r, g + 8 * h));
                  x[i][0] = v.x, x[i][1] = v.y, x[i][2] = v.z, x[i][3] = v.w;
                }
              }
#pragma unroll
              for (int k = 0; k < SPAN / 4; ++k) {
                const uint32_t p0 = __byte_perm(x[0][k], x[1][k], 0x5140), p1 = __byte_perm(x[0][k], x[1][k], 0x7362);
                const uint32_t r0 = __byte_perm(x[2][k], x[3][k], 0x5140), r1 = __byte_perm(x[2][k], x[3][k], 0x7362);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const uint32_t lo = i < 2 ? p0 : p1, hi = i < 2 ? r0 : r1;
                  uint32_t b0 = e4m3_to_half2((uint16_t)((i & 1) ? lo >> 16 : lo)), b1 = e4m3_to_half2((uint16_t)((i & 1) ? hi >> 16 : hi));
                  only(n, b0, b1);
#pragma unroll
                  for (int m = 0; m < MT; ++m) add(m, o[m][h * 16 + 4 * k + i], w[m][n], b0, b1);
                }
              }
            }
          }
        }
      };
      // A key that some rows of the tile see and others do not: 0 x infinity or NaN in its values
      // must not reach the others. Rare, so looked for first: then once for every query, with the
      // values that it does not see taken as zeros, keeping the results of its rows only.
      bool strange = false;
      if (masked && last_limit > first_limit) {
#pragma unroll 1
        for (int i = lane; i < S::TILE / 4; i += 32) {
          const uint32_t x = *reinterpret_cast<const uint32_t*>(smem + (values - shared_address(smem)) + i * 4);
          if constexpr (Q8) {
            const uint32_t m = x & 0x7f7f7f7fu;
            strange = strange || (m & 0xff) == 0x7f || (m >> 8 & 0xff) == 0x7f || (m >> 16 & 0xff) == 0x7f || m >> 24 == 0x7f;
          } else {
            constexpr uint32_t E = std::is_same<A, __half>::value ? 0x7c00u : 0x7f80u;
            strange = strange || (x & E) == E || (x >> 16 & E) == E;
          }
        }
        strange = __any_sync(ALL, strange);
      }
      if (!strange) {
        products([](int, uint32_t&, uint32_t&) {},
                 [](int, float(&d)[4], const uint32_t(&f)[4], uint32_t b0, uint32_t b1) { mma<M>(d, f, b0, b1); });
      } else {
#pragma unroll 1
        for (int l = first_limit; l <= last_limit; ++l) {
          const auto sees = [&](int key) { return key <= l && (p.a.window <= 0 || key > l - p.a.window); };
          products(
              [&](int n, uint32_t& b0, uint32_t& b1) {
                const int key = key0 + n * 16 + 2 * t;
                b0 &= (sees(key) ? 0xffffu : 0u) | (sees(key + 1) ? 0xffff0000u : 0u);
                b1 &= (sees(key + 8) ? 0xffffu : 0u) | (sees(key + 9) ? 0xffff0000u : 0u);
              },
              [&](int m, float(&d)[4], const uint32_t(&f)[4], uint32_t b0, uint32_t b1) {
                float x[4] = {d[0], d[1], d[2], d[3]};
                mma<M>(x, f, b0, b1);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (limit[m][i >> 1] == l) d[i] = x[i];
              });
        }
      }
    }
    copies_wait<0>();

    // ---- the block's sum over its warps ----
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float v = sum[m][i];
        v += __shfl_xor_sync(ALL, v, 1);
        v += __shfl_xor_sync(ALL, v, 2);
        if (v != v && top[m][i] == -INFINITY) top[m][i] = 0.0f;  // every score NaN: not an empty row
        if (t == 0) warp_stats[warp][m * 16 + g + 8 * i] = make_float2(top[m][i], v);
      }
    __syncthreads();  // statistics written, every warp's ring is free
    float* const reduce = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = m * 16 + g + 8 * i;
        float best = -INFINITY;
#pragma unroll
        for (int k = 0; k < WARPS; ++k) best = fmaxf(best, warp_stats[k][r].x);
        const float f = top[m][i] == -INFINITY ? 0.0f : exp2_fast(top[m][i] - best);
        float* to = reduce + (warp * S::ROWS + r) * S::PITCH;
        if (top[m][i] == -INFINITY) {
          // no visible key in this warp: its accumulators are zero
          constexpr int each = D / 4;
#pragma unroll
          for (int d = 0; d < each; d += 4) *reinterpret_cast<float4*>(to + padded(t * each + d)) = make_float4(0, 0, 0, 0);
        } else if constexpr (!Q8) {
#pragma unroll
          for (int j = 0; j < D / 8; ++j)
            *reinterpret_cast<float2*>(to + padded(8 * j + 2 * t)) = make_float2(o[m][j][2 * i] * f, o[m][j][2 * i + 1] * f);
        } else {
          constexpr int SPAN = D == 64 ? 8 : 16;
#pragma unroll
          for (int h = 0; h < imax(1, D / 128); ++h)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int k = 0; k < SPAN; k += 4)
                *reinterpret_cast<float4*>(to + padded(128 * h + SPAN * (2 * t + c) + k)) =
                    make_float4(o[m][16 * h + k][2 * i + c] * f, o[m][16 * h + k + 1][2 * i + c] * f,
                                o[m][16 * h + k + 2][2 * i + c] * f, o[m][16 * h + k + 3][2 * i + c] * f);
        }
      }
    __syncthreads();

    const bool whole = steps == q.steps;
    const int slot = 2 * blockIdx.x + (pos - steps == begin ? 0 : 1);
    const auto store = [&](int r, int d, float4 v, float m, float l) {
      const int row = tile * S::ROWS + r;
      const int64_t token = q.first_row + row / p.group;
      const int h = head * p.group + row % p.group;
      const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
      A* out = static_cast<A*>(p.a.out) + token * p.a.out_token_stride + (int64_t)h * p.a.out_head_stride + d;
      *reinterpret_cast<uint2*>(out) = make_uint2(Pair<A>::pack(v.x * inv, v.y * inv), Pair<A>::pack(v.z * inv, v.w * inv));
      if (d == 0 && p.a.lse)
        p.a.lse[token * p.a.q_heads + h] = l == 0.0f ? -INFINITY : (m - S::SHIFT + log2f(l)) * kLn2;
    };
    for (int i = tid; i < rows * (D / 4); i += NT) {
      const int r = i / (D / 4), d = i % (D / 4) * 4;
      float best = -INFINITY, l = 0.0f;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) best = fmaxf(best, warp_stats[k][r].x);
      float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
      for (int k = 0; k < WARPS; ++k) {
        const float2 st = warp_stats[k][r];
        if (st.x != -INFINITY) l += st.y * exp2_fast(st.x - best);
        const float4 x = *reinterpret_cast<const float4*>(reduce + (k * S::ROWS + r) * S::PITCH + padded(d));
        v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
      }
      if (whole) {
        store(r, d, v, best, l);
      } else {
        __stcg(reinterpret_cast<float4*>(p.ws.parts + (size_t)slot * PART_FLOATS + r * D + d), v);
        if (d == 0) __stcg(p.ws.stats + slot * PART_ROWS + r, make_float2(best, l));
      }
    }
    if (whole) continue;

    // ---- a shared unit: the last CTA to arrive joins its parts ----
    const int c0 = unit_begin / share, c1 = (unit_begin + q.steps - 1) / share;
    const int slot0 = 2 * c0 + (unit_begin == c0 * share ? 0 : 1);
    const int parts = c1 - c0 + 1;
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      const uint32_t arrived = atomicAdd(p.ws.tickets + slot0, 1u);
      is_last = arrived + 1 == (uint32_t)parts;
      if (is_last) p.ws.tickets[slot0] = 0;
    }
    __syncthreads();
    if (!is_last) continue;
    __threadfence();
    const auto part_slot = [&](int k) { return k == 0 ? slot0 : 2 * (c0 + k); };
    float* const weights = reinterpret_cast<float*>(smem);  // [parts][rows]
    for (int r = tid; r < rows; r += NT) {
      float best = -INFINITY, l = 0.0f;
      for (int k = 0; k < parts; ++k) best = fmaxf(best, __ldcg(p.ws.stats + part_slot(k) * PART_ROWS + r).x);
      for (int k = 0; k < parts; ++k) {
        const float2 st = __ldcg(p.ws.stats + part_slot(k) * PART_ROWS + r);
        const float f = st.x == -INFINITY ? 0.0f : exp2_fast(st.x - best);
        weights[k * S::ROWS + r] = f;
        l += st.y * f;
      }
      warp_stats[0][r] = make_float2(best, l);
    }
    __syncthreads();
    for (int i = tid; i < rows * (D / 4); i += NT) {
      const int r = i / (D / 4), d = i % (D / 4) * 4;
      float4 v = make_float4(0, 0, 0, 0);
#pragma unroll 4
      for (int k = 0; k < parts; ++k) {
        const float4 x = __ldcg(reinterpret_cast<const float4*>(p.ws.parts + (size_t)part_slot(k) * PART_FLOATS + r * D + d));
        const float f = weights[k * S::ROWS + r];
        v.x = fmaf(f, x.x, v.x), v.y = fmaf(f, x.y, v.y), v.z = fmaf(f, x.z, v.z), v.w = fmaf(f, x.w, v.w);
      }
      store(r, d, v, warp_stats[0][r].x, warp_stats[0][r].y);
    }
    __syncthreads();
  }
}

template <typename A, bool Q8, int D, int MT>
sonic_status launch_attention(const Launch& p, cudaStream_t stream) {
  using S = Shape<A, Q8, D, MT>;
  static_assert(S::ROWS * D <= PART_FLOATS && S::ROWS <= PART_ROWS, "partial results outgrow their slots");
  // steps the kernel's 32-bit counters can meet: every page-table row full
  const SonicSequences& s = p.a.sequences;
  const double steps = (double)s.table_width * p.a.cache.page_size / S::STEP + 2;
  const double tiles = (double)s.tokens * p.group / S::ROWS + s.requests;
  if (steps * tiles * p.a.cache.kv_heads >= 4.0e9)
    return fail_with(SONIC_ERR_UNSUPPORTED, "the call spans more than 2^32 steps: split it by requests");
  const bool pdl = p.a.flags & SONIC_FLAG_PDL;
  return launch_status(launch_kernel(attention_kernel<A, Q8, D, MT>, dim3(148 * S::OCC), dim3(NT), S::SMEM, stream, pdl, p));
}

template <typename A, bool Q8>
sonic_status launch_shape(const Launch& p, cudaStream_t stream) {
  // two row tiles a CTA where a unit has more than 16 query rows (64 query accumulators a thread
  // and tile leave no room for more, nor for a second at head_dim 256)
  const SonicSequences& s = p.a.sequences;
  const int most = p.a.max_tokens > 0 ? p.a.max_tokens : (s.tokens + s.requests - 1) / s.requests;
  const bool two = (int64_t)most * p.group > 16;
  switch (p.a.cache.head_dim) {
    case 64: return two ? launch_attention<A, Q8, 64, 2>(p, stream) : launch_attention<A, Q8, 64, 1>(p, stream);
    case 128: return two ? launch_attention<A, Q8, 128, 2>(p, stream) : launch_attention<A, Q8, 128, 1>(p, stream);
    default: return launch_attention<A, Q8, 256, 1>(p, stream);
  }
}

}  // namespace
}  // namespace sonic

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
  if (a->sequences.tokens == 0) return SONIC_OK;
  if (!a->queries || !a->out) return fail_with(SONIC_ERR_INVALID_ARGUMENT, "queries and out must not be NULL");
  if (!is_aligned(a->queries, 16) || a->q_token_stride % 8 || a->q_head_stride % 8)
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "query rows must start on 16-byte boundaries");
  if (!is_aligned(a->out, 8) || a->out_token_stride % 4 || a->out_head_stride % 4)
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "output rows must start on 8-byte boundaries");
  if (!a->workspace || a->workspace_bytes < WORKSPACE_BYTES || !is_aligned(a->workspace, 16))
    return fail_with(SONIC_ERR_WORKSPACE, "workspace smaller than sonic_paged_attention_workspace_size(), or not 16-byte aligned");
  Launch p;
  p.a = *a;
  char* w = static_cast<char*>(a->workspace);
  p.ws.error = reinterpret_cast<uint32_t*>(w);
  p.ws.tickets = reinterpret_cast<uint32_t*>(w + HEADER);
  p.ws.stats = reinterpret_cast<float2*>(w + HEADER + TICKET_BYTES);
  p.ws.parts = reinterpret_cast<float*>(w + HEADER + TICKET_BYTES + STAT_BYTES);
  p.group = a->q_heads / a->cache.kv_heads;
  p.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (a->cache.page_size == 1 << i) p.page_shift = i;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool q8 = a->cache.dtype == SONIC_DTYPE_E4M3;
  if (a->dtype == SONIC_DTYPE_BF16) return q8 ? launch_shape<__nv_bfloat16, true>(p, st) : launch_shape<__nv_bfloat16, false>(p, st);
  return q8 ? launch_shape<__half, true>(p, st) : launch_shape<__half, false>(p, st);
}
