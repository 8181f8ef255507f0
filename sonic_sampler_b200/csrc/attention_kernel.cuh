// Attention of a call's new tokens over a paged key-value cache.
//
// With u_j = scale log2(e) q.k_j and any reference m, out = sum_j 2^(u_j - m) v_j / l, l = sum_j
// 2^(u_j - m): the kernel streams the keys once and keeps m, l and the unnormalised out in
// registers. Sums over disjoint key ranges join the same way, so a sequence may be cut anywhere.
// m need not be the maximum: it is raised (and l and out rescaled) only when a score passes it by
// 2^SLACK, so most tiles reduce nothing across lanes.
//
// Bound by memory: G = q_heads / kv_heads query heads share a key, and each cached element takes part in one
// multiply-add a query row, so a cached byte meets G n of them (n new tokens; e4m3) or G n / 2 (16 bits),
// far below the tensor cores' balance of some 125 a byte. The work is laid out for a continuous stream
// of the cache:
// - A unit is (request, kv head, tile of up to 8 NT query rows). All units are laid end to end by
//   their cost (their tiles of KT keys, and START for the unit itself) and cut into equal shares,
//   one a warp, whatever the lengths: a warp finds its place with a scan over `lengths`, and streams
//   its tiles through its own ring of asynchronous 16-byte copies, which runs ahead across units. No
//   block barrier until the end.
// - Where no unit can be long (the page table's width says so), a fixed number of warps takes each
//   unit instead, one warp to a cluster of eight CTAs: no scan, and parts are joined through the
//   cluster's shared memory.
// - A unit inside one warp's share goes straight to the output. One that several warps share is
//   joined in the order of its keys, first by the CTA (through shared memory), then by the last CTA
//   to arrive (by the square root of their number at a time, where many share it), through the
//   workspace. A cut that would leave only a few tiles of a unit on one side moves to the unit's end.
// - The products are transposed: keys (then dimensions) are the 16 rows of the matrix
//   instructions, query rows their 8 columns, so that few query rows waste little. tcgen05 tiles
//   are at least 64 rows by 128 lanes of tensor memory and would take their operands from shared
//   memory, where e4m3 tiles would first have to be widened; these fragments widen in registers.
// - An e4m3 key row is code * scale: the scale multiplies the score after the product. A value row's
//   scale vs multiplies the softmax weight, and m follows u_j + log2 |vs_j|, so that the fp16 weights keep
//   their precision from one value scale to another (below 2^-80 they fade). A weight times scale of less
//   than 2^-24 of the leading one is fp16 subnormal: off by less than 2^-34 of the leading row's values.
//   Codes become fp16 exactly; query rows are brought to fp16's range by a power of two.
//
// Measured (device time of repeated calls, three caches in turn, head_dim 128, 4 query heads a kv head
// unless named): 128 requests of 2048 to 16384 keys, e4m3 cache, one token each 303 us (6.2 TB/s of the
// cache's bytes); 64 requests of 1 to 8192 keys, bf16, 52 us (5.0); 2 requests of 100003 and 131072 keys,
// 8 query heads, e4m3, 89 us (5.4); one request of 700 keys 7.5 us: launch, one trip to memory and the
// join over the cluster (13 us with a page table for 131072 tokens, which takes the equal shares). With
// many query rows the products' latency bounds it, not the memory: two warps a scheduler hold all of its
// registers, and a tile of 16 keys takes a warp some 3000 cycles at 24 rows, 1500 of them the matrix
// instructions' of both warps. 32 requests of up to 4097 keys, 1 to 5 tokens, bf16, 27.5 us (2.4 TB/s, from
// L2 in part); 32 requests of 100 to 8192 keys, 4 tokens of 8 query heads, e4m3, 67 us (1.9). Skipping the
// column tiles that a request's rows do not fill changes neither: the longest shares are full ones.
// A unit's row tiles beyond those that the hint of new tokens foresees are taken one after the other, each
// over all of the request's keys: one prompt of 2000 tokens takes 302 us with its own length as the hint,
// 698 in equal shares with a hint of one token, and 8005 with a fixed number of warps and that hint.

#pragma once

#include <algorithm>
#include <type_traits>

#include "attention.h"
#include "values.cuh"

namespace sonic {
namespace {

constexpr int NT_THREADS = 32 * WARPS;
constexpr int QUEUE = 8;   // pieces a warp's copies may be ahead of its products
constexpr int START = 6;   // cost of a unit beside its tiles, in tiles (3: 32 requests of 4 x 8 query rows, e4m3, 94 us for 89)
constexpr int LEAST = 4;   // cost of a warp's share at least
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr unsigned ALL = 0xffffffffu;

__host__ __device__ constexpr int imax(int a, int b) { return a > b ? a : b; }
__host__ __device__ constexpr int imin(int a, int b) { return a < b ? a : b; }

// What another warp or CTA of this launch wrote (volatile: not from a line that this SM cached
// earlier).
__device__ __forceinline__ float4 load_part(const float4* p) {
  float4 v;
  asm volatile("ld.volatile.global.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
  return v;
}

// the same from either this CTA's shared memory or global memory
__device__ __forceinline__ float4 load_near(const float4* p) {
  float4 v;
  asm volatile("ld.volatile.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
  return v;
}
// and from shared memory of CTA `rank` of the cluster, at this CTA's address `at`
__device__ __forceinline__ float4 load_cluster(uint32_t at, int rank) {
  float4 v;
  asm volatile(
      "{\n\t.reg .u32 r;\n\t"
      "mapa.shared::cluster.u32 r, %4, %5;\n\t"
      "ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [r];\n\t}"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
      : "r"(at), "r"(rank));
  return v;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

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

// 16 bytes global -> shared; the second form writes zeros when !live
__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from));
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(live ? 16 : 0));
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(live ? 4 : 0));
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Shared-memory reads are volatile (in order with the waits above), the arithmetic is not.
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
}
__device__ __forceinline__ void load_matrices_transposed(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
}
__device__ __forceinline__ uint4 load_shared16(uint32_t at) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at));
  return r;
}
__device__ __forceinline__ uint2 load_shared8(uint32_t at) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(at));
  return r;
}
__device__ __forceinline__ uint32_t load_shared4(uint32_t at) {
  uint32_t r;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(at));
  return r;
}

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// transpose of an 8 x 8 matrix of 16-bit values held two a lane
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}

// A: activations; Q8: e4m3 cache; D: head_dim; NT: tiles of 8 query rows.
template <typename A, bool Q8, int D, int NT>
struct Shape {
  using M = std::conditional_t<Q8, __half, A>;  // type of the products' operands
  static constexpr int ROW = D * (Q8 ? 1 : 2);  // bytes of a cached row
  static constexpr int CPR = ROW / 16;          // 16-byte pieces of it
  static constexpr int RPI = 32 / CPR;          // rows one copy instruction of a warp covers
  // keys of a tile: 4 KB of rows, or 16 where four column tiles' accumulators fill the registers (32 keys:
  // 82 us against 78; at three column tiles 49 against 54 with 16)
  static constexpr int KT = Q8 && D == 128 && NT > 3 ? 16 : imin(32, imax(16, 4096 / ROW));
  static constexpr int MK = KT / 16;
  static constexpr int DT = D / 16;
  static constexpr int TILE = KT * ROW;
  static constexpr int COPIES = TILE / 512;     // copy instructions of a tile
  static constexpr int STAGE = 2 * TILE + (Q8 ? imax(2 * KT * 4, 128) : 0);  // keys, values, their scales
  static constexpr int ROWS = 8 * NT;
  // query fragments stay in registers while they and the accumulators take at most 50 of them; beyond,
  // the registers do more for the products in flight (head_dim 128, three column tiles, bf16: 27 us
  // against 33)
  static constexpr bool Q_REGISTERS = NT * DT * 6 <= 50;
  static constexpr int Q_BYTES = Q_REGISTERS ? 0 : NT * DT * 256;  // per warp
  // two CTAs an SM share its 227 KB; 16-bit rows of 256 take one CTA
  static constexpr int BUDGET = (!Q8 && D == 256 ? 54 : 27) * 1024;
  static constexpr int STAGES = imin(6, imax(2, (BUDGET - Q_BYTES) / STAGE));
  static constexpr int WARP_BYTES = STAGES * STAGE + Q_BYTES;
  static constexpr int SMEM = WARPS * WARP_BYTES;
  static constexpr int RECORD = ROWS * D * 4;  // a partial result
  static_assert(WARP_BYTES >= RECORD, "it fits the ring");
  static_assert(STAGE % 128 == 0 && WARP_BYTES % 128 == 0, "the permutations below work on addresses");
  static constexpr int OCC = SMEM <= 108 * 1024 ? 2 : 1;  // (beside 5 KB of static shared memory)
  static constexpr int CTAS = 148 * OCC;
  static_assert(ROWS * D <= PART_FLOATS && ROWS <= PART_ROWS && STAGES < QUEUE, "sizes");
  // m is raised when a score passes it by 2^SLACK; weights of fp16 products lie 2^SHIFT higher, at
  // most 2^14, so that small ones stay above fp16's smallest normal
  static constexpr float SLACK = 4.0f;
  static constexpr float SHIFT = std::is_same<M, __half>::value ? 10.0f : 0.0f;
  // A value scale of zero (or NaN, or a tiny one) counts as 2^LEAST_LOG in m: its key weighs in the sum,
  // with at most 2^(SLACK + SHIFT - LEAST_LOG) = 2^94, which the 2^30 keys of the longest request keep
  // below fp32's largest. (Appended rows have scales of 2^-69 and more.)
  static constexpr float LEAST_LOG = -80.0f;

  // byte offset of piece c of key row r, and of value row r: the pieces are permuted so that the
  // fragment reads below are free of bank conflicts. A row further on by RPI i lies 512 i further
  // on, with the bits key_xor(i), value_xor(i) flipped.
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
  static __host__ __device__ constexpr int key_xor(int i) { return !Q8 ? ((RPI * i) & 7) << 4 : D == 64 ? 0 : ((RPI * i) & 1) << 6; }
  static __host__ __device__ constexpr int value_xor(int i) { return !Q8 ? ((RPI * i) & 7) << 4 : D == 64 ? 0 : ((RPI * i) & 6) << 4; }
  // dimension of accumulator row `row` (0 to 15) of row tile j
  static __device__ __forceinline__ int dimension(int j, int row) {
    const int g = row & 7, half = row >> 3;
    if constexpr (!Q8)
      return 16 * j + row;
    else if constexpr (D == 64)
      return 8 * g + 2 * j + half;
    else
      return 128 * (j >> 3) + 16 * g + 2 * (j & 7) + half;
  }
};

struct Request {
  int new_tokens, first_row, length, begin, tiles, row_tiles;  // begin: first key any query sees
};

template <class S>
__device__ __forceinline__ Request read_request(const AttentionLaunch& p, int b) {
  const SonicSequences& s = p.a.sequences;
  Request q;
  const int length = s.lengths[b];
  if (s.cu_seqlens) {
    q.first_row = min(max(s.cu_seqlens[b], 0), s.tokens);
    q.new_tokens = min(max(s.cu_seqlens[b + 1], q.first_row), s.tokens) - q.first_row;
  } else {
    q.new_tokens = p.each;
    q.first_row = b * p.each;
  }
  q.length = min(max(length, 0), p.room);
  if (length != q.length) atomicOr(p.ws.error, (uint32_t)SONIC_DEVICE_ERR_PAGE);
  q.begin = p.window ? min(max(q.length - q.new_tokens - p.window + 1, 0), q.length) : 0;
  q.tiles = q.new_tokens > 0 && q.begin < q.length ? (q.length + S::KT - 1) / S::KT - q.begin / S::KT : 0;
  q.row_tiles = (q.new_tokens * p.group + S::ROWS - 1) / S::ROWS;
  return q;
}

// A run of tiles of one unit inside one warp's share.
struct alignas(16) Piece {
  int head, row0, rows, first_row;  // kv head; first query row of the tile, and how many; token row of the request's first query
  int offset, key0, tiles, tile0;   // position of that query (length - new); first key; tiles, the first of them
  uint32_t unit;                    // the unit's place by cost
  int unit_tiles, unused[2];
};

// A warp's place: the request that its share begins in, and the cost before that request.
struct Place {
  Request q;
  int b;
  uint32_t base;
};

// The cut at cost `at` (the boundary before warp `index`) through the unit at `unit`: how many of
// its tiles lie before it. A warp's cut keeps 2 tiles on each side, a CTA's 4: joining costs a CTA
// about as much as a tile or two, and several CTAs twice that.
__device__ __forceinline__ int cut(uint32_t at, uint32_t index, uint32_t unit, int tiles) {
  if (at <= unit) return 0;
  const uint32_t y = at - unit;
  if (y >= (uint32_t)tiles + START) return tiles;
  const int v = (int)y - START, keep = index % WARPS == 0 ? 4 : 2;
  return v < keep ? 0 : tiles - v < keep ? tiles : v;
}

// Zeros for rows that see no key, [row, row + rows) of heads [head, head + n), by threads `thread`, `thread` +
// `threads`, ... (Not inlined: rare, and the kernel's registers are not spent on it.)
template <typename A, int D>
__device__ __noinline__ void store_zeros(const AttentionLaunch& p, int row, int rows, int head, int n, int thread, int threads) {
  for (int i = thread; i < rows * n * (D / 4); i += threads) {
    const int d = i % (D / 4) * 4, h = head + i / (D / 4) % n, r = row + i / (D / 4) / n;
    A* out = static_cast<A*>(p.a.out) + (int64_t)r * p.a.out_token_stride + (int64_t)h * p.a.out_head_stride + d;
    *reinterpret_cast<uint2*>(out) = make_uint2(0, 0);
    if (d == 0 && p.a.lse) p.a.lse[(int64_t)r * p.a.q_heads + h] = -INFINITY;
  }
}

template <typename A, bool Q8, int D, int NT>
__global__ void __launch_bounds__(NT_THREADS, (Shape<A, Q8, D, NT>::OCC)) attention_kernel(const __grid_constant__ AttentionLaunch p) {
  using S = Shape<A, Q8, D, NT>;
  using M = typename S::M;
  constexpr int KT = S::KT, MK = S::MK, DT = S::DT;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint32_t scan[WARPS];
  __shared__ Place place[WARPS];
  __shared__ Piece queue[WARPS][QUEUE];
  // what a warp has of units that it shares: its first piece, and its last. The last one's partial
  // result lies in the warp's ring, a first one that others follow in the workspace.
  __shared__ Piece shared_piece[WARPS][2];
  __shared__ int shared_live[WARPS][2];  // 1: in the workspace, 2: in the ring
  __shared__ alignas(16) float2 ring_stats[WARPS][PART_ROWS];
  __shared__ alignas(16) float2 cta_stats[PART_ROWS];  // of a unit's parts in this CTA, joined
  __shared__ uint32_t arrived_last;
  __shared__ alignas(8) float query_back[WARPS][PART_ROWS];
  __shared__ const char* row_address[WARPS][32];  // key rows of a tile that is copied row by row
  constexpr size_t STATIC = sizeof(scan) + sizeof(place) + sizeof(queue) + sizeof(shared_piece) + sizeof(shared_live) + sizeof(ring_stats) +
                            sizeof(cta_stats) + sizeof(arrived_last) + sizeof(query_back) + sizeof(row_address) + 128;
  // (an SM has 228 KB, of which it keeps 1 for each CTA)
  static_assert(S::OCC * (S::SMEM + STATIC + 1024) <= 228 * 1024, "OCC CTAs share an SM");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;  // fragment row, and pair of columns
  const SonicSequences& seq = p.a.sequences;
  const SonicPagedCache& cache = p.a.cache;
  const int heads = cache.kv_heads;

  grid_dependency_trigger();
  if (tid < 2 * WARPS) shared_live[tid >> 1][tid & 1] = 0;
  grid_dependency_wait();

  // k / page_size, for k below 2^31
  const auto page_of = [&](int k) {
    if (p.page_shift < 0) return k;
    const uint32_t high = __umulhi((uint32_t)k, p.page_inverse);
    return (int)((high + (((uint32_t)k - high) >> 1)) >> p.page_shift);
  };
  // query row r of a request belongs to its token r / group
  const auto token_of = [&](int row) { return p.group == 1 ? row : (int)__umulhi((uint32_t)row, p.group_inverse); };
  const auto out_row = [&](const Piece& u, int r) {
    const int row = u.row0 + r, step = token_of(row), token = u.first_row + step, h = u.head * p.group + row - step * p.group;
    return static_cast<A*>(p.a.out) + (int64_t)token * p.a.out_token_stride + (int64_t)h * p.a.out_head_stride;
  };
  const auto store_lse = [&](const Piece& u, int r, float m, float l) {
    if (!p.a.lse) return;
    const int row = u.row0 + r, step = token_of(row), token = u.first_row + step, h = u.head * p.group + row - step * p.group;
    p.a.lse[(int64_t)token * p.a.q_heads + h] = l == 0.0f ? -INFINITY : (m - S::SHIFT + log2f(l)) * kLn2;
  };
  const auto one_over = [](float l) { return l == 0.0f ? 0.0f : __frcp_rn(l); };
  // keys that some row of the piece sees: [from, to); the others of a tile become zeros
  const auto seen = [&](const Piece& u, int& from, int& to) {
    const int first = u.offset + token_of(u.row0), last = u.offset + token_of(u.row0 + u.rows - 1);
    from = p.window ? max(first - p.window + 1, 0) : 0;
    to = last + 1;
  };
  // ---- what this CTA does ----
  Request q{};                                   // the request that the copies' side is in
  int b = 0, direct_head = 0, direct_tile = 0, direct_part = 0;
  uint32_t share = 0, cta_begin = 0, cta_end = 0, base = 0;
  bool any_empty = false;
  const auto unit_cost = [](const Request& r) { return r.tiles > 0 ? (uint32_t)r.tiles + START : 0u; };
  if (p.direct) {
    // one (request, head) and every p.direct'th row tile of it, for unit_warps warps
    const int ctas = p.unit_warps / WARPS;
    int index = ctas ? blockIdx.x / ctas : blockIdx.x * WARPS + warp;
    direct_part = ctas ? (blockIdx.x - index * ctas) * WARPS + warp : 0;
    const int tile_of = index;
    index /= p.direct;
    direct_tile = tile_of - index * p.direct;
    b = index / heads;
    direct_head = index - b * heads;
    if (b >= seq.requests) return;
    q = read_request<S>(p, b);
    if (direct_tile == 0) {  // rows of no request
      const int thread = direct_part * 32 + lane, threads = p.unit_warps * 32, next = q.first_row + q.new_tokens;
      if (b == 0 && q.first_row > 0) store_zeros<A, D>(p, 0, q.first_row, direct_head * p.group, p.group, thread, threads);
      if (b == seq.requests - 1 && next < seq.tokens)
        store_zeros<A, D>(p, next, seq.tokens - next, direct_head * p.group, p.group, thread, threads);
    }
    if (q.tiles == 0) {
      if (direct_tile == 0)
        store_zeros<A, D>(p, q.first_row, q.new_tokens, direct_head * p.group, p.group, direct_part * 32 + lane, p.unit_warps * 32);
      return;
    }
    if (direct_tile >= q.row_tiles) return;
  } else {
    const int per = (seq.requests + NT_THREADS - 1) / NT_THREADS;
    const int b_lo = min(tid * per, seq.requests), b_hi = min(b_lo + per, seq.requests);
    uint32_t mine = 0;
    // The rows before the first request's (even threads) and behind the last one's (odd threads) belong to no
    // request. (Looked at only after the loop, whose loads then come back together with this one: 32 requests
    // of up to 5 tokens take 27.5 us with it and without; 28.3 where the rows are read again when needed.)
    const bool odd = tid & 1;
    int edge = odd ? seq.tokens : 0;
    if (seq.cu_seqlens) edge = seq.cu_seqlens[odd ? seq.requests : 0];
    for (int i = b_lo; i < b_hi; ++i) {
      q = read_request<S>(p, i);
      mine += unit_cost(q) * heads * q.row_tiles;
      any_empty = any_empty || (q.tiles == 0 && q.new_tokens > 0);
    }
    uint32_t upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(ALL, upto, d);
      if (lane >= d) upto += o;
    }
    if (lane == 31) scan[warp] = upto;
    edge = min(max(edge, 0), seq.tokens);
    const int outside = odd ? seq.tokens - edge : edge;
    any_empty = __syncthreads_or(any_empty || outside > 0);
    uint32_t before = upto - mine, total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) before += scan[w];
      total += scan[w];
    }
    share = max((total + S::CTAS * WARPS - 1) / (S::CTAS * WARPS), (uint32_t)LEAST);
    cta_begin = min(blockIdx.x * WARPS * share, total);
    cta_end = min(cta_begin + WARPS * share, total);
#pragma unroll 1
    for (int w = 0; w < WARPS; ++w) {
      const uint32_t at = cta_begin + w * share;
      if (at >= cta_end || at < before || at - before >= mine) continue;
      uint32_t so_far = before;
      Request r = q;
      int i = b_lo;
      if (per > 1)
        for (;; ++i) {
          r = read_request<S>(p, i);
          const uint32_t n = unit_cost(r) * heads * r.row_tiles;
          if (at - so_far < n) break;
          so_far += n;
        }
      place[w] = {r, i, so_far};
    }
    __syncthreads();
    if (any_empty) {
      for (int i = blockIdx.x; i < seq.requests; i += S::CTAS) {
        const Request r = read_request<S>(p, i);
        if (r.tiles == 0) store_zeros<A, D>(p, r.first_row, r.new_tokens, 0, p.a.q_heads, tid, NT_THREADS);
      }
      if (outside > 0)
        store_zeros<A, D>(p, odd ? edge : 0, outside, 0, p.a.q_heads, (blockIdx.x * NT_THREADS + tid) >> 1, S::CTAS * NT_THREADS / 2);
    }
    if (cta_begin >= cta_end) return;
    q = place[warp].q;
    b = place[warp].b;
    base = place[warp].base;
  }

  const float score_scale = p.a.scale * kLog2e;
  const uint32_t ring = shared_address(smem) + warp * S::WARP_BYTES;
  const uint32_t q_smem = ring + S::STAGES * S::STAGE;
  const uint32_t warp0 = blockIdx.x * WARPS;
  // where the pages let 16 or KT consecutive keys be copied as one run of bytes
  const bool whole = MK == 1 ? p.packed >= 1 : p.packed >= 2;
  const int key_lane = whole ? 0 : p.packed ? lane & (KT - 16) : lane & (KT - 1);
  const int key_span = whole ? KT - 1 : p.packed ? 15 : 0;
  // this lane's piece of a copy instruction's rows
  const int row_lane = lane / S::CPR, piece_lane = lane % S::CPR;
  const uint32_t key_to = S::key_at(row_lane, piece_lane), value_to = S::TILE + S::value_at(row_lane, piece_lane);
  const int64_t value_delta = static_cast<const char*>(cache.values) - static_cast<const char*>(cache.keys);

#pragma unroll 1
  while (true) {  // once, or in direct mode once a row tile
    // ---- the copies' side: runs STAGES - 1 tiles ahead ----
    int queued = 0, left = 0, key = 0, from = 0, to = 0, stage_in = 0;
    // Pages of the tiles ahead, asked for a step before they are needed. Runs of keys: lane l holds the
    // page of run l from the batch's first on, from its first use also where the run lies; else of
    // key_lane in the next tile.
    int pages = 0, batch = 0;
    int64_t run_at = 0, run_scale = 0;
    uint32_t runs_there = 0;
    bool ready = false;
    int64_t head_at = 0, scale_head_at = 0;
    const int32_t* table = nullptr;
    // the next unit of request b, and its head and row tile
    int next_head = 0, next_row = 0;
    uint32_t unit = 0, cost = 0;
    const uint32_t begin = cta_begin + warp * share, end = min(begin + share, cta_end);
    const auto enter = [&](int head, int row_tile, int tile, int tiles) {
      Piece u;
      u.head = head;
      u.row0 = row_tile * S::ROWS;
      u.rows = min(S::ROWS, q.new_tokens * p.group - u.row0);
      u.first_row = q.first_row;
      u.offset = q.length - q.new_tokens;
      u.key0 = (q.begin / KT + tile) * KT;
      u.tiles = tiles;
      u.tile0 = tile;
      u.unit = unit;
      u.unit_tiles = q.tiles;
      if (lane == 0) queue[warp][queued % QUEUE] = u;
      ++queued;
      left = tiles;
      batch = 32;
      key = u.key0;
      seen(u, from, to);
      head_at = head * cache.head_stride;
      scale_head_at = head * cache.scale_head_stride;
      table = seq.page_table + (int64_t)b * seq.table_stride;
    };
    if (p.direct) {
      const int each = (q.tiles + p.unit_warps - 1) / p.unit_warps, tile = direct_part * each;
      if (tile < q.tiles) enter(direct_head, direct_tile, tile, min(each, q.tiles - tile));
    } else if (begin < end) {
      cost = unit_cost(q);
      const uint32_t index = (begin - base) / cost;
      unit = base + index * cost;
      next_head = q.row_tiles == 1 ? index : index / q.row_tiles;
      next_row = index - next_head * q.row_tiles;
    } else {
      unit = end;
    }
    // Copy the next tile, and ask for the page of the one after: this lane's key is key_lane further
    // on than the tile's first.
    const auto copy_next = [&]() {
      if (ready) {
        const uint32_t stage = ring + (uint32_t)stage_in * S::STAGE;
        stage_in = stage_in + 1 == S::STAGES ? 0 : stage_in + 1;
        // where key_lane of the tile lies, and whether its page is in the cache
        const auto resolve = [&](int k, int64_t& at, int64_t& scale) {
          const bool wanted = k + key_span >= from && k < to;
          const bool there = wanted && (uint32_t)pages < (uint32_t)cache.pages;
          if (wanted && !there) atomicOr(p.ws.error, (uint32_t)SONIC_DEVICE_ERR_PAGE);
          const int slot = k - page_of(k) * cache.page_size;
          at = there ? (pages * cache.page_stride + head_at + slot * cache.slot_stride) * (Q8 ? 1 : 2) : 0;
          if constexpr (Q8) scale = there ? pages * cache.scale_page_stride + scale_head_at + slot : 0;
          return there;
        };
        int64_t at, scale_at = 0;
        bool there;
        if (key_span) {
          if (batch == 0) runs_there = __ballot_sync(ALL, resolve(key + lane * (key_span + 1), run_at, run_scale));
          const int run = batch + (whole ? 0 : (lane >> 4) & (MK - 1));
          at = __shfl_sync(ALL, run_at, run);
          if constexpr (Q8) scale_at = __shfl_sync(ALL, run_scale, run);
          there = (runs_there >> run) & 1;
          batch += whole ? 1 : MK;
        } else {
          there = resolve(key + key_lane, at, scale_at);
        }
        const bool all = key >= from && key + KT <= to;
        if (whole && all && there) {
          const char* src = static_cast<const char*>(cache.keys) + at + lane * 16;
          const uint32_t kd = stage + key_to, vd = stage + value_to;
#pragma unroll
          for (int i = 0; i < S::COPIES; ++i) {
            copy16((kd ^ S::key_xor(i)) + i * 512, src + i * 512);
            copy16((vd ^ S::value_xor(i)) + i * 512, src + value_delta + i * 512);
          }
        } else if (MK == 2 && key_span && !whole && all && __all_sync(ALL, there)) {
          const char* src[MK];
#pragma unroll
          for (int h = 0; h < MK; ++h) src[h] = static_cast<const char*>(cache.keys) + __shfl_sync(ALL, at, h * 16) + lane * 16;
          const uint32_t kd = stage + key_to, vd = stage + value_to;
#pragma unroll
          for (int i = 0; i < S::COPIES; ++i) {
            const char* from16 = src[i / (S::COPIES / MK)] + i % (S::COPIES / MK) * 512;
            copy16((kd ^ S::key_xor(i)) + i * 512, from16);
            copy16((vd ^ S::value_xor(i)) + i * 512, from16 + value_delta);
          }
        } else {
          // row by row: lane r finds the address of key r
          const int r_lane = lane & (KT - 1);
          const int64_t row_at = key_span ? at + (int64_t)(r_lane - key_lane) * cache.slot_stride * (Q8 ? 1 : 2) : at;
          const bool row_there = there && key + r_lane >= from && key + r_lane < to;
          row_address[warp][lane] = row_there ? static_cast<const char*>(cache.keys) + row_at : nullptr;
          __syncwarp();
          const uint32_t kd = stage + key_to, vd = stage + value_to;
#pragma unroll
          for (int i = 0; i < S::COPIES; ++i) {
            const char* row = row_address[warp][i * S::RPI + row_lane];
            const char* src = row ? row + piece_lane * 16 : static_cast<const char*>(cache.keys);
            copy16((kd ^ S::key_xor(i)) + i * 512, src, row != nullptr);
            copy16((vd ^ S::value_xor(i)) + i * 512, row ? src + value_delta : src, row != nullptr);
          }
        }
        if constexpr (Q8) {
          // lane r copies the scales of key r
          if (lane < KT) {
            const bool live = there && key + lane >= from && key + lane < to;
            const int64_t sat = live ? scale_at + (key_span ? lane - key_lane : 0) : 0;
            copy4(stage + 2 * S::TILE + lane * 4, cache.key_scales + sat, live);
            copy4(stage + 2 * S::TILE + KT * 4 + lane * 4, cache.value_scales + sat, live);
          }
        }
        --left;
        key += KT;
      }
      while (left == 0 && unit < end) {
        if (next_head == heads) {
          do q = read_request<S>(p, ++b);
          while (q.tiles == 0);
          cost = unit_cost(q);
          next_head = next_row = 0;
        }
        const int tile = cut(begin, warp0 + warp, unit, q.tiles);
        const int tiles = cut(end, warp0 + warp + 1, unit, q.tiles) - tile;
        if (tiles > 0) enter(next_head, next_row, tile, tiles);
        unit += cost;
        if (++next_row == q.row_tiles) next_row = 0, ++next_head;
      }
      ready = left > 0;
      if (ready && (!key_span || batch == 32)) {
        // (a run of keys may begin before `from`: its page exists all the same)
        const int k = key + (key_span ? lane * (key_span + 1) : key_lane);
        batch = 0;
        pages = -1;
        if (k + key_span >= from && k < to) pages = table[page_of(k)];
      }
      copies_commit();
    };

    // ---- the products' side ----
    Piece u{};
    // e4m3: undoes the power of two of query columns 2t and 2t + 1 (many: in shared memory)
    float row_scale[S::Q_REGISTERS ? NT : 1][2];
    uint32_t qf[S::Q_REGISTERS ? NT : 1][S::Q_REGISTERS ? DT : 1][2];
    float o[DT][NT][4], ref[NT][2], sum[NT][2];
    int u_from = 0, u_to = 0, all_from = 0, all_to = 0, first_limit = 0, last_limit = 0;
    int stage_out = 0, todo = 0, taken = 0;

    // last key that query column `col` sees
    const auto limit = [&](int col) { return col < u.rows ? u.offset + token_of(u.row0 + col) : -1; };
    const auto begin_piece = [&]() {
      u = queue[warp][taken % QUEUE];
      ++taken;
      todo = u.tiles;
      seen(u, u_from, u_to);
      first_limit = u.offset + token_of(u.row0);
      last_limit = u_to - 1;
      // keys that every row sees: [all_from, all_to)
      all_to = first_limit + 1;
      all_from = p.window ? max(last_limit - p.window + 1, 0) : 0;
      // all of the queries' loads first
      uint2 raw[NT][DT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int r = n * 8 + g, row = u.row0 + r, step = token_of(row);
        const bool live = r < u.rows;
        const A* src = static_cast<const A*>(p.a.queries);
        if (live) src += (int64_t)(u.first_row + step) * p.a.q_token_stride + (int64_t)(u.head * p.group + row - step * p.group) * p.a.q_head_stride;
#pragma unroll
        for (int k = 0; k < DT; ++k) {
          raw[n][k] = make_uint2(0, 0);
          if constexpr (Q8) {
            // a lane's products run over 16 consecutive dimensions (one 16-byte piece of codes), 4 a step
            if (live) raw[n][k] = *reinterpret_cast<const uint2*>(src + 64 * (k / 4) + 16 * t + 4 * (k % 4));
          } else if (live) {
            raw[n][k].x = *reinterpret_cast<const uint32_t*>(src + 16 * k + 2 * t);
            raw[n][k].y = *reinterpret_cast<const uint32_t*>(src + 16 * k + 8 + 2 * t);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float back = 1.0f;
        if constexpr (Q8) {
          uint32_t top = 0;
#pragma unroll
          for (int k = 0; k < DT; ++k) {
            const float2 x = Pair<A>::unpack(raw[n][k].x), y = Pair<A>::unpack(raw[n][k].y);
            top = max(max(top, max(magnitude_bits(x.x), magnitude_bits(x.y))), max(magnitude_bits(y.x), magnitude_bits(y.y)));
          }
          top = max(top, __shfl_xor_sync(ALL, top, 1));
          top = max(top, __shfl_xor_sync(ALL, top, 2));
          // the power of two that brings the row's largest magnitude to [2^14, 2^15); rows of zeros,
          // infinities or NaN stay as they are
          const int exponent = (int)(top >> 23);  // biased
          const int up = exponent == 0 || exponent == 255 ? 0 : min(max(127 + 14 - exponent, -126), 126);
          const float factor = __uint_as_float((uint32_t)(127 + up) << 23);
          back = __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
          for (int k = 0; k < DT; ++k) {
            const float2 x = Pair<A>::unpack(raw[n][k].x), y = Pair<A>::unpack(raw[n][k].y);
            raw[n][k] = make_uint2(Pair<__half>::pack(x.x * factor, x.y * factor), Pair<__half>::pack(y.x * factor, y.y * factor));
          }
        }
#pragma unroll
        for (int k = 0; k < DT; ++k) {
          if constexpr (S::Q_REGISTERS)
            qf[n][k][0] = raw[n][k].x, qf[n][k][1] = raw[n][k].y;
          else
            asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(q_smem + ((n * DT + k) * 32 + lane) * 8), "r"(raw[n][k].x), "r"(raw[n][k].y));
        }
        if constexpr (Q8 && !S::Q_REGISTERS)
          if (t == 0) query_back[warp][n * 8 + g] = back;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if constexpr (Q8 && S::Q_REGISTERS) row_scale[n][c] = __shfl_sync(ALL, back, (2 * t + c) * 4);
          ref[n][c] = -INFINITY;
          sum[n][c] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < DT; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[j][n][i] = 0.0f;
      }
    };

    // Lane offsets of the fragment reads. 16-bit rows: row lane & 15 (keys), or (lane & 7) + 8 (lane
    // >> 4) (values), piece (lane >> 4) or (lane >> 3) & 1; pieces 2 k further on flip bits of the
    // permuted address, 8 further on add 128. Codes: see the products.
    const uint32_t key_read = Q8 ? S::key_at(g, t) : S::key_at(lane & 15, lane >> 4);
    const uint32_t value_read = S::TILE + (!Q8      ? S::value_at((lane & 7) + ((lane >> 4) << 3), (lane >> 3) & 1)
                                           : D == 64 ? S::value_at(2 * t, g >> 1) + (g & 1) * 8
                                                     : S::value_at(2 * t, g));

    const auto tile_products = [&](uint32_t stage, int key0) {
      const uint32_t keys = stage + key_read, values = stage + value_read;
      // ---- scores: s[m][n] has rows (keys) g, g + 8 and columns (queries) 2t, 2t + 1 ----
      float s[MK][NT][4];
#pragma unroll
      for (int m = 0; m < MK; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[m][n][i] = 0.0f;
      const auto query = [&](int n, int k, uint32_t& b0, uint32_t& b1) {
        if constexpr (S::Q_REGISTERS) {
          b0 = qf[n][k][0], b1 = qf[n][k][1];
        } else {
          const uint2 v = load_shared8(q_smem + ((n * DT + k) * 32 + lane) * 8);
          b0 = v.x, b1 = v.y;
        }
      };
      if constexpr (!Q8) {
#pragma unroll
        for (int k = 0; k < DT; ++k) {
          uint32_t b0[NT], b1[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) query(n, k, b0[n], b1[n]);
#pragma unroll
          for (int m = 0; m < MK; ++m) {
            uint32_t kf[4];
            load_matrices(kf, (keys ^ ((2 * k & 7) << 4)) + (k >> 2) * 128 + m * 16 * S::ROW);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma<M>(s[m][n], kf, b0[n], b1[n]);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
          uint4 lo[MK], hi[MK];  // codes of keys g and g + 8, pieces 4 j + t
          const uint32_t at = D == 64 ? keys : (keys ^ ((j & 1) << 6)) + (j >> 1) * 128;
#pragma unroll
          for (int m = 0; m < MK; ++m) {
            lo[m] = load_shared16(at + m * 16 * S::ROW);
            hi[m] = load_shared16(at + (m * 16 + 8) * S::ROW);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t b0[NT], b1[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) query(n, 4 * j + i, b0[n], b1[n]);
#pragma unroll
            for (int m = 0; m < MK; ++m) {
              const uint32_t x = i == 0 ? lo[m].x : i == 1 ? lo[m].y : i == 2 ? lo[m].z : lo[m].w;
              const uint32_t y = i == 0 ? hi[m].x : i == 1 ? hi[m].y : i == 2 ? hi[m].z : hi[m].w;
              const uint32_t kf[4] = {e4m3_to_half2((uint16_t)x), e4m3_to_half2((uint16_t)y), e4m3_to_half2((uint16_t)(x >> 16)),
                                      e4m3_to_half2((uint16_t)(y >> 16))};
#pragma unroll
              for (int n = 0; n < NT; ++n) mma<M>(s[m][n], kf, b0[n], b1[n]);
            }
          }
        }
      }

      // ---- softmax weights ----
      const bool masked = key0 < all_from || key0 + KT > all_to;
      [[maybe_unused]] float back[NT][2];
      if constexpr (Q8) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if constexpr (S::Q_REGISTERS) {
            back[n][0] = row_scale[n][0], back[n][1] = row_scale[n][1];
          } else {
            const uint2 v = load_shared8(shared_address(query_back[warp] + n * 8 + 2 * t));
            back[n][0] = __uint_as_float(v.x), back[n][1] = __uint_as_float(v.y);
          }
        }
      }
      [[maybe_unused]] float vs[MK][2], lv[MK][2];  // value scale of keys g, g + 8, and its logarithm
#pragma unroll
      for (int m = 0; m < MK; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float ks = score_scale;
          lv[m][h] = 0.0f;
          if constexpr (Q8) {
            const uint32_t at = stage + 2 * S::TILE + (m * 16 + 8 * h + g) * 4;
            ks *= __uint_as_float(load_shared4(at));
            vs[m][h] = __uint_as_float(load_shared4(at + KT * 4));
            lv[m][h] = fmaxf(log2_fast(fabsf(vs[m][h])), S::LEAST_LOG);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float v = s[m][n][2 * h + c] * ks;
              if constexpr (Q8) v *= back[n][c];
              s[m][n][2 * h + c] = v;
            }
        }
      if (masked) {
#pragma unroll
        for (int m = 0; m < MK; ++m)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = key0 + m * 16 + g + 8 * (i >> 1), l = limit(n * 8 + 2 * t + (i & 1));
              if (key > l || (p.window && key <= l - p.window)) s[m][n][i] = -INFINITY;
            }
      }
      float top[NT][2];
      bool rise = false;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float v = -INFINITY;
#pragma unroll
          for (int m = 0; m < MK; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) v = fmaxf(v, Q8 ? s[m][n][2 * h + c] + lv[m][h] : s[m][n][2 * h + c]);
          top[n][c] = v;
          rise = rise || v > ref[n][c] + S::SLACK;
        }
      if (__any_sync(ALL, rise)) {
        // An infinite value scale makes the output so, and must leave the sum alone: it counts as 1. (Looked
        // at here alone, where its key always leads: on every key's way it costs 1 % of a long call.)
        if constexpr (Q8) {
#pragma unroll
          for (int m = 0; m < MK; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (lv[m][h] == INFINITY) lv[m][h] = 0.0f;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float alpha[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float v = top[n][c];
            if constexpr (Q8) {
              v = -INFINITY;
#pragma unroll
              for (int m = 0; m < MK; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) v = fmaxf(v, s[m][n][2 * h + c] + lv[m][h]);
            }
            v = fmaxf(v, __shfl_xor_sync(ALL, v, 4));
            v = fmaxf(v, __shfl_xor_sync(ALL, v, 8));
            v = fmaxf(v, __shfl_xor_sync(ALL, v, 16));
            v = fmaxf(v, ref[n][c]);
            alpha[c] = ref[n][c] == -INFINITY ? 0.0f : exp2_fast(ref[n][c] - v);
            ref[n][c] = v;
            sum[n][c] *= alpha[c];
          }
#pragma unroll
          for (int j = 0; j < DT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[j][n][i] *= alpha[i & 1];
        }
      }
      // the weights as the second product's right operand: rows (keys) by pairs, columns (queries) g
      uint32_t wf[MK][NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float low[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) low[c] = (ref[n][c] == -INFINITY ? 0.0f : ref[n][c]) - S::SHIFT;
#pragma unroll
        for (int m = 0; m < MK; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float e0 = exp2_fast(s[m][n][2 * h] - low[0]), e1 = exp2_fast(s[m][n][2 * h + 1] - low[1]);
            sum[n][0] += e0;
            sum[n][1] += e1;
            if constexpr (Q8) {
              e0 *= vs[m][h], e1 *= vs[m][h];
              // a masked key weighs 0 whatever its scale holds
              if (masked) {
                if (s[m][n][2 * h] == -INFINITY) e0 = 0.0f;
                if (s[m][n][2 * h + 1] == -INFINITY) e1 = 0.0f;
              }
            }
            wf[m][n][h] = transpose8(Pair<M>::pack(e0, e1));
          }
      }

      // ---- out += values x weights: o[j][n] has rows (dimensions) g, g + 8, columns (queries) 2t, 2t + 1 ----
      // A key that some rows of the tile see and others do not: 0 x infinity or NaN in its values
      // must not reach the others. Rare, so looked for first.
      if (masked && last_limit > first_limit) {
        bool strange = false;
        const auto look = [&](uint32_t x) {
          if constexpr (Q8) {
            const uint32_t m = x & 0x7f7f7f7fu;
            strange = strange || (m & 0xff) == 0x7f || (m >> 8 & 0xff) == 0x7f || (m >> 16 & 0xff) == 0x7f || m >> 24 == 0x7f;
          } else {
            constexpr uint32_t E = std::is_same<A, __half>::value ? 0x7c00u : 0x7f80u;
            strange = strange || (x & E) == E || (x >> 16 & E) == E;
          }
        };
#pragma unroll 2
        for (int i = lane; i < S::TILE / 16; i += 32) {
          const uint4 x = load_shared16(stage + S::TILE + i * 16);
          look(x.x), look(x.y), look(x.z), look(x.w);
        }
        if (__any_sync(ALL, strange)) {
          // once for every query of the tile, with the values that it does not see taken as zeros,
          // keeping the results of its rows only. The accumulators pass through local memory, so
          // that these loops need not be unrolled.
          float4 acc[DT * NT];
#pragma unroll
          for (int j = 0; j < DT; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[j * NT + n] = make_float4(o[j][n][0], o[j][n][1], o[j][n][2], o[j][n][3]);
#pragma unroll 1
          for (int j = 0; j < DT; ++j) {
#pragma unroll 1
            for (int l = first_limit; l <= last_limit; ++l) {
              const auto sees = [&](int k) { return k <= l && (!p.window || k > l - p.window); };
              float x[NT][4];
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                const float4 v = acc[j * NT + n];
                x[n][0] = v.x, x[n][1] = v.y, x[n][2] = v.z, x[n][3] = v.w;
              }
#pragma unroll
              for (int m = 0; m < MK; ++m) {
                uint32_t vf[4];
                if constexpr (!Q8) {
                  load_matrices_transposed(vf, stage + S::TILE + S::value_at(m * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * j + ((lane >> 3) & 1)));
                } else {
                  // the four keys' words that hold the row tile's two dimensions
                  const int first = S::dimension(j, g), at = first & ~3;
                  uint32_t word[4];
#pragma unroll
                  for (int i = 0; i < 4; ++i)
                    word[i] = load_shared4(stage + S::TILE + S::value_at(m * 16 + 2 * t + (i & 1) + (i >> 1) * 8, at / 16) + at % 16);
                  const uint32_t pick = first & 2 ? 0x7362 : 0x5140;
                  const uint32_t lo = __byte_perm(word[0], word[1], pick), hi = __byte_perm(word[2], word[3], pick);
                  vf[0] = e4m3_to_half2((uint16_t)lo), vf[1] = e4m3_to_half2((uint16_t)(lo >> 16));
                  vf[2] = e4m3_to_half2((uint16_t)hi), vf[3] = e4m3_to_half2((uint16_t)(hi >> 16));
                }
                const int k = key0 + m * 16 + 2 * t;
                const uint32_t lo = (sees(k) ? 0xffffu : 0u) | (sees(k + 1) ? 0xffff0000u : 0u);
                const uint32_t hi = (sees(k + 8) ? 0xffffu : 0u) | (sees(k + 9) ? 0xffff0000u : 0u);
                vf[0] &= lo, vf[1] &= lo, vf[2] &= hi, vf[3] &= hi;
#pragma unroll
                for (int n = 0; n < NT; ++n) mma<M>(x[n], vf, wf[m][n][0], wf[m][n][1]);
              }
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (limit(n * 8 + 2 * t + (i & 1)) == l) reinterpret_cast<float*>(acc + j * NT + n)[i] = x[n][i];
            }
          }
#pragma unroll
          for (int j = 0; j < DT; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const float4 v = acc[j * NT + n];
              o[j][n][0] = v.x, o[j][n][1] = v.y, o[j][n][2] = v.z, o[j][n][3] = v.w;
            }
          return;
        }
      }
#pragma unroll
      for (int m = 0; m < MK; ++m) {
        if constexpr (!Q8) {
#pragma unroll
          for (int j = 0; j < DT; ++j) {
            uint32_t vf[4];
            load_matrices_transposed(vf, (values ^ ((2 * j & 7) << 4)) + (j >> 2) * 128 + m * 16 * S::ROW);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma<M>(o[j][n], vf, wf[m][n][0], wf[m][n][1]);
          }
        } else {
          // lane (g, t) reads keys 2t, 2t + 1, 2t + 8, 2t + 9, dimensions [D/8 g, D/8 (g + 1)) (16
          // at a time): the rows of row tile j are then dimensions 16 g + 2 j and 16 g + 2 j + 1
          constexpr int SPAN = D == 64 ? 8 : 16;
#pragma unroll
          for (int h = 0; h < imax(1, D / 128); ++h) {
            uint32_t x[4][SPAN / 4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if constexpr (D == 64) {
                // rows lie two to 128 bytes: an odd one flips bit 6
                const uint2 v = load_shared8((i & 1 ? values ^ 64u : values) + (m * 16 + (i >> 1) * 8) * S::ROW);
                x[i][0] = v.x, x[i][1] = v.y;
              } else {
                const uint4 v = load_shared16(values + h * 128 + (m * 16 + (i & 1) + (i >> 1) * 8) * S::ROW);
                x[i][0] = v.x, x[i][1] = v.y, x[i][2] = v.z, x[i][3] = v.w;
              }
            }
#pragma unroll
            for (int k = 0; k < SPAN / 4; ++k)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const uint32_t lo = __byte_perm(x[0][k], x[1][k], i == 0 ? 0x5140 : 0x7362);
                const uint32_t hi = __byte_perm(x[2][k], x[3][k], i == 0 ? 0x5140 : 0x7362);
                const uint32_t vf[4] = {e4m3_to_half2((uint16_t)lo), e4m3_to_half2((uint16_t)(lo >> 16)), e4m3_to_half2((uint16_t)hi),
                                        e4m3_to_half2((uint16_t)(hi >> 16))};
#pragma unroll
                for (int n = 0; n < NT; ++n) mma<M>(o[h * 8 + 2 * k + i][n], vf, wf[m][n][0], wf[m][n][1]);
              }
          }
        }
      }
    };

    // Row tile j of 8 query rows (from n8 on) into the output; to0 and to1 are the rows that the lane
    // writes: query row g, or with codes 2t and 2t + 1.
    const auto store_rows = [&](const Piece& x, int n8, A*& to0, A*& to1) {
      const int r0 = n8 + (Q8 ? 2 * t : g);
      to0 = r0 < x.rows ? out_row(x, r0) : nullptr;
      to1 = Q8 && r0 + 1 < x.rows ? out_row(x, r0 + 1) : nullptr;
    };
    const auto store_tile = [&](A* to0, A* to1, int j, const float4& v, float inv0, float inv1) {
      if constexpr (!Q8) {
        // pairs of queries a lane -> pairs of dimensions a lane
        const uint32_t x = transpose8(Pair<A>::pack(v.x * inv0, v.y * inv1));
        const uint32_t y = transpose8(Pair<A>::pack(v.z * inv0, v.w * inv1));
        if (to0) {
          *reinterpret_cast<uint32_t*>(to0 + 16 * j + 2 * t) = x;
          *reinterpret_cast<uint32_t*>(to0 + 16 * j + 8 + 2 * t) = y;
        }
      } else {
        const int d = S::dimension(j, g);
        if (to0) *reinterpret_cast<uint32_t*>(to0 + d) = Pair<A>::pack(v.x * inv0, v.z * inv0);
        if (to1) *reinterpret_cast<uint32_t*>(to1 + d) = Pair<A>::pack(v.y * inv1, v.w * inv1);
      }
    };

    const auto end_piece = [&]() {
      // the columns' sums over the lanes that share them
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float v = sum[n][c];
          v += __shfl_xor_sync(ALL, v, 4);
          v += __shfl_xor_sync(ALL, v, 8);
          v += __shfl_xor_sync(ALL, v, 16);
          sum[n][c] = v;
          if (v != v && ref[n][c] == -INFINITY) ref[n][c] = 0.0f;  // every score NaN: not an empty row
        }
      if (u.tiles == u.unit_tiles) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float inv[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            inv[c] = one_over(sum[n][c]);
            if (g == 0 && n * 8 + 2 * t + c < u.rows) store_lse(u, n * 8 + 2 * t + c, ref[n][c], sum[n][c]);
          }
          A *to0, *to1;
          store_rows(u, n * 8, to0, to1);
#pragma unroll
          for (int j = 0; j < DT; ++j) store_tile(to0, to1, j, make_float4(o[j][n][0], o[j][n][1], o[j][n][2], o[j][n][3]), inv[0], inv[1]);
        }
      } else {
        const int which = taken == 1 ? 0 : 1;  // the share's first piece, or its last
        const bool final = taken == queued && !ready;
        const size_t slot = warp0 + warp;
        if (final) {
          copies_wait<0>();
          __syncwarp();  // the ring is free
        }
        float4* const to = final ? reinterpret_cast<float4*>(smem + warp * S::WARP_BYTES) : p.ws.parts + slot * (PART_FLOATS / 4);
        float2* const stats = final ? ring_stats[warp] : p.ws.stats + slot * PART_ROWS;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (n * 8 + 2 * t >= u.rows) continue;
#pragma unroll
          for (int j = 0; j < DT; ++j) to[(j * NT + n) * 32 + lane] = make_float4(o[j][n][0], o[j][n][1], o[j][n][2], o[j][n][3]);
          if (g == 0)
#pragma unroll
            for (int c = 0; c < 2; ++c) stats[n * 8 + 2 * t + c] = make_float2(ref[n][c], sum[n][c]);
        }
        if (lane == 0) {
          shared_piece[warp][which] = u;
          shared_live[warp][which] = final ? 2 : 1;
        }
      }
    };

    // the first STAGES steps only copy (the very first only asks for the first tile's page)
#pragma unroll 1
    for (int step = -S::STAGES;; ++step) {
      __syncwarp();
      if (step >= 0) {
        if (todo == 0) {
          if (taken == queued) break;  // the copies' side is always a piece ahead
          begin_piece();
        }
        copies_wait<S::STAGES - 2>();
        __syncwarp();
      }
      copy_next();
      if (step < 0) continue;
      const int key0 = u.key0 + (u.tiles - todo) * KT;
      if (key0 < u_to && key0 + KT > u_from) tile_products(ring + (uint32_t)stage_out * S::STAGE, key0);
      stage_out = stage_out + 1 == S::STAGES ? 0 : stage_out + 1;
      if (--todo == 0) end_piece();
    }
    copies_wait<0>();

    // ---- units that several warps share ----
    // Join n_parts parts of piece x, in order, as warp `member` of `members`: one of the column tiles,
    // and of its row tiles j0, j0 + step, ... (J at most), with P parts' loads in flight at once. (A warp
    // for each column tile, not each in turn: those are trips to memory one after the other.)
    // stats(k, i) and values(k, i) give float4 i of part k; into the output, or to `stats_to` and
    // `values_to`.
    constexpr int SIDE = NT > 2 ? 4 : NT;
    const auto join = [&](auto jc, auto pc, const Piece& x, int n_parts, int member, int members, auto&& stats, auto&& values,
                          bool out, float4* stats_to, float4* values_to) {
      constexpr int J = decltype(jc)::value, P = imin(decltype(pc)::value, imax(1, 16 / J));
      const int n = member % SIDE, j0 = member / SIDE, step = members / SIDE;
      if (n < NT && n * 8 < x.rows) {
        const int col = n * 8 + 2 * t;
        const bool live = col < x.rows;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
        float4 v[J];
#pragma unroll
        for (int i = 0; i < J; ++i) v[i] = make_float4(0, 0, 0, 0);
#pragma unroll 1
        for (int k0 = 0; k0 < n_parts; k0 += P) {
          float4 st[P], y[P][J];
#pragma unroll
          for (int k = 0; k < P; ++k) {
            st[k] = make_float4(-INFINITY, 0, -INFINITY, 0);
            const bool there = live && k0 + k < n_parts;
            if (there) st[k] = stats(k0 + k, col / 2);
#pragma unroll
            for (int i = 0; i < J; ++i) {
              y[k][i] = make_float4(0, 0, 0, 0);
              if (there && j0 + i * step < DT) y[k][i] = values(k0 + k, ((j0 + i * step) * NT + n) * 32 + lane);
            }
          }
          float t0 = m0, t1 = m1;
#pragma unroll
          for (int k = 0; k < P; ++k) t0 = fmaxf(t0, st[k].x), t1 = fmaxf(t1, st[k].z);
          const float a0 = m0 == -INFINITY ? 0.0f : exp2_fast(m0 - t0), a1 = m1 == -INFINITY ? 0.0f : exp2_fast(m1 - t1);
          m0 = t0, m1 = t1, l0 *= a0, l1 *= a1;
#pragma unroll
          for (int i = 0; i < J; ++i) v[i].x *= a0, v[i].z *= a0, v[i].y *= a1, v[i].w *= a1;
#pragma unroll
          for (int k = 0; k < P; ++k) {
            const float f0 = st[k].x == -INFINITY ? 0.0f : exp2_fast(st[k].x - m0), f1 = st[k].z == -INFINITY ? 0.0f : exp2_fast(st[k].z - m1);
            l0 = fmaf(st[k].y, f0, l0), l1 = fmaf(st[k].w, f1, l1);
#pragma unroll
            for (int i = 0; i < J; ++i) {
              v[i].x = fmaf(f0, y[k][i].x, v[i].x), v[i].z = fmaf(f0, y[k][i].z, v[i].z);
              v[i].y = fmaf(f1, y[k][i].y, v[i].y), v[i].w = fmaf(f1, y[k][i].w, v[i].w);
            }
          }
        }
        const bool first = j0 == 0 && g == 0 && live;  // this lane also writes the columns' statistics
        if (out) {
          A *to0, *to1;
          store_rows(x, n * 8, to0, to1);
          const float inv0 = one_over(l0), inv1 = one_over(l1);
#pragma unroll
          for (int i = 0; i < J; ++i)
            if (j0 + i * step < DT) store_tile(to0, to1, j0 + i * step, v[i], inv0, inv1);
          if (first) {
            store_lse(x, col, m0, l0);
            if (col + 1 < x.rows) store_lse(x, col + 1, m1, l1);
          }
        } else if (live) {
#pragma unroll
          for (int i = 0; i < J; ++i)
            if (j0 + i * step < DT) values_to[((j0 + i * step) * NT + n) * 32 + lane] = v[i];
          if (first) stats_to[col / 2] = make_float4(m0, l0, m1, l1);
        }
      }
    };
    using PerWarp = std::integral_constant<int, imax(1, DT * SIDE / WARPS)>;  // row tiles of a warp of the CTA
    using PerClusterWarp = std::integral_constant<int, imax(1, DT * SIDE / 8)>;  // of 8 warps or more
    using Few = std::integral_constant<int, WARPS>;
    using Many = std::integral_constant<int, 8>;

    if (p.direct) {
      const int next_tile = direct_tile + p.direct;
      if (p.unit_warps >= WARPS) {
        // a unit's parts lie in the rings of consecutive warps: joined in each CTA, then in the cluster
        const int each = (q.tiles + p.unit_warps - 1) / p.unit_warps, n = (q.tiles + each - 1) / each;
        const int ctas = p.unit_warps / WARPS, rank = direct_part / WARPS;
        Piece x;
        x.head = direct_head;
        x.row0 = direct_tile * S::ROWS;
        x.rows = min(S::ROWS, q.new_tokens * p.group - x.row0);
        x.first_row = q.first_row;
        __syncthreads();
        const int here = min(n - rank * WARPS, WARPS);
        const uint32_t values_at = shared_address(smem), stats_at = shared_address(ring_stats);
        const auto load_here = [](uint32_t at) {
          const uint4 v = load_shared16(at);
          return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
        };
        if (n > 1 && here > 0)
          join(
              PerWarp{}, Few{}, x, here, warp, WARPS, [&](int k, int i) { return load_here(stats_at + k * PART_ROWS * 8 + i * 16); },
              [&](int k, int i) { return load_here(values_at + k * S::WARP_BYTES + i * 16); }, ctas == 1,
              reinterpret_cast<float4*>(cta_stats), reinterpret_cast<float4*>(smem));  // (each thread reads what it overwrites)
        if (ctas > 1) {
          cluster_barrier();
          if (n > 1) {
            const uint32_t cta_stats_at = shared_address(cta_stats);
            join(
                PerClusterWarp{}, Many{}, x, (n + WARPS - 1) / WARPS, direct_part, p.unit_warps,
                [&](int k, int i) { return load_cluster(cta_stats_at + i * 16, k); },
                [&](int k, int i) { return load_cluster(values_at + i * 16, k); }, true, nullptr, nullptr);
          }
          cluster_barrier();  // nobody's shared memory goes before all have read it
        } else if (next_tile < q.row_tiles) {
          __syncthreads();
        }
      }
      direct_tile = next_tile;
      if (direct_tile >= q.row_tiles) return;
      continue;
    }

    __syncthreads();
    // Every warp looks at the CTA's pieces, lane x at piece (w, which) = (x / 2, x % 2): is it the
    // CTA's first of its unit, and how many consecutive warps have a part?
    int parts = 0, part_live, part_last = 0;
    uint32_t part_unit;
    int part_tile0, part_tiles;
    {
      const int x = lane & (2 * WARPS - 1);
      const Piece& piece = shared_piece[x >> 1][x & 1];
      part_live = shared_live[x >> 1][x & 1];
      part_unit = piece.unit, part_tile0 = piece.tile0, part_tiles = piece.unit_tiles;
      part_last = part_tile0 + piece.tiles;
      if (part_live && (x < 2 || part_tile0 == 0)) parts = 1;
#pragma unroll
      for (int k = 1; k < WARPS; ++k) {
        const int from = (x >> 1) + k;  // the first piece of a later warp continues the unit
        const int live = __shfl_sync(ALL, part_live, 2 * from), last = __shfl_sync(ALL, part_last, 2 * from), tile0 = __shfl_sync(ALL, part_tile0, 2 * from);
        const uint32_t unit_there = __shfl_sync(ALL, part_unit, 2 * from);
        if (parts == k && from < WARPS && live && unit_there == part_unit && tile0 > 0 && part_last < part_tiles) parts = k + 1, part_last = last;
      }
      if (lane >= 2 * WARPS) parts = 0;
    }
    const bool mine_crosses = parts > 0 && (part_tile0 > 0 || part_last < part_tiles);
    const uint32_t groups = __ballot_sync(ALL, parts > 0), crossing = __ballot_sync(ALL, mine_crosses);
    const uint32_t in_ring = __ballot_sync(ALL, part_live == 2);
    // The CTAs that have a part of a unit, c0 and the `ctas` from it on; and their slots: 0 is for the
    // unit that an earlier CTA began, 1 for one that the CTA begins.
    int c0 = 0, ctas = 0;  // of piece `lane`
    if (mine_crosses) {
      const auto part_before = [&](uint32_t index) { return cut(index * share, index, part_unit, part_tiles); };
      uint32_t g0 = part_unit / share, g1 = (part_unit + part_tiles + START - 1) / share;
      while (part_before(g0 + 1) == 0) ++g0;
      while (part_before(g1) == part_tiles) --g1;
      c0 = g0 / WARPS;
      ctas = (int)(g1 / WARPS) - c0 + 1;
    }
    const auto cta_slot = [](int c, int k) { return (size_t)(MAX_WARPS + (k == 0 ? 2 * c + 1 : 2 * (c + k))); };

    // -- inside the CTA --
#pragma unroll 1
    for (uint32_t left_groups = groups; left_groups; left_groups &= left_groups - 1) {
      const int x = __ffs(left_groups) - 1, w = x >> 1, n = __shfl_sync(ALL, parts, x);
      const bool out = !((crossing >> x) & 1);
      const int c = __shfl_sync(ALL, c0, x);
      // part k lies in warp w + k's ring, or (a first piece that others followed) in the workspace
      const auto place_of = [&](int k, const float4* ring_at, const float4* slots, size_t slot_size) {
        const int piece = 2 * (w + k) + (k == 0 ? x & 1 : 0);
        return (in_ring >> piece) & 1 ? ring_at : slots + (size_t)(warp0 + w + k) * slot_size;
      };
      const size_t to = out ? 0 : cta_slot(c, (int)blockIdx.x - c);
      join(
          PerWarp{}, Few{}, shared_piece[w][x & 1], n, warp, WARPS,
          [&](int k, int i) {
            return load_near(place_of(k, reinterpret_cast<const float4*>(ring_stats[w + k]), reinterpret_cast<const float4*>(p.ws.stats), PART_ROWS / 2) + i);
          },
          [&](int k, int i) {
            return load_near(place_of(k, reinterpret_cast<const float4*>(smem + (w + k) * S::WARP_BYTES), p.ws.parts, PART_FLOATS / 4) + i);
          },
          out, reinterpret_cast<float4*>(p.ws.stats + to * PART_ROWS), p.ws.parts + to * (PART_FLOATS / 4));
    }
    if (!crossing) return;

    // -- units of several CTAs: the last of them to arrive joins their parts, in sets of `size` where
    // there are many, then the sets. A CTA has at most two such units: both arrive together. --
    int size = max(ctas, 1);
    if (ctas > 12) {
      size = 4;
      while (size * size < ctas) ++size;
    }
    const int sets = (ctas + size - 1) / size, set = ((int)blockIdx.x - c0) / size;
    uint32_t waiting = crossing;  // units whose last arrival at the level before was here
#pragma unroll 1
    for (int level = 1; level <= 2 && waiting; ++level) {
      // (one thread's fence after the barrier covers what the others wrote before it)
      __syncthreads();
      if (warp == 0) {
        int last = 0;
        if ((waiting >> lane) & 1) {
          __threadfence();
          const int members = level == 1 ? min(size, ctas - set * size) : sets;
          uint32_t* const ticket = p.ws.tickets + (level - 1) * 2 * MAX_CTAS + cta_slot(c0, level == 1 ? set * size : 0) - MAX_WARPS;
          last = level == 1 || sets > 1 ? atomicAdd(ticket, 1u) + 1 == (uint32_t)members : 0;
          if (last) {
            *ticket = 0;
            __threadfence();
          }
        }
        const uint32_t arrived = __ballot_sync(ALL, last);
        if (lane == 0) arrived_last = arrived;
      }
      __syncthreads();
      waiting = arrived_last;
#pragma unroll 1
      for (uint32_t todo_groups = waiting; todo_groups; todo_groups &= todo_groups - 1) {
        const int x = __ffs(todo_groups) - 1;
        const int c = __shfl_sync(ALL, c0, x), n = __shfl_sync(ALL, ctas, x), step = __shfl_sync(ALL, size, x);
        const int count = __shfl_sync(ALL, sets, x), mine = __shfl_sync(ALL, set, x);
        const bool out = level == 2 || count == 1;
        // (a set's result goes to a slot of its own: all of its members are being read)
        const auto slot = [&](int k) { return level == 1 ? cta_slot(c, mine * step + k) : cta_slot(c, k * step) + 2 * MAX_CTAS; };
        const size_t to = cta_slot(c, mine * step) + 2 * MAX_CTAS;
        join(
            PerWarp{}, Many{}, shared_piece[x >> 1][x & 1], level == 1 ? min(step, n - mine * step) : count, warp, WARPS,
            [&](int k, int i) { return load_part(reinterpret_cast<const float4*>(p.ws.stats + slot(k) * PART_ROWS) + i); },
            [&](int k, int i) { return load_part(p.ws.parts + slot(k) * (PART_FLOATS / 4) + i); }, out,
            reinterpret_cast<float4*>(p.ws.stats + to * PART_ROWS), p.ws.parts + to * (PART_FLOATS / 4));
        if (out) waiting &= ~(1u << x);
      }
    }
    return;
  }
}

template <typename A, bool Q8, int D, int NT>
sonic_status launch_attention(const AttentionLaunch& launch, cudaStream_t stream) {
  using S = Shape<A, Q8, D, NT>;
  AttentionLaunch p = launch;
  const SonicSequences& s = p.a.sequences;
  const int64_t row_tiles = ((int64_t)p.most * p.group + S::ROWS - 1) / S::ROWS;
  const int64_t units = (int64_t)s.requests * p.a.cache.kv_heads * row_tiles;
  // A fixed number of warps a unit where that leaves a warp at most 16 tiles of the longest possible
  // one and the CTAs run at once (of one warp a unit, in two waves): there the balanced shares' scan
  // and joins cost more than uneven lengths do. (us, fixed against balanced, 8 kv heads, bf16: 37
  // requests of 512 keys 17 against 24, 32 of 1000 26 against 31, of 1 to 1000 16 against 14. Beyond
  // these limits: 32 of 2000 45 against 52, but of 1 to 2000 27 against 18; 64 of 1 to 1000 with 4
  // queries, which take two waves, 28 against 23.)
  const int64_t tiles = ((p.window ? std::min<int64_t>(p.room, (int64_t)p.window + p.most) : p.room) + S::KT - 1) / S::KT + 1;
  const auto ctas_of = [&](int warps) { return (units * warps + WARPS - 1) / WARPS; };
  const auto more = [](int warps) { return warps == 1 ? WARPS : 2 * warps; };
  const auto fits = [&](int warps) {
    return tiles <= 16 * warps && ctas_of(warps) <= (warps == 1 ? 2 : 1) * S::CTAS;
  };
  p.unit_warps = 1;
  while (p.unit_warps < 32 && !fits(p.unit_warps)) p.unit_warps = more(p.unit_warps);
  if (fits(p.unit_warps)) {
    // few units: more warps each, down to two tiles a warp
    while (p.unit_warps < 32 && tiles > 2 * p.unit_warps && ctas_of(more(p.unit_warps)) <= S::CTAS) p.unit_warps = more(p.unit_warps);
    const int64_t ctas = ctas_of(p.unit_warps);
    p.direct = (int)std::max<int64_t>(1, row_tiles);
    return launch_status(launch_kernel(attention_kernel<A, Q8, D, NT>, dim3((unsigned)ctas), dim3(NT_THREADS), S::SMEM, stream,
                                       p.a.flags & SONIC_FLAG_PDL, std::max(1, p.unit_warps / WARPS), p));
  }
  // cost the kernel's 32-bit counters can meet: every page-table row full
  const double most_cost = ((double)p.room / S::KT + 2 + START) * ((double)s.tokens * p.group / S::ROWS + s.requests) * p.a.cache.kv_heads;
  if (most_cost >= 2.0e9) return fail_with(SONIC_ERR_UNSUPPORTED, "the call spans more than 2^32 steps: split it by requests");
  p.direct = 0;
  return launch_status(launch_kernel(attention_kernel<A, Q8, D, NT>, dim3(S::CTAS), dim3(NT_THREADS), S::SMEM, stream,
                                     p.a.flags & SONIC_FLAG_PDL, 1, p));
}

template <typename A, bool Q8>
sonic_status launch_shape(const AttentionLaunch& p, cudaStream_t stream) {
  // query rows of a unit: a tile of 8 for each 8 of them, up to 32 (16 at head_dim 256), which is
  // what the accumulators leave room for
  const int64_t rows = (int64_t)p.most * p.group;
  switch (p.a.cache.head_dim) {
    case 64:
      return rows <= 8    ? launch_attention<A, Q8, 64, 1>(p, stream)
             : rows <= 16 ? launch_attention<A, Q8, 64, 2>(p, stream)
             : rows <= 24 ? launch_attention<A, Q8, 64, 3>(p, stream)
                          : launch_attention<A, Q8, 64, 4>(p, stream);
    case 128:
      return rows <= 8    ? launch_attention<A, Q8, 128, 1>(p, stream)
             : rows <= 16 ? launch_attention<A, Q8, 128, 2>(p, stream)
             : rows <= 24 ? launch_attention<A, Q8, 128, 3>(p, stream)
                          : launch_attention<A, Q8, 128, 4>(p, stream);
    default: return rows <= 8 ? launch_attention<A, Q8, 256, 1>(p, stream) : launch_attention<A, Q8, 256, 2>(p, stream);
  }
}

}  // namespace
}  // namespace sonic
