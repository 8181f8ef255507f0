// Residual root-mean-square norm: r = x + residual, y = r / sqrt(mean(r^2) + eps) * weight, with y
// rounded to the input type or quantised to e4m3 with a scale per row or per 128 columns.
//
// Bound by memory: one pass, the row stays in registers between the sum of squares and the output.
// A row belongs to one CTA, to one warp where a warp's registers hold it (short rows pay no block
// barrier), or to the 8 or 16 lanes of a warp that it fills. Each lane holds N items of P values: P
// consecutive ones in a 16-byte piece where rows are aligned, else 4 values 32 columns apart (a warp then
// still reads consecutive addresses, and an item of a warp is 128 consecutive columns in both layouts of
// a group).
//
// bf16 with a residual to e4m3, device time in a captured graph: 16384 x 8192 138 us with a scale a row, 142 us
// a scale per 128 columns (6.8 and 6.7 TB/s of the bytes that it has to move, above this card's measured copy
// rate of 6.55; as calls one after the other 150 to 158 us); 64 x 4096 2.6 us, launch and one trip to memory.
// 32768 x 128, 16 lanes a row, 7.4 us (a warp a row: 12.0). The strided layout is bound by instructions, some
// 30 a value: 3000 x 5001 takes 30 us, twice what its bytes would. With a division and a maximum by bits for
// every 128 columns in every lane, 16384 x 8192 by groups took 150 us for 141, 3000 x 5001 by groups 36 for 31.

#include <algorithm>

#include "host.h"
#include "values.cuh"

namespace sonic {
namespace {

constexpr int MAX_WARPS = 32;
constexpr int MAX_HIDDEN = 32768;

template <typename T>
__device__ __forceinline__ float to_float(T x) {
  if constexpr (sizeof(T) == 4)
    return x;
  else if constexpr (std::is_same<T, __half>::value)
    return __half2float(x);
  else
    return __bfloat162float(x);
}

template <typename T>
__device__ __forceinline__ T from_float(float x) {
  if constexpr (sizeof(T) == 4)
    return x;
  else if constexpr (std::is_same<T, __half>::value)
    return __float2half_rn(x);
  else
    return __float2bfloat16_rn(x);
}

// values of one 16-byte piece of a row
template <typename T>
struct Piece {
  static constexpr int P = 16 / sizeof(T);
  static __device__ __forceinline__ void unpack(const uint4& x, float (&f)[P]) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = Pair<T>::unpack(w[i]);
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
      }
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[P]) {
    if constexpr (sizeof(T) == 4)
      return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    else
      return make_uint4(Pair<T>::pack(f[0], f[1]), Pair<T>::pack(f[2], f[3]), Pair<T>::pack(f[4], f[5]), Pair<T>::pack(f[6], f[7]));
  }
};

// What the fp32 quotient f = 448 / top leaves of 448 / top, to a few bits: top * (f + rest) = 448. With
// it z * 448 / top is rounded once on its way to a code, so that quotients of short significands that lie
// on the midpoint of two codes are seen to lie there. 0 where the row holds an infinity. (It costs nothing
// that shows here: 16384 x 8192 takes 141 us either way. The cache's append is bound by its instructions
// and keeps the plain product: 20.7 us against 22.1.)
__device__ __forceinline__ float e4m3_rest(float top, float f) {
  return top <= 3.4028235e38f ? fmaf(-f, top, kE4m3Max) * (f * (1.0f / kE4m3Max)) : 0.0f;
}
__device__ __forceinline__ float e4m3_quotient(float x, float f, float rest) { return fmaf(x, f, x * rest); }

// Bits of the largest magnitude of v, ordered as magnitude_bits; a NaN is the largest.
template <int P>
__device__ __forceinline__ uint32_t largest(const float (&v)[P]) {
  float top = v[0];
#pragma unroll
  for (int j = 1; j < P; j += 2)
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(top) : "f"(top), "f"(v[j]), "f"(v[j + 1 < P ? j + 1 : j]));
  return magnitude_bits(top);
}

// Row statistics: over the WIDTH lanes of a row, and over its warps where it has several.
template <int WIDTH>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int d = WIDTH / 2; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
template <int WIDTH>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  if constexpr (WIDTH == 32) {
    return __reduce_max_sync(0xffffffffu, v);
  } else {
#pragma unroll
    for (int d = WIDTH / 2; d >= 1; d >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
  }
}

template <int WIDTH>
__device__ __forceinline__ float row_sum(float v, int warps, float* shared) {
  v = lanes_sum<WIDTH>(v);
  if (WIDTH < 32 || warps == 1) return v;
  const int lane = threadIdx.x & 31;
  if (lane == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  return lanes_sum<32>(lane < warps ? shared[lane] : 0.0f);
}

// Both at once, behind one barrier.
template <int WIDTH>
__device__ __forceinline__ void row_sum_and_max(float& v, uint32_t& top, int warps, float* sums, uint32_t* tops) {
  v = lanes_sum<WIDTH>(v);
  top = lanes_max<WIDTH>(top);
  if (WIDTH < 32 || warps == 1) return;
  const int lane = threadIdx.x & 31;
  if (lane == 0) sums[threadIdx.x >> 5] = v, tops[threadIdx.x >> 5] = top;
  __syncthreads();
  v = lanes_sum<32>(lane < warps ? sums[lane] : 0.0f);
  top = lanes_max<32>(lane < warps ? tops[lane] : 0u);
}

// N: items a lane; VEC: 16-byte pieces; WIDTH: lanes of a row. blockDim.x = WIDTH * warps of a row,
// blockDim.y = rows a CTA (more than one only with one warp a row, or part of one).
template <typename T, bool Q8, bool VEC, int N, int WIDTH>
__global__ void __launch_bounds__(1024) norm_kernel(SonicResidualNormArgs a) {
  constexpr int P = VEC ? Piece<T>::P : 4;
  __shared__ float sums[MAX_WARPS];
  __shared__ uint32_t tops[MAX_WARPS];
  grid_dependency_trigger();
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (WIDTH == 32 && row >= a.rows) return;  // whole warps: a CTA with several rows has one warp a row
  // lanes past the last row share a warp with it: they take part, and hold no columns
  const int hidden = WIDTH == 32 || row < a.rows ? a.hidden : 0;
  const int warps = WIDTH == 32 ? blockDim.x >> 5 : 1, warp = WIDTH == 32 ? threadIdx.x >> 5 : 0, lane = threadIdx.x & (WIDTH - 1);
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
  const T* weight = static_cast<const T*>(a.weight);
  T* res_out = a.residual_out ? static_cast<T*>(a.residual_out) + row * a.residual_out_stride : nullptr;

  // column of value j of item i
  const auto column = [&](int i, int j) {
    if constexpr (VEC) return ((i * warps + warp) * 32 + lane) * P + j;
    return (i * warps + warp) * 128 + lane + 32 * j;
  };

  // An item of the strided layout: all its columns lie in the row, a warp's decision, or each is
  // looked at (0 past the row). One address an item, and no branch between loads in flight.
  const auto whole = [&](int i) { return (i * warps + warp) * 128 + 128 <= hidden; };
  const auto item_of = [&](const T* from, int i, T(&values)[P]) {
    from += column(i, 0);
    if (whole(i)) {
#pragma unroll
      for (int j = 0; j < P; ++j) values[j] = from[32 * j];
    } else {
#pragma unroll
      for (int j = 0; j < P; ++j) values[j] = column(i, j) < hidden ? from[32 * j] : from_float<T>(0.0f);
    }
  };

  float r[N][P];
  grid_dependency_wait();
  if constexpr (VEC) {
    uint4 xs[N], rs[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      xs[i] = rs[i] = make_uint4(0, 0, 0, 0);
      if (column(i, 0) < hidden) {
        xs[i] = *reinterpret_cast<const uint4*>(x + column(i, 0));
        if (res) rs[i] = *reinterpret_cast<const uint4*>(res + column(i, 0));
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      Piece<T>::unpack(xs[i], r[i]);
      if (res) {
        float f[P];
        Piece<T>::unpack(rs[i], f);
#pragma unroll
        for (int j = 0; j < P; ++j) r[i][j] += f[j];
      }
    }
  } else {
    T xs[N][P], rs[N][P];
#pragma unroll
    for (int i = 0; i < N; ++i) item_of(x, i, xs[i]);
    if (res) {
#pragma unroll
      for (int i = 0; i < N; ++i) item_of(res, i, rs[i]);
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < P; ++j) {
        r[i][j] = to_float(xs[i][j]);
        if (res) r[i][j] += to_float(rs[i][j]);
      }
  }
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < P; ++j) s = fmaf(r[i][j], r[i][j], s);
    sum += s;
  }
  if (res_out) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (VEC) {
        if (column(i, 0) < hidden) *reinterpret_cast<uint4*>(res_out + column(i, 0)) = Piece<T>::pack(r[i]);
      } else {
        T* to = res_out + column(i, 0);
        if (whole(i)) {
#pragma unroll
          for (int j = 0; j < P; ++j) to[32 * j] = from_float<T>(r[i][j]);
        } else {
#pragma unroll
          for (int j = 0; j < P; ++j)
            if (column(i, j) < hidden) to[32 * j] = from_float<T>(r[i][j]);
        }
      }
    }
  }
  // z = r * weight; y = z * rstd
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (VEC) {
      float w[P];
      uint4 ws = make_uint4(0, 0, 0, 0);
      if (column(i, 0) < hidden) ws = __ldg(reinterpret_cast<const uint4*>(weight + column(i, 0)));
      Piece<T>::unpack(ws, w);
#pragma unroll
      for (int j = 0; j < P; ++j) r[i][j] = column(i, 0) < hidden ? r[i][j] * w[j] : 0.0f;
    } else {
      T w[P];
      item_of(weight, i, w);
#pragma unroll
      for (int j = 0; j < P; ++j) r[i][j] *= to_float(w[j]);
    }
  }

  if constexpr (!Q8) {
    const float rstd = __frsqrt_rn(__fdiv_rn(row_sum<WIDTH>(sum, warps, sums), (float)a.hidden) + a.eps);
    T* out = static_cast<T*>(a.out) + row * a.out_stride;
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int j = 0; j < P; ++j) r[i][j] *= rstd;
      if constexpr (VEC) {
        if (column(i, 0) < hidden) *reinterpret_cast<uint4*>(out + column(i, 0)) = Piece<T>::pack(r[i]);
      } else {
        T* to = out + column(i, 0);
        if (whole(i)) {
#pragma unroll
          for (int j = 0; j < P; ++j) to[32 * j] = from_float<T>(r[i][j]);
        } else {
#pragma unroll
          for (int j = 0; j < P; ++j)
            if (column(i, j) < hidden) to[32 * j] = from_float<T>(r[i][j]);
        }
      }
    }
  } else {
    // The codes of a row or group do not depend on rstd, which its largest |y| shares: they are
    // e4m3(z * 448 / max |z|), rounded once after z. Only a row whose largest |y| lies below
    // the scales' floor is mapped by rstd * 448 / floor.
    uint8_t* out = static_cast<uint8_t*>(a.out) + row * a.out_stride;
    float rstd, scale, factor, rest;
    // an item's 128 columns lie in 128 / P neighbouring lanes (the whole warp in the strided layout)
    constexpr int LANES = VEC && 128 / P < WIDTH ? 128 / P : WIDTH;
    const auto scale_of = [&](uint32_t top) {
      const float z = __uint_as_float(top), c = z * rstd;
      if (c < kScaleFloor) {
        scale = kScaleFloor / kE4m3Max;
        factor = rstd * (kE4m3Max / kScaleFloor);
        rest = 0.0f;
      } else {
        scale = __fdiv_rn(c, kE4m3Max);
        // (448 / z would overflow for the tiniest z); a NaN makes the whole row NaN
        factor = !(c == c) ? c : z < kScaleFloor ? rstd * __fdiv_rn(kE4m3Max, c) : __fdiv_rn(kE4m3Max, z);
        rest = z < kScaleFloor ? 0.0f : e4m3_rest(z, factor);
      }
    };
    if (a.group == 0) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) top = max(top, largest(r[i]));
      row_sum_and_max<WIDTH>(sum, top, warps, sums, tops);
      rstd = __frsqrt_rn(__fdiv_rn(sum, (float)a.hidden) + a.eps);
      scale_of(top);
      if (threadIdx.x == 0 && hidden) a.scales[row] = scale;
    } else {
      rstd = __frsqrt_rn(__fdiv_rn(row_sum<WIDTH>(sum, warps, sums), (float)a.hidden) + a.eps);
      // lane i of an item's lanes finds the scale and factor of item i: one division each, not one an item
      const int member = lane % LANES;
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        uint32_t t = largest(r[i]);
#pragma unroll
        for (int d = LANES / 2; d >= 1; d >>= 1) t = max(t, __shfl_xor_sync(0xffffffffu, t, d));
        if (member == i) top = t;
      }
      scale_of(top);
      const int at = VEC ? column(member, 0) - member * P : (member * warps + warp) * 128;
      if (member < N && at < hidden) a.scales[row * ((a.hidden + 127) / 128) + at / 128] = scale;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float f = a.group ? __shfl_sync(0xffffffffu, factor, i, LANES) : factor;
      const float f_rest = a.group ? __shfl_sync(0xffffffffu, rest, i, LANES) : rest;
      float q[P];
#pragma unroll
      for (int j = 0; j < P; ++j) q[j] = e4m3_quotient(r[i][j], f, f_rest);
      if constexpr (VEC) {
        if (column(i, 0) < hidden) {
          const uint32_t lo = e4m3_pack4(q[0], q[1], q[2], q[3]);
          if constexpr (P == 8) {
            const uint32_t hi = e4m3_pack4(q[4], q[5], q[6], q[7]);
            *reinterpret_cast<uint2*>(out + column(i, 0)) = make_uint2(lo, hi);
          } else {
            *reinterpret_cast<uint32_t*>(out + column(i, 0)) = lo;
          }
        }
      } else {
        uint8_t* to = out + column(i, 0);
        const uint32_t codes = e4m3_pack4(q[0], q[1], q[2], q[3]);
        if (whole(i)) {
#pragma unroll
          for (int j = 0; j < P; ++j) to[32 * j] = codes >> 8 * j;
        } else {
#pragma unroll
          for (int j = 0; j < P; ++j)
            if (column(i, j) < hidden) to[32 * j] = codes >> 8 * j;
        }
      }
    }
  }
}

template <typename T, bool Q8, bool VEC>
sonic_status run(const SonicResidualNormArgs& a, cudaStream_t stream) {
  constexpr int PER_WARP = 32 * (VEC ? Piece<T>::P : 4);
  const int items = (a.hidden + PER_WARP - 1) / PER_WARP;  // items of a row, over its warps
  // few rows: as many warps as items (latency); many rows: up to 4 items a lane, so that each
  // thread has several loads in flight
  int n = (int64_t)a.rows < 296 ? 1 : std::min(4, items);
  n = n == 3 ? 4 : n;
  while ((items + n - 1) / n > MAX_WARPS) n *= 2;
  const int warps = (items + n - 1) / n;
  int width = 32;
  if (VEC && warps == 1 && a.hidden <= PER_WARP / 2) width = a.hidden <= PER_WARP / 4 ? 8 : 16;
  const int rows = warps > 1 ? 1 : width < 32 ? 128 / width : std::min(a.rows, 4);  // whole warps
  const dim3 block(width * warps, rows), grid((unsigned)(((int64_t)a.rows + rows - 1) / rows));
  const bool pdl = a.flags & SONIC_FLAG_PDL;
  const auto go = [&](auto kernel) { return launch_status(launch_kernel(kernel, grid, block, 0, stream, pdl, 1, a)); };
  if constexpr (VEC) {
    if (width == 8) return go(norm_kernel<T, Q8, VEC, 1, 8>);
    if (width == 16) return go(norm_kernel<T, Q8, VEC, 1, 16>);
  }
  // (the widest row of 16-bit values in 16-byte pieces has 4 items a lane, the others' 8)
  constexpr int MOST = MAX_HIDDEN / PER_WARP / MAX_WARPS;
  static_assert(MOST == 4 || MOST == 8, "the variants below");
  if constexpr (MOST == 8) {
    if (n == 8) return go(norm_kernel<T, Q8, VEC, 8, 32>);
  }
  switch (n) {
    case 1: return go(norm_kernel<T, Q8, VEC, 1, 32>);
    case 2: return go(norm_kernel<T, Q8, VEC, 2, 32>);
    default: return go(norm_kernel<T, Q8, VEC, 4, 32>);
  }
}

template <typename T>
sonic_status run_type(const SonicResidualNormArgs& a, cudaStream_t stream) {
  constexpr int P = Piece<T>::P;
  const bool q8 = a.out_dtype == SONIC_DTYPE_E4M3;
  bool vec = a.hidden % P == 0 && is_aligned(a.x, 16) && a.x_stride % P == 0 && is_aligned(a.weight, 16);
  if (a.residual) vec = vec && is_aligned(a.residual, 16) && a.residual_stride % P == 0;
  if (a.residual_out) vec = vec && is_aligned(a.residual_out, 16) && a.residual_out_stride % P == 0;
  vec = vec && is_aligned(a.out, q8 ? P : 16) && a.out_stride % P == 0;
  if (q8) return vec ? run<T, true, true>(a, stream) : run<T, true, false>(a, stream);
  return vec ? run<T, false, true>(a, stream) : run<T, false, false>(a, stream);
}

}  // namespace
}  // namespace sonic

using namespace sonic;

extern "C" sonic_status sonic_residual_norm(const SonicResidualNormArgs* a, void* stream) {
  if (!a) return fail_with(SONIC_ERR_INVALID_ARGUMENT, "args must not be NULL");
  if (a->rows < 0) return fail_with(SONIC_ERR_INVALID_ARGUMENT, "rows must not be negative");
  if (a->hidden < 1) return fail_with(SONIC_ERR_INVALID_ARGUMENT, "hidden must be positive");
  if (a->hidden > MAX_HIDDEN) return fail_with(SONIC_ERR_UNSUPPORTED, "hidden must be at most 32768");
  if (a->dtype != SONIC_DTYPE_BF16 && a->dtype != SONIC_DTYPE_F16 && a->dtype != SONIC_DTYPE_F32)
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "dtype must be bf16, f16 or f32");
  if (a->out_dtype != a->dtype && a->out_dtype != SONIC_DTYPE_E4M3)
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "out_dtype must be dtype or e4m3");
  if (a->out_dtype == SONIC_DTYPE_E4M3 ? (a->group != 0 && a->group != 128) : a->group != 0)
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "group must be 0, or 128 with an e4m3 output");
  if (a->rows == 0) return SONIC_OK;
  if (!a->x || !a->weight || !a->out) return fail_with(SONIC_ERR_INVALID_ARGUMENT, "x, weight and out must not be NULL");
  if (a->out_dtype == SONIC_DTYPE_E4M3 && !a->scales)
    return fail_with(SONIC_ERR_INVALID_ARGUMENT, "an e4m3 output needs scales");
  const cudaStream_t st = (cudaStream_t)stream;
  if (a->dtype == SONIC_DTYPE_BF16) return run_type<__nv_bfloat16>(*a, st);
  if (a->dtype == SONIC_DTYPE_F16) return run_type<__half>(*a, st);
  return run_type<float>(*a, st);
}
