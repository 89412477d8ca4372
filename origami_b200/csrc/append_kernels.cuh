// Per-head norm, position rotation and append to a paged cache, one launch for a step's
// queries, keys and values.
//
// A row is one head of one token: x[0..D). With a weight w its RMS norm comes first,
//   y_i = x_i * w_i / sqrt(mean(x^2) + eps),
// then the pairs of its first R dims turn by the token's angle,
//   (a, b) -> (a cos - b sin, b cos + a sin),
// the pair of index p being dims (p, p + R/2) (halves) or (2p, 2p + 1) (interleaved), with
// cos / sin from row `position` of the caller's table [max_positions, R] = cos | sin. The
// arithmetic is fp32; the one rounding is the store. Values pass through (converted to the
// cache's type).
//
// Bound: bytes. Every element is read once and written once and nothing else scales with the
// row, so the design only has to keep enough loads in flight and spend few instructions:
// a lane holds 16 elements of a head as two 8-element chunks that contain both members of
// each of its pairs (chunks c and c + R/16 for halves, 2c and 2c + 1 interleaved), so the
// rotation needs no exchange between lanes, the norm is log2(lanes per head) shuffles, and
// the 8 (cos, sin) a lane needs are loaded once for all the heads it walks of its token.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace origami {

// Rows of one tensor [tokens, heads, head_dim], element strides, head_dim contiguous.
struct HeadRows {
  const void* in;
  void* out;  // null: the rows go to the paged cache
  int64_t in_token, in_head, out_token, out_head;
  const void* weight;  // [D] RMS norm weight, null for none
  int32_t heads;
  int32_t weight_dtype;
};

struct AppendArgs {
  HeadRows q, k, v;  // heads = 0 where absent; v has no norm and no rotation
  const void* slots;      // cache rows of the tokens, null without a cache
  const void* positions;  // null without rotation
  const void* table;
  int64_t table_stride, max_positions;
  void* cache;
  int64_t kv_stride, block_stride, token_stride, num_slots, block_size;
  int64_t tokens;
  uint32_t* err;
  int32_t D, R, interleaved, table_dtype, slots64, positions64;
  int32_t lanes_log2;  // lanes per head (fast kernel)
  int32_t groups;      // head walkers per token (fast kernel)
  float eps;
};

namespace app {

constexpr int kF16 = 1, kBF16 = 2, kF32 = 3;
constexpr int kUnroll = 4;  // heads a lane has in flight

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 8 elements as raw 16-byte words.
template <typename T>
struct Raw8 {
  uint4 w[sizeof(T) == 4 ? 2 : 1];
};
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p) {
  Raw8<T> r;
  r.w[0] = *reinterpret_cast<const uint4*>(p);
  if constexpr (sizeof(T) == 4) r.w[1] = *reinterpret_cast<const uint4*>(p + 4);
  return r;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const Raw8<T>& r) {
  *reinterpret_cast<uint4*>(p) = r.w[0];
  if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(p + 4) = r.w[1];
}
template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float* f) {
  const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = to_f<T>(e[i]);
}
template <typename T>
__device__ __forceinline__ Raw8<T> pack8(const float* f) {
  Raw8<T> r;
  T* e = reinterpret_cast<T*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = from_f<T>(f[i]);
  return r;
}

// Element i of a table or weight tensor whose type is known at run time.
__device__ __forceinline__ float small_at(const void* p, int dtype, int64_t i) {
  if (dtype == kF32) return __ldg(static_cast<const float*>(p) + i);
  if (dtype == kBF16) return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(p) + i));
  return __half2float(__ldg(static_cast<const __half*>(p) + i));
}
// 8 consecutive ones; 8-byte aligned (16-byte for fp32).
__device__ __forceinline__ void small8(const void* p, int dtype, int64_t i, float* f) {
  if (dtype == kF32) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const float4 a = __ldg(q), b = __ldg(q + 1);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    return;
  }
  const uint2* q = reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
  const uint2 a = __ldg(q), b = __ldg(q + 1);
  const uint32_t w[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (dtype == kBF16) {
      f[2 * j] = __uint_as_float(w[j] << 16);
      f[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    } else {
      const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      f[2 * j] = h.x;
      f[2 * j + 1] = h.y;
    }
  }
}

__device__ __forceinline__ int64_t index_at(const void* p, int wide, int64_t i) {
  return wide ? __ldg(static_cast<const long long*>(p) + i) : __ldg(static_cast<const int*>(p) + i);
}

__device__ __forceinline__ float inv_rms(float sum, int D, float eps) {
  return __frcp_rn(__fsqrt_rn(sum / static_cast<float>(D) + eps));
}

// A token's place: its cache row (-1: none), whether its position lies in the table, and the
// rows that have to be counted as skipped.
struct Place {
  int64_t cache_row;  // element offset of the token's K row, -1 without one
  int64_t position;
  bool rotates;       // false: position outside the table, no row of the token is written
};
__device__ __forceinline__ Place place_of(const AppendArgs& a, int64_t t, uint32_t& skipped) {
  Place p{-1, 0, true};
  skipped = 0;
  int64_t slot = -1;
  if (a.slots) slot = index_at(a.slots, a.slots64, t);
  const bool in_cache = slot >= 0 && slot < a.num_slots;
  if (a.positions) {
    p.position = index_at(a.positions, a.positions64, t);
    p.rotates = p.position >= 0 && p.position < a.max_positions;
  }
  if (in_cache)
    p.cache_row = (slot / a.block_size) * a.block_stride + (slot % a.block_size) * a.token_stride;
  // slot -1 asks for no cache row; any other slot outside the cache is an error
  if (a.slots && !in_cache && slot != -1) skipped += static_cast<uint32_t>(a.k.heads + a.v.heads);
  if (!p.rotates) {
    skipped += static_cast<uint32_t>(a.q.heads);
    if (!a.slots || in_cache) skipped += static_cast<uint32_t>(a.k.heads + a.v.heads);
  }
  return p;
}

}  // namespace app

// Fast kernel: D % 8 == 0, 16-byte rows, R % 16 == 0 (halves) or R % 8 == 0 (interleaved).
// 1 << lanes_log2 lanes per head; `groups` such walkers share a token's heads (query heads,
// then key heads, then value heads), kUnroll heads in flight each.
template <typename TI, typename TC>
__global__ void __launch_bounds__(256) append_rows(const __grid_constant__ AppendArgs a) {
  using namespace app;
  const int lph = 1 << a.lanes_log2;
  const int lane = threadIdx.x & (lph - 1);
  const int64_t walker = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> a.lanes_log2;
  const int64_t t = walker / a.groups;
  const int g = static_cast<int>(walker - t * a.groups);
  const bool live = t < a.tokens;
  const int total = a.q.heads + a.k.heads + a.v.heads;

  Place pl{-1, 0, false};
  if (live) {
    uint32_t skipped;
    pl = place_of(a, t, skipped);
    if (skipped && g == 0 && lane == 0 && a.err) atomicAdd(a.err, skipped);
  }
  // this lane's two chunks; nchunks may be odd (the last lane then has one)
  const int nchunks = a.D >> 3;
  const bool split = !a.interleaved && lane < (a.R >> 4);
  const int c0 = split ? lane : 2 * lane;
  const int c1 = split ? lane + (a.R >> 4) : 2 * lane + 1;
  const bool has0 = c0 < nchunks, has1 = c1 < nchunks;
  // pairs 8*lane .. 8*lane+7 in both arrangements; the first four and last four may differ
  // in whether they turn (interleaved with R % 16 == 8)
  const bool turn0 = a.positions && (a.interleaved ? 8 * c0 < a.R : split);
  const bool turn1 = a.positions && (a.interleaved ? 8 * c1 < a.R : split);
  float co[8], si[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) co[i] = 1.f, si[i] = 0.f;
  if (live && pl.rotates && turn0) {
    const int64_t row = pl.position * a.table_stride + 8 * lane;
    if (turn1) {
      small8(a.table, a.table_dtype, row, co);
      small8(a.table, a.table_dtype, row + (a.R >> 1), si);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        co[i] = small_at(a.table, a.table_dtype, row + i);
        si[i] = small_at(a.table, a.table_dtype, row + (a.R >> 1) + i);
      }
    }
  }

  // Uniform trip count: walkers of one warp shuffle together.
  for (int u0 = g; u0 - g < total; u0 += kUnroll * a.groups) {
    Raw8<TI> x[kUnroll][2];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const int u = u0 + j * a.groups;
      x[j][0] = Raw8<TI>{};
      x[j][1] = Raw8<TI>{};
      if (!live || u >= total) continue;
      const HeadRows& r = u < a.q.heads ? a.q : u < a.q.heads + a.k.heads ? a.k : a.v;
      const int h = u < a.q.heads ? u : u < a.q.heads + a.k.heads ? u - a.q.heads : u - a.q.heads - a.k.heads;
      const TI* p = static_cast<const TI*>(r.in) + t * r.in_token + h * r.in_head;
      if (has0) x[j][0] = load8(p + 8 * c0);
      if (has1) x[j][1] = load8(p + 8 * c1);
    }
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const int u = u0 + j * a.groups;
      const bool is_q = u < a.q.heads, is_k = !is_q && u < a.q.heads + a.k.heads;
      const HeadRows& r = is_q ? a.q : is_k ? a.k : a.v;
      const int h = is_q ? u : is_k ? u - a.q.heads : u - a.q.heads - a.k.heads;
      float f[16];
      unpack8(x[j][0], f);
      unpack8(x[j][1], f + 8);
      // the branch is taken by the whole warp or the shuffles run anyway: any weight at all
      if (a.q.weight || a.k.weight) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s = fmaf(f[i], f[i], s);
        for (int o = lph >> 1; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (r.weight && u < total) {
          const float inv = inv_rms(s, a.D, a.eps);
          float w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = 0.f;
          if (has0) small8(r.weight, r.weight_dtype, 8 * c0, w);
          if (has1) small8(r.weight, r.weight_dtype, 8 * c1, w + 8);
#pragma unroll
          for (int i = 0; i < 16; ++i) f[i] = f[i] * inv * w[i];
        }
      }
      if (!live || u >= total || !pl.rotates) continue;
      if (!is_q && !r.out && pl.cache_row < 0) continue;
      if (is_q || is_k) {
        if (a.interleaved) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (i < 4 ? turn0 : turn1) {
              const float x0 = f[2 * i], x1 = f[2 * i + 1];
              f[2 * i] = fmaf(x0, co[i], -(x1 * si[i]));
              f[2 * i + 1] = fmaf(x1, co[i], x0 * si[i]);
            }
          }
        } else if (turn0) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float x0 = f[i], x1 = f[i + 8];
            f[i] = fmaf(x0, co[i], -(x1 * si[i]));
            f[i + 8] = fmaf(x1, co[i], x0 * si[i]);
          }
        }
      }
      if (r.out) {
        TI* o = static_cast<TI*>(r.out) + t * r.out_token + h * r.out_head;
        if (has0) store8(o + 8 * c0, pack8<TI>(f));
        if (has1) store8(o + 8 * c1, pack8<TI>(f + 8));
      } else {
        TC* o = static_cast<TC*>(a.cache) + (is_k ? 0 : a.kv_stride) + pl.cache_row + static_cast<int64_t>(h) * a.D;
        if (has0) store8(o + 8 * c0, pack8<TC>(f));
        if (has1) store8(o + 8 * c1, pack8<TC>(f + 8));
      }
    }
  }
}

// Any head_dim, any even R, element-aligned rows: one warp per row, a lane reads and writes
// both members of its pairs (so a row may be rewritten in place).
template <typename TI, typename TC>
__global__ void __launch_bounds__(256) append_rows_any(const __grid_constant__ AppendArgs a) {
  using namespace app;
  const int lane = threadIdx.x & 31;
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int total = a.q.heads + a.k.heads + a.v.heads;
  const int64_t t = row / total;
  if (t >= a.tokens) return;
  const int u = static_cast<int>(row - t * total);
  const bool is_q = u < a.q.heads, is_k = !is_q && u < a.q.heads + a.k.heads;
  const HeadRows& r = is_q ? a.q : is_k ? a.k : a.v;
  const int h = is_q ? u : is_k ? u - a.q.heads : u - a.q.heads - a.k.heads;
  uint32_t skipped;
  const Place pl = place_of(a, t, skipped);
  if (u == 0 && lane == 0 && skipped && a.err) atomicAdd(a.err, skipped);
  if (!pl.rotates || (!r.out && pl.cache_row < 0)) return;
  const TI* x = static_cast<const TI*>(r.in) + t * r.in_token + h * r.in_head;
  float inv = 1.f;
  if (r.weight) {
    float s = 0.f;
    for (int i = lane; i < a.D; i += 32) {
      const float v = to_f<TI>(x[i]);
      s = fmaf(v, v, s);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    inv = inv_rms(s, a.D, a.eps);
  }
  auto value = [&](int i) {
    const float v = to_f<TI>(x[i]);
    return r.weight ? v * inv * small_at(r.weight, r.weight_dtype, i) : v;
  };
  TI* rows_out = static_cast<TI*>(r.out) + t * r.out_token + h * r.out_head;
  TC* cache_out = static_cast<TC*>(a.cache) + (is_k ? 0 : a.kv_stride) + pl.cache_row + static_cast<int64_t>(h) * a.D;
  auto put = [&](int i, float v) {
    if (r.out) rows_out[i] = from_f<TI>(v);
    else cache_out[i] = from_f<TC>(v);
  };
  const int turned = (is_q || is_k) && a.positions ? a.R : 0;
  for (int p = lane; p < turned / 2; p += 32) {
    const int i0 = a.interleaved ? 2 * p : p, i1 = a.interleaved ? 2 * p + 1 : p + turned / 2;
    const float x0 = value(i0), x1 = value(i1);
    const float co = small_at(a.table, a.table_dtype, pl.position * a.table_stride + p);
    const float si = small_at(a.table, a.table_dtype, pl.position * a.table_stride + (turned >> 1) + p);
    put(i0, fmaf(x0, co, -(x1 * si)));
    put(i1, fmaf(x1, co, x0 * si));
  }
  for (int i = turned + lane; i < a.D; i += 32) put(i, value(i));
}

}  // namespace origami
