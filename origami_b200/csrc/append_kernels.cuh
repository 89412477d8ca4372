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
// - a lane holds 16 elements of a head as two 8-element chunks that contain both members of
//   each of its pairs (chunks c and c + R/16 for halves, 2c and 2c + 1 interleaved), so the
//   rotation needs no exchange between lanes and the norm is log2(lanes per head) shuffles;
//   chunks of 4 halve the registers but double the instructions (147 us instead of 98 for
//   16384 tokens of 32 + 8 heads of 128, both with one token per walker);
// - a walker steps through tokens with a fixed set of heads: addresses, weights (fp32, in shared
//   memory) and roles are set up once, the next token's position and slot are loaded a token
//   ahead, its rows copied to shared memory by cp.async, each row's place refilled as soon as it
//   has been read, so that a walker never waits with nothing requested (16384 tokens: 78 us with
//   loads into registers, 68 so, 72 with two tokens ahead; calls one by one, cold L2);
// - fp32 arithmetic in pairs (f32x2).
// Measured on bf16, halves, with norm: 16384 tokens of 32 query and 8 KV heads of 128, 344 MB,
// 62 to 67 us (5.1 to 5.5 TB/s, 0.80 to 0.86 of the copy rate); append of 32768 such tokens, 822
// MB, 134 to 147 us (5.6 to 6.1 TB/s, 0.87 to 0.95). 8192 tokens in fp32, 340 MB: 82 us (0.64);
// 16384 of heads of 64 / 80 / 96: 34 / 73 / 73 us (0.78 / 0.46 / 0.55: 5 and 6 of 8 lanes have
// work), 8192 of 256: 64 us (0.84). (The lower figures: twenty calls in a graph, L2 flushed before
// each; the higher ones: calls one by one.)
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "f32x2.cuh"

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
  int32_t step;        // tokens from one of a walker's to the next
  float eps, inv_d;
};

namespace app {

constexpr int kF16 = 1, kBF16 = 2, kF32 = 3;
// Rows of a token that a walker of the streaming form has at most (key, value, query heads), and
// the shared memory for one token's of each: 48 KB a CTA of 16-bit rows, 96 KB of fp32.
constexpr int kQueryRows = 4, kWalkerRows = 2 + kQueryRows;
template <typename TI>
constexpr int kStreamSmem = kWalkerRows * 256 * 16 * static_cast<int>(sizeof(TI));

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
// Words of two 16-bit elements to and from floats.
template <typename T>
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xFFFF0000u);
  } else {
    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = h.x;
    hi = h.y;
  }
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float* f) {
#pragma unroll
  for (int k = 0; k < static_cast<int>(sizeof(T)) / 2; ++k) {
    const uint32_t w[4] = {r.w[k].x, r.w[k].y, r.w[k].z, r.w[k].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) f[4 * k + i] = __uint_as_float(w[i]);
      else unpack2<T>(w[i], f[2 * i], f[2 * i + 1]);
    }
  }
}
template <typename T>
__device__ __forceinline__ Raw8<T> pack8(const float* f) {
  Raw8<T> r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      r.w[k] = make_uint4(__float_as_uint(f[4 * k]), __float_as_uint(f[4 * k + 1]), __float_as_uint(f[4 * k + 2]),
                          __float_as_uint(f[4 * k + 3]));
  } else {
    r.w[0] = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
  }
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

// 1 / sqrt(sum / D + eps): rsqrt and one Newton step (within an ulp or two; 0 and infinity as they are).
__device__ __forceinline__ float inv_rms(float sum, float inv_d, float eps) {
  const float x = fmaf(sum, inv_d, eps), r = rsqrtf(x);
  const float n = fmaf(r * 0.5f, fmaf(-x * r, r, 1.f), r);
  return x > 0.f && x < INFINITY ? n : r;
}

// A token's place: its cache row (-1: none), whether its position lies in the table, and the
// rows that have to be counted as skipped.
struct Place {
  int64_t cache_row;  // element offset of the token's K row, -1 without one
  int64_t position;
  bool rotates;       // false: position outside the table, no row of the token is written
};
// What the lists hold for a token; loaded a token ahead by the kernel that steps through them.
struct Listed {
  int64_t slot, position;
  __device__ __forceinline__ Listed(const AppendArgs& a, int64_t t)
      : slot(a.slots ? index_at(a.slots, a.slots64, t) : -1), position(a.positions ? index_at(a.positions, a.positions64, t) : 0) {}
};
__device__ __forceinline__ Place place_of(const AppendArgs& a, const Listed& listed, uint32_t& skipped) {
  Place p{-1, listed.position, true};
  skipped = 0;
  const int64_t slot = listed.slot;
  const bool in_cache = slot >= 0 && slot < a.num_slots;
  if (a.positions) p.rotates = p.position >= 0 && p.position < a.max_positions;
  if (in_cache) {
    int64_t block;
    if (((slot | a.block_size) >> 31) == 0) block = static_cast<uint32_t>(slot) / static_cast<uint32_t>(a.block_size);
    else block = slot / a.block_size;
    p.cache_row = block * a.block_stride + (slot - block * a.block_size) * a.token_stride;
  }
  // slot -1 asks for no cache row; any other slot outside the cache is an error
  if (a.slots && !in_cache && slot != -1) skipped += static_cast<uint32_t>(a.k.heads + a.v.heads);
  if (!p.rotates) {
    skipped += static_cast<uint32_t>(a.q.heads);
    if (!a.slots || in_cache) skipped += static_cast<uint32_t>(a.k.heads + a.v.heads);
  }
  return p;
}

}  // namespace app

// Fast kernel: D % 8 == 0, 16-byte rows, R % 16 == 0. 1 << lanes_log2 lanes ("a walker") per
// head. STREAM: `groups` walkers share a token's heads, walker g taking up to kQueryRows query
// heads, key head g and value head groups - 1 - g, and step through the tokens, so that all but
// the rows, the position and the slot is set up once (the weights in shared memory, in fp32).
// Else a walker for each head of each token. FULL: every lane has both chunks (D is 16 <<
// lanes_log2).
template <typename TI, typename TC, bool FULL, bool STREAM>
__global__ void __launch_bounds__(256, 2) append_rows(const __grid_constant__ AppendArgs a) {
  using namespace app;
  __shared__ __align__(16) float w_sm[2][512];
  const int lph = 1 << a.lanes_log2;
  const int lane = threadIdx.x & (lph - 1);
  const int walker = static_cast<int>((blockIdx.x * blockDim.x + threadIdx.x) >> a.lanes_log2);
  const int first = walker / a.groups, g = walker - first * a.groups;
  // this walker's heads
  const int kh = STREAM ? g : g - a.q.heads;
  const int vh = STREAM ? a.groups - 1 - g : g - a.q.heads - a.k.heads;
  const bool has_k = kh >= 0 && kh < a.k.heads, has_v = vh >= 0 && vh < a.v.heads;
  const int q_per = STREAM ? (a.q.heads + a.groups - 1) / a.groups : 1;
  const int q0 = g * q_per, q1 = min(q0 + q_per, a.q.heads);

  // this lane's two chunks; D / 8 may be odd (the last lane then has one)
  const bool split = !a.interleaved && lane < (a.R >> 4);
  const int e0 = 8 * (split ? lane : 2 * lane), e1 = 8 * (split ? lane + (a.R >> 4) : 2 * lane + 1);
  const bool has0 = FULL || e0 < a.D, has1 = FULL || e1 < a.D;
  // pairs 8 lane .. 8 lane + 7 in both arrangements
  const bool turns = a.positions && 16 * lane < a.R;
  const int64_t k_in = (has_k ? kh : 0) * a.k.in_head, v_in = (has_v ? vh : 0) * a.v.in_head;
  for (int i = threadIdx.x; i < a.D; i += blockDim.x) {
    if (a.q.weight) w_sm[0][i] = small_at(a.q.weight, a.q.weight_dtype, i);
    if (a.k.weight) w_sm[1][i] = small_at(a.k.weight, a.k.weight_dtype, i);
  }
  __syncthreads();
  auto put = [&](auto* o, const float (&f)[16]) {
    using T = std::remove_reference_t<decltype(*o)>;
    if (has0) store8(o + e0, pack8<T>(f));
    if (has1) store8(o + e1, pack8<T>(f + 8));
  };
  float co[8], si[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) co[i] = 1.f, si[i] = 0.f;
  // norm and rotation of one head's 16 elements (the whole warp takes part in the shuffles)
  auto turn = [&](const float* w, bool norm, bool scale, bool rotate, const Raw8<TI> (&x)[2], float (&f)[16]) {
    unpack8(x[0], f);
    unpack8(x[1], f + 8);
    if (norm) {
      uint64_t s2 = 0ull, s3 = 0ull;
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        s2 = fma2(pair2(f[i], f[i + 1]), pair2(f[i], f[i + 1]), s2);
        s3 = fma2(pair2(f[i + 8], f[i + 9]), pair2(f[i + 8], f[i + 9]), s3);
      }
      float s0, s1;
      split2(add2(s2, s3), s0, s1);
      float s = s0 + s1;
#pragma unroll 1
      for (int o = lph >> 1; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      const float inv = inv_rms(s, a.inv_d, a.eps);
      const uint64_t inv2 = pair2(inv, inv);
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        if (scale && (i < 8 ? has0 : has1)) {
          const float4 v = *reinterpret_cast<const float4*>(w + (i < 8 ? e0 + i : e1 + i - 8));
          split2(mul2(mul2(pair2(f[i], f[i + 1]), inv2), pair2(v.x, v.y)), f[i], f[i + 1]);
          split2(mul2(mul2(pair2(f[i + 2], f[i + 3]), inv2), pair2(v.z, v.w)), f[i + 2], f[i + 3]);
        }
      }
    }
    if (!turns || !rotate) return;
    if (a.interleaved) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x0 = f[2 * i], x1 = f[2 * i + 1];
        f[2 * i] = fmaf(x0, co[i], -(x1 * si[i]));
        f[2 * i + 1] = fmaf(x1, co[i], x0 * si[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const uint64_t x0 = pair2(f[i], f[i + 1]), x1 = pair2(f[i + 8], f[i + 9]);
        const uint64_t c = pair2(co[i], co[i + 1]), s = pair2(si[i], si[i + 1]);
        split2(sub2(mul2(x0, c), mul2(x1, s)), f[i], f[i + 1]);
        split2(fma2(x0, s, mul2(x1, c)), f[i + 8], f[i + 9]);
      }
    }
  };
  // (walkers beyond the last whole token of a pass have none)
  int64_t t = first < a.step ? first : a.tokens;
  Listed listed(a, min64(t, a.tokens - 1));
  auto table = [&](const Listed& at, float (&c)[8], float (&s)[8]) {
    if (turns && at.position >= 0 && at.position < a.max_positions) {
      const int64_t row = at.position * a.table_stride + 8 * lane;
      small8(a.table, a.table_dtype, row, c);
      small8(a.table, a.table_dtype, row + (a.R >> 1), s);
    }
  };
  if constexpr (STREAM) {
    // Row r of a token: 0 the key, 1 the value, then query heads. A lane requests the 16-byte
    // pieces of its own chunks into its own places of shared memory and reads no other's, so
    // nothing but its own copies' groups (one a row, in order) has to be waited for.
    extern __shared__ __align__(16) uint8_t stream_sm[];
    constexpr int kHalfPieces = static_cast<int>(sizeof(TI)) / 2, kPer16 = 16 / static_cast<int>(sizeof(TI));
    uint8_t* mine = stream_sm + threadIdx.x * 16;
    auto request = [&](int r, int64_t at_t) {
      const bool want = at_t < a.tokens && (r == 0 ? has_k : r == 1 ? has_v : q0 + r - 2 < q1);
      if (want) {
        const HeadRows& rows = r == 0 ? a.k : r == 1 ? a.v : a.q;
        const TI* p = static_cast<const TI*>(rows.in) + at_t * rows.in_token +
                      (r == 0 ? k_in : r == 1 ? v_in : (q0 + r - 2) * a.q.in_head);
        uint8_t* dst = mine + r * 2 * kHalfPieces * 4096;
#pragma unroll
        for (int c = 0; c < kHalfPieces; ++c) {
          if (has0) cp_async16(dst + c * 4096, p + e0 + c * kPer16);
          if (has1) cp_async16(dst + (kHalfPieces + c) * 4096, p + e1 + c * kPer16);
        }
      }
      asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
    auto take = [&](int r, Raw8<TI> (&x)[2]) {
      asm volatile("cp.async.wait_group %0;\n" ::"n"(kWalkerRows - 1) : "memory");
      const uint8_t* src = mine + r * 2 * kHalfPieces * 4096;
      if (!FULL) x[0] = x[1] = Raw8<TI>{};
#pragma unroll
      for (int c = 0; c < kHalfPieces; ++c) {
        if (has0) x[0].w[c] = *reinterpret_cast<const uint4*>(src + c * 4096);
        if (has1) x[1].w[c] = *reinterpret_cast<const uint4*>(src + (kHalfPieces + c) * 4096);
      }
    };
#pragma unroll
    for (int r = 0; r < kWalkerRows; ++r) request(r, t);
    Listed next(a, min64(t + a.step, a.tokens - 1));
    table(listed, co, si);
#pragma unroll 1
    for (; __any_sync(0xffffffffu, t < a.tokens); t += a.step) {
      Place pl{-1, 0, false};
      if (t < a.tokens) {
        uint32_t skipped;
        pl = place_of(a, listed, skipped);
        if (skipped && g == 0 && lane == 0 && a.err) atomicAdd(a.err, skipped);
      }
      float co_next[8], si_next[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) co_next[i] = 1.f, si_next[i] = 0.f;
      table(next, co_next, si_next);
      listed = next;
      next = Listed(a, min64(t + 2 * static_cast<int64_t>(a.step), a.tokens - 1));
      TC* cache_row = static_cast<TC*>(a.cache) + pl.cache_row;
      Raw8<TI> x[2];
      float f[16];
      take(0, x);
      turn(w_sm[1], a.k.weight != nullptr, true, true, x, f);
      if (has_k && pl.rotates) {
        if (a.k.out) put(static_cast<TI*>(a.k.out) + t * a.k.out_token + kh * a.k.out_head, f);
        else if (pl.cache_row >= 0) put(cache_row + static_cast<int64_t>(kh) * a.D, f);
      }
      request(0, t + a.step);
      if (a.v.heads > 0) {
        take(1, x);
        unpack8(x[0], f);
        unpack8(x[1], f + 8);
        if (has_v && pl.rotates && pl.cache_row >= 0) put(cache_row + a.kv_stride + static_cast<int64_t>(vh) * a.D, f);
      }
      request(1, t + a.step);
      TI* out = static_cast<TI*>(a.q.out) + t * a.q.out_token + q0 * a.q.out_head;
#pragma unroll 1
      for (int j = 0; j < kQueryRows; ++j) {
        if (j < q_per) {
          take(2 + j, x);
          turn(w_sm[0], a.q.weight != nullptr, true, true, x, f);
          if (q0 + j < q1 && pl.rotates) put(out + j * a.q.out_head, f);
        }
        request(2 + j, t + a.step);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) co[i] = co_next[i], si[i] = si_next[i];
    }
    return;
  }
  // One head of one token a walker, in one pass.
  const bool live = t < a.tokens, is_q = q0 < q1;
  Place pl{-1, 0, false};
  if (live) {
    uint32_t skipped;
    pl = place_of(a, listed, skipped);
    if (skipped && g == 0 && lane == 0 && a.err) atomicAdd(a.err, skipped);
  }
  const HeadRows& rows = is_q ? a.q : has_k ? a.k : a.v;
  const int64_t head = is_q ? q0 : has_k ? kh : vh;
  Raw8<TI> x[2] = {Raw8<TI>{}, Raw8<TI>{}};
  if (live) {
    const TI* p = static_cast<const TI*>(rows.in) + t * rows.in_token + head * rows.in_head;
    if (has0) x[0] = load8(p + e0);
    if (has1) x[1] = load8(p + e1);
  }
  if (is_q || has_k) table(listed, co, si);
  float f[16];
  turn(w_sm[is_q ? 0 : 1], a.q.weight || a.k.weight, rows.weight != nullptr, is_q || has_k, x, f);
  if (!pl.rotates) return;
  if (rows.out) put(static_cast<TI*>(rows.out) + t * rows.out_token + head * rows.out_head, f);
  else if (pl.cache_row >= 0) put(static_cast<TC*>(a.cache) + pl.cache_row + (has_k ? 0 : a.kv_stride) + head * a.D, f);
}

// Any head_dim, any even R, element-aligned rows: one warp per row, a lane reads and writes
// both members of its pairs (so a row may be rewritten in place). Bound by its instructions: loads
// of single elements, a branch on the type for each entry of the table and the weights, rows read
// twice for a norm. 16384 tokens of 32 + 8 heads of 80 with 40 dims turned, bf16: 468 us with norm,
// 378 without (0.07 and 0.09 of the copy rate); heads of 128 at an odd element: 478 and 472 (0.11).
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
  const Place pl = place_of(a, Listed(a, t), skipped);
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
    inv = inv_rms(s, a.inv_d, a.eps);
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
