// Attention of a ragged batch over a paged prefix that all its requests share and each
// request's own paged suffix.
//
// Mathematics. Row (token t, query head qh) of KV head h: with scores s_k = scale q.k over
// its visible keys, out = sum_k e^(s_k - m) v_k / sum_k e^(s_k - m). The keys are split into
// pieces; a piece leaves (O, m, l) = (sum e^(s - m) v, reference maximum, sum e^(s - m)) and
// pieces join as O = sum O_i e^(m_i - m), l = sum l_i e^(m_i - m). Softmax statistics, O and
// the joins are fp32; the probabilities are rounded to the type of V for the product (the
// tensor cores take both operands in one type; half a step, 2^-8 bf16 / 2^-11 fp16, of each
// probability at most, which averages over the keys: measured against 64 bits, 2.2e-3 of the
// output's norm in bf16 where the output's own rounding is 1.7e-3). In fp16 that holds down to
// 2^-23 of the piece's largest probability; smaller ones are off by up to 2^-34 of it each.
//
// Work. The prefix is one attention problem per KV head whose rows are the new tokens of ALL
// requests x the query heads of the group: its K and V are read once for every 128 or 256
// rows instead of once per request. The suffixes are one small problem per (KV head, request).
// Both are cut into "items" (rows x one key range), every item into tiles of 128 keys, and the
// tiles of all items, laid end to end with a cost each, are dealt to one persistent CTA per SM
// in equal contiguous shares: no tail, no atomics, a fixed order of summation. A share's piece
// of an item (a "segment") writes one partial; merge_partials joins each row's partials.
//
// A CTA: 4 loader warps gather K and V tiles through the block tables into a ring of
// 128-byte-swizzled tiles, by TMA where a block's rows come in eights (a box per block), else
// and where a tile ends inside with 16-byte cp.async (rows past the end become zeros, so
// garbage there cannot reach the products; all by cp.async: 94 / 147 / 219 us for the three cases
// measured below); one warp per stream issues its tcgen05.mma; two softmax
// warpgroups own one stream each, a stream being, in TMEM, 64 keys' scores, two buffers of P and O:
//   S_s [128 rows x 64 keys] = Q K^T (shared memory operands),
//   O_s [128 rows x D]      += P V   (P in TMEM, V the N-major B operand).
// The next scores are begun as soon as a step has read its own, so a stream's chain is its
// softmax alone. One thread owns one row: the softmax needs no exchange. O is rescaled only when the
// maximum grew by more than a few powers of two (`Reference`; each time it grows, the batch of 256
// takes 245 us).
// With more than 128 rows an item has two row tiles, one per stream, that share each K and V
// tile ("pair"); with fewer, the streams take one half of each key tile for one row tile and
// join at the end of the segment ("split"); segments of one tile go to the streams in turn
// ("solo"), so that one's epilogue runs under the other's work.
//
// Measured (both launches, twenty calls in a graph, L2 flushed before each; all figures here and at
// the constants below are by this): 64 requests over 32768 shared keys and up to 1024 own, 32 / 8
// heads of 128, 282 MB, 35 GFLOP: 83 us, the prefix alone 57, the suffixes alone 47 (512 items with
// 4 live rows of 128); 8 requests over 131072, 64 / 8 heads, 616 MB: 125 us (4.9 TB/s, 0.76 of the
// copy rate, by the ring's stages in flight); 256 requests over 32768, 138 GFLOP: 194 to 208 us,
// the prefix alone 152, the suffixes alone 64. In the prefix a pair of streams' steps of 64 keys
// takes about 1850 clocks, its products alone 1304 (Q K^T at N = 64 takes 49 clocks per 16 dims,
// bound by its shared-memory operands, where N = 128 takes 65), softmax 1027 of ex2: the products'
// chain bounds. Steps of 128 keys have cheaper products but leave TMEM for one S a stream, with P
// over it: 223 us at the batch of 256 when steps of 64 took 211 (one call each).
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attention_kernels.cuh"
#include "common.cuh"
#include "f32x2.cuh"

namespace origami {

namespace spa {

constexpr int kThreadsS = 512;  // warps 0-3 / 4-7: softmax of stream 0 / 1; 8-11: loaders; 12 / 14: products of
                                // stream 0 / 1; 13: scheduler
constexpr uint32_t kQueryStartFlag = 0x40000000u;  // of d_error_flags: query_start decreases
constexpr int kTile = 128;      // keys per tile, rows per row tile
constexpr int kHalf = 64;       // keys per softmax step
// Cost units of the deal: a tile that is read for one row tile, one for a pair, the fixed cost of
// an item of either kind (its prologue, epilogue and partial). Chunks (13 requests of up to 300
// tokens, D 64) / batch of 64 / batch of 256 over 32768 keys, us: 68 / 83 / 199 so; a pair's tile
// at 8: 73 / 95 / 223, at 16: 78 / 83 / 221; items for nothing: 80 / 81 / 261, a pair's at 8:
// 70 / 86 / 203, a single's at 16: 70 / 87 / 219.
constexpr int kCostTile = 8, kCostPair = 12, kCostItem = 8, kCostPairItem = 22;
// The probabilities as the products take them: p = 2^(s log2(e) - m), where the reference m lies
// `up` below the largest score (in powers of two) when it is set and follows it once the largest
// has grown by more than `grow`, so that p stays below 2^(up + grow). fp16 ends at 2^16 and loses
// bits below 2^-14: the largest begins at 2^9 there, which puts that end 23 bits below it (with
// `up` 0, keys 17 nats behind one that stands out came to nothing in the products). Of the range,
// growth by 2^6 costs nothing (batch of 64 / of 256 in fp16: 83 / 194 us, with 8 83 / 203), by 2^4
// 88 / 212, by 2^2 95 / 223.
template <bool BF16>
struct Reference {
  static constexpr float up = BF16 ? 0.f : 9.f, grow = BF16 ? 8.f : 6.f;
  static_assert(BF16 || up + grow <= 15.f, "fp16 holds p");
};

// Shared memory: Q tiles, then the ring of K / V tiles (each [128][D] 16-bit), then scalars.
template <int D>
struct Smem {
  static constexpr int tile = kTile * D * 2;
  static constexpr int stages = D == 128 ? 5 : 10;
  static constexpr int lag = 2;  // stages of a warp's own copies in flight before the oldest is signalled
  static constexpr int ring = 2 * tile;
  static constexpr int scalars = ring + stages * tile;
  static constexpr int bytes = scalars + 2 * kTile * 8 + 1024;
};

}  // namespace spa

struct SharedArgs {
  CUtensorMap map;  // the cache as [token rows, heads, D], boxes of tma_rows x 1 x 64; see tma_rows
  const uint16_t* query;
  uint16_t* output;
  float* lse;
  int64_t q_token, q_head, o_token, o_head;
  const uint16_t* cache;
  int64_t kv_stride, row_elems;  // elements from K to V; elements of one token row (heads * D)
  int64_t num_blocks;
  int32_t block_size, block_rows;  // token rows from one block to the next
  const int32_t* prefix_blocks;
  const int32_t* suffix_blocks;
  int64_t suffix_stride;
  const int32_t* suffix_lens;
  const int32_t* query_start;
  int32_t tokens, requests, prefix, suffix_cap;
  int32_t q_heads, kv_heads, group, tile_tokens;  // tokens per row tile
  int32_t item_rows_p, item_rows_s;               // partial rows a CTA may need for a prefix / suffix item
  int32_t q_vec, o_vec, ctas;
  int32_t merge_rows;  // rows a warp of merge_partials joins
  int32_t tma_rows;   // token rows per TMA box (divides the block size), 0: no TMA
  int32_t all_rows, v_rows;  // token rows of the cache; rows from a token's K to its V
  uint32_t inv_ctas;         // floor(2^32 / ctas)
  float scale_log2;
  // workspace
  int32_t* head;      // suffix cost of one head, -1 if the call is refused
  int32_t* req_cost;  // [requests] suffix cost of the requests before this one
  float* ml;          // [rows][2]
  float* o;           // [rows][D]
  uint32_t* err;
};

namespace spa {

using attn::pack2;
using attn::proxy_fence;
using attn::tc_fence_after;
using attn::tc_fence_before;

// ---------------------------------------------------------------------------------------
// The deal: items in order (prefix items of head 0, 1, ..; then suffix items of head 0, 1,
// .. by request and row tile), each with a start on the cost axis (below 2^31: the host checks).
// ---------------------------------------------------------------------------------------
struct Item {
  int32_t start;   // on the cost axis
  int32_t tok0;    // first token
  int32_t ntok;    // its tokens
  int32_t kend;    // keys its last row sees
  int32_t vis0;    // suffix: keys its first token sees (may be negative)
  int32_t h, b;    // KV head; request, -1 for the prefix
  bool pair;
  __device__ __forceinline__ int tiles() const { return (kend + kTile - 1) / kTile; }
  __device__ __forceinline__ int cost() const {
    return kend > 0 ? (pair ? kCostPairItem + tiles() * kCostPair : kCostItem + tiles() * kCostTile) : 0;
  }
  // First tile that a share beginning at w takes.
  __device__ __forceinline__ int tile_at(int w) const {
    const int x = w - start - (pair ? kCostPairItem : kCostItem);
    if (x <= 0) return 0;
    return min(pair ? (x + kCostPair - 1) / kCostPair : (x + kCostTile - 1) / kCostTile, tiles());
  }
};

// Where CTA c's share begins: monotone in c, 0 and `all` at the ends.
__device__ __forceinline__ int share_begin(const SharedArgs& a, int all, int c) {
  return c >= a.ctas ? all : static_cast<int>(__umulhi(static_cast<uint32_t>(all), static_cast<uint32_t>(c) * a.inv_ctas));
}
__device__ __forceinline__ int clamp32(int v, int lo, int hi) { return min(max(v, lo), hi); }
// An entry of the device lists, or of the costs that the first kernel leaves for the join. The
// kernel before on the stream may still be writing them when this one starts, so the load has to
// stay behind the dependent wait: one through the read-only path, which asks for data that nobody
// writes while the kernel lives, may be moved ahead of it.
__device__ __forceinline__ int list_at(const int32_t* p) {
  int v;
  asm volatile("ld.global.s32 %0, [%1];\n" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ int used_tokens(const SharedArgs& a) {
  return clamp32(list_at(a.query_start + a.requests), 0, a.tokens);
}
__device__ __forceinline__ int prefix_item_tokens(const SharedArgs& a, int used) {
  return used > a.tile_tokens ? 2 * a.tile_tokens : a.tile_tokens;
}
__device__ __forceinline__ Item prefix_item(const SharedArgs& a, int used, int h, int tok0, int start) {
  Item it;
  it.start = start;
  it.tok0 = tok0;
  it.ntok = clamp32(used - tok0, 0, prefix_item_tokens(a, used));
  it.kend = a.prefix;
  it.vis0 = a.prefix;
  it.h = h;
  it.b = -1;
  it.pair = it.ntok > a.tile_tokens;
  return it;
}
// Cost of all prefix items of one head.
__device__ __forceinline__ int prefix_cost(const SharedArgs& a, int used) {
  if (used == 0 || a.prefix == 0) return 0;
  const int per = prefix_item_tokens(a, used), before = (used - 1) / per;
  return before * prefix_item(a, used, 0, 0, 0).cost() + prefix_item(a, used, 0, before * per, 0).cost();
}

struct Request {
  int32_t begin, n, len;
};
__device__ __forceinline__ Request request_at(const SharedArgs& a, int b, bool& falls) {
  const int begin = list_at(a.query_start + b), end = list_at(a.query_start + b + 1), len = list_at(a.suffix_lens + b);
  Request r;
  r.begin = clamp32(begin, 0, a.tokens);
  r.n = clamp32(end, r.begin, a.tokens) - r.begin;
  r.len = clamp32(len, 0, a.suffix_cap);
  falls = end < begin;
  return r;
}
__device__ __forceinline__ Request request_at(const SharedArgs& a, int b) {
  bool falls;
  return request_at(a, b, falls);
}
__device__ __forceinline__ Item suffix_item(const SharedArgs& a, const Request& r, int h, int b, int tile, int start) {
  Item it;
  it.start = start;
  const int t0 = tile * a.tile_tokens;
  it.tok0 = r.begin + t0;
  it.ntok = min(a.tile_tokens, r.n - t0);
  it.vis0 = r.len - r.n + t0 + 1;
  it.kend = clamp32(it.vis0 + it.ntok - 1, 0, r.len);
  it.h = h;
  it.b = b;
  it.pair = false;
  return it;
}
// Cost of a request's row tiles.
__device__ __forceinline__ int request_cost(const SharedArgs& a, const Request& r) {
  int c = 0;
#pragma unroll 1
  for (int t = 0; t * a.tile_tokens < r.n; ++t) c += suffix_item(a, r, 0, 0, t, 0).cost();
  return c;
}

// Where a CTA's share begins and ends, and its first suffix item.
struct Deal {
  int32_t wp;      // cost of one head's prefix items
  int32_t w0, w1;  // this CTA's share
  int32_t used;
  int32_t h, b, tile, start;
};

// Walks the segments of a CTA's share (one warp of the CTA).
struct Walk {
  const SharedArgs& a;
  const Deal& d;
  Item it;
  int t0, t1;      // tiles of the segment
  int next;        // start of the item after `it`
  int h, b, tile;  // next suffix item
  int ph, ptok;    // next prefix item: head and first token
  bool in_prefix;
  Request r;
  __device__ __forceinline__ Walk(const SharedArgs& args, const Deal& deal) : a(args), d(deal), r(request_at(args, deal.b)) {
    in_prefix = d.w0 < d.wp * a.kv_heads;
    h = d.h;
    b = d.b;
    tile = d.tile;
    next = d.start;
    ph = 0;
    ptok = 0;
    if (in_prefix) {
      const int per = prefix_item_tokens(a, d.used), first = prefix_item(a, d.used, 0, 0, 0).cost();
      ph = d.w0 / d.wp;
      const int i = min((d.w0 - ph * d.wp) / first, (d.used - 1) / per);
      ptok = i * per;
      next = ph * d.wp + i * first;
    }
  }
  __device__ __forceinline__ bool step() {
#pragma unroll 1
    while (next < d.w1) {
      if (in_prefix) {
        it = prefix_item(a, d.used, ph, ptok, next);
        ptok += it.ntok;
        if (ptok >= d.used) {
          ptok = 0;
          ++ph;
        }
        if (ph >= a.kv_heads) {
          in_prefix = false;
          h = b = tile = 0;
          r = request_at(a, 0);
        }
      } else {
        // past the last head there is nothing (requests without any tile cost nothing)
        if (h >= a.kv_heads) return false;
        if (tile * a.tile_tokens >= r.n) {
          tile = 0;
          if (++b >= a.requests) {
            b = 0;
            ++h;
          }
          r = request_at(a, b);
          continue;
        }
        it = suffix_item(a, r, h, b, tile, next);
        ++tile;
      }
      next += it.cost();
      if (it.kend <= 0) continue;
      t0 = it.tile_at(d.w0);
      t1 = it.tile_at(d.w1);
      if (t1 > t0) return true;
    }
    return false;
  }
};

// A segment as the other warps read it from shared memory.
struct Segment {
  int64_t prow;       // partial row of its first row
  int32_t t0, n;      // first tile, tiles; n = 0 ends the share
  int32_t halves;     // 64-key halves of its tiles that hold keys
  int32_t mode, h, b;  // kSplit .. kSolo + 1; KV head; request, -1 for the prefix
  int32_t tok0, ntok, kend, vis0;
};
constexpr int kSplit = 0, kPair = 1, kSolo = 2;  // how the streams share a segment; kSolo + s: stream s alone
// The readers of a segment's tiles: stream 0, stream 1, or 2 for both.
__device__ __forceinline__ uint32_t readers(int mode) { return mode < kSolo ? 2u : static_cast<uint32_t>(mode - kSolo); }
constexpr int kSegments = 4;  // in the ring between the scheduler and the others

// Partial rows: an item's rows begin at its place among all rows of its kind plus its CTA's
// index times the rows one item may have. Two segments never overlap: a later CTA's segment of
// one item lies item_rows further, a later item at least this item's rows further.
__device__ __forceinline__ int64_t partial_base(const SharedArgs& a, const Item& it, int cta) {
  const int64_t rows = (static_cast<int64_t>(it.h) * a.tokens + it.tok0) * a.group;
  if (it.b < 0) return rows + static_cast<int64_t>(cta) * a.item_rows_p;
  return static_cast<int64_t>(a.q_heads) * a.tokens + static_cast<int64_t>(a.ctas) * a.item_rows_p + rows +
         static_cast<int64_t>(cta) * a.item_rows_s;
}

// ---------------------------------------------------------------------------------------
// tcgen05 helpers
// ---------------------------------------------------------------------------------------
// Descriptors of 128-byte-swizzled tiles [rows][64 elements] (8-row groups 1024 bytes apart).
// K-major (Q, K): a further 64 dims are another 16 KB tile, addressed by the start.
// N-major (V): 64-dim columns of the tile lie 16 KB (the leading byte offset) apart.
__device__ __forceinline__ uint64_t desc128(uint32_t addr, uint32_t lbo) {
  return (static_cast<uint64_t>(addr >> 4) & 0x3FFFull) | (static_cast<uint64_t>(lbo >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// The warp that issues products runs as one, so that descriptors stay in uniform registers;
// `lead` is 1 in the elected thread, whose products and commits these are.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t lead;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(lead));
  return lead;
}
__device__ __forceinline__ void mma_ss(uint32_t lead, uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(da), "l"(db), "r"(idesc), "r"(acc), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t lead, uint32_t d, uint32_t ta, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(ta), "l"(db), "r"(idesc), "r"(acc), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t lead, uint32_t bar) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar),
      "r"(lead)
      : "memory");
}

// 32 TMEM columns of this thread's lane from each of two addresses: two loads in flight, one
// wait. The empty statements tie every value to the wait, so that none is used before it.
__device__ __forceinline__ void ld64(uint32_t a0, uint32_t a1, uint32_t (&r)[64]) {
#pragma unroll
  for (int c = 0; c < 64; c += 32)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
        "%30,%31}, [%32];\n"
        : "=r"(r[c]), "=r"(r[c + 1]), "=r"(r[c + 2]), "=r"(r[c + 3]), "=r"(r[c + 4]), "=r"(r[c + 5]), "=r"(r[c + 6]),
          "=r"(r[c + 7]), "=r"(r[c + 8]), "=r"(r[c + 9]), "=r"(r[c + 10]), "=r"(r[c + 11]), "=r"(r[c + 12]),
          "=r"(r[c + 13]), "=r"(r[c + 14]), "=r"(r[c + 15]), "=r"(r[c + 16]), "=r"(r[c + 17]), "=r"(r[c + 18]),
          "=r"(r[c + 19]), "=r"(r[c + 20]), "=r"(r[c + 21]), "=r"(r[c + 22]), "=r"(r[c + 23]), "=r"(r[c + 24]),
          "=r"(r[c + 25]), "=r"(r[c + 26]), "=r"(r[c + 27]), "=r"(r[c + 28]), "=r"(r[c + 29]), "=r"(r[c + 30]),
          "=r"(r[c + 31])
        : "r"(c == 0 ? a0 : a1)
        : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
  for (int j = 0; j < 64; ++j) asm volatile("" : "+r"(r[j]));
}
__device__ __forceinline__ void ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      " tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A warp's bounded wait, agreed by its lanes, that gives up early when another role has. The
// ready barrier costs one poll and one vote; the loop is kept short, as every role has several.
__device__ __forceinline__ uint32_t try_bar(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done;
}
__device__ __forceinline__ bool poll(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, try_bar(smem_u32(bar), parity) != 0) != 0;
}
constexpr uint32_t kPolls = 1u << 19;  // about 2 s, far beyond any copy or product
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort) {
#pragma unroll 1
  for (uint32_t i = 0; i < kPolls; ++i) {
    if (poll(bar, parity)) return true;
    if (__any_sync(0xffffffffu, *abort)) return false;
  }
  *abort = 1;
  return false;
}

// One arrival for a warp (arrivals of single lanes on one barrier would queue up).
__device__ __forceinline__ void arrive_warp(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// Copy of 16 bytes, or 16 zero bytes where `valid` is false (the source is then not read).
__device__ __forceinline__ void cp16_or_zero(uint32_t dst, const void* src, bool valid) {
  const uint32_t n = valid ? 16u : 0u;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

// The first n of o as consecutive floats of a partial row, whole 32-byte sectors a store.
__device__ __forceinline__ void store_o(float* p, const uint32_t (&o)[64], int n) {
#pragma unroll
  for (int j = 0; j < 64; j += 8)
    if (j < n)
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(p + j), "r"(o[j]), "r"(o[j + 1]),
                   "r"(o[j + 2]), "r"(o[j + 3]), "r"(o[j + 4]), "r"(o[j + 5]), "r"(o[j + 6]), "r"(o[j + 7])
                   : "memory");
}

__device__ __forceinline__ void cp_async16_at(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}

// Byte offset of 16-byte chunk c of row r in a swizzled [128][D] tile.
__device__ __forceinline__ uint32_t chunk_off(int r, int c) {
  return static_cast<uint32_t>((c >> 3) * (kTile * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// TMA: a box of the cache's token rows from row z, one head, 64 dims from x; the elected thread's
// (lanes that each issue their own take 65 clocks a box, an elected one 18).
__device__ __forceinline__ void tma_rows(uint32_t lead, uint32_t dst, const CUtensorMap* map, int x, int head, int z, uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %6, 0;\n"
      " @q cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n}\n" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(head), "r"(z), "r"(smem_u32(bar)), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;\n" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

// A parity tells a barrier's last phase from the one before only, so whoever waits on a barrier
// has to see each of its phases. S begins anew only when every warp has read the last (s_empty),
// and P's two buffers have a barrier each. A stage's tile is read by stream 0, by stream 1 or by
// both: its arrival goes to the barrier of that set of readers.
struct Bars {
  uint64_t full[3][10], empty[10], q_empty[2], s_full[2], s_empty[2], p_full[4], pv[4], seg_full[kSegments], seg_empty[kSegments];
  uint64_t o_free[2], xch, done;
};

}  // namespace spa

// ---------------------------------------------------------------------------------------
// One persistent CTA per SM.
// ---------------------------------------------------------------------------------------
template <typename QT, int D>
__global__ void __launch_bounds__(spa::kThreadsS, 1) shared_prefix_attention(const __grid_constant__ SharedArgs a) {
  using namespace spa;
  using S = Smem<D>;
  extern __shared__ __align__(1024) uint8_t spa_smem[];
  uint8_t* sm = spa_smem;
  float2* ml_sm = reinterpret_cast<float2*>(sm + S::scalars);  // [2 streams][128 rows]
  Bars* bars = reinterpret_cast<Bars*>(ml_sm + 2 * kTile);
  uint32_t* tslot = reinterpret_cast<uint32_t*>(bars + 1);
  int* abort_sm = reinterpret_cast<int*>(tslot + 1);
  Deal* deal_sm = reinterpret_cast<Deal*>(tslot + 2);
  Segment* segs = reinterpret_cast<Segment*>(deal_sm + 1);
  static_assert(sizeof(Bars) + 8 + sizeof(Deal) + kSegments * sizeof(Segment) <= 1024, "scalars fit");
  static_assert(S::bytes <= 227 * 1024, "shared memory of one SM");
  constexpr bool kBf16 = attn::is_bf16<QT>();
  using Ref = Reference<kBf16>;
  constexpr uint32_t kIdescS = attn::instr_desc(kBf16, kHalf);
  constexpr uint32_t kIdescO = attn::instr_desc(kBf16, D) | (1u << 16);  // B (V) is N-major
  constexpr uint32_t kP = 64, kO = 128;  // of stream s: S at column 256 s, P at + 64 and + 96, O at + 128

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = static_cast<int>(blockIdx.x);
  // the tiles' swizzle is a function of the address: they must begin on a 1024-byte boundary
  if (smem_u32(sm) & 1023) {
    if (tid == 0 && a.err) atomicOr(a.err, kWaitTimeoutFlag);
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < S::stages; ++i) {
      for (int r = 0; r < 3; ++r) mbar_init(&bars->full[r][i], 4);
      mbar_init(&bars->empty[i], 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->q_empty[i], 2);
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->s_empty[i], 4);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&bars->pv[i], 1);
      mbar_init(&bars->p_full[i], 4);
    }
    for (int i = 0; i < kSegments; ++i) {
      mbar_init(&bars->seg_full[i], 1);
      mbar_init(&bars->seg_empty[i], 8 + 4 + 2);  // softmax, loader and product warps
    }
    mbar_init(&bars->o_free[0], 8);
    mbar_init(&bars->o_free[1], 8);
    mbar_init(&bars->xch, 8);
    mbar_init(&bars->done, 2);
    *abort_sm = 0;
    fence_mbar_init();
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tslot)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
  }
  // dependent launch: everything above overlaps the kernel before this one
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");

  // The deal: suffix costs of contiguous runs of requests, scanned over the CTA.
  {
    int* scan = reinterpret_cast<int*>(sm);  // [16] warp sums
    const int per = (a.requests + kThreadsS - 1) / kThreadsS;
    const int b0 = min(tid * per, a.requests), b1 = min(b0 + per, a.requests);
    const int used = used_tokens(a);
    int sum = 0;
    bool falls = false;  // query_start does: requests would share tokens, and their costs have no bound
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
      bool here;
      sum += request_cost(a, request_at(a, b, here));
      falls |= here;
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) scan[warp] = incl;
    const bool refused = __syncthreads_or(falls) != 0;
    int before = lane < kThreadsS / 32 ? scan[lane] : 0, total = before;
    if (lane >= warp) before = 0;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      before += __shfl_xor_sync(0xffffffffu, before, o);
      total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    before = __shfl_sync(0xffffffffu, before, 0);
    total = refused ? 0 : __shfl_sync(0xffffffffu, total, 0);
    const int excl = before + incl - sum;
    const int wp = refused ? 0 : prefix_cost(a, used), all_p = wp * a.kv_heads, all = all_p + total * a.kv_heads;
    const int w0 = share_begin(a, all, cta);
    // the share's first suffix item lies in the run of requests that holds its cost
    const int y = max(w0 - all_p, 0), fh = total > 0 ? y / total : a.kv_heads, rem = total > 0 ? y - fh * total : 0;
    if (tid == 0) {
      deal_sm->wp = wp;
      deal_sm->w0 = w0;
      deal_sm->w1 = share_begin(a, all, cta + 1);
      deal_sm->used = used;
      if (total == 0) {  // no suffix anywhere
        deal_sm->h = fh;
        deal_sm->b = deal_sm->tile = 0;
        deal_sm->start = all_p;
      }
      if (cta == 0) *a.head = refused ? -1 : total;
      if (cta == 0 && refused && a.err) atomicOr(a.err, kQueryStartFlag);
    }
    if (!refused && ((sum > 0 && rem >= excl && rem < excl + sum) || cta == 0)) {
      int at = excl;
#pragma unroll 1
      for (int b = b0; b < b1; ++b) {
        const Request r = request_at(a, b);
        const int c = request_cost(a, r);
        if (cta == 0) a.req_cost[b] = at;
        if (c > 0 && rem >= at && rem < at + c) {
          int t = 0, start = at;
#pragma unroll 1
          for (;; ++t) {
            const int x = suffix_item(a, r, 0, 0, t, 0).cost();
            if (rem < start + x) break;
            start += x;
          }
          deal_sm->h = fh;
          deal_sm->b = b;
          deal_sm->tile = t;
          deal_sm->start = all_p + fh * total + start;
        }
        at += c;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tslot;
  volatile int* abort = abort_sm;

  if (warp >= 8 && warp < 12) {
    // ---------------------------------------------------------------- loaders
    // Warp lw fills rows 32 lw .. 32 lw + 31 of every tile; lane l knows row 32 lw + l.
    constexpr int kChunks = D / 8;          // 16-byte chunks per row
    constexpr int kRowsPer = 32 / kChunks;  // rows a warp copies at once
    const int lw = __shfl_sync(0xffffffffu, warp - 8, 0);
    const uint32_t lead = elect_one();
    const int sub = lane / kChunks, chunk = lane % kChunks;
    // this lane's chunk of row 32 lw + sub; kRowsPer rows on, the row's swizzle changes
    const uint32_t base = smem_u32(sm);
    uint32_t ring = 0, signalled = 0;  // stages begun, stages whose arrival this warp has made
    uint32_t slot = 0, q_used = 0u, q_phase = 0u, q_next = 0u;
    // a segment's first tile is signalled with its Q: held back until Q is requested, and then
    // until it has landed (q_wait)
    bool ok = true, q_hold = false, q_wait = false;
    uint32_t hold = 0, sets = 0;  // sets: the readers of each stage, two bits
    // Copies of this warp's own threads are generic-proxy writes: the fence that orders the
    // products' reads behind them is made here, once they have landed (in the products' warp it
    // would wait for the products under way). TMA stages need none and arrive at once unless an
    // older stage is still to be signalled.
    auto signal = [&](uint32_t upto) {
      if (signalled == upto) return;
      proxy_fence();
      __syncwarp();
      if (lane == 0)
        for (uint32_t i = signalled; i < upto; ++i) {
          const uint32_t st = i % S::stages;
          mbar_arrive(&bars->full[(sets >> (2 * st)) & 3u][st]);
        }
      signalled = upto;
    };
    auto drain = [&]() {
      asm volatile("cp.async.wait_all;\n" ::: "memory");
      signal(q_hold ? hold : ring);
      q_wait = q_wait && q_hold;
    };
    // Waits with nothing unsignalled behind: whoever makes the arrival may need it.
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (poll(bar, parity)) return true;
      drain();
      return wait_warp(bar, parity, abort);
    };
    for (;; ++slot) {
      ok = ok && wait(&bars->seg_full[slot % kSegments], (slot / kSegments) & 1u);
      if (!ok) break;
      const Segment seg = segs[slot % kSegments];
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->seg_empty[slot % kSegments]);
      if (seg.n == 0) break;
      const int head = __shfl_sync(0xffffffffu, seg.h, 0);
      const int32_t* table = seg.b < 0 ? a.prefix_blocks : a.suffix_blocks + seg.b * a.suffix_stride;
      // cache row of key `key`, negative past the end of the item or outside the cache
      auto row_of = [&](int key) -> int {
        if (key >= seg.kend) return -1;
        const uint32_t page = static_cast<uint32_t>(key) / static_cast<uint32_t>(a.block_size);
        const int pb = list_at(table + page);
        return pb < 0 || pb >= a.num_blocks ? -1 : pb * a.block_rows + (key - static_cast<int>(page) * a.block_size);
      };
      int key = seg.t0 * kTile + 32 * lw + lane;
      int row = row_of(key);
      if (signalled != ring) drain();
      q_hold = true;
      hold = ring;
      const uint32_t set = readers(seg.mode);
#pragma unroll 1
      for (int i = 0; i < seg.n && ok; ++i) {
        const bool tma = a.tma_rows > 0 && __all_sync(0xffffffffu, key < seg.kend);
        key += kTile;
        const int next_row = i + 1 < seg.n ? row_of(key) : -1;
        // Waits until stage `ring` may be refilled, copies this warp's rows of K (which = 0) and
        // of V: all inside the item by TMA, else row by row. The stage is full when every
        // loader warp's rows have landed (Q's with the first K's).
#pragma unroll 1
        for (int which = 0; which < 2; ++which) {
          const uint32_t st = ring % S::stages, use = ring / S::stages;
          if (use > 0 && !wait(&bars->empty[st], (use - 1) & 1u)) {
            ok = false;
            break;
          }
          const uint32_t dst = base + S::ring + st * S::tile + lw * (32 * 128);  // this warp's rows
          uint64_t* full = &bars->full[set][st];
          sets = (sets & ~(3u << (2 * st))) | (set << (2 * st));
          if (tma) {
            if (lead) expect_tx(full, 32 * D * 2);
            __syncwarp();
            const int z = row < 0 ? a.all_rows : row + which * a.v_rows;  // past the last row: zeros
#pragma unroll 1
            for (int r = 0; r < 32; r += a.tma_rows) {
              const int zr = __shfl_sync(0xffffffffu, z, r);
#pragma unroll
              for (int x = 0; x < D; x += 64)
                tma_rows(lead, dst + (x >> 6) * (kTile * 128) + r * 128, &a.map, x, head, zr, full);
            }
          } else {
            const uint16_t* src = a.cache + which * a.kv_stride + static_cast<int64_t>(seg.h) * D + chunk * 8;
#pragma unroll 4
            for (int j = 0; j < 32 / kRowsPer; ++j) {
              const int r = j * kRowsPer + sub;
              const int cr = __shfl_sync(0xffffffffu, row, r);
              cp16_or_zero(dst + chunk_off(r, chunk), src + (cr < 0 ? 0 : cr) * a.row_elems, cr >= 0);
            }
          }
          asm volatile("cp.async.commit_group;\n" ::: "memory");
          ++ring;
          if (q_hold) continue;
          if (q_wait) {
            drain();
          } else if (tma && signalled + 1 == ring) {
            if (lead) mbar_arrive(full);
            signalled = ring;
          } else if (ring - signalled > S::lag) {
            asm volatile("cp.async.wait_group %0;\n" ::"n"(S::lag) : "memory");
            signal(ring - S::lag);
          }
        }
        row = next_row;
        if (i > 0) continue;
        // Q, behind the first tile's requests: one row tile, into the buffer after the last one
        // used, or both for a pair. Rows past the end keep what lies there: they reach nothing but
        // their own rows of S and O.
        if (seg.mode == kPair) q_next = 0;
#pragma unroll 1
        for (int q = 0; q <= (seg.mode == kPair); ++q) {
          const uint32_t buf = q_next;
          q_next ^= 1u;
          if ((q_used >> buf) & 1u) {
            ok = wait(&bars->q_empty[buf], (q_phase >> buf) & 1u);
            if (!ok) break;
            q_phase ^= 1u << buf;
          }
          q_used |= 1u << buf;
          // lane l finds the query row of tile row 32 lw + l
          const int mine = min(a.tile_tokens, seg.ntok - q * a.tile_tokens) * a.group - 32 * lw;  // rows of this warp
          if (mine <= 0) continue;
          const int tile_row = 32 * lw + lane, tl = tile_row / a.group;
          const int64_t at = (seg.tok0 + static_cast<int64_t>(q) * a.tile_tokens + tl) * a.q_token +
                             (seg.h * a.group + tile_row - tl * a.group) * a.q_head;
          const uint32_t dst = base + buf * S::tile;
#pragma unroll 1
          for (int i = 0; i < min(mine, 32); i += 2 * kRowsPer) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int r = i + j * kRowsPer + sub;
              const uint16_t* src = a.query + __shfl_sync(0xffffffffu, at, r & 31) + chunk * 8;
              if (r >= mine || r >= 32) continue;
              if (a.q_vec) {
                cp_async16_at(dst + chunk_off(32 * lw + r, chunk), src);
              } else {
                uint32_t v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = src[2 * e] | (static_cast<uint32_t>(src[2 * e + 1]) << 16);
                *reinterpret_cast<uint4*>(sm + buf * S::tile + chunk_off(32 * lw + r, chunk)) =
                    make_uint4(v[0], v[1], v[2], v[3]);
              }
            }
          }
        }
        q_hold = false;
        q_wait = true;
      }
    }
    drain();
    // every stage was waited for by the products; after a timeout, time for the copies in flight to land
    if (*abort) {
      const long long begin = clock64();
      while (clock64() - begin < 2000000) {
      }
    }
  } else if (warp >= 12) {
    if (warp == 13) {
      // -------------------------------------------------------------- scheduler
      const Deal deal = *deal_sm;
      Walk w(a, deal);
      uint32_t solos = 0u;
      for (uint32_t slot = 0;; ++slot) {
        const uint32_t at = slot % kSegments, use = slot / kSegments;
        const bool more = w.step();
        if (use > 0 && !wait_warp(&bars->seg_empty[at], (use - 1) & 1u, abort)) break;
        if (lane == 0) {
          Segment& g = segs[at];
          g.n = more ? w.t1 - w.t0 : 0;
          g.t0 = w.t0;
          g.halves = (min(w.it.kend - w.t0 * kTile, g.n * kTile) + kHalf - 1) / kHalf;
          // one tile: a stream of its own, unless it is all that this CTA has and both can work at it
          const bool solo = !w.it.pair && g.n == 1 && (g.halves == 1 || slot > 0 || w.next < deal.w1);
          g.mode = w.it.pair ? kPair : solo ? kSolo + static_cast<int>(solos++ & 1u) : kSplit;
          g.h = w.it.h;
          g.b = w.it.b;
          g.tok0 = w.it.tok0;
          g.ntok = w.it.ntok;
          g.kend = w.it.kend;
          g.vis0 = w.it.vis0;
          g.prow = more ? partial_base(a, w.it, cta) : 0;
          mbar_arrive(&bars->seg_full[at]);
        }
        if (!more) break;
      }
    } else if (warp == 12 || warp == 14) {
      // -------------------------------------------------------------- products of stream s
      const uint32_t s = warp == 12 ? 0u : 1u;
      const uint32_t base = __shfl_sync(0xffffffffu, smem_u32(sm), 0), tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t lead = elect_one();
      auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_warp(bar, parity, abort); };
      auto at = [&](const void* bar) { return __shfl_sync(0xffffffffu, smem_u32(bar), 0); };
      const uint32_t full_own = at(&bars->full[s][0]), full_both = at(&bars->full[2][0]), empty = at(&bars->empty[0]);
      const uint32_t s_full = at(&bars->s_full[s]), s_empty = at(&bars->s_empty[s]);
      const uint32_t p_full = at(&bars->p_full[2 * s]), pv = at(&bars->pv[2 * s]);
      // stages of the tiles that S and P V use next (K and V alternate in the ring); phases of this
      // stream's own full barriers and of the shared ones, a bit per stage
      uint32_t k_stage = 0u, v_stage = 1u, own = 0u, both = 0u;
      auto next_tile = [](uint32_t& stage) {
        stage += 2;
        if (stage >= S::stages) stage -= S::stages;
      };
      uint32_t n_s = 0u, n_pv = 0u, n_seg = 0u, q_next = 0u;  // S and P V products begun, segments ended
      bool ok = true;
#pragma unroll 1
      for (uint32_t slot = 0;; ++slot) {
        if (!ok || !wait(&bars->seg_full[slot % kSegments], (slot / kSegments) & 1u)) break;
        const int n = __shfl_sync(0xffffffffu, segs[slot % kSegments].n, 0);
        const int mode = __shfl_sync(0xffffffffu, segs[slot % kSegments].mode, 0);
        const int halves = __shfl_sync(0xffffffffu, segs[slot % kSegments].halves, 0);
        if (lead) mbar_arrive(&bars->seg_empty[slot % kSegments]);
        if (n == 0) break;
        if (mode == kPair) q_next = 0;
        const uint32_t qb = mode == kPair ? s : q_next;
        if (mode != kPair) q_next ^= 1u;
        if (mode >= kSolo && mode - kSolo != static_cast<int>(s)) {  // one tile, the other stream's
          next_tile(k_stage);
          next_tile(v_stage);
          continue;
        }
        // Step g of the stream is half s of tile g (split) or half g & 1 of tile g >> 1.
        const int steps = mode == kSplit ? (halves + 1 - static_cast<int>(s)) / 2 : halves;
        const int odd = mode == kSplit ? 0 : 1;  // a tile's first step has (g & odd) == 0, its last odd, or ends the segment
        const uint32_t half0 = mode == kSplit ? s * (kHalf * 128) : 0u;
        const uint64_t qd = desc128(base + qb * S::tile, 16);
        const bool solo = mode >= kSolo;
        const uint32_t full = solo ? full_own : full_both;
        uint32_t bits = solo ? own : both;  // phases of the full barriers of these tiles' readers
        // A tile and a Q buffer are freed by two arrivals: one of each stream that reads it, or
        // both of the only one.
        auto free_tile = [&](uint32_t stage) {
          commit(lead, empty + 8 * stage);
          if (solo) commit(lead, empty + 8 * stage);
          bits ^= 1u << stage;
        };
        auto free_q = [&]() {
          commit(lead, smem_u32(&bars->q_empty[qb]));
          if (mode != kSplit) commit(lead, smem_u32(&bars->q_empty[qb]));
        };
        // The two barriers that a product waits for are tried together: ready, as they mostly are,
        // they cost one vote.
        auto wait2 = [&](uint32_t b0, uint32_t parity0, bool need0, uint32_t b1, uint32_t parity1, bool need1) {
#pragma unroll 1
          for (uint32_t i = 0; i < kPolls; ++i) {
            const uint32_t d0 = need0 ? try_bar(b0, parity0) : 1u, d1 = need1 ? try_bar(b1, parity1) : 1u;
            if (__all_sync(0xffffffffu, (d0 & d1) != 0)) return true;
            if (__any_sync(0xffffffffu, *abort)) return false;
          }
          *abort = 1;
          return false;
        };
        // S of step g + 1 is begun before P V of step g
#pragma unroll 1
        for (int g = -1; g < steps; ++g) {
          if (g + 1 < steps) {
            const int x = g + 1;
            // the tile is there and the last S has been read
            ok = wait2(full + 8 * k_stage, (bits >> k_stage) & 1u, (x & odd) == 0, s_empty, (n_s - 1) & 1u, n_s > 0);
            if (!ok) break;
            tc_fence_after();
            const uint32_t d = tm + 256 * s;
            const uint64_t kd = desc128(base + S::ring + k_stage * S::tile + half0 + (x & odd) * (kHalf * 128), 16);
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              const uint64_t off = ((k >> 2) * (kTile * 128) + (k & 3) * 32) >> 4;
              mma_ss(lead, d, qd + off, kd + off, kIdescS, k > 0 ? 1u : 0u);
            }
            commit(lead, s_full);
            ++n_s;
            if ((x & odd) == odd || x == steps - 1) {
              free_tile(k_stage);
              next_tile(k_stage);
            }
            if (x == steps - 1) free_q();
          }
          if (g >= 0) {
            if (g == 0 && n_seg > 0) {  // the last segment's O has been read
              ok = wait(&bars->o_free[s], (n_seg - 1) & 1u);
              if (!ok) break;
            }
            ok = wait2(full + 8 * v_stage, (bits >> v_stage) & 1u, (g & odd) == 0, p_full + 8 * (n_pv & 1u),
                       (n_pv >> 1) & 1u, true);
            if (!ok) break;
            tc_fence_after();
            const uint32_t d = tm + 256 * s + kO, p = tm + 256 * s + kP + 32 * (n_pv & 1u);
            const uint64_t vd =
                desc128(base + S::ring + v_stage * S::tile + half0 + (g & odd) * (kHalf * 128), kTile * 128);
#pragma unroll
            for (int k = 0; k < kHalf / 16; ++k)
              mma_ts(lead, d, p + k * 8, vd + k * (2048 >> 4), kIdescO, (g > 0 || k > 0) ? 1u : 0u);
            commit(lead, pv + 8 * (n_pv & 1u));
            ++n_pv;
            if ((g & odd) == odd || g == steps - 1) {
              free_tile(v_stage);
              next_tile(v_stage);
            }
          }
        }
        if (!ok) break;
        ++n_seg;
        if (mode == kSplit && steps < n) {  // the last tile has no keys for this stream: seen and freed
          ok = wait2(full + 8 * k_stage, (bits >> k_stage) & 1u, true, full + 8 * v_stage, (bits >> v_stage) & 1u, true);
          free_tile(k_stage);
          free_tile(v_stage);
          next_tile(k_stage);
          next_tile(v_stage);
        }
        if (solo) own = bits;
        else both = bits;
      }
      // nothing may be in flight when the columns are released
      commit(lead, smem_u32(&bars->done));
      mbar_wait_bounded(&bars->done, 0u, kPolls);
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax of stream s
    const int s = warp >> 2;
    const int row = tid & (kTile - 1);
    const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t ts = lane_base + 256 * s, to = ts + kO;
    const int token_in_tile = row / a.group;
    uint32_t count = 0u, x_phase = 0u;  // steps so far
    bool ok = true;
    for (uint32_t slot = 0;; ++slot) {
      ok = ok && wait_warp(&bars->seg_full[slot % kSegments], (slot / kSegments) & 1u, abort);
      if (!ok) break;
      const Segment seg = segs[slot % kSegments];
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->seg_empty[slot % kSegments]);
      if (seg.n == 0) break;
      if (seg.mode >= kSolo && seg.mode - kSolo != s) continue;
      const bool split = seg.mode == kSplit;
      const int steps = !split ? seg.halves : s == 0 ? (seg.halves + 1) / 2 : seg.halves / 2;
      const int first_tok = seg.mode == kPair ? s * a.tile_tokens : 0;
      const int rows = min(a.tile_tokens, seg.ntok - first_tok) * a.group;
      const bool warp_live = (warp & 3) * 32 < rows;
      // keys of the item this row sees, less those before the current step's
      int lim = 0;
      if (row < rows) lim = seg.b < 0 ? seg.kend : clamp32(seg.vis0 + token_in_tile, 0, seg.kend);
      lim -= seg.t0 * kTile + (split ? s * kHalf : 0);
      float m = -INFINITY, l = 0.f;
#pragma unroll 1
      for (int i = 0; i < steps; ++i) {
        const uint32_t buf = count & 1u;
        ok = wait_warp(&bars->s_full[s], count & 1u, abort);
        if (!ok) break;
        tc_fence_after();
        if (warp_live) {
          uint32_t x[kHalf];
          ld64(ts, ts + 32, x);
          tc_fence_before();
          arrive_warp(&bars->s_empty[s]);
          if (!__all_sync(0xffffffffu, lim >= kHalf || row >= rows)) {
#pragma unroll
            for (int j = 0; j < kHalf; ++j)
              if (j >= lim) x[j] = 0xFF800000u;  // -inf: not seen
          }
          float mx[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) mx[k] = __uint_as_float(x[k]);
#pragma unroll
          for (int j = 4; j + 8 <= kHalf; j += 8) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mx[k] = max3(mx[k], __uint_as_float(x[j + 2 * k]), __uint_as_float(x[j + 2 * k + 1]));
          }
          mx[0] = max3(mx[0], __uint_as_float(x[kHalf - 4]), __uint_as_float(x[kHalf - 3]));
          mx[1] = max3(mx[1], __uint_as_float(x[kHalf - 2]), __uint_as_float(x[kHalf - 1]));
          // directed roundings: no score lies above mt, no reference more than up + grow below one
          const float mt = __fmul_ru(fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]), a.scale_log2);
          const float ref = __fsub_ru(mt, Ref::up);
          const bool grow = row < rows && (mt > __fadd_rd(m, Ref::up + Ref::grow) || (m == -INFINITY && mt > -INFINITY));
          if (__any_sync(0xffffffffu, grow)) {
            const float alpha = grow ? (m == -INFINITY ? 0.f : ex2(m - ref)) : 1.f;
            if (i > 0) {  // O is at rest once the product of the step before has ended
              const uint32_t last = count - 1;
              ok = wait_warp(&bars->pv[2 * s + (last & 1u)], (last >> 1) & 1u, abort);
              if (!ok) break;
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < D; c += 16) {
                uint32_t o[16];
                ld16(to + c, o);
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
                st16(to + c, o);
              }
            }
            l *= alpha;
            m = grow ? ref : m;
          }
          // P's buffer is free: S of this step was begun after the product of two steps before,
          // and its barrier tells that all products begun before it have ended
          const float neg = m == -INFINITY ? 0.f : -m;
          const uint64_t scale2 = pair2(a.scale_log2, a.scale_log2), neg2 = pair2(neg, neg);
          uint64_t sum[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint32_t p[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const uint64_t arg =
                  fma2(pair2(__uint_as_float(x[32 * q + 2 * j]), __uint_as_float(x[32 * q + 2 * j + 1])), scale2, neg2);
              float p0, p1;
              split2(arg, p0, p1);
              p0 = ex2(p0);
              p1 = ex2(p1);
              sum[j & 3] = add2(sum[j & 3], pair2(p0, p1));
              p[j] = pack2<QT>(p0, p1);
            }
            st16(ts + kP + 32 * buf + 16 * q, p);
          }
          float l0, l1;
          split2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), l0, l1);
          l += l0 + l1;
          st_wait();
        } else {
          arrive_warp(&bars->s_empty[s]);
        }
        tc_fence_before();
        arrive_warp(&bars->p_full[2 * s + buf]);
        lim -= split ? kTile : kHalf;
        ++count;
      }
      if (!ok) break;
      // ------------------------------------------------------------ the segment's partial
      // scores that are all NaN leave no maximum: any reference carries their NaN on
      if (l != l && m == -INFINITY) m = 0.f;
      {
        const uint32_t last = count - 1;
        ok = wait_warp(&bars->pv[2 * s + (last & 1u)], (last >> 1) & 1u, abort);
        if (!ok) break;
      }
      if (split) {
        // Both streams' sums belong to the same rows: exchange (m, l), then each stream joins and
        // writes half of the dims. (m, l) of the split segment before were read before a stream's
        // next product into O could begin.
        ml_sm[s * kTile + row] = make_float2(m, l);
        tc_fence_before();
        arrive_warp(&bars->xch);
        ok = wait_warp(&bars->xch, x_phase, abort);
        if (!ok) break;
        x_phase ^= 1u;
      }
      tc_fence_after();
      if (warp_live) {
        const int64_t prow = seg.prow + first_tok * a.group + row;
        if (!split) {
#pragma unroll 1
          for (int c = 0; c < D; c += 64) {
            uint32_t o[64];
            ld64(to + c, to + c + 32, o);
            if (row < rows) store_o(a.o + prow * D + c, o, 64);
          }
          if (row < rows) reinterpret_cast<float2*>(a.ml)[prow] = make_float2(m, l);
        } else {
          const float2 ml0 = ml_sm[row], ml1 = ml_sm[kTile + row];
          const float mm = fmaxf(ml0.x, ml1.x);
          const float w0 = ml0.x == -INFINITY ? 0.f : ex2(ml0.x - mm), w1 = ml1.x == -INFINITY ? 0.f : ex2(ml1.x - mm);
#pragma unroll 1
          for (int c = 0; c < D / 2; c += 32) {
            const int col = s * (D / 2) + c;
            uint32_t o[64];  // 32 dims of each stream's O
            ld64(lane_base + kO + col, lane_base + 256 + kO + col, o);
#pragma unroll
            for (int j = 0; j < 32; ++j)
              o[j] = __float_as_uint(fmaf(__uint_as_float(o[j]), w0, __uint_as_float(o[32 + j]) * w1));
            if (row < rows) store_o(a.o + prow * D + col, o, 32);
          }
          if (row < rows && s == 0) reinterpret_cast<float2*>(a.ml)[prow] = make_float2(mm, fmaf(ml0.y, w0, ml1.y * w1));
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {  // 8 arrivals free an O: of all warps that read it
        if (split) {
          mbar_arrive(&bars->o_free[0]);
          mbar_arrive(&bars->o_free[1]);
        } else {
          mbar_arrive(&bars->o_free[s]);
          mbar_arrive(&bars->o_free[s]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_sm && tid == 0 && a.err) atomicOr(a.err, kWaitTimeoutFlag);
  if (warp == 12) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512u));
  }
}

// ---------------------------------------------------------------------------------------
// Joins the partials of the rows: a warp takes merge_rows rows (query heads) of one token and
// KV head, which share their list of partials. A lane stands for one partial (its place and
// weight) and, in the sum, for D / 32 dims.
// ---------------------------------------------------------------------------------------
namespace spa {

// The shares that can hold a tile of an item, and where its partial rows lie.
struct Parts {
  Item it;
  int32_t first, count, stride;
  int32_t row0;  // (the host keeps partial rows below 2^31)
  __device__ __forceinline__ Parts(const SharedArgs& a, const Item& item, int t, int all, float shares) : it(item) {
    // (float: off by less than one share)
    first = max(static_cast<int>(static_cast<float>(it.start) * shares) - 2, 0);
    const int last = min(static_cast<int>(static_cast<float>(it.start + it.cost()) * shares) + 2, a.ctas - 1);
    count = it.kend > 0 ? last - first + 1 : 0;
    stride = it.b < 0 ? a.item_rows_p : a.item_rows_s;
    row0 = static_cast<int32_t>(partial_base(a, it, first)) + (t - it.tok0) * a.group;
  }
};

}  // namespace spa

// MANY: several rows a warp.
template <typename QT, int D, bool MANY>
__global__ void __launch_bounds__(256, 2) merge_partials(const __grid_constant__ SharedArgs a) {
  constexpr int kAhead = 16;  // partials' loads in flight (8: 69.5 us for 68.4 in the chunks)
  using namespace spa;
  constexpr int kPer = D / 32;  // dims per lane
  const int lane = threadIdx.x & 31;
  const int per_head = (a.group + a.merge_rows - 1) / a.merge_rows, per_token = a.kv_heads * per_head;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int t = static_cast<int>(unit / per_token), in_token = static_cast<int>(unit - static_cast<int64_t>(t) * per_token);
  const int h = in_token / per_head, g0 = (in_token - h * per_head) * a.merge_rows;
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  // The request: token t itself in a step of one token each (everything that such a step has to know
  // is asked for at once), else searched for, 32 places of the range at a time.
  int b = clamp32(t, 0, a.requests - 1), step = (a.requests + 31) >> 5;
  const int used = used_tokens(a), first = list_at(a.query_start), ws = list_at(a.head);
  int before = list_at(a.req_cost + b), probe = list_at(a.query_start + min(lane * step, a.requests));
  Request r = request_at(a, b);
  if (ws < 0 || t >= used || t < first) return;
  if (t < r.begin || t >= r.begin + r.n) {
    int lo = 0, hi = a.requests;  // query_start[lo] <= t < query_start[hi]
    for (;;) {
      const bool below = lane == 0 || (lo + lane * step < hi && probe <= t);
      lo += (31 - __clz(__ballot_sync(0xffffffffu, below))) * step;
      hi = min(lo + step, hi);
      if (hi - lo <= 1) break;
      step = (hi - lo + 31) >> 5;
      probe = list_at(a.query_start + min(lo + lane * step, hi));
    }
    b = lo;
    r = request_at(a, b);
    before = list_at(a.req_cost + b);
  }
  const int tile = (t - r.begin) / a.tile_tokens;
  if (tile > 0) {  // the cost of the request's row tiles before this one
    int c = 0;
    for (int j = lane; j < tile; j += 32) c += suffix_item(a, r, h, b, j, 0).cost();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
    before += c;
  }
  const int wp = prefix_cost(a, used), per = prefix_item_tokens(a, used), pi = t / per;
  const int all = (wp + ws) * a.kv_heads;
  const float shares = static_cast<float>(a.ctas) / static_cast<float>(all);
  const Parts pre(a, prefix_item(a, used, h, pi * per, h * wp + pi * prefix_item(a, used, 0, 0, 0).cost()), t, all, shares);
  const Parts suf(a, suffix_item(a, r, h, b, tile, a.kv_heads * wp + h * ws + before), t, all, shares);
  const int parts = pre.count + suf.count;
  // partial row of the token's first row in partial i of the list, -1 where the share holds none
  auto place = [&](int i) -> int {
    if (i >= parts) return -1;
    const bool p = i < pre.count;
    const Item& it = p ? pre.it : suf.it;
    const int k = p ? i : i - pre.count, c = (p ? pre.first : suf.first) + k;
    if (it.tile_at(share_begin(a, all, c + 1)) <= it.tile_at(share_begin(a, all, c))) return -1;
    return (p ? pre.row0 : suf.row0) + k * (p ? pre.stride : suf.stride);
  };
  const int mine = place(lane);
  auto load_ml = [&](int row) {
    return row < 0 ? make_float2(-INFINITY, 0.f) : __ldcg(reinterpret_cast<const float2*>(a.ml) + row);
  };
  const int g_end = min(g0 + a.merge_rows, a.group);
  uint16_t* out_t = a.output + static_cast<int64_t>(t) * a.o_token + static_cast<int64_t>(h) * a.group * a.o_head + lane * kPer;
  auto put = [&](int g, const float* f) {
    uint16_t* out = out_t + g * a.o_head;
    uint32_t packed[kPer / 2];
#pragma unroll
    for (int i = 0; i < kPer / 2; ++i) packed[i] = pack2<QT>(f[2 * i], f[2 * i + 1]);
    if (a.o_vec) {
      if constexpr (kPer == 4) *reinterpret_cast<uint2*>(out) = make_uint2(packed[0], packed[1]);
      else *reinterpret_cast<uint32_t*>(out) = packed[0];
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) out[i] = static_cast<uint16_t>(packed[i / 2] >> (16 * (i & 1)));
    }
  };
  auto put_lse = [&](int g, float m, float l) {
    a.lse[static_cast<int64_t>(t) * a.q_heads + h * a.group + g] =
        l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
  };
  const float* o_lane = a.o + lane * kPer;
  auto load_o = [&](int row, float (&v)[kPer]) {
    const float* p = o_lane + static_cast<int64_t>(row) * D;
    if constexpr (kPer == 4) {
      const float4 f = __ldcg(reinterpret_cast<const float4*>(p));
      v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else {
      const float2 f = __ldcg(reinterpret_cast<const float2*>(p));
      v[0] = f.x, v[1] = f.y;
    }
  };
  // At most four partials, as mostly in a large batch: eight rows' weights at once, a lane for one
  // row's one partial (chunks of 2100 tokens x 16 heads: 89 us without this, 68 so).
  unsigned held = MANY ? __ballot_sync(0xffffffffu, mine >= 0) : 0u;
  if (MANY && parts <= 32 && __popc(held) <= 4) {
    int rows[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = __shfl_sync(0xffffffffu, mine, held ? __ffs(held) - 1 : 0);
      rows[i] = held ? row : -1;
      held &= held - 1;
    }
    const int part = lane & 3;
    const int my_row = part == 0 ? rows[0] : part == 1 ? rows[1] : part == 2 ? rows[2] : rows[3];
#pragma unroll 1
    for (int gb = g0; gb < g_end; gb += 8) {
      const int my_g = gb + (lane >> 2);
      const float2 ml = load_ml(my_g < g_end && my_row >= 0 ? my_row + my_g : -1);
      float m = fmaxf(ml.x, __shfl_xor_sync(0xffffffffu, ml.x, 1));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
      float wgt = ml.x == -INFINITY ? 0.f : ex2(ml.x - m);
      float l = wgt * ml.y;
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      // l > 0 wherever a key has weight; NaN stays NaN
      wgt *= l == 0.f ? 0.f : 1.f / l;
      const unsigned live = __ballot_sync(0xffffffffu, ml.x != -INFINITY);
      if (a.lse && part == 0 && my_g < g_end) put_lse(my_g, m, l);
      constexpr int kRows = kAhead / 4;  // rows in flight
#pragma unroll 1
      for (int r = 0; r < min(8, g_end - gb); r += kRows) {
        float v[kRows][4][kPer];
#pragma unroll
        for (int u = 0; u < kRows; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int e = 0; e < kPer; ++e) v[u][i][e] = 0.f;
            if ((live >> (4 * (r + u) + i)) & 1u) load_o(rows[i] + gb + r + u, v[u][i]);
          }
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
          float acc[kPer];
#pragma unroll
          for (int e = 0; e < kPer; ++e) acc[e] = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float w = __shfl_sync(0xffffffffu, wgt, (4 * (r + u) + i) & 31);
            // (a NaN of the sum reaches the row through the weights)
#pragma unroll
            for (int e = 0; e < kPer; ++e) acc[e] = fmaf(v[u][i][e], w, acc[e]);
          }
          if (gb + r + u < g_end) put(gb + r + u, acc);
        }
      }
    }
    return;
  }
  float2 ml_next = load_ml(mine < 0 ? mine : mine + g0);
#pragma unroll 1
  for (int g = g0; g < g_end; ++g) {
    const float2 ml_mine = ml_next;
    if (g + 1 < g_end) ml_next = load_ml(mine < 0 ? mine : mine + g + 1);
    float acc[kPer], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
#pragma unroll 1
    for (int i0 = 0; i0 < parts; i0 += 32) {
      const int row = i0 == 0 ? mine : place(i0 + lane);
      const float2 ml = i0 == 0 ? ml_mine : load_ml(row < 0 ? row : row + g);
      float mn = fmaxf(m, ml.x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      if (mn == -INFINITY) continue;  // nothing with weight here
      const float alpha = m == -INFINITY ? 0.f : ex2(m - mn);
      const float wgt = ml.x == -INFINITY ? 0.f : ex2(ml.x - mn);
      float sum = wgt * ml.y;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l = fmaf(l, alpha, sum);
      m = mn;
      if (i0 > 0) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) acc[i] *= alpha;
      }
      unsigned live = __ballot_sync(0xffffffffu, ml.x != -INFINITY);
      while (live) {
        float v[kAhead][kPer], wv[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int src = live ? __ffs(live) - 1 : 0;
          const float w = __shfl_sync(0xffffffffu, wgt, src);
          const int at = __shfl_sync(0xffffffffu, row, src) + g;
          wv[u] = live ? w : 0.f;
          if (live) {
            load_o(at, v[u]);
          } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i) v[u][i] = 0.f;
          }
          live &= live - 1;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
          for (int i = 0; i < kPer; ++i) acc[i] = fmaf(v[u][i], wv[u], acc[i]);
      }
    }
    // l > 0 wherever a key has weight; NaN stays NaN
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] *= inv;
    put(g, acc);
    if (a.lse && lane == 0) put_lse(g, m, l);
  }
}

}  // namespace origami
