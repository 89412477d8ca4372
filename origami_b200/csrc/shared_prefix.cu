// C ABI of the shared-prefix attention (shared_prefix_kernels.cuh): validation, the workspace
// and the two launches.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/origami_b200.h"
#include "host_common.h"
#include "shared_prefix_kernels.cuh"

using namespace origami_host;

namespace {

constexpr int64_t kAlign = 256;
int64_t round_up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

int32_t device_sms(int& sms) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return e == cudaSuccess ? ORIGAMI_OK : cuda_fail(e, "cudaDeviceGetAttribute");
}

struct Workspace {
  int64_t req_cost, ml, o, bytes;  // byte offsets
  int32_t item_rows_p, item_rows_s;
};

int32_t check_shape(int64_t tokens, int64_t query_heads, int64_t kv_heads, int64_t head_dim, int64_t requests) {
  if (tokens < 0 || query_heads <= 0) return fail(ORIGAMI_ERR_INVALID, "query token and head counts must be positive");
  if (kv_heads <= 0 || query_heads % kv_heads != 0)
    return fail(ORIGAMI_ERR_INVALID, "query_heads must be divisible by kv_heads");
  if (query_heads / kv_heads > origami::spa::kTile)
    return fail(ORIGAMI_ERR_UNSUPPORTED, "at most %d query heads per KV head are supported", origami::spa::kTile);
  if (head_dim != 64 && head_dim != 128)
    return fail(ORIGAMI_ERR_UNSUPPORTED, "shared-prefix attention supports head_dim 64 and 128");
  if (requests <= 0) return fail(ORIGAMI_ERR_INVALID, "at least one request is needed");
  if (requests > (1 << 24) || tokens > (1 << 24) || query_heads > (1 << 15) || tokens * query_heads > (1 << 29))
    return fail(ORIGAMI_ERR_UNSUPPORTED, "too many query rows");
  return ORIGAMI_OK;
}

Workspace plan(int64_t tokens, int64_t query_heads, int64_t kv_heads, int64_t head_dim, int64_t requests, int sms) {
  const int64_t group = query_heads / kv_heads, per = origami::spa::kTile / group;
  Workspace w{};
  w.item_rows_p = static_cast<int32_t>(std::min(2 * per, tokens) * group);
  w.item_rows_s = static_cast<int32_t>(std::min(per, tokens) * group);
  const int64_t rows = 2 * query_heads * tokens + static_cast<int64_t>(sms) * (w.item_rows_p + w.item_rows_s);
  w.req_cost = kAlign;
  w.ml = w.req_cost + round_up(requests * 4, kAlign);
  w.o = w.ml + round_up(rows * 8, kAlign);
  w.bytes = w.o + round_up(rows * head_dim * 4, kAlign) + 16;  // 16: to a 32-byte boundary, for whole-sector stores
  return w;
}

template <typename F, typename... Args>
int32_t launch_dependent(F* fn, dim3 grid, int threads, int smem, cudaStream_t st, const char* what, const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, args...);
  if (e != cudaSuccess) return cuda_fail(e, what);
  return after_launch(what);
}

template <typename QT, int D>
int32_t launch(const origami::SharedArgs& a, cudaStream_t st) {
  auto* fn = &origami::shared_prefix_attention<QT, D>;
  constexpr int smem = origami::spa::Smem<D>::bytes;
  int resident = 0;
  int32_t rc = persistent_slots(reinterpret_cast<const void*>(fn), smem, resident);  // raises the shared-memory limit
  if (rc) return rc;
  rc = launch_dependent(fn, dim3(static_cast<unsigned>(a.ctas)), origami::spa::kThreadsS, smem, st,
                        "shared_prefix_attention launch", a);
  if (rc) return rc;
  const int64_t warps = static_cast<int64_t>(a.tokens) * a.kv_heads * ((a.group + a.merge_rows - 1) / a.merge_rows);
  auto* merge = a.merge_rows == 1 ? &origami::merge_partials<QT, D, false> : &origami::merge_partials<QT, D, true>;
  return launch_dependent(merge, dim3(static_cast<unsigned>((warps + 7) / 8)), 256, 0, st, "merge_partials launch", a);
}

int32_t check_head_rows(const origami_head_rows* r, const char* name, int64_t tokens, int64_t head_dim, bool written) {
  if (r == nullptr || r->d_data == nullptr) return fail(ORIGAMI_ERR_INVALID, "%s is null", name);
  if (r->dtype != ORIGAMI_DTYPE_F16 && r->dtype != ORIGAMI_DTYPE_BF16)
    return fail(ORIGAMI_ERR_INVALID, "%s must be float16 or bfloat16", name);
  if (!aligned(r->d_data, 2)) return fail(ORIGAMI_ERR_INVALID, "%s must be 2-byte aligned", name);
  if (r->token_stride < 0 || r->head_stride < 0) return fail(ORIGAMI_ERR_INVALID, "%s has a negative stride", name);
  if (written && rows_overlap(*r, head_dim, tokens))
    return fail(ORIGAMI_ERR_INVALID, "%s has rows that overlap", name);
  return ORIGAMI_OK;
}

bool rows_vec(const origami_head_rows* r) {
  return aligned(r->d_data, 16) && r->token_stride % 8 == 0 && r->head_stride % 8 == 0;
}

}  // namespace

extern "C" {

int32_t origami_shared_prefix_attention_workspace(int64_t tokens, int64_t query_heads, int64_t kv_heads,
                                                  int64_t head_dim, int64_t requests, int64_t* workspace_bytes) {
  if (workspace_bytes == nullptr) return fail(ORIGAMI_ERR_INVALID, "workspace_bytes is null");
  int32_t rc = check_shape(tokens, query_heads, kv_heads, head_dim, requests);
  if (rc) return rc;
  int sms = 0;
  if ((rc = device_sms(sms))) return rc;
  *workspace_bytes = plan(tokens, query_heads, kv_heads, head_dim, requests, sms).bytes;
  return ORIGAMI_OK;
}

int32_t origami_shared_prefix_attention(
    const origami_head_rows* query, const origami_head_rows* output, float* d_lse, int64_t tokens, int64_t head_dim,
    const origami_paged_kv* cache, int32_t cache_dtype, const int32_t* d_prefix_blocks, int64_t num_prefix_blocks,
    int64_t prefix_tokens, const int32_t* d_suffix_blocks, int64_t suffix_stride, int64_t suffix_width,
    const int32_t* d_suffix_lens, const int32_t* d_query_start, int64_t requests, double softmax_scale,
    void* d_workspace, int64_t workspace_bytes, uint32_t* d_error_flags, origami_stream_t stream) {
  PagedGeom g;
  int32_t rc = validate_cache(cache, g);
  if (rc) return rc;
  if (query == nullptr || output == nullptr) return fail(ORIGAMI_ERR_INVALID, "query and output are both needed");
  if ((rc = check_shape(tokens, query->num_heads, cache->num_heads, head_dim, requests))) return rc;
  if (cache->head_dim != head_dim) return fail(ORIGAMI_ERR_INVALID, "kv_cache head_dim does not match query");
  if (prefix_tokens < 0 || num_prefix_blocks < 0 || suffix_width < 0)
    return fail(ORIGAMI_ERR_INVALID, "prefix and suffix lengths must not be negative");
  if (prefix_tokens > 0x3FFFFFFF) return fail(ORIGAMI_ERR_UNSUPPORTED, "the prefix is too long");
  if (num_prefix_blocks < (prefix_tokens + cache->block_size - 1) / cache->block_size)
    return fail(ORIGAMI_ERR_INVALID, "prefix_blocks is too short for prefix_tokens");
  if (!(softmax_scale > 0.0) || std::isinf(softmax_scale))
    return fail(ORIGAMI_ERR_INVALID, "softmax_scale must be finite and positive");
  const float scale_log2 = static_cast<float>(softmax_scale * 1.4426950408889634);
  if (!std::isnormal(scale_log2))  // zero or infinite, it would make NaN of scores that are not seen or zero
    return fail(ORIGAMI_ERR_INVALID, "softmax_scale is too small or too large for 32 bits");
  if (cache->block_size > 0x3FFFFFFF || cache->num_blocks * cache->block_size > 0x3FFFFFFF)
    return fail(ORIGAMI_ERR_UNSUPPORTED, "the cache has too many token rows");
  if (tokens == 0) return ORIGAMI_OK;
  if ((rc = check_head_rows(query, "query", tokens, head_dim, false))) return rc;
  if ((rc = check_head_rows(output, "output", tokens, head_dim, true))) return rc;
  if (output->num_heads != query->num_heads) return fail(ORIGAMI_ERR_INVALID, "output must have the heads of query");
  if (output->dtype != query->dtype) return fail(ORIGAMI_ERR_INVALID, "output dtype must match query dtype");
  if (cache_dtype != query->dtype) return fail(ORIGAMI_ERR_INVALID, "kv_cache dtype must match query dtype");
  if (d_query_start == nullptr || d_suffix_lens == nullptr || !aligned(d_query_start, 4) || !aligned(d_suffix_lens, 4))
    return fail(ORIGAMI_ERR_INVALID, "query_start and suffix_lens must be int32 device arrays");
  if ((prefix_tokens > 0 && d_prefix_blocks == nullptr) || !aligned(d_prefix_blocks, 4))
    return fail(ORIGAMI_ERR_INVALID, "prefix_blocks must be an int32 device array");
  if ((suffix_width > 0 && d_suffix_blocks == nullptr) || !aligned(d_suffix_blocks, 4))
    return fail(ORIGAMI_ERR_INVALID, "suffix_blocks must be an int32 device array");
  if (suffix_stride < 0) return fail(ORIGAMI_ERR_INVALID, "suffix_blocks has a negative stride");
  if (d_lse != nullptr && !aligned(d_lse, 4)) return fail(ORIGAMI_ERR_INVALID, "lse must be a float32 device array");
  // every item's cost, at most, has to fit the 31-bit cost axis of the deal
  const int64_t per_tile = origami::spa::kTile / (query->num_heads / cache->num_heads);
  const int64_t row_tiles = (tokens + per_tile - 1) / per_tile;
  const int64_t suffix_cap = std::min<int64_t>(suffix_width, 0x3FFFFFFF / cache->block_size) * cache->block_size;
  auto cost = [](int64_t keys, int64_t tile) {
    return origami::spa::kCostPairItem + (keys + origami::spa::kTile - 1) / origami::spa::kTile * tile;
  };
  const double most = static_cast<double>(cache->num_heads) *
                      (static_cast<double>(row_tiles) * cost(prefix_tokens, origami::spa::kCostPair) +
                       static_cast<double>(row_tiles + requests) * cost(suffix_cap, origami::spa::kCostTile));
  if (most >= 2147483648.0) return fail(ORIGAMI_ERR_UNSUPPORTED, "too many tiles of keys and query rows for one call");
  int sms = 0;
  if ((rc = device_sms(sms))) return rc;
  const Workspace w = plan(tokens, query->num_heads, cache->num_heads, head_dim, requests, sms);
  if (d_workspace == nullptr || workspace_bytes < w.bytes || !aligned(d_workspace, 16))
    return fail(ORIGAMI_ERR_INVALID, "workspace must be 16-byte aligned and hold %lld bytes",
                static_cast<long long>(w.bytes));

  origami::SharedArgs a{};
  a.query = static_cast<const uint16_t*>(query->d_data);
  a.output = static_cast<uint16_t*>(output->d_data);
  a.lse = d_lse;
  a.q_token = query->token_stride;
  a.q_head = query->head_stride;
  a.o_token = output->token_stride;
  a.o_head = output->head_stride;
  a.cache = static_cast<const uint16_t*>(cache->d_data);
  a.kv_stride = g.kv_stride;
  a.row_elems = g.token_stride;
  a.num_blocks = cache->num_blocks;
  a.block_size = static_cast<int32_t>(cache->block_size);
  a.block_rows = static_cast<int32_t>(g.block_stride / g.token_stride);
  a.prefix_blocks = d_prefix_blocks;
  a.suffix_blocks = d_suffix_blocks;
  a.suffix_stride = suffix_stride;
  a.suffix_lens = d_suffix_lens;
  a.query_start = d_query_start;
  a.tokens = static_cast<int32_t>(tokens);
  a.requests = static_cast<int32_t>(requests);
  a.prefix = static_cast<int32_t>(prefix_tokens);
  a.suffix_cap = static_cast<int32_t>(suffix_cap);
  a.q_heads = static_cast<int32_t>(query->num_heads);
  a.kv_heads = static_cast<int32_t>(cache->num_heads);
  a.group = a.q_heads / a.kv_heads;
  a.tile_tokens = origami::spa::kTile / a.group;
  a.item_rows_p = w.item_rows_p;
  a.item_rows_s = w.item_rows_s;
  a.all_rows = static_cast<int32_t>(2 * cache->num_blocks * cache->block_size);
  a.v_rows = static_cast<int32_t>(g.kv_stride / g.token_stride);
  a.inv_ctas = static_cast<uint32_t>(0x100000000ull / static_cast<uint64_t>(std::max(sms, 2)));  // (unused for one CTA)
  // TMA boxes of at least one swizzle atom (8 rows) that lie inside one block and one warp's 32 rows
  a.tma_rows = 32;
  while (a.tma_rows >= 8 && cache->block_size % a.tma_rows != 0) a.tma_rows /= 2;
  if (a.tma_rows < 8) a.tma_rows = 0;
  if (a.tma_rows > 0) {
    auto encode = tensor_map_encoder();
    if (encode == nullptr) return fail(ORIGAMI_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(cache->num_heads),
                                static_cast<cuuint64_t>(a.all_rows)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(head_dim * 2), static_cast<cuuint64_t>(g.token_stride * 2)};
    const cuuint32_t box[3] = {64, 1, static_cast<cuuint32_t>(a.tma_rows)}, estr[3] = {1, 1, 1};
    const CUresult r = encode(&a.map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, cache->d_data, dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(ORIGAMI_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
  }
  a.q_vec = rows_vec(query);
  a.o_vec = rows_vec(output);
  a.ctas = sms;
  // One row a warp while the rows are few (their latency counts: twice as many rows a warp take the
  // batch of 64 over 32768 keys from 83 to 88 us), more when their lists' lookup would be what an SM
  // spends its issue slots on (half as many change nothing beyond the spread of the batch of 256;
  // one each: chunks of 2100 tokens of 16 heads 110 us instead of 68).
  a.merge_rows = static_cast<int32_t>(std::clamp<int64_t>(tokens * a.q_heads / (8 * sms), 1, a.group));
  a.scale_log2 = scale_log2;
  uint8_t* ws = reinterpret_cast<uint8_t*>(round_up(reinterpret_cast<int64_t>(d_workspace), 32));
  a.head = reinterpret_cast<int32_t*>(ws);
  a.req_cost = reinterpret_cast<int32_t*>(ws + w.req_cost);
  a.ml = reinterpret_cast<float*>(ws + w.ml);
  a.o = reinterpret_cast<float*>(ws + w.o);
  a.err = d_error_flags;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (query->dtype == ORIGAMI_DTYPE_BF16)
    return head_dim == 128 ? launch<__nv_bfloat16, 128>(a, st) : launch<__nv_bfloat16, 64>(a, st);
  return head_dim == 128 ? launch<__half, 128>(a, st) : launch<__half, 64>(a, st);
}

}  // extern "C"
