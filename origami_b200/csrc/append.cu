// C ABI of the per-head norm + rotation and of the append to a paged cache
// (append_kernels.cuh): validation, the choice of kernel and the launch.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/origami_b200.h"
#include "append_kernels.cuh"
#include "host_common.h"

using namespace origami_host;

namespace {

int64_t dtype_bytes(int32_t dtype) {
  switch (dtype) {
    case ORIGAMI_DTYPE_F16:
    case ORIGAMI_DTYPE_BF16: return 2;
    case ORIGAMI_DTYPE_F32: return 4;
    default: return 0;
  }
}

int32_t check_rows(const origami_head_rows* r, const char* name, int64_t head_dim, int64_t tokens, bool written) {
  const int64_t es = dtype_bytes(r->dtype);
  if (es == 0) return fail(ORIGAMI_ERR_INVALID, "%s must be float16, bfloat16 or float32", name);
  if (r->num_heads <= 0 || r->num_heads > 0xFFFF) return fail(ORIGAMI_ERR_INVALID, "%s must have 1..65535 heads", name);
  if (r->d_data == nullptr) return fail(ORIGAMI_ERR_INVALID, "%s is null", name);
  if (!aligned(r->d_data, static_cast<uintptr_t>(es)))
    return fail(ORIGAMI_ERR_INVALID, "%s is not aligned to its element type", name);
  if (r->token_stride < 0 || r->head_stride < 0) return fail(ORIGAMI_ERR_INVALID, "%s has a negative stride", name);
  if (written && rows_overlap(*r, head_dim, tokens))
    return fail(ORIGAMI_ERR_INVALID, "%s has rows that overlap", name);
  return ORIGAMI_OK;
}

int32_t check_pair(const origami_head_rows* in, const origami_head_rows* out, const char* in_name, const char* out_name,
                   int64_t head_dim, int64_t tokens) {
  if (in == nullptr || out == nullptr) return fail(ORIGAMI_ERR_INVALID, "%s and %s are both needed", in_name, out_name);
  int32_t rc = check_rows(in, in_name, head_dim, tokens, false);
  if (rc) return rc;
  if ((rc = check_rows(out, out_name, head_dim, tokens, true))) return rc;
  if (in->dtype != out->dtype) return fail(ORIGAMI_ERR_INVALID, "%s must have the type of %s", out_name, in_name);
  if (in->num_heads != out->num_heads) return fail(ORIGAMI_ERR_INVALID, "%s must have the heads of %s", out_name, in_name);
  if (in->d_data == out->d_data && (in->token_stride != out->token_stride || in->head_stride != out->head_stride))
    return fail(ORIGAMI_ERR_INVALID, "%s starts where %s does and must then have its strides", out_name, in_name);
  return ORIGAMI_OK;
}

int32_t check_norm(const origami_head_norm* n) {
  if (n == nullptr) return ORIGAMI_OK;
  if (!(n->eps >= 0.0) || std::isinf(n->eps)) return fail(ORIGAMI_ERR_INVALID, "eps must be finite and not negative");
  const void* w[2] = {n->d_query_weight, n->d_key_weight};
  const int32_t dt[2] = {n->query_weight_dtype, n->key_weight_dtype};
  for (int i = 0; i < 2; ++i) {
    if (w[i] == nullptr) continue;
    const int64_t es = dtype_bytes(dt[i]);
    if (es == 0) return fail(ORIGAMI_ERR_INVALID, "norm weights must be float16, bfloat16 or float32");
    if (!aligned(w[i], static_cast<uintptr_t>(es)))
      return fail(ORIGAMI_ERR_INVALID, "norm weights are not aligned to their element type");
  }
  return ORIGAMI_OK;
}

int32_t check_rotation(const origami_rotation* r, int64_t head_dim) {
  const int64_t es = dtype_bytes(r->table_dtype);
  if (r->d_cos_sin == nullptr || r->d_positions == nullptr)
    return fail(ORIGAMI_ERR_INVALID, "rotation needs a cos_sin table and positions");
  if (es == 0) return fail(ORIGAMI_ERR_INVALID, "cos_sin must be float16, bfloat16 or float32");
  if (!aligned(r->d_cos_sin, static_cast<uintptr_t>(es)))
    return fail(ORIGAMI_ERR_INVALID, "cos_sin is not aligned to its element type");
  if (r->rotary_dim <= 0 || r->rotary_dim % 2 != 0 || r->rotary_dim > head_dim)
    return fail(ORIGAMI_ERR_INVALID, "the rotated dims must be even in number and at most head_dim (%lld)",
                static_cast<long long>(head_dim));
  if (r->max_positions <= 0) return fail(ORIGAMI_ERR_INVALID, "cos_sin has no rows");
  if (r->row_stride < r->rotary_dim) return fail(ORIGAMI_ERR_INVALID, "cos_sin rows overlap");
  if (r->position_bytes != 4 && r->position_bytes != 8) return fail(ORIGAMI_ERR_INVALID, "positions must be int32 or int64");
  if (!aligned(r->d_positions, static_cast<uintptr_t>(r->position_bytes)))
    return fail(ORIGAMI_ERR_INVALID, "positions are not aligned to their element type");
  return ORIGAMI_OK;
}

// (the token stride of one token and the head stride of one head are never used: 0, so that they
// do not count in the choice of kernel)
void set_rows(origami::HeadRows& r, const origami_head_rows* in, const origami_head_rows* out, int64_t tokens,
              const void* weight, int32_t weight_dtype) {
  r.in = in->d_data;
  r.in_token = tokens > 1 ? in->token_stride : 0;
  r.in_head = in->num_heads > 1 ? in->head_stride : 0;
  r.heads = static_cast<int32_t>(in->num_heads);
  if (out) {
    r.out = out->d_data;
    r.out_token = tokens > 1 ? out->token_stride : 0;
    r.out_head = out->num_heads > 1 ? out->head_stride : 0;
  }
  r.weight = weight;
  r.weight_dtype = weight_dtype;
}

void set_shared(origami::AppendArgs& a, int64_t tokens, int64_t head_dim, const origami_rotation* rot,
                const origami_head_norm* norm, uint32_t* err) {
  a.tokens = tokens;
  a.D = static_cast<int32_t>(head_dim);
  a.err = err;
  if (rot) {
    a.positions = rot->d_positions;
    a.positions64 = rot->position_bytes == 8;
    a.table = rot->d_cos_sin;
    a.table_dtype = rot->table_dtype;
    a.table_stride = rot->row_stride;
    a.max_positions = rot->max_positions;
    a.R = static_cast<int32_t>(rot->rotary_dim);
    a.interleaved = rot->interleaved != 0;
  }
  a.eps = norm ? static_cast<float>(norm->eps) : 0.f;
  a.inv_d = 1.f / static_cast<float>(head_dim);
}

bool rows16(const origami::HeadRows& r, int64_t es) {
  if (r.heads == 0) return true;
  return aligned(r.in, 16) && (r.in_token * es) % 16 == 0 && (r.in_head * es) % 16 == 0 && aligned(r.out, 16) &&
         (r.out_token * es) % 16 == 0 && (r.out_head * es) % 16 == 0;
}

// The fast kernel's conditions (append_kernels.cuh); everything else takes the kernel for
// any layout.
bool fast_rows(const origami::AppendArgs& a, int64_t es) {
  if (a.D % 8 != 0 || a.D > 512) return false;
  if (!rows16(a.q, es) || !rows16(a.k, es) || !rows16(a.v, es) || !aligned(a.cache, 16)) return false;
  if (a.positions == nullptr) return true;
  const int64_t ts = dtype_bytes(a.table_dtype);
  return a.R % 16 == 0 && aligned(a.table, 16) && (a.table_stride * ts) % 16 == 0;
}

template <typename TI, typename TC>
int32_t launch(origami::AppendArgs& a, cudaStream_t st) {
  const int total = a.q.heads + a.k.heads + a.v.heads;
  if (fast_rows(a, sizeof(TI))) {
    const int lanes = (a.D / 8 + 1) / 2;
    while ((1 << a.lanes_log2) < lanes) ++a.lanes_log2;
    // One walker per head while that many threads fit the device at once (the step of a few
    // tokens is bound by latency); else kQueryRows query heads a walker beside a key and a value
    // head (two of them took 162 us for the 32768-token append that four take 139 for, cold L2).
    int sms = 0, dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceGetAttribute");
    const int64_t resident = static_cast<int64_t>(sms) * 512;
    a.groups = a.tokens * total << a.lanes_log2 <= resident ? total : std::max(a.k.heads, (a.q.heads + origami::app::kQueryRows - 1) / origami::app::kQueryRows);
    const bool full = a.D == 16 << a.lanes_log2;
    const bool stream = a.groups != total;
    auto* fn = stream ? (full ? &origami::append_rows<TI, TC, true, true> : &origami::append_rows<TI, TC, false, true>)
                      : (full ? &origami::append_rows<TI, TC, true, false> : &origami::append_rows<TI, TC, false, false>);
    const int smem = stream ? origami::app::kStreamSmem<TI> : 0;
    int slots = 0;
    const int32_t rc = persistent_slots(reinterpret_cast<const void*>(fn), smem, slots);
    if (rc) return rc;
    const int64_t per_cta = 256 >> a.lanes_log2;  // walkers
    const int64_t needed = (a.tokens * a.groups + per_cta - 1) / per_cta;
    // as many CTAs as fit at once, but at least one token's walkers (without steps: all); whole tokens per pass
    const int64_t ctas = stream ? std::min(needed, std::max<int64_t>(slots, (a.groups + per_cta - 1) / per_cta)) : needed;
    a.step = static_cast<int32_t>(ctas * per_cta / a.groups);
    fn<<<static_cast<unsigned>(ctas), 256, smem, st>>>(a);
    return after_launch("append_rows launch");
  }
  const int64_t ctas = (a.tokens * total + 7) / 8;
  if (ctas > 0x7FFFFFFF) return fail(ORIGAMI_ERR_UNSUPPORTED, "too many rows");
  origami::append_rows_any<TI, TC><<<static_cast<unsigned>(ctas), 256, 0, st>>>(a);
  return after_launch("append_rows_any launch");
}

template <typename TI>
int32_t launch_cache(origami::AppendArgs& a, int32_t cache_dtype, cudaStream_t st) {
  return cache_dtype == ORIGAMI_DTYPE_F16 ? launch<TI, __half>(a, st) : launch<TI, __nv_bfloat16>(a, st);
}

int32_t check_tokens(int64_t tokens, int64_t head_dim) {
  if (tokens < 0 || tokens > 0x3FFFFFFF) return fail(ORIGAMI_ERR_INVALID, "tokens must be in [0, 2^30)");
  if (head_dim <= 0 || head_dim > 65536) return fail(ORIGAMI_ERR_INVALID, "head_dim must be in [1, 65536]");
  return ORIGAMI_OK;
}

}  // namespace

extern "C" {

int32_t origami_norm_rope(const origami_head_rows* query, const origami_head_rows* query_out,
                          const origami_head_rows* key, const origami_head_rows* key_out, int64_t tokens,
                          int64_t head_dim, const origami_rotation* rotation, const origami_head_norm* norm,
                          uint32_t* d_error_count, origami_stream_t stream) {
  int32_t rc = check_tokens(tokens, head_dim);
  if (rc) return rc;
  if (tokens == 0) return ORIGAMI_OK;
  if ((rc = check_pair(query, query_out, "query", "query_out", head_dim, tokens))) return rc;
  if ((rc = check_pair(key, key_out, "key", "key_out", head_dim, tokens))) return rc;
  if (query->dtype != key->dtype) return fail(ORIGAMI_ERR_INVALID, "query and key must have the same type");
  if (query_out->d_data == key_out->d_data) return fail(ORIGAMI_ERR_INVALID, "query_out and key_out are the same rows");
  if (rotation == nullptr) return fail(ORIGAMI_ERR_INVALID, "rotation is null");
  if ((rc = check_rotation(rotation, head_dim)) || (rc = check_norm(norm))) return rc;
  origami::AppendArgs a{};
  set_shared(a, tokens, head_dim, rotation, norm, d_error_count);
  set_rows(a.q, query, query_out, tokens, norm ? norm->d_query_weight : nullptr, norm ? norm->query_weight_dtype : 0);
  set_rows(a.k, key, key_out, tokens, norm ? norm->d_key_weight : nullptr, norm ? norm->key_weight_dtype : 0);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (query->dtype) {
    case ORIGAMI_DTYPE_F16: return launch<__half, __half>(a, st);
    case ORIGAMI_DTYPE_BF16: return launch<__nv_bfloat16, __nv_bfloat16>(a, st);
    default: return launch<float, __half>(a, st);
  }
}

int32_t origami_append_kv(const origami_head_rows* key, const origami_head_rows* value, const origami_head_rows* query,
                          const origami_head_rows* query_out, const origami_paged_kv* cache, int32_t cache_dtype,
                          const void* d_slots, int32_t slot_bytes, int64_t tokens, const origami_rotation* rotation,
                          const origami_head_norm* norm, uint32_t* d_error_count, origami_stream_t stream) {
  PagedGeom g;
  int32_t rc = validate_cache(cache, g);
  if (rc) return rc;
  const int64_t head_dim = cache->head_dim;
  if ((rc = check_tokens(tokens, head_dim))) return rc;
  if (cache_dtype != ORIGAMI_DTYPE_F16 && cache_dtype != ORIGAMI_DTYPE_BF16)
    return fail(ORIGAMI_ERR_INVALID, "the paged cache must be float16 or bfloat16");
  if (slot_bytes != 4 && slot_bytes != 8) return fail(ORIGAMI_ERR_INVALID, "slots must be int32 or int64");
  if (tokens == 0) return ORIGAMI_OK;
  if (key == nullptr || value == nullptr) return fail(ORIGAMI_ERR_INVALID, "key and value are both needed");
  if ((rc = check_rows(key, "key", head_dim, tokens, false))) return rc;
  if ((rc = check_rows(value, "value", head_dim, tokens, false))) return rc;
  if (key->dtype != value->dtype) return fail(ORIGAMI_ERR_INVALID, "key and value must have the same type");
  if (key->num_heads != cache->num_heads || value->num_heads != cache->num_heads)
    return fail(ORIGAMI_ERR_INVALID, "key and value must have the cache's %lld heads",
                static_cast<long long>(cache->num_heads));
  if (query != nullptr || query_out != nullptr) {
    if ((rc = check_pair(query, query_out, "query", "query_out", head_dim, tokens))) return rc;
    if (query->dtype != key->dtype) return fail(ORIGAMI_ERR_INVALID, "query and key must have the same type");
  }
  if (d_slots == nullptr || !aligned(d_slots, static_cast<uintptr_t>(slot_bytes)))
    return fail(ORIGAMI_ERR_INVALID, "slots are null or not aligned to their element type");
  if (rotation != nullptr && (rc = check_rotation(rotation, head_dim))) return rc;
  if ((rc = check_norm(norm))) return rc;
  origami::AppendArgs a{};
  set_shared(a, tokens, head_dim, rotation, norm, d_error_count);
  if (query) set_rows(a.q, query, query_out, tokens, norm ? norm->d_query_weight : nullptr, norm ? norm->query_weight_dtype : 0);
  set_rows(a.k, key, nullptr, tokens, norm ? norm->d_key_weight : nullptr, norm ? norm->key_weight_dtype : 0);
  set_rows(a.v, value, nullptr, tokens, nullptr, 0);
  a.slots = d_slots;
  a.slots64 = slot_bytes == 8;
  a.cache = cache->d_data;
  a.kv_stride = g.kv_stride;
  a.block_stride = g.block_stride;
  a.token_stride = g.token_stride;
  a.block_size = cache->block_size;
  a.num_slots = cache->num_blocks * cache->block_size;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (key->dtype) {
    case ORIGAMI_DTYPE_F16: return launch_cache<__half>(a, cache_dtype, st);
    case ORIGAMI_DTYPE_BF16: return launch_cache<__nv_bfloat16>(a, cache_dtype, st);
    default: return launch_cache<float>(a, cache_dtype, st);
  }
}

}  // extern "C"
