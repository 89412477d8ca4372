// Host helpers shared by the translation units of liborigami_b200.so: the per-thread
// error message, CUDA error mapping, paged-cache validation and the persistent-grid
// occupancy cache.
#pragma once

#include <cstdint>

#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include "../../include/origami_b200.h"

namespace origami_host {

constexpr int kThreads = 256;

// Records a printf-style message for origami_last_error() and returns `code`.
int32_t fail(int32_t code, const char* fmt, ...);
int32_t cuda_fail(cudaError_t e, const char* what);
// cudaGetLastError() after a launch, as an ORIGAMI_ERR_CUDA status.
int32_t after_launch(const char* what);

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// Element strides of one layer's paged cache.
struct PagedGeom {
  int64_t kv_stride, block_stride, token_stride, head_stride;
};
int32_t validate_cache(const origami_paged_kv* kv, PagedGeom& g);

// Whether rows share elements; rows that are written must not.
inline bool rows_overlap(const origami_head_rows& r, int64_t head_dim, int64_t tokens) {
  const int64_t heads = r.num_heads;
  const bool token_outer = (heads == 1 || r.head_stride >= head_dim) &&
                           (tokens == 1 || r.token_stride >= (heads - 1) * r.head_stride + head_dim);
  const bool head_outer = (tokens == 1 || r.token_stride >= head_dim) &&
                          (heads == 1 || r.head_stride >= (tokens - 1) * r.token_stride + head_dim);
  return !token_outer && !head_outer;
}

// Raises the kernel's dynamic shared-memory limit to `smem` (once per kernel and device)
// and returns the CTAs of kThreads threads resident on the whole device.
int32_t persistent_slots(const void* fn, int smem, int& resident);

// The driver's cuTensorMapEncodeTiled, null where the driver has none.
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

}  // namespace origami_host
