// The paged key-value cache as the kernels see it, its argument checks, and
// the device guard of the serving entry points.
//
// Layout: K and V pages [num_blocks][n_kv_heads][block_size][head_dim], a
// page `block_stride` elements after the one before it. Inside a page the
// rows of one head are contiguous, so a head's tokens are read in whole
// lines; with num_blocks = 1 and block_size = max_seq it is the per-sequence
// cache [n_kv_heads][max_seq][64] that mc_proj3_gemv_scatter writes. Every
// offset is 64-bit.
#pragma once
#include "mc_internal.cuh"

#define MC_KV_SLOT_NONE 0xffffffffffffffffull

// Makes ctx's device current for the launches of one call and puts the
// caller's device back: the stream belongs to ctx's device, whatever device
// the calling thread has current.
class McDeviceGuard {
 public:
  explicit McDeviceGuard(int device) {
    if (cudaGetDevice(&prev_) != cudaSuccess) {
      (void)cudaGetLastError();
      prev_ = -1;
    }
    if (prev_ != device) {
      err_ = cudaSetDevice(device);
      if (err_ != cudaSuccess) (void)cudaGetLastError();
      moved_ = err_ == cudaSuccess;
    }
  }
  ~McDeviceGuard() {
    if (moved_ && prev_ >= 0) (void)cudaSetDevice(prev_);
  }
  McDeviceGuard(const McDeviceGuard&) = delete;
  McDeviceGuard& operator=(const McDeviceGuard&) = delete;
  cudaError_t error() const { return err_; }

 private:
  int prev_ = -1;
  bool moved_ = false;
  cudaError_t err_ = cudaSuccess;
};

// Checks a cache description; `name` is the entry point.
static inline int mc_check_kv_cache(const char* name, const void* k, const void* v, int dtype,
                                    int num_blocks, int block_size, size_t block_stride,
                                    int n_kv_heads, int head_dim, const float* k_scale,
                                    const float* v_scale) {
  MC_REQUIRE(dtype == MC_DTYPE_BF16 || dtype == MC_DTYPE_E4M3, "%s: cache dtype %d", name, dtype);
  if (head_dim != 64 && head_dim != 128)
    return mc_fail(MC_EUNSUPPORTED, "%s: head_dim %d (64 and 128 are built)", name, head_dim);
  MC_REQUIRE(n_kv_heads >= 1 && n_kv_heads <= 1024, "%s: n_kv_heads %d out of range", name,
             n_kv_heads);
  MC_REQUIRE(num_blocks >= 1 && block_size >= 1, "%s: %d blocks of %d tokens", name, num_blocks,
             block_size);
  MC_REQUIRE(k && v, "%s: null cache", name);
  MC_REQUIRE(mc_aligned(k, 16) && mc_aligned(v, 16), "%s: the cache must be 16-byte aligned", name);
  const size_t page = (size_t)n_kv_heads * (size_t)block_size * (size_t)head_dim;
  MC_REQUIRE(block_stride >= page || num_blocks == 1,
             "%s: block stride %zu below a page of %zu elements", name, block_stride, page);
  MC_REQUIRE(block_stride % (size_t)head_dim == 0,
             "%s: block stride %zu not a multiple of head_dim", name, block_stride);
  // rows are numbered in 32 bits (the memory of a GPU holds fewer of 64 bytes); the stride by
  // itself first, so that its product stays in 64
  const size_t most = 0xffffffffull, step = num_blocks > 1 ? block_stride / head_dim : 0;
  MC_REQUIRE(page / head_dim < most && step < most &&
                 step * (num_blocks - 1) + page / head_dim < most,
             "%s: a cache of more than 2^32 - 2 rows", name);
  MC_REQUIRE(dtype == MC_DTYPE_E4M3 || (!k_scale && !v_scale),
             "%s: scales belong to an e4m3 cache", name);
  MC_REQUIRE(mc_aligned(k_scale, 4) && mc_aligned(v_scale, 4), "%s: scales misaligned", name);
  return MC_OK;
}
